// A step's rows of the fused projection into a cache in 8 bits (cache8.h): per-head RMSNorm and rotation of q and k, q to its rows,
// k and v to the blocks that the step writes to.
//
//   x <- x / sqrt(mean(x^2) + eps) * w          per head of q and k, if there is a norm
//   (x_a, x_b) <- (x_a cos - x_b sin, x_a sin + x_b cos)   per pair of the first rotary_dim channels
//   block: e = max(e of what it holds, the least e with max |x| <= 448 * 2^e of the new ones); byte = e4m3(x * 2^-e)
//
// A workgroup takes a (block, kv head): a block's scale needs all of its tokens, and its earlier bytes move when the scale grows, so
// whoever else wrote to the block in the same step would race.  Workgroups behind those take q's heads.  All arithmetic is float32; k and
// v are rounded once, to 8 bits, and never to bfloat16 in between.  Bound: decoding, a launch's latency and the chain work list ->
// rows -> largest value -> bytes; prompts, the reading of the projection and the writing of q.
#include "cache8.h"

#include <algorithm>

namespace {

constexpr int THREADS = 256;
constexpr int MAX_DIM = 512;

struct StoreArgs {
    int nq, nkv, d, tokens;
    int64_t row_stride, q_stride;
    float eps;
    int rotary_dim, pairing;     // rotary_dim 0: no rotation; pairing 0: (2i, 2i+1)  1: (i, i + rotary_dim/2)
    int norm;                    // 0: none   1: with the weights q_w / k_w   2: without weights
    int v_head0;                 // the values of kv head g are columns (v_head0 + g) * d .. of a row
    float temp_coef;             // q *= 1 + temp_coef * ln(floor((pos + 1) / temp_every) + 1); temp_every 0: none
    int temp_every;
    int n_blocks, blocks_per_page, block, page_size;
    int64_t all_blocks;          // of the pool
    int lanes;                   // lanes a head, a power of two: 8 channels each
};

// Channels of the pair p: neighbours, or half the rotated channels apart; behind the rotated ones neighbours again.
__device__ __forceinline__ void channels_of(const StoreArgs& a, int p, int& ia, int& ib) {
    const int half = a.rotary_dim / 2;
    if (p < half) {
        ia = a.pairing == 0 ? 2 * p : p;
        ib = a.pairing == 0 ? 2 * p + 1 : p + half;
    } else {
        ia = a.rotary_dim + 2 * (p - half);
        ib = ia + 1;
    }
}

// Four pairs (lane c: 4 c .. 4 c + 3) of a head's row as float32, x[i] and y[i] the pair's two.  WHOLE: d and rotary_dim are multiples of
// 8 and rows are aligned, so that the eight channels lie in one piece of 8 or two of 4.
template <typename T, bool WHOLE>
__device__ __forceinline__ void read_pairs(const StoreArgs& a, const T* row, int c, float (&x)[4], float (&y)[4]) {
    if constexpr (WHOLE) {
        const bool apart = a.pairing == 1 && 8 * c < a.rotary_dim;
        const int first = apart ? 4 * c : 8 * c, second = apart ? first + a.rotary_dim / 2 : first + 4;
        float one[4], two[4];
        if constexpr (sizeof(T) == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(row + first), w = *reinterpret_cast<const uint2*>(row + second);
            one[0] = __uint_as_float(u.x << 16), one[1] = __uint_as_float(u.x & 0xffff0000u);
            one[2] = __uint_as_float(u.y << 16), one[3] = __uint_as_float(u.y & 0xffff0000u);
            two[0] = __uint_as_float(w.x << 16), two[1] = __uint_as_float(w.x & 0xffff0000u);
            two[2] = __uint_as_float(w.y << 16), two[3] = __uint_as_float(w.y & 0xffff0000u);
        } else {
            const float4 u = *reinterpret_cast<const float4*>(row + first), w = *reinterpret_cast<const float4*>(row + second);
            one[0] = u.x, one[1] = u.y, one[2] = u.z, one[3] = u.w;
            two[0] = w.x, two[1] = w.y, two[2] = w.z, two[3] = w.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = apart ? one[i] : (i < 2 ? one[2 * i] : two[2 * i - 4]);
            y[i] = apart ? two[i] : (i < 2 ? one[2 * i + 1] : two[2 * i - 3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int ia, ib;
            channels_of(a, 4 * c + i, ia, ib);
            const bool on = 2 * (4 * c + i) < a.d;
            x[i] = on ? to_f32<T>(row[ia]) : 0.f;
            y[i] = on ? to_f32<T>(row[ib]) : 0.f;
        }
    }
}

// Norm and rotation of those pairs; the sum of squares runs over the head's `lanes` neighbouring lanes.
template <typename TW, bool WHOLE>
__device__ __forceinline__ void prepare_pairs(const StoreArgs& a, const TW* w, const float* cos_t, const float* sin_t, int64_t t, int c,
                                              float factor, float (&x)[4], float (&y)[4]) {
    const int half = a.rotary_dim / 2;
    if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += x[i] * x[i] + y[i] * y[i];
        for (int step = 1; step < a.lanes; step *= 2) ss += __shfl_xor(ss, step);
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.d) + a.eps);
        float wx[4], wy[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) wx[i] = wy[i] = 1.f;
        if (w && 8 * c < a.d) read_pairs<TW, WHOLE>(a, w, c, wx, wy);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = x[i] * inv * wx[i];
            y[i] = y[i] * inv * wy[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] *= factor;
        y[i] *= factor;
        const int p = 4 * c + i;
        if (p < half) {
            const float cs = cos_t[t * half + p], sn = sin_t[t * half + p];
            const float u = x[i] * cs - y[i] * sn, v = x[i] * sn + y[i] * cs;
            x[i] = u;
            y[i] = v;
        }
    }
}

template <typename T, typename TW, bool WHOLE>
__global__ __launch_bounds__(THREADS) void store8_kernel(const T* qkv, T* q_out, const TW* __restrict__ q_w,
                                                         const TW* __restrict__ k_w, const float* __restrict__ cos_t,
                                                         const float* __restrict__ sin_t, uint8_t* __restrict__ keys,
                                                         uint8_t* __restrict__ values, float* __restrict__ scales,
                                                         const int* __restrict__ positions, const int4* __restrict__ work, StoreArgs a) {
    const int tid = threadIdx.x;
    const int c = tid % a.lanes;
    const int heads_at_once = THREADS / a.lanes;
    const bool on = 8 * c < a.d;
    const int block_groups = a.n_blocks * a.nkv;
    if (static_cast<int>(blockIdx.x) >= block_groups) {
        // q: neighbouring groups of lanes take neighbouring heads of the rows in turn
        const int64_t i = static_cast<int64_t>(blockIdx.x - block_groups) * heads_at_once + tid / a.lanes;
        const bool live = i < static_cast<int64_t>(a.tokens) * a.nq;
        const int64_t t = live ? i / a.nq : 0;
        const int h = live ? static_cast<int>(i - t * a.nq) : 0;
        const T* row = qkv + t * a.row_stride + static_cast<int64_t>(h) * a.d;
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
        if (on) read_pairs<T, WHOLE>(a, row, c, x, y);
        float factor = 1.f;
        if (a.temp_every > 0) factor = 1.f + a.temp_coef * logf(static_cast<float>((positions[t] + 1) / a.temp_every) + 1.f);
        prepare_pairs<TW, WHOLE>(a, q_w, cos_t, sin_t, t, c, factor, x, y);
        if (!on || !live) return;
        T* to = q_out + t * a.q_stride + static_cast<int64_t>(h) * a.d;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            int ia, ib;
            channels_of(a, 4 * c + i4, ia, ib);
            if (2 * (4 * c + i4) < a.d) {
                to[ia] = from_f32<T>(x[i4]);
                to[ib] = from_f32<T>(y[i4]);
            }
        }
        return;
    }

    __shared__ float s_max[2][THREADS / PULSE_WAVE];
    __shared__ int s_bad;
    const int4 job = work[blockIdx.x / a.nkv];
    const int g = blockIdx.x % a.nkv;
    const int first = job.x, rows = job.y, at = job.w;
    // (a list that says anything else is not followed)
    if (rows <= 0 || job.z < 0 || job.z >= a.all_blocks || at < 0 || at + rows > a.block || first < 0 || first + rows > a.tokens) return;
    const int64_t page = job.z / a.blocks_per_page;
    const int inner = job.z - static_cast<int>(page) * a.blocks_per_page;
    const int64_t head = page * a.nkv + g;
    uint8_t* kb = keys + (head * a.page_size + static_cast<int64_t>(inner) * a.block) * a.d;      // [token][channel]
    uint8_t* vb = values + (head * a.page_size + static_cast<int64_t>(inner) * a.block) * a.d;    // [channel][token]
    float* sc = scales + (head * a.blocks_per_page + inner) * 2;
    const bool fresh = at == 0;
    const float had_k = fresh ? 0.f : sc[0], had_v = fresh ? 0.f : sc[1];

    auto key_pairs = [&](int j, float (&x)[4], float (&y)[4]) {
        const int64_t t = first + min(j, rows - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = y[i] = 0.f;
        if (on) read_pairs<T, WHOLE>(a, qkv + t * a.row_stride + static_cast<int64_t>(a.nq + g) * a.d, c, x, y);
        prepare_pairs<TW, WHOLE>(a, k_w, cos_t, sin_t, t, c, 1.f, x, y);
    };
    // values: a thread takes a pair of neighbouring channels and every `groups`-th token
    const int pairs = a.d / 2, groups = max(1, THREADS / pairs);
    const int vc = 2 * (tid % pairs), vg = tid / pairs;
    const bool v_on = vg < groups;
    const T* vrow = qkv + static_cast<int64_t>(a.v_head0 + g) * a.d + vc;

    float kmax = 0.f, vmax = 0.f;
    int bad = 0;
    for (int j0 = 0; j0 < rows; j0 += heads_at_once) {
        float x[4], y[4];
        key_pairs(j0 + tid / a.lanes, x, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kmax = fmaxf(kmax, cache8::finite(x[i]) ? fabsf(x[i]) : 0.f);
            kmax = fmaxf(kmax, cache8::finite(y[i]) ? fabsf(y[i]) : 0.f);
        }
    }
    for (int j = vg; j < rows && v_on; j += groups) {
        const T* v = vrow + (first + j) * a.row_stride;
        const float x = to_f32<T>(v[0]), y = to_f32<T>(v[1]);
        vmax = fmaxf(vmax, fmaxf(cache8::finite(x) ? fabsf(x) : 0.f, cache8::finite(y) ? fabsf(y) : 0.f));
        bad |= !cache8::finite(x) | !cache8::finite(y);
    }
    kmax = wave_max(kmax);
    vmax = wave_max(vmax);
    if (tid == 0) s_bad = 0;
    __syncthreads();
    if (bad) s_bad = 1;
    if (tid % PULSE_WAVE == 0) {
        s_max[0][tid / PULSE_WAVE] = kmax;
        s_max[1][tid / PULSE_WAVE] = vmax;
    }
    __syncthreads();
    kmax = vmax = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / PULSE_WAVE; ++w) {
        kmax = fmaxf(kmax, s_max[0][w]);
        vmax = fmaxf(vmax, s_max[1][w]);
    }
    const int was_k = fresh ? cache8::LEAST : cache8::exponent_of(had_k), was_v = fresh ? cache8::LEAST : cache8::exponent_of(had_v);
    const int ek = max(was_k, cache8::exponent_for(kmax)), ev = max(was_v, cache8::exponent_for(vmax));
    const float by_k = cache8::pow2(-ek), by_v = cache8::pow2(-ev);

    // what the block holds besides the new tokens: nothing (a block that is begun: zeros behind them), or earlier bytes at their scale
    if (fresh || ek != was_k) {
        const float down = cache8::pow2(max(was_k - ek, -126));
        for (int i = tid; i < a.block * a.d; i += THREADS) {
            const int token = i / a.d;
            if (token < at || token >= at + rows) kb[i] = fresh ? 0 : static_cast<uint8_t>(cache8::moved(kb[i], down));
        }
    }
    if (fresh || ev != was_v) {
        const float down = cache8::pow2(max(was_v - ev, -126));
        for (int i = tid; i < a.block * a.d; i += THREADS) {
            const int token = i % a.block;
            if (token < at || token >= at + rows) vb[i] = fresh ? 0 : static_cast<uint8_t>(cache8::moved(vb[i], down));
        }
    }
    for (int j0 = 0; j0 < rows; j0 += heads_at_once) {
        float x[4], y[4];
        const int j = j0 + tid / a.lanes;
        key_pairs(j, x, y);
        if (j >= rows || !on) continue;
        uint8_t* to = kb + static_cast<int64_t>(at + j) * a.d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int ia, ib;
            channels_of(a, 4 * c + i, ia, ib);
            if (2 * (4 * c + i) < a.d) {
                const uint32_t both = cache8::to_e4m3x2(x[i] * by_k, y[i] * by_k);
                to[ia] = static_cast<uint8_t>(both);
                to[ib] = static_cast<uint8_t>(both >> 8);
            }
        }
    }
    for (int j = vg; j < rows && v_on; j += groups) {
        const T* v = vrow + (first + j) * a.row_stride;
        const uint32_t both = cache8::to_e4m3x2(to_f32<T>(v[0]) * by_v, to_f32<T>(v[1]) * by_v);
        uint8_t* to = vb + static_cast<int64_t>(vc) * a.block + at + j;
        to[0] = static_cast<uint8_t>(both);
        to[a.block] = static_cast<uint8_t>(both >> 8);
    }
    if (tid == 0) {
        const bool marked = s_bad || (!fresh && had_v < 0.f);
        sc[0] = cache8::pow2(ek);
        sc[1] = marked ? -cache8::pow2(ev) : cache8::pow2(ev);
    }
}

}  // namespace

extern "C" int pulse_store8(const void* qkv, int x_dtype, int64_t row_stride, void* q_out, int64_t q_stride, const void* q_w,
                            const void* k_w, int w_dtype, float eps, const float* cos_t, const float* sin_t, int rotary_dim, int pairing,
                            void* keys, void* values, float* scales, int num_pages, int page_size, const int* positions, const int* work,
                            int n_blocks, int tokens, int nq, int nkv, int d, int plain_norm, int v_head0, float temp_coef,
                            int temp_every, hipStream_t stream) {
    PULSE_REQUIRE(pulse_dtype_ok(x_dtype) && pulse_dtype_ok(w_dtype), "store8: unknown storage type");
    PULSE_REQUIRE(tokens >= 0 && n_blocks >= 0 && nq > 0 && nkv > 0 && num_pages > 0 && page_size > 0 && v_head0 >= 0, "store8: bad sizes");
    PULSE_REQUIRE(d >= 2 && d % 2 == 0 && d <= MAX_DIM, "store8: heads of %d channels (even, up to %d)", d, MAX_DIM);
    PULSE_REQUIRE(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= d && (pairing == 0 || pairing == 1), "store8: bad rotation");
    PULSE_REQUIRE(rotary_dim == 0 || (cos_t && sin_t), "store8: the rotation's tables are missing");
    PULSE_REQUIRE(!(q_w == nullptr) == !(k_w == nullptr) && !(plain_norm && q_w), "store8: bad norm options");
    PULSE_REQUIRE(temp_every >= 0 && (temp_every == 0 || positions), "store8: bad query temperature");
    PULSE_REQUIRE(qkv && q_out && keys && values && scales && (n_blocks == 0 || work), "store8: an operand is missing");
    PULSE_REQUIRE((reinterpret_cast<uintptr_t>(work) & 15) == 0, "store8: the work list must be aligned to 16 bytes");
    if (tokens == 0) return 0;
    const int block = cache8::block_tokens(page_size);
    int lanes = 1;
    while (lanes * 8 < d) lanes *= 2;
    StoreArgs a{nq, nkv, d, tokens, row_stride, q_stride, eps, rotary_dim, pairing, q_w ? 1 : plain_norm ? 2 : 0, v_head0, temp_coef, temp_every,
                n_blocks, page_size / block, block, page_size, static_cast<int64_t>(num_pages) * (page_size / block), lanes};
    const int64_t q_groups = (static_cast<int64_t>(tokens) * nq + THREADS / lanes - 1) / (THREADS / lanes);
    const int64_t grid = q_groups + static_cast<int64_t>(n_blocks) * nkv;
    PULSE_REQUIRE(grid <= 0x7fffffff, "store8: too many rows");
    const int size = x_dtype == PULSE_F32 ? 4 : 2, w_size = w_dtype == PULSE_F32 ? 4 : 2;
    auto aligned = [](const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
    const bool whole = d % 8 == 0 && rotary_dim % 8 == 0 && row_stride % 4 == 0 && aligned(qkv, 4 * size) && aligned(q_w, 4 * w_size) &&
                       aligned(k_w, 4 * w_size);
    auto go = [&](auto x, auto w, auto v) {
        using T = decltype(x);
        using TW = decltype(w);
        store8_kernel<T, TW, decltype(v)::value><<<static_cast<int>(grid), THREADS, 0, stream>>>(
            static_cast<const T*>(qkv), static_cast<T*>(q_out), static_cast<const TW*>(q_w), static_cast<const TW*>(k_w), cos_t, sin_t,
            static_cast<uint8_t*>(keys), static_cast<uint8_t*>(values), scales, positions, reinterpret_cast<const int4*>(work), a);
    };
    auto by_weight = [&](auto x, auto v) {
        if (w_dtype == PULSE_F32) go(x, float(), v);
        else go(x, bf16_t(), v);
    };
    auto by_type = [&](auto v) {
        if (x_dtype == PULSE_F32) by_weight(float(), v);
        else by_weight(bf16_t(), v);
    };
    if (whole) by_type(std::true_type());
    else by_type(std::false_type());
    PULSE_LAUNCH_CHECK("store8");
    return 0;
}

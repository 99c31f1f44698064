// A step's rows of the fused projection into a cache in 8 bits (cache8.h): per-head RMSNorm and rotation of q and k, q to its rows,
// k and v to the blocks that the step writes to.
//
//   x <- x / sqrt(mean(x^2) + eps) * w          per head of q and k, if there is a norm
//   (x_a, x_b) <- (x_a cos - x_b sin, x_a sin + x_b cos)   per pair of the first rotary_dim channels
//   block: e = max(e of what it holds, the least e with max |x| <= 448 * 2^e of the new ones); byte = e4m3(x * 2^-e)
//
// A workgroup takes a (block, kv head): a block's scale needs all of its tokens, and its earlier bytes move when the scale grows, so
// whoever else wrote to the block in the same step would race.  Workgroups behind those take q's heads.  All arithmetic is float32; k and
// v are rounded once, to 8 bits, and never to bfloat16 in between.  Some tens to 256 rows may come as the projection's shares: a prompt of
// 23 tokens, 36 layers of 32 heads on 8 of 128, takes 3,640 us with them and 4,048 from a product that adds them up itself.
//
// Bound: decoding, a launch's latency and the chain work list -> rows -> largest value -> bytes (32 heads on 8 of 128, in a recording: one
// token 4.4 us, 64 tokens 5.7); prompts, the reading of the projection and the writing of q (2,048 tokens 14.3 us for 46 MB, 3.2 TB/s of
// the 4.8 that a copy of 2 GB reaches; 15.3 with the hardware's divisions in the place of multiplications and shifts).  Two or four heads
// of q a thread: 15.6 and 17.8 us for 15.3.
#include "cache8.h"

#include <algorithm>

namespace {

constexpr int THREAD_BITS = 8, THREADS = 1 << THREAD_BITS;
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
    int n_blocks, block, page_size;
    cache8::Div blocks_per_page, q_heads, kv_heads, pairs;      // (pairs: d / 2)
    int64_t all_blocks;          // of the pool
    int lanes, lane_bits;        // lanes a head, a power of two: 8 channels each
    const float* parts;          // the rows as float32 shares of the projection, added up here in their order; null: qkv's
    int shares;
    int64_t part_stride, part_row;
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

// The same of a row that comes as shares: whole pieces, the shares asked for together.
__device__ __forceinline__ void read_shares(const StoreArgs& a, const float* row, int c, float (&x)[4], float (&y)[4]) {
    read_pairs<float, true>(a, row, c, x, y);
#pragma unroll 4
    for (int s = 1; s < a.shares; ++s) {
        float u[4], v[4];
        read_pairs<float, true>(a, row + s * a.part_stride, c, u, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] += u[i];
            y[i] += v[i];
        }
    }
}
template <typename T, bool WHOLE, bool PARTS>
__device__ __forceinline__ void read_head(const StoreArgs& a, const T* qkv, int64_t t, int64_t head, int c, float (&x)[4], float (&y)[4]) {
    if constexpr (PARTS) read_shares(a, a.parts + t * a.part_row + head * a.d, c, x, y);
    else read_pairs<T, WHOLE>(a, qkv + t * a.row_stride + head * a.d, c, x, y);
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
    }
    auto turn = [&](int i, float cs, float sn) {
        const float u = x[i] * cs - y[i] * sn, v = x[i] * sn + y[i] * cs;
        x[i] = u;
        y[i] = v;
    };
    if constexpr (WHOLE) {       // (four pairs are rotated, or none of them)
        if (4 * c < half) {
            const float4 cs = *reinterpret_cast<const float4*>(cos_t + t * half + 4 * c), sn = *reinterpret_cast<const float4*>(sin_t + t * half + 4 * c);
            turn(0, cs.x, sn.x), turn(1, cs.y, sn.y), turn(2, cs.z, sn.z), turn(3, cs.w, sn.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * c + i < half) turn(i, cos_t[t * half + 4 * c + i], sin_t[t * half + 4 * c + i]);
    }
}

// Those pairs of a row of q to their places.
template <typename T, bool WHOLE>
__device__ __forceinline__ void write_pairs(const StoreArgs& a, T* to, int c, const float (&x)[4], const float (&y)[4]) {
    if constexpr (WHOLE) {
        const bool apart = a.pairing == 1 && 8 * c < a.rotary_dim;
        float one[4], two[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            one[i] = apart ? x[i] : (i % 2 ? y[i / 2] : x[i / 2]);
            two[i] = apart ? y[i] : (i % 2 ? y[2 + i / 2] : x[2 + i / 2]);
        }
        const int first = apart ? 4 * c : 8 * c, second = apart ? first + a.rotary_dim / 2 : first + 4;
        if constexpr (sizeof(T) == 2) {
            auto pack = [](const float* v) {
                return make_uint2(f32_to_bf16(v[0]) | static_cast<uint32_t>(f32_to_bf16(v[1])) << 16, f32_to_bf16(v[2]) | static_cast<uint32_t>(f32_to_bf16(v[3])) << 16);
            };
            *reinterpret_cast<uint2*>(to + first) = pack(one);
            *reinterpret_cast<uint2*>(to + second) = pack(two);
        } else {
            *reinterpret_cast<float4*>(to + first) = make_float4(one[0], one[1], one[2], one[3]);
            *reinterpret_cast<float4*>(to + second) = make_float4(two[0], two[1], two[2], two[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int ia, ib;
            channels_of(a, 4 * c + i, ia, ib);
            if (2 * (4 * c + i) < a.d) {
                to[ia] = from_f32<T>(x[i]);
                to[ib] = from_f32<T>(y[i]);
            }
        }
    }
}

// A workgroup's share of q: neighbouring groups of lanes take neighbouring heads of the rows in turn.
template <typename T, typename TW, bool WHOLE, bool PARTS>
__device__ __forceinline__ void rows_of_q(const StoreArgs& a, int first, const T* qkv, T* q_out, const TW* q_w, const float* cos_t,
                                          const float* sin_t, const int* positions) {
    const int tid = threadIdx.x, c = tid & (a.lanes - 1);
    const int i = (first << (THREAD_BITS - a.lane_bits)) + (tid >> a.lane_bits);       // (rows times heads are less than 2^31)
    const bool live = i < a.tokens * a.nq, on = 8 * c < a.d;
    const int row = live ? a.q_heads.over(i) : 0, h = live ? i - row * a.nq : 0;
    const int64_t t = row;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    if (on) read_head<T, WHOLE, PARTS>(a, qkv, t, h, c, x, y);
    float factor = 1.f;
    if (a.temp_every > 0) factor = 1.f + a.temp_coef * logf(static_cast<float>((positions[t] + 1) / a.temp_every) + 1.f);
    prepare_pairs<TW, WHOLE>(a, q_w, cos_t, sin_t, t, c, factor, x, y);
    if (on && live) write_pairs<T, WHOLE>(a, q_out + t * a.q_stride + static_cast<int64_t>(h) * a.d, c, x, y);
}

// The largest finite |x| of the keys and of the values that the workgroup's threads have, and whether a value is none.
__device__ __forceinline__ void largest(float& kmax, float& vmax, bool& bad) {
    __shared__ float s_max[2][THREADS / PULSE_WAVE];
    __shared__ int s_bad[THREADS / PULSE_WAVE];
    const int wave = threadIdx.x / PULSE_WAVE;
    kmax = wave_max(kmax);
    vmax = wave_max(vmax);
    const bool any = __any(bad);
    if (threadIdx.x % PULSE_WAVE == 0) {
        s_max[0][wave] = kmax;
        s_max[1][wave] = vmax;
        s_bad[wave] = any;
    }
    __syncthreads();
    kmax = vmax = 0.f;
    bad = false;
#pragma unroll
    for (int w = 0; w < THREADS / PULSE_WAVE; ++w) {
        kmax = fmaxf(kmax, s_max[0][w]);
        vmax = fmaxf(vmax, s_max[1][w]);
        bad |= s_bad[w] != 0;
    }
}
__device__ __forceinline__ float size_of(float x) { return cache8::finite(x) ? fabsf(x) : 0.f; }

// What a workgroup of a (block, kv head) has to do, or nothing (a list that says what cannot be is not followed).
struct Job {
    int first, rows, at, g;
    uint8_t *keys, *values;      // the block's, of this head: [token][channel], [channel][token]
    float* scale;
};
__device__ __forceinline__ bool job_of(const StoreArgs& a, const int4* work, uint8_t* keys, uint8_t* values, float* scales, Job& j) {
    const int place = a.kv_heads.over(blockIdx.x);
    const int4 w = work[place];
    j.g = blockIdx.x - place * a.nkv;
    j.first = w.x, j.rows = w.y, j.at = w.w;
    if (w.y <= 0 || w.z < 0 || w.z >= a.all_blocks || w.w < 0 || w.w >= a.block || w.y > a.block - w.w || w.x < 0 || w.y > a.tokens ||
        w.x > a.tokens - w.y)
        return false;
    const int page = a.blocks_per_page.over(w.z), inner = w.z - page * a.blocks_per_page.b;
    const int64_t head = static_cast<int64_t>(page) * a.nkv + j.g;
    j.keys = keys + (head * a.page_size + static_cast<int64_t>(inner) * a.block) * a.d;
    j.values = values + (head * a.page_size + static_cast<int64_t>(inner) * a.block) * a.d;
    j.scale = scales + (head * a.blocks_per_page.b + inner) * 2;
    return true;
}

// Blocks of 16 tokens and heads of a multiple of 8 channels, NP * 128 at most, in whole pieces: what is read is kept in registers until
// the scale is known.  Keys: a group of lanes takes a token's row.  Values: a thread takes a pair of channels and four of the block's
// tokens, whose bytes are a word; a word that holds earlier tokens too is put together with them.  PARTS: the rows are shares.
template <typename T, typename TW, int NP, bool PARTS>
__global__ __launch_bounds__(THREADS) void store8_blocks_kernel(const T* qkv, T* q_out, const TW* __restrict__ q_w, const TW* __restrict__ k_w,
                                                                const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                                uint8_t* keys, uint8_t* values, float* scales, const int* __restrict__ positions,
                                                                const int4* __restrict__ work, StoreArgs a) {
    const int tid = threadIdx.x, block_groups = a.n_blocks * a.nkv;
    if (static_cast<int>(blockIdx.x) >= block_groups) {
        rows_of_q<T, TW, true, PARTS>(a, blockIdx.x - block_groups, qkv, q_out, q_w, cos_t, sin_t, positions);
        return;
    }
    Job j;
    if (!job_of(a, work, keys, values, scales, j)) return;
    const int c = tid & (a.lanes - 1), at_once = THREADS >> a.lane_bits, of_lanes = tid >> a.lane_bits, d = a.d;
    const bool on = 8 * c < d, fresh = j.at == 0;
    const float had_k = fresh ? 0.f : j.scale[0], had_v = fresh ? 0.f : j.scale[1];
    const int pairs = d / 2, quad = a.pairs.over(tid), vc = 2 * (tid - quad * pairs);      // (of the first NP; the others are THREADS / pairs quads further on)
    const int quads_at_once = a.pairs.over(THREADS);

    // everything that is read is asked for before anything waits
    float kx[NP][4], ky[NP][4], vx[NP][4], vy[NP][4];
    uint32_t old[NP][2];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int i = n * at_once + of_lanes;
#pragma unroll
        for (int e = 0; e < 4; ++e) kx[n][e] = ky[n][e] = vx[n][e] = vy[n][e] = 0.f;
        if (on && i < j.rows) read_head<T, true, PARTS>(a, qkv, j.first + i, a.nq + j.g, c, kx[n], ky[n]);
        const int qd = quad + n * quads_at_once;
        old[n][0] = old[n][1] = 0;
        if (quad < quads_at_once && qd < 4) {
            if (!fresh) {
                old[n][0] = *reinterpret_cast<const uint32_t*>(j.values + vc * 16 + qd * 4);
                old[n][1] = *reinterpret_cast<const uint32_t*>(j.values + vc * 16 + 16 + qd * 4);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 4 * qd + e - j.at;
                if (row >= 0 && row < j.rows) {
                    const int64_t column = static_cast<int64_t>(a.v_head0 + j.g) * d + vc;
                    const T* v = qkv + static_cast<int64_t>(j.first + row) * a.row_stride + column;
                    if constexpr (PARTS) {
                        const float* part = a.parts + static_cast<int64_t>(j.first + row) * a.part_row + column;
#pragma unroll 4
                        for (int s = 0; s < a.shares; ++s) {
                            const float2 u = *reinterpret_cast<const float2*>(part + s * a.part_stride);
                            vx[n][e] += u.x, vy[n][e] += u.y;
                        }
                    } else if constexpr (sizeof(T) == 2) {
                        const uint32_t u = *reinterpret_cast<const uint32_t*>(v);
                        vx[n][e] = __uint_as_float(u << 16), vy[n][e] = __uint_as_float(u & 0xffff0000u);
                    } else {
                        const float2 u = *reinterpret_cast<const float2*>(v);
                        vx[n][e] = u.x, vy[n][e] = u.y;
                    }
                }
            }
        }
    }
    float kmax = 0.f, vmax = 0.f;
    bool bad = false;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int i = n * at_once + of_lanes;
        prepare_pairs<TW, true>(a, k_w, cos_t, sin_t, j.first + min(i, j.rows - 1), c, 1.f, kx[n], ky[n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i < j.rows) kmax = fmaxf(kmax, fmaxf(size_of(kx[n][e]), size_of(ky[n][e])));
            vmax = fmaxf(vmax, fmaxf(size_of(vx[n][e]), size_of(vy[n][e])));
            bad |= !cache8::finite(vx[n][e]) | !cache8::finite(vy[n][e]);
        }
    }
    largest(kmax, vmax, bad);
    const int was_k = fresh ? cache8::LEAST : cache8::exponent_of(had_k), was_v = fresh ? cache8::LEAST : cache8::exponent_of(had_v);
    const int ek = max(was_k, cache8::exponent_for(kmax)), ev = max(was_v, cache8::exponent_for(vmax));
    const float by_k = cache8::pow2(-ek), by_v = cache8::pow2(-ev);
    const bool grew_k = !fresh && ek != was_k, grew_v = !fresh && ev != was_v;
    const float down_k = cache8::pow2(max(was_k - ek, -126)), down_v = cache8::pow2(max(was_v - ev, -126));

#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int i = n * at_once + of_lanes;
        if (on && i < j.rows) {
            const bool apart = a.pairing == 1 && 8 * c < a.rotary_dim;
            const int first = apart ? 4 * c : 8 * c, second = apart ? first + a.rotary_dim / 2 : first + 4;
            uint32_t lo = 0, hi = 0;
            if (apart) {
                lo = cache8::to_e4m3x4(kx[n][0] * by_k, kx[n][1] * by_k, kx[n][2] * by_k, kx[n][3] * by_k);
                hi = cache8::to_e4m3x4(ky[n][0] * by_k, ky[n][1] * by_k, ky[n][2] * by_k, ky[n][3] * by_k);
            } else {
                lo = cache8::to_e4m3x4(kx[n][0] * by_k, ky[n][0] * by_k, kx[n][1] * by_k, ky[n][1] * by_k);
                hi = cache8::to_e4m3x4(kx[n][2] * by_k, ky[n][2] * by_k, kx[n][3] * by_k, ky[n][3] * by_k);
            }
            uint8_t* to = j.keys + (j.at + i) * d;
            *reinterpret_cast<uint32_t*>(to + first) = cache8::at_exponent(ek, lo);
            *reinterpret_cast<uint32_t*>(to + second) = cache8::at_exponent(ek, hi);
        }
        const int qd = quad + n * quads_at_once;
        if (quad < quads_at_once && qd < 4) {
            uint32_t fill = 0;       // the bytes of the new tokens
#pragma unroll
            for (int e = 0; e < 4; ++e) fill |= 4 * qd + e >= j.at && 4 * qd + e < j.at + j.rows ? 0xffu << (8 * e) : 0u;
            if (fill || fresh || grew_v) {
                uint32_t x = old[n][0], y = old[n][1];
                if (grew_v) x = cache8::moved(x, down_v), y = cache8::moved(y, down_v);
                x = (x & ~fill) | (cache8::to_e4m3x4(vx[n][0] * by_v, vx[n][1] * by_v, vx[n][2] * by_v, vx[n][3] * by_v) & fill);
                y = (y & ~fill) | (cache8::to_e4m3x4(vy[n][0] * by_v, vy[n][1] * by_v, vy[n][2] * by_v, vy[n][3] * by_v) & fill);
                *reinterpret_cast<uint32_t*>(j.values + vc * 16 + qd * 4) = cache8::at_exponent(ev, x);
                *reinterpret_cast<uint32_t*>(j.values + vc * 16 + 16 + qd * 4) = cache8::at_exponent(ev, y);
            }
        }
    }
    if ((fresh && j.rows < 16) || grew_k) {
        // the keys around the new ones: zeros in a block that is begun, else at their new scale
        uint32_t* all = reinterpret_cast<uint32_t*>(j.keys);
        const int begin = j.at * d / 4, end = (j.at + j.rows) * d / 4;
        for (int i = tid; i < 4 * d; i += THREADS)
            if (i < begin || i >= end) all[i] = fresh ? 0u : cache8::moved(all[i], down_k);
    }
    if (tid == 0) {
        j.scale[0] = cache8::pow2(ek);
        j.scale[1] = bad || (!fresh && had_v < 0.f) ? -cache8::pow2(ev) : cache8::pow2(ev);
    }
}

// Every size: two readings, the first for the scale, and bytes one by one (32 heads on 8 of 128, pages of 8, us: one token 7.2, 64 single ones 10,
// 2,048 tokens 41; in blocks of 16 4.4, 5.7, 14.3).
template <typename T, typename TW>
__global__ __launch_bounds__(THREADS) void store8_kernel(const T* qkv, T* q_out, const TW* __restrict__ q_w, const TW* __restrict__ k_w,
                                                         const float* __restrict__ cos_t, const float* __restrict__ sin_t, uint8_t* keys,
                                                         uint8_t* values, float* scales, const int* __restrict__ positions,
                                                         const int4* __restrict__ work, StoreArgs a) {
    const int tid = threadIdx.x, block_groups = a.n_blocks * a.nkv;
    if (static_cast<int>(blockIdx.x) >= block_groups) {
        rows_of_q<T, TW, false, false>(a, blockIdx.x - block_groups, qkv, q_out, q_w, cos_t, sin_t, positions);
        return;
    }
    Job j;
    if (!job_of(a, work, keys, values, scales, j)) return;
    const int c = tid & (a.lanes - 1), at_once = THREADS >> a.lane_bits, of_lanes = tid >> a.lane_bits, d = a.d;
    const bool on = 8 * c < d, fresh = j.at == 0;
    const float had_k = fresh ? 0.f : j.scale[0], had_v = fresh ? 0.f : j.scale[1];
    auto key_pairs = [&](int i, float (&x)[4], float (&y)[4]) {
        const int64_t t = j.first + min(i, j.rows - 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = y[e] = 0.f;
        if (on) read_pairs<T, false>(a, qkv + t * a.row_stride + static_cast<int64_t>(a.nq + j.g) * d, c, x, y);
        prepare_pairs<TW, false>(a, k_w, cos_t, sin_t, t, c, 1.f, x, y);
    };
    // values: a thread takes a pair of neighbouring channels and every `groups`-th token
    const int groups = a.pairs.over(THREADS), vg = a.pairs.over(tid), vc = 2 * (tid - vg * (d / 2));
    const T* vrow = qkv + static_cast<int64_t>(j.first) * a.row_stride + static_cast<int64_t>(a.v_head0 + j.g) * d + vc;
    float kmax = 0.f, vmax = 0.f;
    bool bad = false;
    for (int i0 = 0; i0 < j.rows; i0 += at_once) {
        float x[4], y[4];
        key_pairs(i0 + of_lanes, x, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) kmax = fmaxf(kmax, fmaxf(size_of(x[e]), size_of(y[e])));
    }
    for (int i = vg; i < j.rows && vg < groups; i += groups) {
        const float x = to_f32<T>(vrow[i * a.row_stride]), y = to_f32<T>(vrow[i * a.row_stride + 1]);
        vmax = fmaxf(vmax, fmaxf(size_of(x), size_of(y)));
        bad |= !cache8::finite(x) | !cache8::finite(y);
    }
    largest(kmax, vmax, bad);
    const int was_k = fresh ? cache8::LEAST : cache8::exponent_of(had_k), was_v = fresh ? cache8::LEAST : cache8::exponent_of(had_v);
    const int ek = max(was_k, cache8::exponent_for(kmax)), ev = max(was_v, cache8::exponent_for(vmax));
    const float by_k = cache8::pow2(-ek), by_v = cache8::pow2(-ev);

    // what the block holds besides the new tokens: nothing (a block that is begun: zeros behind them), or earlier bytes at their scale
    auto around = [&](uint8_t* bytes, bool by_channel, float down) {
        for (int i = tid; i < a.block * d; i += THREADS) {
            const int token = by_channel ? i % a.block : i / d;
            if (token < j.at || token >= j.at + j.rows) bytes[i] = fresh ? 0 : static_cast<uint8_t>(cache8::moved(bytes[i], down));
        }
    };
    if (fresh || ek != was_k) around(j.keys, false, cache8::pow2(max(was_k - ek, -126)));
    if (fresh || ev != was_v) around(j.values, true, cache8::pow2(max(was_v - ev, -126)));
    for (int i0 = 0; i0 < j.rows; i0 += at_once) {
        float x[4], y[4];
        const int i = i0 + of_lanes;
        key_pairs(i, x, y);
        if (i >= j.rows || !on) continue;
        uint8_t* to = j.keys + static_cast<int64_t>(j.at + i) * d;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int ia, ib;
            channels_of(a, 4 * c + e, ia, ib);
            if (2 * (4 * c + e) < d) {
                const uint32_t both = cache8::at_exponent(ek, cache8::to_e4m3x2(x[e] * by_k, y[e] * by_k));
                to[ia] = static_cast<uint8_t>(both);
                to[ib] = static_cast<uint8_t>(both >> 8);
            }
        }
    }
    for (int i = vg; i < j.rows && vg < groups; i += groups) {
        const uint32_t both = cache8::at_exponent(ev, cache8::to_e4m3x2(to_f32<T>(vrow[i * a.row_stride]) * by_v, to_f32<T>(vrow[i * a.row_stride + 1]) * by_v));
        uint8_t* to = j.values + static_cast<int64_t>(vc) * a.block + j.at + i;
        to[0] = static_cast<uint8_t>(both);
        to[a.block] = static_cast<uint8_t>(both >> 8);
    }
    if (tid == 0) {
        j.scale[0] = cache8::pow2(ek);
        j.scale[1] = bad || (!fresh && had_v < 0.f) ? -cache8::pow2(ev) : cache8::pow2(ev);
    }
}

}  // namespace

// The entry point's arguments (ops/cache8.py fills it; the same fields in the same order).
struct PulseStore8 {
    const void* qkv;
    int64_t row_stride;
    void* q_out;
    int64_t q_stride;
    const void *q_w, *k_w;
    const float *cos_t, *sin_t;
    void *keys, *values;
    float* scales;
    const int *positions, *work;
    int x_dtype, w_dtype, rotary_dim, pairing, num_pages, page_size, n_blocks, tokens, nq, nkv, d, plain_norm, v_head0, temp_every;
    float eps, temp_coef;
    const float* parts;
    int64_t part_stride, part_row, shares;
};

extern "C" int pulse_store8(const PulseStore8* args, hipStream_t stream) {
    PULSE_REQUIRE(args != nullptr, "store8: no arguments");
    const PulseStore8& in = *args;
    const void *qkv = in.qkv, *q_w = in.q_w, *k_w = in.k_w;
    void *q_out = in.q_out, *keys = in.keys, *values = in.values;
    const float *cos_t = in.cos_t, *sin_t = in.sin_t;
    float* scales = in.scales;
    const int *positions = in.positions, *work = in.work;
    const int64_t row_stride = in.row_stride, q_stride = in.q_stride;
    const int x_dtype = in.x_dtype, w_dtype = in.w_dtype, rotary_dim = in.rotary_dim, pairing = in.pairing, num_pages = in.num_pages,
              page_size = in.page_size, n_blocks = in.n_blocks, tokens = in.tokens, nq = in.nq, nkv = in.nkv, d = in.d,
              plain_norm = in.plain_norm, v_head0 = in.v_head0, temp_every = in.temp_every;
    const float eps = in.eps, temp_coef = in.temp_coef;
    PULSE_REQUIRE(pulse_dtype_ok(x_dtype) && pulse_dtype_ok(w_dtype), "store8: unknown storage type");
    PULSE_REQUIRE(tokens >= 0 && n_blocks >= 0 && nq > 0 && nkv > 0 && num_pages > 0 && page_size > 0 && v_head0 >= 0, "store8: bad sizes");
    PULSE_REQUIRE(d >= 2 && d % 2 == 0 && d <= MAX_DIM, "store8: heads of %d channels (even, up to %d)", d, MAX_DIM);
    PULSE_REQUIRE(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= d && (pairing == 0 || pairing == 1), "store8: bad rotation");
    PULSE_REQUIRE(rotary_dim == 0 || (cos_t && sin_t), "store8: the rotation's tables are missing");
    PULSE_REQUIRE(!(q_w == nullptr) == !(k_w == nullptr) && !(plain_norm && q_w), "store8: bad norm options");
    PULSE_REQUIRE(temp_every >= 0 && (temp_every == 0 || positions), "store8: bad query temperature");
    PULSE_REQUIRE(qkv && q_out && keys && values && scales && (n_blocks == 0 || work), "store8: an operand is missing");
    const int64_t columns = static_cast<int64_t>(std::max(nq + nkv, v_head0 + nkv)) * d;
    PULSE_REQUIRE((reinterpret_cast<uintptr_t>(work) & 15) == 0, "store8: the work list must be aligned to 16 bytes");
    if (tokens == 0) return 0;
    const int block = cache8::block_tokens(page_size);
    int lanes = 1, lane_bits = 0;
    while (lanes * 8 < d) lanes *= 2, ++lane_bits;
    PULSE_REQUIRE(static_cast<int64_t>(tokens) * nq + THREADS <= 0x7fffffff, "store8: too many rows");
    StoreArgs a{nq, nkv, d, tokens, row_stride, q_stride, eps, rotary_dim, pairing, q_w ? 1 : plain_norm ? 2 : 0, v_head0, temp_coef, temp_every,
                n_blocks, block, page_size, cache8::div_by(page_size / block), cache8::div_by(nq), cache8::div_by(nkv), cache8::div_by(d / 2),
                static_cast<int64_t>(num_pages) * (page_size / block), lanes, lane_bits,
                in.parts, static_cast<int>(in.shares), in.part_stride, in.part_row};
    const int64_t q_groups = (static_cast<int64_t>(tokens) * nq + THREADS / lanes - 1) / (THREADS / lanes);
    const int64_t grid = q_groups + static_cast<int64_t>(n_blocks) * nkv;
    PULSE_REQUIRE(grid <= 0x7fffffff, "store8: too many rows");
    const int size = x_dtype == PULSE_F32 ? 4 : 2, w_size = w_dtype == PULSE_F32 ? 4 : 2;
    auto aligned = [](const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
    const bool whole = block == cache8::BLOCK && d % 8 == 0 && rotary_dim % 8 == 0 && row_stride % 4 == 0 && q_stride % 4 == 0 &&
                       aligned(qkv, 4 * size) && aligned(q_out, 4 * size) && aligned(q_w, 4 * w_size) && aligned(k_w, 4 * w_size) &&
                       aligned(cos_t, 16) && aligned(sin_t, 16) && aligned(keys, 4) && aligned(values, 4);
    PULSE_REQUIRE(!in.parts || (whole && x_dtype == PULSE_BF16 && in.shares > 0 && in.shares <= 64 && in.part_row >= columns &&
                                in.part_row % 4 == 0 && in.part_stride % 4 == 0 && aligned(in.parts, 16)),
                  "store8: shares need bfloat16 rows, aligned, in chunks of eight channels, and pages of a multiple of 16 tokens");
    auto go = [&](auto x, auto w) {
        using T = decltype(x);
        using TW = decltype(w);
        auto run = [&](auto kernel) {
            kernel<<<static_cast<int>(grid), THREADS, 0, stream>>>(
                static_cast<const T*>(qkv), static_cast<T*>(q_out), static_cast<const TW*>(q_w), static_cast<const TW*>(k_w), cos_t, sin_t,
                static_cast<uint8_t*>(keys), static_cast<uint8_t*>(values), scales, positions, reinterpret_cast<const int4*>(work), a);
        };
        auto by_width = [&](auto parts) {
            if (d <= 128) run(store8_blocks_kernel<T, TW, 1, decltype(parts)::value>);
            else if (d <= 256) run(store8_blocks_kernel<T, TW, 2, decltype(parts)::value>);
            else run(store8_blocks_kernel<T, TW, 4, decltype(parts)::value>);
        };
        if (!whole) {
            run(store8_kernel<T, TW>);
        } else {
            if constexpr (sizeof(T) == 2) {
                if (in.parts) return by_width(std::true_type());
            }
            by_width(std::false_type());
        }
    };
    auto by_weight = [&](auto x) {
        if (w_dtype == PULSE_F32) go(x, float());
        else go(x, bf16_t());
    };
    if (x_dtype == PULSE_F32) by_weight(float());
    else by_weight(bf16_t());
    PULSE_LAUNCH_CHECK("store8");
    return 0;
}

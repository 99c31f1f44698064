// Attention over a cache in 8 bits (cache8.h) for every size and storage type: a workgroup a (row, head), its four wavefronts share the
// keys, float32 throughout.
//
//   s_j = scale * q . k_j, capped: cap * tanh(s_j / cap);  seen: low <= j <= position, in pages that are there
//   o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m)), one pass with the running maximum m and sum
//
// A lane takes a key's score (its row of bytes in pieces of 16) and then channels of the sum, for which the weights go from lane to lane.
// A row that sees no key is zeros; a row of no entry (token_entry outside the table) is left as it is.  Keys and values that a row does
// not see are not multiplied, so that what is not finite stays with those who see it.
// It serves what the matrix-core kernels do not: float32 rows, heads that are no multiple of 32 channels, pages that are no multiple
// of 16 tokens.
#include "cache8_attn.h"

namespace {

constexpr int THREADS = 256, WAVES = THREADS / PULSE_WAVE, MAX_DIM = 512;

// 16 bytes from their place, whatever its alignment
template <bool WHOLE>
__device__ __forceinline__ uint4 piece(const uint8_t* p, int stride) {
    if constexpr (WHOLE) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = p[(4 * i) * stride] | (p[(4 * i + 1) * stride] << 8) | (p[(4 * i + 2) * stride] << 16) | (static_cast<uint32_t>(p[(4 * i + 3) * stride]) << 24);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// CH: channels a lane sums.  WHOLE: blocks of 16 tokens and heads of a multiple of 16 channels.
template <typename T, int CH, bool WHOLE>
__global__ __launch_bounds__(THREADS) void attn8_plain_kernel(PulseAttn8 a) {
    __shared__ float s_q[MAX_DIM];
    __shared__ float s_o[WAVES][MAX_DIM];
    __shared__ float s_m[WAVES], s_l[WAVES];
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid % PULSE_WAVE, wave = tid / PULSE_WAVE;
    const int entry = a.token_entry[row];
    if (entry < 0 || entry >= a.entries) return;
    const int pos = a.positions[row];
    const int g = h / (a.nq / a.nkv), d = a.d;
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride + static_cast<int64_t>(h) * d;
    for (int c = tid; c < MAX_DIM; c += THREADS) s_q[c] = c < d ? to_f32<T>(q[c]) : 0.f;
    __syncthreads();
    const int block = cache8::block_tokens(a.page_size), nb = a.page_size / block;
    const int lo = cache8::low_key(a.window, a.chunk, pos);
    const int* bt = a.table + static_cast<int64_t>(entry) * a.table_width;
    float m = -INFINITY, l = 0.f, acc[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = 0.f;

    for (int j0 = lo / PULSE_WAVE * PULSE_WAVE + wave * PULSE_WAVE; j0 <= pos; j0 += WAVES * PULSE_WAVE) {
        const int j = j0 + lane;
        const int pi = j / a.page_size;
        const int page = pi < a.table_width ? bt[pi] : -1;
        const bool seen = j >= lo && j <= pos && page >= 0 && page < a.num_pages;
        const int64_t head = static_cast<int64_t>(seen ? page : 0) * a.nkv + g;
        const int slot = seen ? j - pi * a.page_size : 0;
        const int64_t bn = head * nb + slot / block;
        float s = 0.f;
        const uint8_t* k = a.keys + (head * a.page_size + slot) * d;
        if (WHOLE) {
            for (int c = 0; c < d; c += 16) {
                const uint4 u = piece<true>(k + c, 1);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x[4];
                    cache8::from_e4m3x4(w[i], x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s += x[e] * s_q[c + 4 * i + e];
                }
            }
        } else {
            for (int c = 0; c < d; ++c) s += cache8::from_e4m3(k[c]) * s_q[c];
        }
        s *= a.scales[2 * bn] * a.scale;
        if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
        s = seen ? s : -INFINITY;
        const float top = fmaxf(m, wave_max(s));
        const float shift = top == -INFINITY ? 0.f : top;
        const float again = __expf(m - shift);       // (0 while nothing has been seen)
        const float p = __expf(s - shift);
        l = l * again + wave_sum(p);
        m = top;
#pragma unroll
        for (int i = 0; i < CH; ++i) acc[i] *= again;
        const uint64_t seen_keys = __ballot(seen);
        const float pv = seen ? p * fabsf(a.scales[2 * bn + 1]) : 0.f;
        if constexpr (WHOLE) {
#pragma unroll
            for (int b = 0; b < PULSE_WAVE / 16; ++b) {
                const uint32_t some = static_cast<uint32_t>(seen_keys >> (16 * b)) & 0xffffu;
                if (!some) continue;
                // (a block's keys lie in one page: the first that is seen says where)
                const int64_t at = __shfl(head, 16 * b + __builtin_ctz(some));
                const int inner = __shfl(slot, 16 * b + __builtin_ctz(some)) / 16;
                const uint8_t* v = a.values + (at * a.page_size + inner * 16) * d;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int c = lane + i * PULSE_WAVE;
                    const uint4 u = piece<true>(v + (c < d ? c : 0) * 16, 1);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x[4];
                        cache8::from_e4m3x4(w[e], x);
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            if (some >> (4 * e + f) & 1) acc[i] += __shfl(pv, 16 * b + 4 * e + f) * x[f];
                    }
                }
            }
        } else {
            for (uint64_t left = seen_keys; left; left &= left - 1) {
                const int n = __builtin_ctzll(left);
                const int64_t at = __shfl(head, n);
                const int sl = __shfl(slot, n);
                const float w = __shfl(pv, n);
                const uint8_t* v = a.values + (at * a.page_size + sl / block * block) * d + sl % block;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int c = lane + i * PULSE_WAVE;
                    if (c < d) acc[i] += w * cache8::from_e4m3(v[static_cast<int64_t>(c) * block]);
                }
            }
        }
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (lane + i * PULSE_WAVE < d) s_o[wave][lane + i * PULSE_WAVE] = acc[i];
    __syncthreads();
    const float sink = a.sink ? a.sink[h] : -INFINITY;
    float top = sink;
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s_m[w]);
    const float shift = top == -INFINITY ? 0.f : top;
    float total = a.sink ? __expf(sink - shift) : 0.f;
    for (int w = 0; w < WAVES; ++w) total += s_l[w] * __expf(s_m[w] - shift);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const T* gate = static_cast<const T*>(a.gate);
    T* out = static_cast<T*>(a.out) + row * a.o_stride + static_cast<int64_t>(h) * d;
    for (int c = tid; c < d; c += THREADS) {
        float o = 0.f;
        for (int w = 0; w < WAVES; ++w) o += s_o[w][c] * __expf(s_m[w] - shift);
        o *= inv;
        if (gate && a.gate_width == 0) o *= cache8::sigmoid_of(to_f32<T>(gate[row * a.gate_stride + h]));
        if (gate && c < a.gate_width) o *= cache8::sigmoid_of(to_f32<T>(gate[row * a.gate_stride + static_cast<int64_t>(h) * a.gate_width + c]));
        out[c] = from_f32<T>(o);
    }
}

}  // namespace

// What every entry point of this attention asks of its arguments.
int pulse_attn8_check(const PulseAttn8* a, const char* what) {
    PULSE_REQUIRE(a != nullptr, "%s: no arguments", what);
    PULSE_REQUIRE(pulse_dtype_ok(a->dtype), "%s: unknown storage type", what);
    PULSE_REQUIRE(a->tokens >= 0 && a->entries > 0 && a->table_width > 0 && a->nq > 0 && a->nkv > 0 && a->nq % a->nkv == 0 && a->d > 0 &&
                      a->page_size > 0 && a->num_pages > 0, "%s: bad sizes", what);
    PULSE_REQUIRE(a->window >= 0 && a->chunk >= 0 && !(a->window && a->chunk), "%s: a window and chunks at once, or a negative one", what);
    PULSE_REQUIRE(a->scale > 0.f && a->softcap >= 0.f, "%s: the scale must be positive and the cap not negative", what);
    PULSE_REQUIRE(a->gate_width >= 0 && a->gate_width <= a->d, "%s: %d gated channels of a head of %d", what, a->gate_width, a->d);
    PULSE_REQUIRE(((reinterpret_cast<uintptr_t>(a->keys) | reinterpret_cast<uintptr_t>(a->values)) & 15) == 0, "%s: pages must be aligned to 16 bytes", what);
    PULSE_REQUIRE(a->q && a->out && a->keys && a->values && a->scales && a->positions && a->table, "%s: an operand is missing", what);
    return 0;
}

extern "C" int pulse_attn8_plain(const PulseAttn8* a, hipStream_t stream) {
    if (int rc = pulse_attn8_check(a, "attn8_plain")) return rc;
    PULSE_REQUIRE(a->token_entry, "attn8_plain: an operand is missing");
    PULSE_REQUIRE(a->d <= MAX_DIM, "attn8_plain: heads of %d channels (up to %d)", a->d, MAX_DIM);
    PULSE_REQUIRE(a->nq <= 65535, "attn8_plain: too many heads");
    if (a->tokens == 0) return 0;
    const bool whole = a->page_size % cache8::BLOCK == 0 && a->d % 16 == 0;
    auto go = [&](auto t, auto ch, auto w) {
        attn8_plain_kernel<decltype(t), decltype(ch)::value, decltype(w)::value><<<dim3(a->tokens, a->nq), THREADS, 0, stream>>>(*a);
    };
    auto by_width = [&](auto t, auto w) {
        if (a->d <= 64) go(t, std::integral_constant<int, 1>(), w);
        else if (a->d <= 128) go(t, std::integral_constant<int, 2>(), w);
        else if (a->d <= 256) go(t, std::integral_constant<int, 4>(), w);
        else go(t, std::integral_constant<int, 8>(), w);
    };
    auto by_form = [&](auto t) {
        if (whole) by_width(t, std::true_type());
        else by_width(t, std::false_type());
    };
    if (a->dtype == PULSE_F32) by_form(float());
    else by_form(bf16_t());
    PULSE_LAUNCH_CHECK("attn8_plain");
    return 0;
}

// Attention over a cache in 8 bits (cache8.h) for every size and storage type: a workgroup a (row, head), its wavefronts share the
// keys, float32 throughout.
//
//   s_j = scale * q . k_j, capped: cap * tanh(s_j / cap);  seen: low <= j <= position, in pages that are there
//   o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m)), one pass with the running maximum m and sum
//
// A lane takes a key's score (its row of bytes in pieces of 16) and then channels of the sum, for which the weights come as scalars.
// A row that sees no key is zeros; a row of no entry (token_entry outside the table) is left as it is.  Keys and values that a row does
// not see are not multiplied, so that what is not finite stays with those who see it.
// Bound by trips to memory (keys, then values, a wavefront's 64 keys at a time: 24 tokens behind 2,000 to 600, 32 heads on 8 of 128, pages of 8, 53 us,
// of which its wavefronts wait for data 47 %) and, with many rows, by its own arithmetic, for nothing is shared between rows or heads (float32 prompts
// of 512 / 1,024 tokens 110 / 357 us, the vector units busy 83 %; 280 rows of up to 90 keys, 6 heads of 32, float32, 8.0).
// It serves what the matrix-core kernels do not: float32 rows, heads that are no multiple of 16 channels from 32 on (of 32 above 128), pages that are
// no multiple of 16 tokens, caps above 256.
#include "cache8_attn.h"

namespace {

constexpr int MAX_DIM = 512;

__device__ __forceinline__ float of_lane(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

// 0xff in the bytes whose bit is set
__device__ __forceinline__ uint32_t spread(uint32_t bits) { return ((bits * 0x00204081u) & 0x01010101u) * 0xffu; }

// CH: channels a lane sums.  WIDE: heads of a multiple of 16 channels, a key's row in pieces of 16 bytes.  VQ: tokens of a channel that are
// read together: 16 (blocks of 16), 4 (blocks of a multiple of 4) or 1.
template <typename T, int CH, bool WIDE, int VQ, int WAVES>
__global__ __launch_bounds__(WAVES * PULSE_WAVE) void attn8_plain_kernel(PulseAttn8 a) {
    constexpr int THREADS = WAVES * PULSE_WAVE;
    __shared__ __attribute__((aligned(16))) float s_q[MAX_DIM];
    __shared__ float s_o[WAVES][MAX_DIM];
    __shared__ float s_m[WAVES], s_l[WAVES];
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid % PULSE_WAVE, wave = tid / PULSE_WAVE;
    const int entry = a.token_entry[row];
    if (entry < 0 || entry >= a.entries) return;
    // (no key lies behind the table, and no position so far on that the next one leaves 32 bits)
    const int pos = static_cast<int>(min(static_cast<int64_t>(a.positions[row]),
                                         min(static_cast<int64_t>(a.table_width) * a.page_size, static_cast<int64_t>(0x7fffffff - 2 * THREADS)) - 1));
    const int g = h / (a.nq / a.nkv), d = a.d;
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride + static_cast<int64_t>(h) * d;
    for (int c = tid; c < MAX_DIM; c += THREADS) s_q[c] = c < d ? to_f32<T>(q[c]) : 0.f;
    __syncthreads();
    const int block = cache8::block_tokens(a.page_size), nb = a.page_size / block;
    const int lo = max(0, min(cache8::low_key(a.window, a.chunk, a.positions[row]), pos + 1));      // (so that no wavefront's first key leaves 32 bits)
    const int* bt = a.table + static_cast<int64_t>(entry) * a.table_width;
    float m = -INFINITY, l = 0.f, acc[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = 0.f;

    for (int j0 = lo / PULSE_WAVE * PULSE_WAVE + wave * PULSE_WAVE; j0 <= pos; j0 += WAVES * PULSE_WAVE) {
        const int j = j0 + lane;
        const int pi = j / a.page_size;
        const int page = pi < a.table_width ? bt[pi] : -1;
        const bool seen = j >= lo && j <= pos && page >= 0 && page < a.num_pages;
        const uint64_t seen_keys = __ballot(seen);
        if (seen_keys == 0) continue;
        const int slot = seen ? j - pi * a.page_size : 0;
        // the key's number in the cache, and its block's
        const int64_t head = static_cast<int64_t>(seen ? page : 0) * a.nkv + g;
        const int64_t bn = head * nb + slot / block;
        const float ks = a.scales[2 * bn], vs = a.scales[2 * bn + 1];
        float s = 0.f;
        const uint8_t* k = a.keys + (head * a.page_size + slot) * d;
        if constexpr (WIDE) {
#pragma unroll 4
            for (int c = 0; c < d; c += 16) {
                const uint4 u = *reinterpret_cast<const uint4*>(k + c);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x[4];
                    cache8::from_e4m3x4(w[i], x);
                    const float4 y = *reinterpret_cast<const float4*>(&s_q[c + 4 * i]);
                    s += x[0] * y.x;
                    s += x[1] * y.y;
                    s += x[2] * y.z;
                    s += x[3] * y.w;
                }
            }
        } else {
            for (int c = 0; c < d; ++c) s += cache8::from_e4m3(k[c]) * s_q[c];
        }
        s *= ks * a.scale;
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
        const float pv = seen ? p * fabsf(vs) : 0.f;
        // (VQ keys from a multiple of VQ on are of one block: the first that is seen says where it lies)
        const uint32_t place_lo = static_cast<uint32_t>(bn), place_hi = static_cast<uint32_t>(bn >> 32);
        const int in_block = slot % block;
        // so many groups of VQ keys are asked for together (a trip to memory for all of them, registers allowing)
        constexpr int WORDS = VQ < 4 ? 1 : VQ / 4, SOME = WORDS * CH >= 16 ? 1 : 16 / (WORDS * CH) < 8 ? 16 / (WORDS * CH) : 8;
        constexpr uint64_t MASK = SOME * VQ >= 64 ? ~0ull : (1ull << (SOME * VQ % 64)) - 1;
        const int any = __builtin_ctzll(seen_keys);
        for (int b0 = 0; b0 < PULSE_WAVE; b0 += SOME * VQ) {
            if (!(seen_keys >> b0 & MASK)) continue;
            uint32_t bytes[SOME][CH][WORDS], some[SOME];
#pragma unroll
            for (int u = 0; u < SOME; ++u) {
                const int b = b0 + u * VQ;
                some[u] = static_cast<uint32_t>(seen_keys >> b) & ((1u << VQ) - 1u);
                const int one = some[u] ? b + __builtin_ctz(some[u]) : any;      // (none is seen: others are read, and count as zeros)
                const int64_t at = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(place_hi, one))) << 32 |
                                                        static_cast<uint32_t>(__builtin_amdgcn_readlane(place_lo, one)));
                const uint8_t* v = a.values + at * block * d + (__builtin_amdgcn_readlane(in_block, one) & ~(VQ - 1));
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int c = lane + i * PULSE_WAVE;
                    const uint8_t* from = v + static_cast<int64_t>(c < d ? c : 0) * block;
                    if constexpr (VQ == 16) {
                        const uint4 w = *reinterpret_cast<const uint4*>(from);
                        bytes[u][i][0] = w.x, bytes[u][i][1] = w.y, bytes[u][i][2] = w.z, bytes[u][i][3] = w.w;
                    } else if constexpr (VQ == 4) {
                        bytes[u][i][0] = *reinterpret_cast<const uint32_t*>(from);
                    } else {
                        bytes[u][i][0] = *from;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < SOME; ++u) {
                float w[VQ];
#pragma unroll
                for (int e = 0; e < VQ; ++e) w[e] = of_lane(pv, b0 + u * VQ + e);
#pragma unroll
                for (int i = 0; i < CH; ++i) {
#pragma unroll
                    for (int e = 0; e < WORDS; ++e) {
                        float x[4];
                        // what is not seen is not multiplied: its bytes are zeros (a block that is seen whole keeps its own)
                        cache8::from_e4m3x4(bytes[u][i][e] & spread(some[u] >> (4 * e) & 15u), x);
#pragma unroll
                        for (int f = 0; f < (VQ < 4 ? 1 : 4); ++f) acc[i] += w[VQ < 4 ? 0 : 4 * e + f] * x[f];
                    }
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
    const int block = cache8::block_tokens(a->page_size);
    // A workgroup a compute unit at the most: as many wavefronts as it can have share a row's keys, so that each walks a quarter.  Tokens of 32
    // heads on 8 of 128 behind 2,000 (200), us, 4 / 16 wavefronts: 8 tokens, 256 workgroups, pages of 8 31.5 / 21.9 (6.3 / 6.7), float32 rows
    // 26.1 / 17.8 (5.6 / 6.0); 14 tokens 49.7 / 51.0 (9.7 / 13.0), 43.3 / 44.2 (8.9 / 11.6); 16 tokens 47.9 / 47.4 (8.9 / 12.0), 40.7 / 38.9 (7.8 / 10.6); 18
    // tokens 65 / 71 (11.5 / 17.6), 55 / 62 (10.3 / 15.6).
    const bool few = static_cast<int64_t>(a->tokens) * a->nq <= 256;
    auto go = [&](auto t, auto ch, auto wide, auto vq) {
        const dim3 grid(a->tokens, a->nq);
        if (few) attn8_plain_kernel<decltype(t), decltype(ch)::value, decltype(wide)::value, decltype(vq)::value, 16><<<grid, 16 * PULSE_WAVE, 0, stream>>>(*a);
        else attn8_plain_kernel<decltype(t), decltype(ch)::value, decltype(wide)::value, decltype(vq)::value, 4><<<grid, 4 * PULSE_WAVE, 0, stream>>>(*a);
    };
    auto by_block = [&](auto t, auto ch, auto wide) {
        if (block == 16) go(t, ch, wide, std::integral_constant<int, 16>());
        else if (block % 4 == 0) go(t, ch, wide, std::integral_constant<int, 4>());
        else go(t, ch, wide, std::integral_constant<int, 1>());
    };
    auto by_width = [&](auto t, auto wide) {
        if (a->d <= 64) by_block(t, std::integral_constant<int, 1>(), wide);
        else if (a->d <= 128) by_block(t, std::integral_constant<int, 2>(), wide);
        else if (a->d <= 256) by_block(t, std::integral_constant<int, 4>(), wide);
        else by_block(t, std::integral_constant<int, 8>(), wide);
    };
    auto by_form = [&](auto t) {
        if (a->d % 16 == 0) by_width(t, std::true_type());
        else by_width(t, std::false_type());
    };
    if (a->dtype == PULSE_F32) by_form(float());
    else by_form(bf16_t());
    PULSE_LAUNCH_CHECK("attn8_plain");
    return 0;
}

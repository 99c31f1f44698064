// Attention over a cache in 8 bits (cache8.h) on the matrix cores: bfloat16 rows, heads of a multiple of 16 channels from 32 to 128 and of 32 up
// to 256, pages of a multiple of 16 tokens.  Bytes become bfloat16 on their way into the matrix cores' operands (three bits of fraction: exactly), with the
// block's scale applied by the same instruction; products, maxima, sums and accumulators are float32.  Weights are rounded to bfloat16
// for the second product (a relative 2^-8 at most, as q was), the sum that divides them is of the unrounded ones.
//
// A piece of work is an item (some rows of one request that share a kv head: "columns", a head of a row each) and a stretch of tiles of
// 64 keys.  Everything is kept transposed, so that a column stays in its lanes:
//   S^T[key, col] = K[key, :] . q[col, :]      P^T = exp2(S^T c - m[col])      O^T[ch, col] += V^T[ch, key] P^T[key, col]
//
// attn8_cut      shares the tiles of all items out over a number of pieces: T = the least length for which sum ceil(tiles / T) fits (by
//                bisection), an item in equal pieces of at most T.  Made on the device from the positions, once a step for all layers, so that a
//                recorded step's replays bring their own lengths.
// attn8_few      up to 16 columns an item (a decoded token's heads; a few tokens).  Its four wavefronts take every fourth tile and
//                meet at the end.  Bound by reading the cache: 64 contexts of 4,096, 32 heads on 8 of 128, 539 MB in 95 us, 5.7 TB/s (a copy
//                reaches 4.8, read and written); one context of 4,096 by the chain of trips piece -> table -> keys -> join, 10 us.
// attn8_many     128 columns an item (portions of prompts).  A tile is converted once for all and lies in LDS as bfloat16.  2,048 tokens,
//                32 heads on 8 of 128, 63 us (0.55 PFLOP/s, its longest walks), 8,192 590 to 640 (0.86 to 0.93, the power limit).
// attn8_join     joins the pieces of items of attn8_many that were cut into many; else the piece that comes last does.
#include "cache8_attn.h"

#include <algorithm>
#include <type_traits>

int pulse_attn8_check(const PulseAttn8* a, const char* what);

namespace {

using cache8::TILE;

constexpr int THREADS = 256, WAVES = THREADS / PULSE_WAVE;
constexpr int FEW = 16, MANY = 128;
constexpr float LOG2E = 1.44269504088896340736f;

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A number that nothing in the launch writes; ONE: the same for the wavefront, read by the scalar unit.
template <bool ONE, typename T>
__device__ __forceinline__ T read_only(const T* p) {
    if constexpr (ONE) return *reinterpret_cast<const __attribute__((address_space(4))) T*>(reinterpret_cast<uintptr_t>(p));
    return *p;
}

// Eight bytes times a power of two, as a matrix-core operand.
__device__ __forceinline__ bf16x8 operand(uint32_t lo, uint32_t hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The same with nothing in the place of what is not a number, and ones (else zeros) in those places.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {    // 0xff in every byte that is NaN (0x7f, 0xff)
    const uint32_t m = w & 0x7f7f7f7fu, t = (m + 0x01010101u) & 0x80808080u;
    return (t >> 7) * 0xffu;
}
__device__ __forceinline__ bf16x8 ones_at(uint32_t lo, uint32_t hi) {     // 0x38: one
    return operand(nan_bytes(lo) & 0x38383838u, nan_bytes(hi) & 0x38383838u, 1.f);
}

// A score in the units of exp2; a cap takes the place of the factor: cap tanh(x / cap) log2 e = c - 2 c / (exp(2 x / cap) + 1) with
// c = cap log2 e.  (The hardware's reciprocal: its error and the difference's are some 2^-22 of the cap.)
struct Score {
    float factor, in, out;
    __device__ __forceinline__ float operator()(float s) const {
        return fmaf(-2.f * out, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * in) + 1.f), out);
    }
};
__device__ __forceinline__ Score score_of(const PulseAttn8& a) {
    if (a.softcap > 0.f) return {1.f, 2.f * LOG2E * a.scale / a.softcap, a.softcap * LOG2E};
    return {a.scale * LOG2E, 0.f, 0.f};
}

// What a column's sums are multiplied by at the end: its denominator with the sink in it, and its head's gate.
__device__ __forceinline__ float finish(const PulseAttn8& a, float m, float l, int row, int head) {
    if (a.sink) l += __builtin_amdgcn_exp2f(a.sink[head] * LOG2E - (m == -INFINITY ? 0.f : m));
    float inv = l == 0.f ? 0.f : 1.f / l;
    if (a.gate && a.gate_width == 0) inv *= cache8::sigmoid_of(bf16_to_f32(static_cast<const bf16_t*>(a.gate)[row * a.gate_stride + head]));
    return inv;
}
__device__ __forceinline__ float channel_gate(const PulseAttn8& a, int row, int head, int ch) {
    if (!a.gate || ch >= a.gate_width) return 1.f;
    return cache8::sigmoid_of(bf16_to_f32(static_cast<const bf16_t*>(a.gate)[row * a.gate_stride + static_cast<int64_t>(head) * a.gate_width + ch]));
}

// Four channels of a row, each times its factor.
template <typename F>
__device__ __forceinline__ void store4(bf16_t* to, f32x4 x, F factor) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = f32_to_bf16(x[e] * factor(e));
    *reinterpret_cast<uint2*>(to) = make_uint2(y[0] | y[1] << 16, y[2] | y[3] << 16);
}

// ------------------------------------------------------------------------------------------------------------------ the cut
__device__ __forceinline__ cache8::Piece piece_of(const PulseAttn8& a, int w) {
    cache8::Piece x;
    const int* from = a.cut + w * cache8::PIECE_INTS;
    int* to = &x.row0;
#pragma unroll
    for (int i = 0; i < 10; ++i) to[i] = read_only<true>(from + i);
    return x;
}

// Where a piece's tiles end: at the table's end at the latest, however far on the positions are.
__device__ __forceinline__ int tiles_end(const PulseAttn8& a, const cache8::Piece& job, const cache8::Div& blocks) {
    return static_cast<int>(min(static_cast<int64_t>(job.tile_end), (static_cast<int64_t>(a.table_width) * blocks.b + 3) / 4));
}

__global__ __launch_bounds__(THREADS) void attn8_cut_kernel(const int4* __restrict__ items, int n, const int* __restrict__ positions,
                                                            int window, int chunk, int slots, int least, int max_work, int groups, int even, int shrink,
                                                            int* cut) {
    __shared__ int s_sum[WAVES], s_max[WAVES];
    const int tid = threadIdx.x, lane = tid % PULSE_WAVE, wave = tid / PULSE_WAVE;
    cache8::Piece* work = reinterpret_cast<cache8::Piece*>(cut);
    int2* info = reinterpret_cast<int2*>(cut + cache8::PIECE_INTS * max_work);
    int* arrived = cut + cache8::PIECE_INTS * max_work + 2 * n;
    // A thread's part of a sum ends here, so that no sum and none with the slots in it leaves 32 bits: of lengths it only says where the search
    // begins and whether items are alike, and as a number of pieces it is more than the slots in any case.
    constexpr int FULL = 0x7fff0000 / THREADS;
    auto walk = [&](int i) {
        const int4 it = items[i];
        const int hi = positions[it.x + it.y - 1], pos0 = positions[it.x], first = cache8::low_key(window, chunk, pos0) / TILE;
        const int count = max(hi / TILE + 1 - first, 1);
        return cache8::Piece{it.x, it.y, it.z, i, first, first + count, 0, 0, hi, pos0, {0, 0}};
    };
    // over all threads
    auto both = [&](int& sum, int& most) {
        sum = wave_sum(sum);
        most = wave_reduce(most, [](int x, int y) { return max(x, y); });
        __syncthreads();
        if (lane == 0) s_sum[wave] = sum, s_max[wave] = most;
        __syncthreads();
        sum = most = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += s_sum[w], most = max(most, s_max[w]);
    };
    // (a thread's first item's tiles are kept: with up to 256 items the search reads nothing)
    cache8::Piece mine = {};
    if (tid < n) mine = walk(tid);
    auto tiles = [&](int i) {
        if (i == tid) return mine.tile_end - mine.tile;
        const cache8::Piece x = walk(i);
        return x.tile_end - x.tile;
    };
    int total = 0, most = 0;
    for (int i = tid; i < n; i += THREADS) {
        const int t = tiles(i);
        total = min(total + t, FULL);
        most = max(most, t);
    }
    both(total, most);
    // the least length for which the pieces are no more than the slots (where the items are more than that: nothing is cut)
    int lo = max(least, (total + slots - 1) / slots), hi = max(lo, most);
    // Of `tiles` in P pieces, walk and join take about tiles / (4 P) 0.75 us + P / 8 us, least for P = sqrt(1.5 tiles) (one context of 32,000 in
    // 64 pieces 21.3 us, in 28 18.6).
    if (shrink) lo = min(max(lo, static_cast<int>(sqrtf(static_cast<float>(most) * (2.f / 3.f)))), hi);
    if (max_work == n || static_cast<int64_t>(most) * n * 100 <= static_cast<int64_t>(total) * even) lo = hi;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        int pieces = 0, unused = 0;
        for (int i = tid; i < n; i += THREADS) pieces = min(pieces + (tiles(i) + mid - 1) / mid, FULL);
        both(pieces, unused);
        if (pieces <= slots) hi = mid;
        else lo = mid + 1;
    }
    int before = 0;
    for (int base = 0; base < n; base += THREADS) {
        const int i = base + tid;
        cache8::Piece x = i == tid ? mine : i < n ? walk(i) : cache8::Piece{};
        const int count = x.tile_end - x.tile;
        int pieces = 0, each = 1;
        if (i < n) {
            each = (count + (count + lo - 1) / lo - 1) / ((count + lo - 1) / lo);
            pieces = (count + each - 1) / each;
        }
        int sum = pieces;
#pragma unroll
        for (int step = 1; step < PULSE_WAVE; step *= 2) {
            const int other = __shfl_up(sum, step);
            sum += lane >= step ? other : 0;
        }
        __syncthreads();
        if (lane == PULSE_WAVE - 1) s_sum[wave] = sum;
        __syncthreads();
        int at = before + sum - pieces, all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            at += w < wave ? s_sum[w] : 0;
            all += s_sum[w];
        }
        before += all;
        if (i < n) {
            info[i] = make_int2(at, pieces);
            const int end = x.tile_end;
            x.first = at;
            x.pieces = pieces;
            for (int z = 0; z < pieces && at + z < max_work; ++z) {
                x.tile_end = min(end, x.tile + each);
                work[at + z] = x;
                x.tile += each;
            }
        }
    }
    for (int w = before + tid; w < max_work; w += THREADS) work[w] = cache8::Piece{};
    for (int i = tid; i < n * groups; i += THREADS) arrived[i] = 0;
}

// Two numbers to and from memory that workgroups of one launch share: past the caches that belong to one die (relaxed atomics of the
// device's scope), so that neither side has to write a cache back or to empty it.
__device__ __forceinline__ void share2(float* to, float x, float y) {
    const uint64_t both = static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool SHARED>
__device__ __forceinline__ float2 shared2(const float* from) {
    if constexpr (!SHARED) return *reinterpret_cast<const float2*>(from);
    const uint64_t both = __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float(static_cast<uint32_t>(both)), __uint_as_float(static_cast<uint32_t>(both >> 32)));
}

// Whether this workgroup's piece is the last of its item's (in column `x` of `width`).  A wavefront has its sums where all dies see them
// before it meets the others, and only then is the piece counted; the counter is left at zero for the next launch.  (By a release and an
// acquire, which write a die's cache back for every piece, 24 requests of one token took 82 us for 42.)
__device__ __forceinline__ bool arrive_last(const PulseAttn8& a, const cache8::Piece& job, int width, int x) {
    __shared__ int s_last;
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    int* arrived = const_cast<int*>(a.cut) + cache8::PIECE_INTS * a.max_work + 2 * a.n_items + job.item * width + x;
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = before == job.pieces - 1;
        if (s_last) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return s_last != 0;
}

// The join: out = sum_z w_z o_z / sum_z w_z l_z, w_z = exp2(m_z - max m), over an item's pieces (pieces of one column are COLS columns
// and the launch's `heads_x` apart).  A thread takes four channels of one of the columns c0 .. c0 + each - 1 and, where the threads are
// more than that, every ZS-th piece, eight at a time under a running maximum: one trip to memory for eight; the threads' sums meet in LDS.
// The order is fixed by the sizes alone.  SHARED: the pieces are this launch's.
template <int COLS, bool SHARED>
__device__ __forceinline__ void join_columns(const PulseAttn8& a, int first, int pieces, int heads_x, int x, int c0, int each, int row0, int cols,
                                             int head0, int heads) {
    __shared__ f32x4 s_sum[THREADS];
    __shared__ float2 s_ml[THREADS];
    const int tid = threadIdx.x, d = a.d, quads = d / 4, units = each * quads, zs = max(1, THREADS / units);
    const int64_t step = static_cast<int64_t>(heads_x) * COLS, at0 = static_cast<int64_t>(first) * step + static_cast<int64_t>(x) * COLS;
    for (int u0 = 0; u0 < units; u0 += THREADS) {
        const int unit = zs > 1 ? tid % units : u0 + tid, z0 = zs > 1 ? tid / units : 0;
        const int c = c0 + unit / quads, ch = unit % quads * 4;
        const bool on = unit < units && z0 < zs && c < cols;
        const int64_t at = at0 + (on ? c : c0);
        float m = -INFINITY, l = 0.f;
        f32x4 all = {0.f, 0.f, 0.f, 0.f};
        auto add = [&](float pm, float pl, f32x4 po) __attribute__((always_inline)) {     // (nothing yet: all is zeros, or NaN to be kept)
            const float now = fmaxf(m, pm), ref = now == -INFINITY ? 0.f : now;
            const float f = __builtin_amdgcn_exp2f(m - ref), g = __builtin_amdgcn_exp2f(pm - ref);
            l = l * f + pl * g;
            all = all * f + po * g;
            m = now;
        };
        constexpr int BATCH = 8;
        for (int z = z0; z < pieces && on; z += BATCH * zs) {
            float2 ml[BATCH], lo[BATCH], hi[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int64_t piece = at + min(z + i * zs, pieces - 1) * step;       // (past the last: the last again, for nobody)
                ml[i] = shared2<SHARED>(a.part_ml + 2 * piece);
                lo[i] = shared2<SHARED>(a.part_o + piece * d + ch);
                hi[i] = shared2<SHARED>(a.part_o + piece * d + ch + 2);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
                if (z + i * zs < pieces) add(ml[i].x, ml[i].y, f32x4{lo[i].x, lo[i].y, hi[i].x, hi[i].y});
        }
        if (zs > 1) {
            s_sum[tid] = all;
            s_ml[tid] = make_float2(m, l);
            __syncthreads();
            for (int z = 1; z < zs && z0 == 0 && on; ++z) add(s_ml[unit + z * units].x, s_ml[unit + z * units].y, s_sum[unit + z * units]);
        }
        if (on && z0 == 0) {
            const int row = row0 + c / heads, hd = head0 + c % heads;
            const float inv = finish(a, m, l, row, hd);
            bf16_t* to = static_cast<bf16_t*>(a.out) + row * a.o_stride + static_cast<int64_t>(hd) * d + ch;
            store4(to, all, [&](int e) { return inv * channel_gate(a, row, hd, ch + e); });
        }
    }
}

// --------------------------------------------------------------------------------------------------------- up to 16 columns
// Lane l holds row l % 16 of an operand and its 8 numbers 8 (l / 16) .., and gets back rows 4 (l / 16) .. of column l % 16.  Which key or
// channel a row or number stands for is free as long as both operands agree, so that every load is of 16 neighbouring bytes and no
// weight changes its lane: row 4 b + i of score tile t is key 4 t + i of the tile's block b, so that lane group b holds the 16 keys of block
// b; those are, eight by eight, the numbers of the second product, whose other operand is a channel's 16 bytes of the block.
template <int D>
struct Few {
    // (What is left behind 64s: 48 channels are three quarters of such a piece, 32 one of 8 bytes a lane, 16 half of that.  The lanes beyond
    // hold numbers of q that are zero, against others of the key's own row.)
    static constexpr int LEFT = D % 64, K16 = D / 64 + (LEFT == 48 ? 1 : 0), K8 = LEFT == 16 || LEFT == 32 ? 1 : 0, STEPS = 2 * K16 + K8, MT = D / 16;
    u32x4 k[4][K16 ? K16 : 1];
    uint2 k8[4];
    u32x4 v[MT];
    float ks, vs;          // of the lane's row's block, of the lane's own block (negative: it holds values that are not finite)
    bool there;            // the lane's own block
};

template <int D, bool CAP>
__global__ __launch_bounds__(THREADS, 2) void attn8_few_kernel(PulseAttn8 a, cache8::Div blocks, int head_groups) {
    using F = Few<D>;
    __shared__ float s_o[WAVES][FEW][D + 4];
    __shared__ float s_m[WAVES][FEW], s_l[WAVES][FEW];
    const int w = blockIdx.y;
    const cache8::Piece job = piece_of(a, w);
    if (job.rows <= 0) return;
    const int row0 = job.row0, ntok = job.rows, entry = job.entry, tile_end = tiles_end(a, job, blocks);
    const bool whole = job.pieces == 1;
    const int g = blockIdx.x / head_groups, part = blockIdx.x % head_groups;
    const int group = a.nq / a.nkv, heads = min(group - part * FEW, FEW);
    const int tid = threadIdx.x, lane = tid % PULSE_WAVE, wave = uniform(tid / PULSE_WAVE);
    const int r = lane % 16, b = lane / 16, hi = job.hi, pos0 = job.pos0;
    const int lo = cache8::low_key(a.window, a.chunk, pos0), lo_last = cache8::low_key(a.window, a.chunk, hi);

    // this lane's column: token r / heads, head r % heads
    const int tok = r / heads;
    const bool col_ok = tok < ntok;
    const int col_row = row0 + (col_ok ? tok : 0), head = g * group + part * FEW + r % heads;
    const int pos = col_ok ? a.positions[col_row] : -1, low = cache8::low_key(a.window, a.chunk, pos);
    bf16x8 q[F::STEPS];
    {
        const bf16_t* from = static_cast<const bf16_t*>(a.q) + col_row * a.q_stride + static_cast<int64_t>(head) * D;
        const bf16x8 none = {};
#pragma unroll
        for (int j = 0; j < F::K16; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) q[2 * j + s] = col_ok && 64 * j + 16 * b < D ? *reinterpret_cast<const bf16x8*>(from + 64 * j + 16 * b + 8 * s) : none;
        if constexpr (F::K8) q[F::STEPS - 1] = col_ok && 64 * F::K16 + 8 * b < D ? *reinterpret_cast<const bf16x8*>(from + 64 * F::K16 + 8 * b) : none;
    }
    const Score score = score_of(a);
    const int* bt = a.table + static_cast<int64_t>(entry) * a.table_width;
    const int b_last = F::LEFT == 48 && b == 3 ? 0 : b, b_8 = F::LEFT == 16 ? b % 2 : b;      // (a lane's part of a key's last piece)

    // where a tile's blocks lie: of the lane's row (block r / 4) and its own (block b)
    struct Place { int pk, pv; };
    auto find = [&](int tile) {
        const int ik = blocks.over(4 * tile + r / 4), iv = blocks.over(4 * tile + b);
        return Place{bt[min(ik, a.table_width - 1)], bt[min(iv, a.table_width - 1)]};
    };
    auto load = [&](int tile, Place at, F& x) {
        const int nk = 4 * tile + r / 4, nv = 4 * tile + b;
        auto there = [&](int n, int page) {
            return page >= 0 && page < a.num_pages && blocks.over(n) < a.table_width && 16 * n <= hi && 16 * n + 15 >= lo;
        };
        const bool on_k = there(nk, at.pk);
        x.there = there(nv, at.pv);
        const uint32_t bk = on_k ? (static_cast<uint32_t>(at.pk) * a.nkv + g) * blocks.b + blocks.rest(nk) : 0u;
        const uint32_t bv = x.there ? (static_cast<uint32_t>(at.pv) * a.nkv + g) * blocks.b + blocks.rest(nv) : 0u;
        const uint8_t* kp = a.keys + static_cast<uint64_t>(bk) * (16 * D) + (r % 4) * D;
        const uint8_t* vp = a.values + static_cast<uint64_t>(bv) * (16 * D) + r * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int j = 0; j < F::K16; ++j) x.k[t][j] = *reinterpret_cast<const u32x4*>(kp + 4 * t * D + 64 * j + 16 * (j == F::K16 - 1 ? b_last : b));
            if constexpr (F::K8) x.k8[t] = *reinterpret_cast<const uint2*>(kp + 4 * t * D + 64 * F::K16 + 8 * b_8);
        }
#pragma unroll
        for (int m = 0; m < F::MT; ++m) x.v[m] = *reinterpret_cast<const u32x4*>(vp + m * 256);
        x.ks = a.scales[2ull * bk];
        x.vs = a.scales[2ull * bv + 1];
    };

    f32x4 o[F::MT];
#pragma unroll
    for (int m = 0; m < F::MT; ++m) o[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, l = 0.f;

    auto compute = [&](int tile, F& x) {
        const int j0 = tile * TILE;
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < F::K16; ++j) {
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(x.k[t][j][0], x.k[t][j][1], x.ks), q[2 * j], s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(x.k[t][j][2], x.k[t][j][3], x.ks), q[2 * j + 1], s[t], 0, 0, 0);
            }
            if constexpr (F::K8) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(x.k8[t].x, x.k8[t].y, x.ks), q[F::STEPS - 1], s[t], 0, 0, 0);
        }
        if constexpr (CAP) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = score(s[t][i]);
        }
        // key j0 + 16 b + 4 t + i
        const int from = low - j0 - 16 * b, to = x.there ? pos - j0 - 16 * b : -1;
        const bool masked = j0 + TILE - 1 > pos0 || j0 < lo_last || __any(!x.there);
        if (masked) {
            asm volatile("");
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = 4 * t + i >= from && 4 * t + i <= to ? s[t][i] : -INFINITY;
            // (what was read in the place of a block that is not there)
#pragma unroll
            for (int m = 0; m < F::MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[m][i] = x.there ? x.v[m][i] : 0u;
        }
        float best = s[0][0];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) best = fmaxf(best, s[t][i]);
        best = across_rows(best, LaneMax()) * score.factor;
        const float now = fmaxf(top, best);
        if (__any(now > top)) {
            asm volatile("");
            const float again = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
            l *= again;
#pragma unroll
            for (int m = 0; m < F::MT; ++m) o[m] *= again;
            top = now;
        }
        const float shift = top == -INFINITY ? 0.f : -top;
        bf16x8 p[2];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[t][i], score.factor, shift));
                l += e;
                p[t / 2][4 * (t % 2) + i] = static_cast<__bf16>(e);
            }
        const float vs = x.there ? fabsf(x.vs) : 1.f;       // (in the place of a block that is not there one was read that nobody need have written)
        if (__builtin_expect(__any(x.there && x.vs < 0.f), 0)) {
            asm volatile("");
            // Values that are not finite belong to those who see them alone: they are left out of the sums, and a column that sees one
            // in a channel (a product of ones says so) gets NaN there.
            bf16x8 see[2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) see[t / 2][4 * (t % 2) + i] = static_cast<__bf16>(4 * t + i >= from && 4 * t + i <= to ? 1.f : 0.f);
#pragma unroll
            for (int m = 0; m < F::MT; ++m) {
                f32x4 bad = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    bad = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones_at(x.v[m][2 * u], x.v[m][2 * u + 1]), see[u], bad, 0, 0, 0);
                    x.v[m][2 * u] &= ~nan_bytes(x.v[m][2 * u]);
                    x.v[m][2 * u + 1] &= ~nan_bytes(x.v[m][2 * u + 1]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[m][i] = bad[i] > 0.f ? __builtin_nanf("") : o[m][i];
            }
        }
#pragma unroll
        for (int m = 0; m < F::MT; ++m) {
            o[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(x.v[m][0], x.v[m][1], vs), p[0], o[m], 0, 0, 0);
            o[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(x.v[m][2], x.v[m][3], vs), p[1], o[m], 0, 0, 0);
        }
    };

    // A wavefront takes its tiles in turn from one on that differs from item to item: where requests' pages lie one after the other, walks
    // that all start at their first tile ask the same channels of memory at the same time (64 contexts of 8,192, pages in order, 202 -> 185 us;
    // of 4,096 109 -> 101; pages at random, or fewer requests than fill the GPU: no difference).
    const int mine = (tile_end - job.tile - wave + WAVES - 1) / WAVES;
    if (mine > 0) {
        const int turn = job.item % mine;
        auto at = [&](int i) {
            const int n = min(i, mine - 1) + turn;
            return job.tile + wave + WAVES * (n < mine ? n : n - mine);
        };
        // One tile's registers a wavefront and three workgroups a unit (two from 192 channels on), whose wavefronts read while others
        // compute, in the place of two tiles' and two (one): 64 contexts of 4,096, heads of 64 / 128 / 192 / 256 channels 45.5 / 103 / 160 /
        // 267 -> 43 / 95 / 141 / 187 us, 5.6 to 5.9 TB/s.
        F x;
        Place ahead = find(at(0));
        for (int i = 0; i < mine; ++i) {
            load(at(i), ahead, x);
            ahead = find(at(i + 1));
            compute(at(i), x);
        }
    }
    l = across_rows(l, LaneSum());

    // the four wavefronts' columns meet
    if (b == 0) {
        s_m[wave][r] = top;
        s_l[wave][r] = l;
    }
#pragma unroll
    for (int m = 0; m < F::MT; ++m) *reinterpret_cast<f32x4*>(&s_o[wave][r][16 * m + 4 * b]) = o[m];
    __syncthreads();
    const int64_t at = (static_cast<int64_t>(w) * gridDim.x + blockIdx.x) * FEW;
    constexpr int QUADS = D / 4;
    for (int i = tid; i < FEW * QUADS; i += THREADS) {
        const int c = i / QUADS, ch = i % QUADS * 4;
        if (c >= ntok * heads) break;
        float m = s_m[0][c], sum = 0.f;
#pragma unroll
        for (int v = 1; v < WAVES; ++v) m = fmaxf(m, s_m[v][c]);
        f32x4 all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            const float f = s_m[v][c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[v][c] - m);
            // (a wavefront that has seen no key has zeros, or NaN for a column that saw a value that is none: kept)
            sum += s_l[v][c] * f;
            all += *reinterpret_cast<const f32x4*>(&s_o[v][c][ch]) * f;
        }
        const int row = row0 + c / heads, hd = g * group + part * FEW + c % heads;
        if (whole) {
            const float inv = finish(a, m, sum, row, hd);
            bf16_t* to = static_cast<bf16_t*>(a.out) + row * a.o_stride + static_cast<int64_t>(hd) * D + ch;
            store4(to, all, [&](int e) { return inv * channel_gate(a, row, hd, ch + e); });
        } else {
            share2(a.part_o + (at + c) * D + ch, all[0], all[1]);
            share2(a.part_o + (at + c) * D + ch + 2, all[2], all[3]);
            if (ch == 0) share2(a.part_ml + 2 * (at + c), m, sum);
        }
    }
    if (whole) return;
    // The piece that comes last joins them all.  (Its sums go by the pieces' order: who comes last changes nothing.)
    if (arrive_last(a, job, gridDim.x, blockIdx.x))
        join_columns<FEW, true>(a, job.first, job.pieces, gridDim.x, blockIdx.x, 0, ntok * heads, row0, ntok * heads, g * group + part * FEW, heads);
}

// ------------------------------------------------------------------------------------------------------------ 128 columns
// A wavefront takes 32 columns: lane l supplies row l % 32 of an operand and its 8 numbers 8 (l / 32) .., and gets back rows
// 8 (i / 4) + 4 (l / 32) + i % 4, i < 16, of column l % 32.  The values lie in LDS in the order in which the weights come out of the
// first product: of 16 keys the lanes of half h hold 4 h .. and 8 + 4 h .., which are one piece of 16 bytes.  Rows are 16 bytes longer than
// they have to be, so that the eight rows that are read in a cycle lie in different banks.
//
// A thread brings piece n of a tile's keys and of its values: 16 bytes at the same place of the same block (a row's 16 channels, a
// channel's 16 tokens), asked for while the tile before is computed, and converts them into the other of two stages.  What is rare (caps,
// masks, blocks that are not there or hold what is not finite, a maximum that grew) stands behind real branches: left to itself the
// compiler computes both sides.
// Heads of 160 to 224 channels take 32 keys at a time, for which a unit's registers hold two workgroups (with 64, one; 2 portions of 600 behind
// 2,000, 16 heads on 4 of 160 / 192 / 224 channels 80 / 89 / 105 -> 60 / 66 / 83 us).  256 channels have no room for two either way (32
// keys, spilled: 2,048 tokens 94 -> 99), and up to 128 fewer keys a step cost more than a third workgroup gives (128 channels, 512 tokens behind
// 8,192 98 -> 106, 2,048 alone 62 -> 58).
template <int D>
constexpr bool SMALL_STEPS = D > 128 && D < 256;
template <int D, bool CAP>
__global__ __launch_bounds__(THREADS, D < 256 ? 2 : 1) void attn8_many_kernel(PulseAttn8 a, cache8::Div blocks) {
    constexpr int KEYS = SMALL_STEPS<D> ? 32 : 64, BLOCKS = KEYS / 16, HALVES = KEYS / 32;
    constexpr int KROW = D + 8, VROW = KEYS + 8;                 // in bfloat16 numbers
    constexpr int PIECES = BLOCKS * D, TURNS = (PIECES + THREADS - 1) / THREADS, STEPS = D / 16, MT = (D + 31) / 32;
    using NoneWord = std::conditional_t<BLOCKS == 4, uint64_t, uint32_t>;
    __shared__ __attribute__((aligned(16))) bf16_t s_k[2][KEYS * KROW];
    __shared__ __attribute__((aligned(16))) bf16_t s_v[2][MT * 32 * VROW];      // (of 16 channels too many nothing is kept)
    // the tile + 1 in which something is out of the ordinary; in which a block is not there; in which it holds values that are none, and which
    __shared__ int s_odd[2], s_gone[2][BLOCKS], s_bad[2][BLOCKS];
    __shared__ __attribute__((aligned(8))) uint16_t s_none[2][MT * 32][BLOCKS];
    const int w = blockIdx.y;
    const cache8::Piece job = piece_of(a, w);
    if (job.rows <= 0) return;
    const int row0 = job.row0, ntok = job.rows, entry = job.entry, begin = job.tile * (TILE / KEYS), end = tiles_end(a, job, blocks) * (TILE / KEYS);
    const bool whole = job.pieces == 1;
    const int g = blockIdx.x, group = a.nq / a.nkv;
    const int tid = threadIdx.x, lane = tid % PULSE_WAVE, wave = uniform(tid / PULSE_WAVE);
    const int r = lane % 32, half = lane / 32, hi = job.hi, pos0 = job.pos0;
    const int lo = cache8::low_key(a.window, a.chunk, pos0);

    const int col = wave * 32 + r, tok = col / group;
    const bool col_ok = tok < ntok;
    const int col_row = row0 + (col_ok ? tok : 0), head = g * group + (col_ok ? col - tok * group : 0);
    const int pos = col_ok ? a.positions[col_row] : -1, low = cache8::low_key(a.window, a.chunk, pos);
    // the wavefront's first and last position (its columns' tokens follow each other), -1 where it has no column
    const int w_tok0 = wave * 32 / group, w_tok1 = min((wave * 32 + 31) / group, ntok - 1);
    const bool w_any = w_tok0 < ntok;
    const int w_first = w_any ? uniform(a.positions[row0 + w_tok0]) : -1, w_last = w_any ? uniform(a.positions[row0 + w_tok1]) : -1;
    const int w_low = cache8::low_key(a.window, a.chunk, w_first), w_low_last = cache8::low_key(a.window, a.chunk, w_last);

    bf16x8 q[STEPS];
    {
        const bf16_t* from = static_cast<const bf16_t*>(a.q) + col_row * a.q_stride + static_cast<int64_t>(head) * D;
        const bf16x8 none = {};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) q[s] = col_ok ? *reinterpret_cast<const bf16x8*>(from + 16 * s + 8 * half) : none;
    }
    const Score score = score_of(a);
    const int* bt = a.table + static_cast<int64_t>(entry) * a.table_width;

    // Piece n = tid + 256 i is of the tile's block n / D.  Where D is a multiple of 64 that is one block for a wavefront: its page, its
    // scales and its address are then scalars (asked for by the scalar unit), and what is left of a lane's address never changes.  (A
    // last turn that not all threads take brings the others a piece for nobody.)
    constexpr bool ONE = D % 64 == 0;
    struct Spot { int n, page_index, rest, page; };       // a block of the context: its number, its page's and its place in it, the page
    struct Raw {
        u32x4 k[TURNS], v[TURNS];
        float2 scale[TURNS];
        int there[TURNS];      // -1: beyond what the item sees, 0: not there, 1: there
    };
    Spot spot[TURNS];          // of the tile whose pages are asked for next
    const int page_step = blocks.over(BLOCKS), rest_step = BLOCKS - page_step * blocks.b;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const int in_tile = min((tid + i * THREADS) / D, BLOCKS - 1);
        spot[i].n = BLOCKS * begin + (ONE ? uniform(in_tile) : in_tile);
        spot[i].page_index = blocks.over(spot[i].n);
        spot[i].rest = spot[i].n - spot[i].page_index * blocks.b;
        spot[i].page = 0;
    }
    auto find = [&](Spot (&to)[TURNS]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            Spot& s = spot[i];
            to[i] = s;
            to[i].page = read_only<ONE>(bt + min(s.page_index, a.table_width - 1));
            if (s.page_index >= a.table_width) to[i].page = -1;
            s.n += BLOCKS;
            s.page_index += page_step;
            s.rest += rest_step;
            if (s.rest >= blocks.b) {
                s.rest -= blocks.b;
                ++s.page_index;
            }
        }
    };
    auto load = [&](const Spot (&from)[TURNS], Raw& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const Spot& s = from[i];
            const bool ours = 16 * s.n <= hi && 16 * s.n + 15 >= lo;
            const bool there = ours && s.page >= 0 && s.page < a.num_pages;
            x.there[i] = there ? 1 : ours ? 0 : -1;
            const uint32_t at = there ? (static_cast<uint32_t>(s.page) * a.nkv + g) * blocks.b + s.rest : 0u;
            const uint64_t byte = static_cast<uint64_t>(at) * (16 * D);
            const uint32_t mine = (tid + i * THREADS) % D * 16;
            x.k[i] = *reinterpret_cast<const u32x4*>(a.keys + byte + mine);
            x.v[i] = *reinterpret_cast<const u32x4*>(a.values + byte + mine);
            const float* sc = a.scales + 2 * static_cast<uint64_t>(at);
            x.scale[i] = make_float2(read_only<ONE>(sc), read_only<ONE>(sc + 1));
        }
    };
    auto put = [&](Raw& x, int stage, int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int n = tid + i * THREADS;
            if (PIECES % THREADS == 0 || n < PIECES) {
                const int kr = n / (D / 16), kc = n % (D / 16), vb = n / D, vc = n % D;
                if (__builtin_expect(x.there[i] <= 0 || x.scale[i].y < 0.f, 0)) {
                    asm volatile("");
                    if (x.there[i] <= 0) {       // (what was read in its place nobody need have written)
                        x.k[i] = x.v[i] = u32x4{0u, 0u, 0u, 0u};
                        x.scale[i] = make_float2(1.f, 1.f);
                    }
                    if (x.there[i] >= 0) s_odd[stage] = tile + 1;       // (every thread that writes it writes the same)
                    if (x.there[i] == 0) s_gone[stage][vb] = tile + 1;
                    if (x.there[i] > 0) {
                        // Values that are not finite belong to those who see them alone: they leave the sums here, and a column that sees
                        // one gets NaN in its channel.
                        s_bad[stage][vb] = tile + 1;
                        uint32_t none = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t bytes = nan_bytes(x.v[i][e]);
                            none |= ((bytes & 1u) | (bytes >> 7 & 2u) | (bytes >> 14 & 4u) | (bytes >> 21 & 8u)) << (4 * e);
                            x.v[i][e] &= ~bytes;
                        }
                        s_none[stage][vc][vb] = static_cast<uint16_t>(none);
                    }
                }
                const float ks = x.scale[i].x, vs = fabsf(x.scale[i].y);
                bf16_t* k = &s_k[stage][kr * KROW + kc * 16];
                *reinterpret_cast<bf16x8*>(k) = operand(x.k[i][0], x.k[i][1], ks);
                *reinterpret_cast<bf16x8*>(k + 8) = operand(x.k[i][2], x.k[i][3], ks);
                bf16_t* v = &s_v[stage][vc * VROW + vb * 16];
                *reinterpret_cast<bf16x8*>(v) = operand(x.v[i][0], x.v[i][2], vs);
                *reinterpret_cast<bf16x8*>(v + 8) = operand(x.v[i][1], x.v[i][3], vs);
            }
        }
    };

    f32x16 o[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) o[m] = f32x16{};
    float top = -INFINITY, l = 0.f;

    auto compute = [&](int tile, int stage) __attribute__((always_inline)) {
        const int j0 = tile * KEYS;
        if (j0 > w_last || j0 + KEYS - 1 < w_low) return;       // no column of this wavefront sees a key of the tile
        const bf16_t* sk = s_k[stage] + r * KROW + 8 * half;
        const bf16_t* sv = s_v[stage] + r * VROW + 8 * half;
        const bool odd = uniform(s_odd[stage]) == tile + 1;
        constexpr int AHEAD = SMALL_STEPS<D> ? 2 : 4;       // operand reads run that many products ahead
        auto key = [&](int i) __attribute__((always_inline)) { return *reinterpret_cast<const bf16x8*>(sk + i / STEPS * (32 * KROW) + i % STEPS * 16); };
        auto value = [&](int i) __attribute__((always_inline)) { return *reinterpret_cast<const bf16x8*>(sv + i / BLOCKS * (32 * VROW) + i % BLOCKS * 16); };
        bf16x8 ak[HALVES * STEPS], av[BLOCKS * MT];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ak[i] = key(i);
        f32x16 s[HALVES] = {};
#pragma unroll
        for (int i = 0; i < HALVES * STEPS; ++i) {
            if (i + AHEAD < HALVES * STEPS) ak[i + AHEAD] = key(i + AHEAD);
            else if (i + AHEAD - HALVES * STEPS < BLOCKS * MT) av[i + AHEAD - HALVES * STEPS] = value(i + AHEAD - HALVES * STEPS);
            s[i / STEPS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ak[i], q[i % STEPS], s[i / STEPS], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (CAP) {
#pragma unroll
            for (int t = 0; t < HALVES; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = score(s[t][i]);
        }
        // s[t][i] is of key j0 + 32 t + 8 (i / 4) + 4 half + i % 4, of block 2 t + i / 8
        const int from = low - j0 - 4 * half, to = pos - j0 - 4 * half;
        uint32_t gone = 0;
        auto seen = [&](int t, int i) __attribute__((always_inline)) {
            const int j = 32 * t + 8 * (i / 4) + i % 4;
            return j >= from && j <= to && !(gone >> (2 * t + i / 8) & 1u);
        };
        if (j0 + KEYS - 1 > w_first || j0 < w_low_last || !w_any || odd) {
            asm volatile("");
            if (odd) {
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) gone |= (uniform(s_gone[stage][b]) == tile + 1 ? 1u : 0u) << b;
            }
#pragma unroll
            for (int t = 0; t < HALVES; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = seen(t, i) ? s[t][i] : -INFINITY;
        }
        float best = s[0][0];
#pragma unroll
        for (int t = 0; t < HALVES; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) best = fmaxf(best, s[t][i]);
        const WaveTwo two = wave_two<32>(__float_as_uint(best));
        best = fmaxf(__uint_as_float(two.a), __uint_as_float(two.b)) * score.factor;
        // the sums move to a new maximum only when it is 2^8 above the old one: weights stay below 2^8 until then
        if (__any(best > top + 8.f || (top == -INFINITY && best > -INFINITY))) {
            asm volatile("");
            const float now = fmaxf(top, best);
            const float again = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
            l *= again;
#pragma unroll
            for (int m = 0; m < MT; ++m) o[m] *= again;
            top = now;
        }
        const float shift = top == -INFINITY ? 0.f : -top;
        bf16x8 p[BLOCKS];
#pragma unroll
        for (int t = 0; t < HALVES; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[t][i], score.factor, shift));
                l += e;
                p[2 * t + i / 8][i % 8] = static_cast<__bf16>(e);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < BLOCKS * MT; ++i) {
            if (i + AHEAD < BLOCKS * MT) av[i + AHEAD] = value(i + AHEAD);
            o[i / BLOCKS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av[i], p[i % BLOCKS], o[i / BLOCKS], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(odd, 0)) {
            asm volatile("");
            // the keys of the tile that this column sees, and of those the ones whose value in a channel is none
            const int first = max(low - j0, 0), last = min(pos - j0 + 1, KEYS);
            uint64_t seen_keys = last > first ? (~0ull >> (64 - (last - first))) << first : 0ull;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
                if (uniform(s_gone[stage][b]) == tile + 1 || uniform(s_bad[stage][b]) != tile + 1) seen_keys &= ~(0xffffull << (16 * b));
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const NoneWord none = *reinterpret_cast<const NoneWord*>(s_none[stage][32 * m + 8 * (i / 4) + 4 * half + i % 4]);
                    if (none & static_cast<NoneWord>(seen_keys)) o[m][i] = __builtin_nanf("");
                }
        }
    };

    {
        Raw raw;
        Spot next[TURNS];
        find(next);
        if (tid < 2) s_odd[tid] = 0;
        if (tid < 2 * BLOCKS) s_gone[tid / BLOCKS][tid % BLOCKS] = s_bad[tid / BLOCKS][tid % BLOCKS] = 0;
        __syncthreads();
        load(next, raw);
        find(next);
        put(raw, 0, begin);
        __syncthreads();
        int stage = 0;
        for (int tile = begin; tile < end; ++tile, stage ^= 1) {
            const bool more = tile + 1 < end;
            if (more) {
                load(next, raw);
                find(next);
            }
            compute(tile, stage);
            if (more) put(raw, stage ^ 1, tile + 1);       // (that stage was read before the last barrier)
            __syncthreads();
        }
    }
    const WaveTwo two = wave_two<32>(__float_as_uint(l));
    l = __uint_as_float(two.a) + __uint_as_float(two.b);
    if (!whole && a.join_here) {
        // The piece that comes last joins them, as in attn8_few; the others' sums lie in the order of the threads, a pair of channels each.
        const int64_t step = static_cast<int64_t>(gridDim.x) * MANY, first = static_cast<int64_t>(job.first) * step + static_cast<int64_t>(blockIdx.x) * MANY;
        const int own = w - job.first;
        auto sums_of = [&](int z) __attribute__((always_inline)) { return a.part_o + (first + z * step) * D + 2 * tid; };
        auto state_of = [&](int z) __attribute__((always_inline)) { return a.part_ml + 2 * (first + z * step + col); };
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (32 * m + 8 * (i / 2) < D) share2(sums_of(own) + (8 * m + i) * (2 * THREADS), o[m][2 * i], o[m][2 * i + 1]);
        if (half == 0) share2(state_of(own), top, l);
        if (!arrive_last(a, job, gridDim.x, blockIdx.x)) return;
        float most = top;
        for (int z = 0; z < job.pieces; ++z) most = fmaxf(most, shared2<true>(state_of(z)).x);
        const float shift = most == -INFINITY ? 0.f : most;
        constexpr int SOME = D <= 128 ? MT : 1;       // (32 channels at a time: wider heads have no registers for more)
        float sum = 0.f;
#pragma unroll
        for (int m0 = 0; m0 < MT; m0 += SOME) {
            f32x16 all[SOME] = {};
            for (int z = 0; z < job.pieces; ++z) {       // (in their order, whoever came last)
                const float2 ml = shared2<true>(state_of(z));
                const float f = __builtin_amdgcn_exp2f(ml.x - shift);
                if (m0 == 0) sum += ml.y * f;
                if (z == own) {
#pragma unroll
                    for (int m = 0; m < SOME; ++m)
#pragma unroll
                        for (int i = 0; i < 16; ++i) all[m][i] = fmaf(o[m0 + m][i], f, all[m][i]);
                } else {
#pragma unroll
                    for (int m = 0; m < SOME; ++m) {
                        float2 x[8] = {};
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (32 * (m0 + m) + 8 * (i / 2) < D) x[i] = shared2<true>(sums_of(z) + (8 * (m0 + m) + i) * (2 * THREADS));
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            all[m][2 * i] = fmaf(x[i].x, f, all[m][2 * i]);
                            all[m][2 * i + 1] = fmaf(x[i].y, f, all[m][2 * i + 1]);
                        }
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < SOME; ++m) o[m0 + m] = all[m];
        }
        top = most;
        l = sum;
    }
    if (!col_ok) return;
    if (whole || a.join_here) {
        const float inv = finish(a, top, l, col_row, head);
        bf16_t* to = static_cast<bf16_t*>(a.out) + col_row * a.o_stride + static_cast<int64_t>(head) * D;
        if (__builtin_expect(a.gate_width > 0, 0)) {
            asm volatile("");
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[m][i] *= channel_gate(a, col_row, head, 32 * m + 8 * (i / 4) + 4 * half + i % 4);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < 4 && 32 * m + 8 * c < D; ++c)
                store4(to + 32 * m + 8 * c + 4 * half, f32x4{o[m][4 * c], o[m][4 * c + 1], o[m][4 * c + 2], o[m][4 * c + 3]}, [&](int) { return inv; });
    } else {
        const int64_t at = (static_cast<int64_t>(w) * gridDim.x + blockIdx.x) * MANY + col;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < 4 && 32 * m + 8 * c < D; ++c)
                *reinterpret_cast<f32x4*>(a.part_o + at * D + 32 * m + 8 * c + 4 * half) =
                    f32x4{o[m][4 * c], o[m][4 * c + 1], o[m][4 * c + 2], o[m][4 * c + 3]};
        if (half == 0) {
            a.part_ml[2 * at] = top;
            a.part_ml[2 * at + 1] = l;
        }
    }
}

// The portions' pieces where there are many of an item, 16 columns a workgroup (128 columns of ten pieces take one workgroup longer
// than a launch and its spread).
__global__ __launch_bounds__(THREADS) void attn8_join_kernel(PulseAttn8 a) {
    const int item = blockIdx.y;
    const int2 info = reinterpret_cast<const int2*>(a.cut + cache8::PIECE_INTS * a.max_work)[item];
    const int first = uniform(info.x), pieces = uniform(info.y);
    if (pieces <= 1) return;
    const int4 it = reinterpret_cast<const int4*>(a.items)[item];
    const int group = a.nq / a.nkv;
    join_columns<MANY, false>(a, first, pieces, gridDim.x, blockIdx.x, blockIdx.z * 16, 16, it.x, it.y * group, blockIdx.x * group, group);
}

int check_matrix(const PulseAttn8* a, const char* what) {
    if (int rc = pulse_attn8_check(a, what)) return rc;
    PULSE_REQUIRE(a->dtype == PULSE_BF16 && a->d % 16 == 0 && a->d >= 32 && (a->d % 32 == 0 || a->d < 128) && a->d <= 256 && a->page_size % cache8::BLOCK == 0,
                  "%s: bfloat16 rows, heads of a multiple of 16 channels from 32 to 128, of 32 up to 256, and pages of a multiple of 16 tokens are served", what);
    PULSE_REQUIRE(static_cast<int64_t>(a->num_pages) * a->nkv * (a->page_size / cache8::BLOCK) <= 0x7fffffff, "%s: too many pages", what);
    PULSE_REQUIRE(a->items && a->cut && a->n_items > 0 && a->max_work > 0 && a->max_work <= 65535 && a->n_items <= 65535, "%s: bad work list", what);
    PULSE_REQUIRE(a->q_stride % 8 == 0 && a->o_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a->q) & 15) == 0 &&
                      (reinterpret_cast<uintptr_t>(a->out) & 7) == 0, "%s: rows must be aligned to 16 bytes", what);
    PULSE_REQUIRE(a->max_work == a->n_items || (a->part_o && a->part_ml), "%s: the room for pieces is missing", what);
    return 0;
}

template <typename F>
int by_width(int d, F go) {
    switch (d) {
        case 32: go(std::integral_constant<int, 32>()); break;
        case 48: go(std::integral_constant<int, 48>()); break;
        case 64: go(std::integral_constant<int, 64>()); break;
        case 80: go(std::integral_constant<int, 80>()); break;
        case 96: go(std::integral_constant<int, 96>()); break;
        case 112: go(std::integral_constant<int, 112>()); break;
        case 128: go(std::integral_constant<int, 128>()); break;
        case 160: go(std::integral_constant<int, 160>()); break;
        case 192: go(std::integral_constant<int, 192>()); break;
        case 224: go(std::integral_constant<int, 224>()); break;
        default: go(std::integral_constant<int, 256>()); break;
    }
    return 0;
}

}  // namespace

// `groups`: the kv heads (and sixteens of their heads) that there are counters of arrived pieces for; 0 where a launch of its own joins.
// `even`: nothing is cut where the longest item is at most that many hundredths of the mean (0: no such rule).  `shrink`: pieces of long items
// are longer than they had to be, for a shorter join.
extern "C" int pulse_attn8_cut(const int* items, int n_items, const int* positions, int window, int chunk, int slots, int least,
                               int max_work, int groups, int even, int shrink, int* cut, hipStream_t stream) {
    PULSE_REQUIRE(items && positions && cut && n_items > 0 && slots > 0 && least > 0 && groups >= 0, "attn8_cut: bad work list");
    PULSE_REQUIRE(max_work == n_items || max_work >= n_items + slots, "attn8_cut: room for %d pieces, %d are possible", max_work, n_items + slots);
    PULSE_REQUIRE((reinterpret_cast<uintptr_t>(items) & 15) == 0 && (reinterpret_cast<uintptr_t>(cut) & 15) == 0, "attn8_cut: lists must be aligned to 16 bytes");
    // (no room for more pieces than items: one each)
    attn8_cut_kernel<<<1, THREADS, 0, stream>>>(reinterpret_cast<const int4*>(items), n_items, positions, window, chunk, slots,
                                                least, max_work, groups, even, shrink, cut);
    PULSE_LAUNCH_CHECK("attn8_cut");
    return 0;
}

extern "C" int pulse_attn8_few(const PulseAttn8* a, hipStream_t stream) {
    if (int rc = check_matrix(a, "attn8_few")) return rc;
    const int head_groups = (a->nq / a->nkv + FEW - 1) / FEW;
    const cache8::Div blocks = cache8::div_by(a->page_size / cache8::BLOCK);
    const dim3 grid(a->nkv * head_groups, a->max_work);
    by_width(a->d, [&](auto d) {
        if (a->softcap > 0.f) attn8_few_kernel<decltype(d)::value, true><<<grid, THREADS, 0, stream>>>(*a, blocks, head_groups);
        else attn8_few_kernel<decltype(d)::value, false><<<grid, THREADS, 0, stream>>>(*a, blocks, head_groups);
    });
    PULSE_LAUNCH_CHECK("attn8_few");
    return 0;
}

extern "C" int pulse_attn8_many(const PulseAttn8* a, hipStream_t stream) {
    if (int rc = check_matrix(a, "attn8_many")) return rc;
    PULSE_REQUIRE(a->nq / a->nkv <= MANY, "attn8_many: %d heads on one (up to %d)", a->nq / a->nkv, MANY);
    const cache8::Div blocks = cache8::div_by(a->page_size / cache8::BLOCK);
    const dim3 grid(a->nkv, a->max_work);
    by_width(a->d, [&](auto d) {
        if (a->softcap > 0.f) attn8_many_kernel<decltype(d)::value, true><<<grid, THREADS, 0, stream>>>(*a, blocks);
        else attn8_many_kernel<decltype(d)::value, false><<<grid, THREADS, 0, stream>>>(*a, blocks);
    });
    PULSE_LAUNCH_CHECK("attn8_many");
    if (a->max_work > a->n_items && !a->join_here) {
        attn8_join_kernel<<<dim3(a->nkv, a->n_items, MANY / 16), THREADS, 0, stream>>>(*a);
        PULSE_LAUNCH_CHECK("attn8_join");
    }
    return 0;
}

// What a step's kernels have to know about rows and pages, made on the GPU from the requests' lengths.
//
//   first_row[b] = sum of count[i], i < b                    position[t] = start[b] + t - first_row[b]     token_entry[t] = b
//   held[b] = ceil((start[b] + count[b]) / page_size)        table[b, j] = pages[at[b] + j], j < held[b], else -1; at = sums of held
//   slot[t] = page of its position * page_size + place in it, -1 where the page is none of the pool's
//   blocks: for every request the blocks that [start, start + count) reaches into, in order: (its first row, rows, the block's number
//   page * blocks a page + block in the page or -1, the place in the block that the first row takes); left-over places: no rows, -1
//
// One launch.  The sums over the requests (a few hundred additions) are made by every workgroup for itself in LDS, which costs less
// than a second launch or a wait between workgroups would; a row finds its request by bisection there.  All of it is integers that are
// read once and written once: a launch's latency bounds it (64 requests 4.5 us, 64 with 9,648 rows 5.0, an empty launch 2 to 3).
#include "cache8.h"

#include <algorithm>

namespace {

using cache8::Div;

constexpr int THREADS = 256;
constexpr int MAX_REQUESTS = 4096;      // three sums a request in LDS: 48 KB

struct MapArgs {
    const int *start, *count;
    int requests;
    const int* pages;          // null: the pages are read from `table`
    int n_pages;
    Div page, block;
    int blocks_per_page, num_pages;
    int* first_row;
    int *positions, *token_entry, *slots;
    int rows;
    int* table;
    int width;
    int4* blocks;
    int n_blocks;
};

// the sum of a value over all threads below this one, and over all of them
__device__ __forceinline__ int below(int v, int* waves, int& total) {
    const int lane = threadIdx.x % PULSE_WAVE, wave = threadIdx.x / PULSE_WAVE;
    int sum = v;
#pragma unroll
    for (int step = 1; step < PULSE_WAVE; step *= 2) {
        const int other = __shfl_up(sum, step);
        sum += lane >= step ? other : 0;
    }
    __syncthreads();     // (the words may still be read)
    if (lane == PULSE_WAVE - 1) waves[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / PULSE_WAVE; ++w) {
        before += w < wave ? waves[w] : 0;
        total += waves[w];
    }
    return before + sum - v;
}

__global__ __launch_bounds__(THREADS) void step_maps_kernel(MapArgs a) {
    extern __shared__ int sums[];       // first rows, first pages, first blocks: requests + 1 each
    __shared__ int waves[THREADS / PULSE_WAVE];
    const int n = a.requests, tid = threadIdx.x;
    int *row0 = sums, *page0 = sums + (n + 1), *block0 = sums + 2 * (n + 1);
    int rows = 0, pages = 0, blocks = 0;
    for (int base = 0; base < n; base += THREADS) {
        const int b = base + tid;
        const int s = b < n ? max(a.start[b], 0) : 0, c = b < n ? max(a.count[b], 0) : 0;
        const int held = s + c > 0 ? a.page.over(s + c - 1) + 1 : 0;
        const int touched = c > 0 ? a.block.over(s + c - 1) - a.block.over(s) + 1 : 0;
        int all_rows, all_pages, all_blocks;
        const int r = below(c, waves, all_rows), p = below(held, waves, all_pages), k = below(touched, waves, all_blocks);
        if (b < n) {
            row0[b] = rows + r;
            page0[b] = pages + p;
            block0[b] = blocks + k;
        }
        rows += all_rows;
        pages += all_pages;
        blocks += all_blocks;
    }
    if (tid == 0) {
        row0[n] = rows;
        page0[n] = pages;
        block0[n] = blocks;
    }
    __syncthreads();
    if (blockIdx.x == 0 && a.first_row)
        for (int b = tid; b <= n; b += THREADS) a.first_row[b] = row0[b];

    // the last request whose sum is at most i (requests without any are passed over)
    auto find = [&](const int* first, int i) {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= i) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    auto page_at = [&](int b, int j) {
        int p = -1;
        if (a.pages) {
            const int at = page0[b] + j;
            if (at >= 0 && at < min(page0[b + 1], a.n_pages)) p = a.pages[at];
        } else if (j >= 0 && j < a.width) {
            p = a.table[static_cast<int64_t>(b) * a.width + j];
        }
        return p;
    };
    auto of_pool = [&](int p) { return p >= 0 && p < a.num_pages; };

    const int stride = gridDim.x * THREADS;
    if (a.pages && a.table) {
        const int64_t cells = static_cast<int64_t>(n) * a.width;
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + tid; i < cells; i += stride) {
            const int b = static_cast<int>(i / a.width), j = static_cast<int>(i - static_cast<int64_t>(b) * a.width);
            a.table[i] = page_at(b, j);
        }
    }
    if (a.rows > 0) {
        for (int t = blockIdx.x * THREADS + tid; t < min(a.rows, rows); t += stride) {
            const int b = find(row0, t);
            const int pos = max(a.start[b], 0) + t - row0[b];
            if (a.positions) a.positions[t] = pos;
            if (a.token_entry) a.token_entry[t] = b;
            if (a.slots) {
                const int p = page_at(b, a.page.over(pos));
                a.slots[t] = of_pool(p) ? p * a.page.b + a.page.rest(pos) : -1;
            }
        }
    }
    for (int i = blockIdx.x * THREADS + tid; i < a.n_blocks; i += stride) {
        int4 out = make_int4(0, 0, -1, 0);
        if (i < blocks) {
            const int b = find(block0, i);
            const int s = max(a.start[b], 0), c = max(a.count[b], 0);
            const int number = a.block.over(s) + i - block0[b];
            const int from = max(number * a.block.b, s), at = from - number * a.block.b;      // (the block may end behind the last position)
            const int p = page_at(b, number / a.blocks_per_page);
            out = make_int4(row0[b] + from - s, min(a.block.b - at, s + c - from), of_pool(p) ? p * a.blocks_per_page + number % a.blocks_per_page : -1, at);
        }
        a.blocks[i] = out;
    }
}

}  // namespace

// The entry point's arguments (ops/cache8.py fills it; the same fields in the same order).
struct PulseStepMaps {
    const int *start, *count, *pages;
    int *first_row, *positions, *token_entry, *slots, *table, *blocks;
    int requests, n_pages, page_size, num_pages, block, rows, width, n_blocks;
};

extern "C" int pulse_step_maps(const PulseStepMaps* args, hipStream_t stream) {
    PULSE_REQUIRE(args != nullptr, "step_maps: no arguments");
    const auto [start, count, pages, first_row, positions, token_entry, slots, table, blocks, requests, n_pages, page_size, num_pages, block,
                rows, width, n_blocks] = *args;
    PULSE_REQUIRE(requests > 0 && requests <= MAX_REQUESTS, "step_maps: %d requests (1 to %d are served)", requests, MAX_REQUESTS);
    PULSE_REQUIRE(start && count && page_size > 0 && num_pages > 0 && rows >= 0 && width >= 0 && n_blocks >= 0, "step_maps: bad sizes");
    PULSE_REQUIRE(static_cast<int64_t>(num_pages) * page_size <= 0x7fffffff, "step_maps: %d pages of %d tokens have no slot numbers in 32 bits",
                  num_pages, page_size);
    PULSE_REQUIRE(block > 0 && page_size % block == 0, "step_maps: blocks of %d tokens do not divide pages of %d", block, page_size);
    PULSE_REQUIRE(pages || table || !(slots || n_blocks), "step_maps: slots and blocks need the pages or the table");
    PULSE_REQUIRE((reinterpret_cast<uintptr_t>(blocks) & 15) == 0, "step_maps: the blocks must be aligned to 16 bytes");
    MapArgs a{start, count, requests, pages, n_pages, cache8::div_by(page_size), cache8::div_by(block), page_size / block, num_pages,
              first_row, positions, token_entry, slots, positions || token_entry || slots ? rows : 0, table, width,
              reinterpret_cast<int4*>(blocks), blocks ? n_blocks : 0};
    const int64_t most = std::max<int64_t>({pages && table ? static_cast<int64_t>(requests) * width : 0, a.rows, a.n_blocks, 1});
    const int grid = static_cast<int>(std::min<int64_t>((most + THREADS - 1) / THREADS, 1024));
    step_maps_kernel<<<grid, THREADS, 3 * (requests + 1) * sizeof(int), stream>>>(a);
    PULSE_LAUNCH_CHECK("step_maps");
    return 0;
}

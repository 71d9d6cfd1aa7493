// K-g: a matrix product in equal shares of the chip -- which workgroup takes which part of which tile, and where its sums go.  Arithmetic
// on sizes alone, for host and device; no HIP in it, so that it can be walked without a GPU.
#pragma once
#include <cstddef>
#include <cstdint>

namespace xent {

constexpr int TB = 128;          // k of one unit; sizes of slices and paddings are multiples of this

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 256-wide tiles in 16 bits (a 128-wide one asks LDS for 1.5 times as much per product), 128-wide ones where one side has no more rows,
// and in 32 bits, whose matrix instructions are 16 times slower and whose smaller tiles fill the chip more evenly
constexpr int tile_of(int size, int64_t rows_a, int64_t rows_b) { return size == 2 && rows_a > 128 && rows_b > 128 ? 256 : 128; }

// workgroups of these kernels that the chip holds at once: one of 8 waves per compute unit, or two of 4
constexpr int64_t places_of(int tile) { return tile == 256 ? 256 : 512; }

// The units are (tile, step of TB in k), the steps of a tile together; every worker takes `share` consecutive ones.
struct ProductPlan {
    int tile;
    int64_t tiles_m, tiles_n, steps, units, share, workers;
    size_t floats;                    // of the workers' places
};

constexpr ProductPlan product_plan(int size, int64_t M, int64_t N, int64_t K)
{
    ProductPlan q{};
    q.tile = tile_of(size, M, N);
    q.tiles_m = ceil_div(M, q.tile);
    q.tiles_n = ceil_div(N, q.tile);
    q.steps = ceil_div(K, TB);
    q.units = q.tiles_m * q.tiles_n * q.steps;
    q.share = ceil_div(q.units, places_of(q.tile));
    q.workers = ceil_div(q.units, q.share);
    q.floats = (size_t)q.workers * 2 * q.tile * q.tile;
    return q;
}

// What a worker does of one tile, from unit u on: `count` steps from `step`.  A whole tile is finished by its worker.  Of the others a
// share has two at most: the one it ends (it began in an earlier share, step > 0) and the one it begins (step 0) without ending it.
struct TilePart {
    int64_t tile, step, count;
};

constexpr TilePart tile_part(int64_t u, int64_t end, int64_t steps)
{
    const int64_t tile = u / steps, step = u - tile * steps;
    return TilePart{tile, step, end - u < steps - step ? end - u : steps - step};
}

// Where the 32-bit sums of a part go that is not a whole tile: a worker has two places
constexpr int64_t place_of_part(int64_t worker, bool begins_tile) { return worker * 2 + (begins_tile ? 1 : 0); }

// The workers that have parts of a tile: first == last where one has all of it
struct Workers {
    int64_t first, last;
};

constexpr Workers workers_of(int64_t tile, int64_t steps, int64_t share) { return Workers{tile * steps / share, ((tile + 1) * steps - 1) / share}; }

}  // namespace xent

// K-f: embedding lookup with a scale, and the gradient of the table, gfx950.  Both are HBM-bound.
//
//   out[t, :]    = scale * table[id_t, :]
//   dtable[v, :] = scale * sum over {t : id_t = v, v != padding} of dout[t, :]        (rows that no id names are zero)
//
// Counterpart of nn.Embedding.__call__ and its backward pass     src/helpers/ncf_model.py:207-208,220-221
//
// The gradient sorts (id, position) pairs, so that every table row's terms lie together in order of position, and adds them in
// 32 bits in an order that depends on the sizes alone: no atomic adds, the same bits on every run.  Ids of `padding` sort behind
// all others and are never read.
//   sort     least-significant-digit radix sort, stable; up to SMALL_SORT ids in the LDS of one workgroup, else tile by tile
//            (count, scan, scatter per digit).  Workgroups beside the sorting ones write the zeros of the whole gradient meanwhile.
//   sum      the sorted list is cut into chunks of equal length, whatever the ids are, so that a very frequent id is shared out
//            as evenly as the rest: a run that lies in one chunk is finished there, one that crosses chunks leaves 32-bit partial
//            rows, and join_kernel adds those in chunk order.
#include "types16.h"

#include <type_traits>

namespace {

constexpr int RADIX_BITS = 11;
constexpr int BINS = 1 << RADIX_BITS;
constexpr int SORT_THREADS = 256;
constexpr int SMALL_SORT = 4096;        // ids that one workgroup sorts by itself
constexpr int SMALL_THREADS = 1024;

__device__ __forceinline__ int64_t clamp_row(int64_t id, int64_t n) { return id < 0 ? 0 : id >= n ? n - 1 : id; }

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
// Bound by HBM: 1,000,003 ids x 128 bf16 out of 1 M rows in 96 us, 5.3 TB/s read and written, as a copy has.  Up to 256 lanes share a row,
// 16 bytes each where every row start allows it, so that a row is whole lines; grid-stride over the ids.
// lanes_sh: log2 of the lanes that share a row (a power of two, at most 256); a row of `packs` accesses of N values
template <typename T, int N>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ table, int64_t rows, int64_t ld, int packs, int lanes_sh,
                                                     const int64_t* __restrict__ ids, int64_t n, float scale, T* __restrict__ out,
                                                     int32_t* oob)
{
    typedef Pack<T, N> P;
    const int lanes = 1 << lanes_sh;
    const int c0 = threadIdx.x & (lanes - 1);
    const int64_t step = (int64_t)gridDim.x << (8 - lanes_sh);
    for (int64_t t = ((int64_t)blockIdx.x << (8 - lanes_sh)) + (threadIdx.x >> lanes_sh); t < n; t += step) {
        const int64_t id = ids[t];
        if (oob && c0 == 0 && (id < 0 || id >= rows)) atomicAdd(oob, 1);
        const T* src = table + clamp_row(id, rows) * ld;
        T* dst = out + t * ((int64_t)packs * N);
        for (int c = c0; c < packs; c += lanes) {
            P v = *reinterpret_cast<const P*>(src + c * N);
#pragma unroll
            for (int i = 0; i < N; ++i) v.v[i] = (T)((float)v.v[i] * scale);
            *reinterpret_cast<P*>(dst + c * N) = v;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------------------------
struct SortPass {
    const int64_t* ids;      // first pass: the caller's ids; NULL afterwards
    const uint32_t* key_in;
    const uint32_t* pos_in;
    uint32_t* key_out;
    uint32_t* pos_out;
    uint32_t* counts;        // [bins][tiles]: ids of a digit per tile, then (scan) those of the digit in earlier tiles
    uint32_t* totals;        // [bins]
    int64_t n;
    int64_t rows, padding;
    int shift, bits, tiles;
    int per_tile;            // ids per workgroup and pass: a multiple of SORT_THREADS, at most 16 of them per thread
};

__device__ __forceinline__ uint32_t id_key(int64_t id, int64_t rows, int64_t padding)
{
    const int64_t r = clamp_row(id, rows);
    return r == padding ? (uint32_t)rows : (uint32_t)r;          // padding sorts behind every row
}

__device__ __forceinline__ uint32_t load_key(const SortPass& a, int64_t t)
{
    return a.ids ? id_key(a.ids[t], a.rows, a.padding) : a.key_in[t];
}

struct Fill {                // the gradient: 16-byte pieces, then what is left of the last one in 2-byte words
    f32x4* p;
    int64_t packs;
    int words;
};

__device__ __forceinline__ void zero_fill(const Fill& f, int64_t first, int64_t step)
{
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    for (int64_t i = first; i < f.packs; i += step) f.p[i] = z;
    if (first < f.words) reinterpret_cast<uint16_t*>(f.p + f.packs)[first] = 0;
}

// The sort leaves most of the memory's time unused: each of its launches has workgroups behind its own `work` ones that write a part of
// the gradient's zeros (16 bytes at a time).  All three kernels have 256 threads.
__device__ __forceinline__ bool fills(const Fill& fill, int work)
{
    if ((int)blockIdx.x < work) return false;
    zero_fill(fill, (int64_t)(blockIdx.x - work) * 256 + threadIdx.x, (int64_t)(gridDim.x - work) * 256);
    return true;
}

// The three launches of a digit are short (524,289 ids, two digits of 10 bits: 12 + 10 + 18 us each with a sixth of 256 MB of zeros beside
// them) and bound by latency; ids, keys and positions are 12 bytes each.
// a tile's digit counts
__global__ __launch_bounds__(SORT_THREADS) void count_kernel(SortPass a, Fill fill)
{
    __shared__ uint32_t bin[BINS];
    if (fills(fill, a.tiles)) return;
    const int bins = 1 << a.bits;
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) bin[b] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * a.per_tile;
#pragma unroll 4
    for (int i = 0; i < a.per_tile; i += SORT_THREADS) {
        const int64_t t = t0 + i + threadIdx.x;
        if (t < a.n) atomicAdd(&bin[(load_key(a, t) >> a.shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) a.counts[(int64_t)b * a.tiles + blockIdx.x] = bin[b];
}

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v, int lane)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// one wave per digit: how many of its ids lie in earlier tiles
__global__ __launch_bounds__(256) void scan_kernel(SortPass a, Fill fill)
{
    if (fills(fill, ((1 << a.bits) + 3) / 4)) return;
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (b >= (1 << a.bits)) return;
    uint32_t* row = a.counts + (int64_t)b * a.tiles;
    uint32_t run = 0;
    for (int t0 = 0; t0 < a.tiles; t0 += 64) {
        const uint32_t v = t0 + lane < a.tiles ? row[t0 + lane] : 0;
        const uint32_t inc = wave_inclusive(v, lane);
        if (t0 + lane < a.tiles) row[t0 + lane] = run + inc - v;
        run += __shfl(inc, 63, 64);
    }
    if (lane == 0) a.totals[b] = run;
}

// Exclusive scan of v[0 .. count) in LDS by the whole workgroup (count <= BINS); scratch: one word per wave.
template <int THREADS> __device__ void block_exclusive(uint32_t* v, int count, uint32_t* scratch)
{
    constexpr int PER = BINS / THREADS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t x[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = tid * PER + i;
        x[i] = j < count ? v[j] : 0;
        sum += x[i];
    }
    const uint32_t inc = wave_inclusive(sum, lane);
    if (lane == 63) scratch[wave] = inc;
    __syncthreads();
    uint32_t base = inc - sum;
    for (int w = 0; w < wave; ++w) base += scratch[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = tid * PER + i;
        if (j < count) v[j] = base;
        base += x[i];
    }
    __syncthreads();
}

// lanes of the wave that hold the same digit (only lanes of `active` count)
__device__ __forceinline__ unsigned long long same_digit(uint32_t d, int bits, unsigned long long active)
{
    unsigned long long m = active;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((d >> b) & 1u);
        m &= ((d >> b) & 1u) ? set : ~set;
    }
    return m;
}

// Orders the LDS accesses of one wave's lanes: the hardware keeps them in order, the compiler has to as well.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Destination of every id of one tile: wave w holds STEPS * 64 consecutive ids; `at` [waves][bins] comes in as the first place of
// wave w's ids of a digit and counts up.  LDS accesses of one wave complete in order, so the waves need no barrier among themselves.
__device__ __forceinline__ uint32_t place_of(uint32_t* at, uint32_t digit, int bits, bool valid, int lane)
{
    const unsigned long long active = __ballot(valid);
    const unsigned long long same = same_digit(digit, bits, active);
    uint32_t base = 0;
    if (valid) base = at[digit];
    const uint32_t rank = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
    wave_fence();
    if (valid && rank == 0) at[digit] = base + (uint32_t)__popcll(same);
    wave_fence();
    return base + rank;
}

template <int STEPS>
__global__ __launch_bounds__(SORT_THREADS) void scatter_kernel(SortPass a, Fill fill)
{
    constexpr int WAVES = SORT_THREADS / 64;
    __shared__ uint32_t first[BINS];
    __shared__ uint32_t at[WAVES][BINS];
    __shared__ uint32_t scratch[WAVES];
    if (fills(fill, a.tiles)) return;
    const int bins = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int b = tid; b < bins; b += SORT_THREADS) {
        first[b] = a.totals[b];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) at[w][b] = 0;
    }
    __syncthreads();
    block_exclusive<SORT_THREADS>(first, bins, scratch);
    const int64_t t0 = (int64_t)blockIdx.x * a.per_tile + wave * (STEPS * 64);
    uint32_t key[STEPS], pos[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int64_t t = t0 + i * 64 + lane;
        key[i] = t < a.n ? load_key(a, t) : 0;
        pos[i] = t < a.n ? (a.ids ? (uint32_t)t : a.pos_in[t]) : 0;
        if (t < a.n) atomicAdd(&at[wave][(key[i] >> a.shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = tid; b < bins; b += SORT_THREADS) {
        uint32_t base = first[b] + a.counts[(int64_t)b * a.tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t c = at[w][b];
            at[w][b] = base;
            base += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int64_t t = t0 + i * 64 + lane;
        const uint32_t p = place_of(at[wave], (key[i] >> a.shift) & (bins - 1), a.bits, t < a.n, lane);
        if (t < a.n) {
            a.key_out[p] = key[i];
            a.pos_out[p] = pos[i];
        }
    }
}

// Up to SMALL_SORT ids: every pass in the LDS of workgroup 0; the other workgroups write the zeros.  4096 ids in 12 us, bound by the
// latency of its passes (two of 7 bits for 6,038 rows); by tiles it would be six launches.
__global__ __launch_bounds__(SMALL_THREADS) void small_sort_kernel(SortPass a, int passes, Fill fill)
{
    constexpr int WAVES = SMALL_THREADS / 64, STEPS = SMALL_SORT / SMALL_THREADS;
    __shared__ uint16_t place[WAVES][BINS];           // first place of a wave's ids of a digit
    __shared__ uint32_t first[BINS];
    __shared__ uint32_t keys[SMALL_SORT];
    __shared__ uint16_t poss[SMALL_SORT];
    __shared__ uint32_t scratch[WAVES];
    if (blockIdx.x) {
        zero_fill(fill, (int64_t)(blockIdx.x - 1) * SMALL_THREADS + threadIdx.x, (int64_t)(gridDim.x - 1) * SMALL_THREADS);
        return;
    }
    const int bins = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = (int)a.n;
    const int per = ((n + SMALL_THREADS - 1) / SMALL_THREADS) * 64;      // ids of one wave: consecutive, 64 a step
    uint32_t key[STEPS];
    uint16_t pos[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int t = wave * per + i * 64 + lane;
        key[i] = i * 64 < per && t < n ? id_key(a.ids[t], a.rows, a.padding) : 0;
        pos[i] = (uint16_t)t;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * a.bits;
        for (int b = tid; b < bins * WAVES; b += SMALL_THREADS) place[b / bins][b & (bins - 1)] = 0;
        __syncthreads();
        uint32_t rank[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {                                // rank inside the wave, counts per wave
            const int t = wave * per + i * 64 + lane;
            const bool valid = i * 64 < per && t < n;
            const uint32_t d = (key[i] >> shift) & (bins - 1);
            const unsigned long long same = same_digit(d, a.bits, __ballot(valid));
            const uint32_t below = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
            uint32_t seen = 0;
            if (valid) seen = place[wave][d];
            wave_fence();
            if (valid && below == 0) place[wave][d] = (uint16_t)(seen + __popcll(same));
            wave_fence();
            rank[i] = seen + below;
        }
        __syncthreads();
        for (int b = tid; b < bins; b += SMALL_THREADS) {
            uint32_t run = 0;
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t c = place[w][b];
                place[w][b] = (uint16_t)run;
                run += c;
            }
            first[b] = run;
        }
        __syncthreads();
        block_exclusive<SMALL_THREADS>(first, bins, scratch);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int t = wave * per + i * 64 + lane;
            if (i * 64 < per && t < n) {
                const uint32_t d = (key[i] >> shift) & (bins - 1);
                const uint32_t p = first[d] + place[wave][d] + rank[i];
                keys[p] = key[i];
                poss[p] = pos[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int t = wave * per + i * 64 + lane;
            if (i * 64 < per && t < n) {
                key[i] = keys[t];
                pos[i] = poss[t];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int t = wave * per + i * 64 + lane;
        if (i * 64 < per && t < n) {
            a.key_out[t] = key[i];
            a.pos_out[t] = pos[i];
        }
    }
}

// ---------------------------------------------------------------------------------------------
// sum
// ---------------------------------------------------------------------------------------------
struct SumArgs {
    const uint32_t* key;
    const uint32_t* pos;
    int64_t n, rows;
    int chunk;               // sorted places per chunk
    int64_t chunks;
    int packs;               // accesses of N values per row
    int dim;
    int64_t ldg;
    float scale;
    float* part;             // [chunks][2][dim]: the run that came in from the left, the run that goes on to the right
};

template <typename T, int N> __device__ __forceinline__ void store_row(T* dst, const float* acc, float scale)
{
    Pack<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = (T)(acc[i] * scale);
    *reinterpret_cast<Pack<T, N>*>(dst) = v;
}

// 1 << lanes_sh lanes walk one chunk for one block of columns, eight rows under way at once.  Bound by HBM: every row of the gradient is
// read once, every row of the table that an id names is written once (524,289 ids, 0.6 of them counting, x 128 bf16: 38 us).
template <typename T, int N>
__global__ __launch_bounds__(256) void sum_kernel(SumArgs a, const T* __restrict__ grad, T* __restrict__ out, int lanes_sh)
{
    constexpr int AHEAD = 8;
    typedef Pack<T, N> P;
    const int lanes = 1 << lanes_sh;
    const int64_t c = ((int64_t)blockIdx.x << (8 - lanes_sh)) + (threadIdx.x >> lanes_sh);
    const int col = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    if (c >= a.chunks || col >= a.packs) return;
    const int64_t i0 = c * a.chunk, i1 = i0 + a.chunk < a.n ? i0 + a.chunk : a.n;
    const uint32_t last = (uint32_t)a.rows;                     // the key of padding: nothing from here on
    uint32_t cur = a.key[i0];
    if (cur >= last) return;
    bool from_left = i0 > 0 && a.key[i0 - 1] == cur;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    float* part = a.part + c * 2 * (int64_t)a.dim + col * N;
    // places are read one batch before their rows
    uint32_t key[AHEAD], next_key[AHEAD], next_pos[AHEAD];
    auto places = [&](int64_t i) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t at = i + u < i1 ? i + u : i1 - 1;
            next_key[u] = i + u < i1 ? a.key[at] : last;
            next_pos[u] = a.pos[at];
        }
    };
    places(i0);
    for (int64_t i = i0; i < i1; i += AHEAD) {
        P v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            key[u] = next_key[u];
            // behind the chunk and for padding: row 0 of the gradient is read and not used
            const int64_t p = key[u] < last ? next_pos[u] : 0;
            v[u] = *reinterpret_cast<const P*>(grad + p * a.ldg + col * N);
        }
        if (i + AHEAD < i1) places(i + AHEAD);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (i + u < i1 && cur < last) {
                if (key[u] != cur) {
                    if (from_left) {
#pragma unroll
                        for (int j = 0; j < N; ++j) part[j] = acc[j];
                    } else {
                        store_row<T, N>(out + cur * (int64_t)a.dim + col * N, acc, a.scale);
                    }
                    from_left = false;
                    cur = key[u];
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] = 0.f;
                }
                if (cur < last) {
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += (float)v[u].v[j];
                }
            }
        }
        if (cur >= last) return;
    }
    const bool to_right = i1 < a.n && a.key[i1] == cur;
    if (!from_left && !to_right) {
        store_row<T, N>(out + cur * (int64_t)a.dim + col * N, acc, a.scale);
        return;
    }
    if (!from_left) part += a.dim;
#pragma unroll
    for (int j = 0; j < N; ++j) part[j] = acc[j];
}

// A run that starts in chunk c and goes on: its partial rows are [c][1], then [c + 1][0] .. [e][0] with e the chunk it ends in.
// One workgroup looks at `per` consecutive chunks (at most 8); the groups of lanes take the partial rows in turn and their sums are added in
// group order.  A very frequent id has thousands of partial rows for each group; equal ones round the same way each time (2,000,003 equal rows
// of 512 values: 2.5e-5 off when they were added one after the other).
template <typename T, int N>
__global__ __launch_bounds__(256) void join_kernel(SumArgs a, int per, T* __restrict__ out, int lanes_sh)
{
    __shared__ int goes_on[8];
    __shared__ int window_end;
    __shared__ float sums[256 * N];
    const int lanes = 1 << lanes_sh, groups = 256 >> lanes_sh;
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_sh;
    const int col = blockIdx.y * lanes + lane;
    if ((int)threadIdx.x < per) {
        const int64_t c = (int64_t)blockIdx.x * per + threadIdx.x;
        bool run = false;
        if (c + 1 < a.chunks) {
            const int64_t i0 = c * a.chunk, i1 = i0 + a.chunk;
            const uint32_t k = a.key[i1 - 1];
            run = k < (uint32_t)a.rows && a.key[i1] == k && (i0 == 0 || a.key[i0 - 1] != k);
        }
        goes_on[threadIdx.x] = run;
    }
    __syncthreads();
    for (int j = 0; j < per; ++j) {
        if (!goes_on[j]) continue;                               // the same for the whole workgroup
        const int64_t c = (int64_t)blockIdx.x * per + j;
        // the last chunk that begins with the run's key, looked for 256 chunks at a time
        const uint32_t k = a.key[(c + 1) * a.chunk];
        int64_t e = c + 1;
        for (;;) {
            const int64_t at = e + 1 + threadIdx.x;
            const bool out = at >= a.chunks || a.key[at * a.chunk] != k;
            const unsigned long long outs = __ballot(out);
            if (threadIdx.x == 0) window_end = 256;
            __syncthreads();
            if ((threadIdx.x & 63) == 0 && outs) atomicMin(&window_end, (int)(threadIdx.x + __ffsll(outs) - 1));
            __syncthreads();
            const int more = window_end;
            __syncthreads();
            e += more;
            if (more < 256) break;
        }
        Sum acc[N];
        if (col < a.packs) {
            // four rows at a time, all on their way at once (behind the end the last one, not used)
            for (int64_t p = c + group; p <= e; p += 4 * groups) {
                float v[4][N], four[N];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int64_t q = p + k * groups < e ? p + k * groups : e;
                    const float* src = a.part + (2 * q + (q == c ? 1 : 0)) * (int64_t)a.dim + col * N;
#pragma unroll
                    for (int i = 0; i < N; ++i) v[k][i] = src[i];
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    four[i] = v[0][i];
#pragma unroll
                    for (int k = 1; k < 4; ++k) four[i] += p + k * groups <= e ? v[k][i] : 0.f;
                    acc[i].template add<true>(four[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) sums[threadIdx.x * N + i] = acc[i].s;
        __syncthreads();
        if (group == 0 && col < a.packs) {
            const int busy = e - c + 1 < groups ? (int)(e - c + 1) : groups;        // most runs have two partial rows
            for (int g = 1; g < busy; ++g)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i].template add<true>(sums[(g * lanes + lane) * N + i]);
            float total[N];
#pragma unroll
            for (int i = 0; i < N; ++i) total[i] = acc[i].s;
            store_row<T, N>(out + k * (int64_t)a.dim + col * N, total, a.scale);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// The widest access (in bytes) that every row start allows: rows lie `ld` values apart, `dim` values long
int access_bytes(const void* p, int64_t ld, int dim, int size)
{
    int b = 16;
    while (b > size && ((uintptr_t)p % b || (ld * size) % b || ((int64_t)dim * size) % b)) b >>= 1;
    return b;
}

template <typename T, typename F> int with_access(int bytes, F&& fn)
{
    switch (bytes / (int)sizeof(T)) {
    case 8: return fn(std::integral_constant<int, sizeof(T) == 2 ? 8 : 4>());
    case 4: return fn(std::integral_constant<int, 4>());
    case 2: return fn(std::integral_constant<int, 2>());
    default: return fn(std::integral_constant<int, 1>());
    }
}

int lanes_shift(int packs, int most)
{
    int sh = 0;
    while ((1 << sh) < packs && sh < most) ++sh;
    return sh;
}

int bit_length(int64_t v)
{
    int b = 1;
    while (v >> b) ++b;
    return b;
}

struct GradPlan {
    int per_tile, tiles, passes, bits, chunk, join;
    int64_t chunks;
    size_t keys, poss, counts, totals, part, total;
};

GradPlan grad_plan(int64_t n, int64_t rows, int dim)
{
    GradPlan p{};
    const int need = bit_length(rows);                 // keys 0 .. rows, the last one being padding
    p.passes = (need + RADIX_BITS - 1) / RADIX_BITS;
    p.bits = (need + p.passes - 1) / p.passes;
    // Measured (us, gradients in bf16, 5,000 x 64 / 70,001 x 50 / 200,000 x 64 / 524,289 x 128 / 2,000,003 x 64 ids x values):
    //   as chosen here            35 / 43 / 76 / 159 / 240
    //   tiles of 1024 always      35 / 43 / 76 / 159 / 293        of 4096 always  57 / 65 / 99 / 165 / 241
    //   chunks of 8 always        35 / 45 / 80 / 175 / 343        of 64 always    49 / 47 / 79 / 153 / 241
    //   join of 1 chunk always    35 / 42 / 74 / 162 / 253        of 4 always     39 / 43 / 76 / 159 / 241
    // Small tiles fill the chip, large ones keep the counts [digits][tiles] small; short chunks hide latency, long ones leave less to join.
    p.per_tile = n <= (1 << 20) ? 1024 : 4096;
    p.tiles = (int)ceil_div64(n, p.per_tile);
    p.chunk = n <= 16384 ? 8 : n <= (1 << 17) ? 16 : n <= (1 << 20) ? 32 : 64;
    p.chunks = ceil_div64(n, p.chunk);
    p.join = p.chunks <= 4096 ? 1 : 4;
    const bool small = n <= SMALL_SORT;
    const size_t copies = small ? 1 : 2;
    const size_t list = align_up((size_t)n * 4, 256);
    p.keys = 0;
    p.poss = copies * list;
    p.counts = 2 * copies * list;
    p.totals = p.counts + (small ? 0 : align_up(((size_t)p.tiles << p.bits) * 4, 256));
    p.part = p.totals + (small ? 0 : align_up((size_t)4 << p.bits, 256));
    p.total = p.part + (size_t)p.chunks * 2 * dim * 4;
    return p;
}

}  // namespace

extern "C" int reco_embedding(const void* table, int64_t rows, int64_t ld, int dim, int dtype, const int64_t* ids, int64_t n, float scale,
                              void* out, int32_t* oob, void* stream)
{
    if (n <= 0) return RECO_OK;
    RECO_REQUIRE(table && ids && out, "embedding: null pointer");
    RECO_REQUIRE(rows > 0 && dim > 0 && ld >= dim, "embedding: bad table shape (%lld rows of %d, stride %lld)", (long long)rows, dim, (long long)ld);
    return reco_with_type(dtype, [&](auto zero) -> int {
        typedef decltype(zero) T;
        const int bytes = access_bytes(table, ld, dim, sizeof(T)), out_bytes = access_bytes(out, dim, dim, sizeof(T));
        return with_access<T>(bytes < out_bytes ? bytes : out_bytes, [&](auto width) -> int {
            constexpr int N = decltype(width)::value;
            const int packs = dim / N, sh = lanes_shift(packs, 8);
            int64_t blocks = ceil_div64(n, 256 >> sh);
            if (blocks > 2048) blocks = 2048;
            ProfScope prof((hipStream_t)stream, RECO_PROF_EMBEDDING);
            hipLaunchKernelGGL((lookup_kernel<T, N>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, (const T*)table, rows, ld, packs, sh,
                               ids, n, scale, (T*)out, oob);
            RECO_CHECK_LAUNCH();
            return RECO_OK;
        });
    });
}

extern "C" size_t reco_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int dim)
{
    return n > 0 && rows > 0 && dim > 0 ? grad_plan(n, rows, dim).total : 0;
}

extern "C" int reco_embedding_grad(const int64_t* ids, int64_t n, const void* grad, int64_t ldg, int dim, int dtype, int64_t rows, float scale,
                                   int64_t padding, void* out, void* ws, size_t ws_bytes, void* stream)
{
    RECO_REQUIRE(n >= 0 && n < (int64_t)1 << 31, "embedding_grad: %lld ids (at most 2^31 - 1)", (long long)n);
    RECO_REQUIRE(rows > 0 && rows < ((int64_t)1 << 31) - 1 && dim > 0, "embedding_grad: bad table shape (%lld rows of %d)", (long long)rows, dim);
    RECO_REQUIRE(out && (n == 0 || (ids && grad)), "embedding_grad: null pointer");
    RECO_REQUIRE(n == 0 || ldg >= dim, "embedding_grad: gradient row stride %lld below the width %d", (long long)ldg, dim);
    RECO_REQUIRE(dtype >= RECO_DT_F32 && dtype <= RECO_DT_F16, "unknown element type %d", dtype);
    RECO_REQUIRE((uintptr_t)out % 16 == 0, "embedding_grad: the output must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const int size = dtype == RECO_DT_F32 ? 4 : 2;
    const int64_t out_bytes = rows * dim * size;
    const Fill fill{(f32x4*)out, out_bytes / 16, (int)(out_bytes % 16 / 2)};
    const int64_t fill_want = fill.packs ? ceil_div64(fill.packs, 4 * SORT_THREADS) : 1;
    const GradPlan p = n ? grad_plan(n, rows, dim) : GradPlan{};
    RECO_REQUIRE(n == 0 || (ws && (uintptr_t)ws % 16 == 0), "embedding_grad: the workspace is missing or not 16-byte aligned");
    if (n && ws_bytes < p.total) {
        reco_set_error("embedding_grad: workspace of %zu bytes, %zu needed", ws_bytes, p.total);
        return RECO_ENOMEM;
    }
    SortPass a{};
    a.ids = ids; a.n = n; a.rows = rows; a.padding = padding; a.bits = p.bits; a.tiles = p.tiles; a.per_tile = p.per_tile;
    char* w = (char*)ws;
    const uint32_t *key = nullptr, *pos = nullptr;
    if (n <= SMALL_SORT) {
        const int64_t blocks = fill_want < 1024 ? fill_want : 1024;
        a.key_out = (uint32_t*)(w + p.keys);
        a.pos_out = (uint32_t*)(w + p.poss);
        ProfScope prof(s, RECO_PROF_EMBEDDING);
        hipLaunchKernelGGL(small_sort_kernel, dim3((unsigned)(1 + blocks)), dim3(SMALL_THREADS), 0, s, a, p.passes, fill);
        RECO_CHECK_LAUNCH();
        if (n == 0) return RECO_OK;
        key = a.key_out;
        pos = a.pos_out;
    } else {
        const size_t list = align_up((size_t)n * 4, 256);
        a.counts = (uint32_t*)(w + p.counts);
        a.totals = (uint32_t*)(w + p.totals);
        // the zeros in proportion to the time that the launches take (10 : 6 : 14 measured at 524,289 ids, 10-bit digits); the last one
        // takes the rest
        int64_t filled = 0;
        int share = 0;
        auto part = [&](int weight, int64_t* blocks) {
            share += weight;
            const int64_t to = share == 30 * p.passes ? fill.packs : fill.packs * share / (30 * p.passes);
            const Fill f{fill.p + filled, to - filled, share == 30 * p.passes ? fill.words : 0};
            filled = to;
            const int64_t want = ceil_div64(f.packs, 4 * 256);
            *blocks = want < 1 ? (f.words ? 1 : 0) : want < 1024 ? want : 1024;
            return f;
        };
        for (int pass = 0; pass < p.passes; ++pass) {
            a.shift = pass * p.bits;
            a.key_out = (uint32_t*)(w + p.keys + (pass & 1) * list);
            a.pos_out = (uint32_t*)(w + p.poss + (pass & 1) * list);
            ProfScope prof(s, RECO_PROF_EMBEDDING);
            int64_t extra;
            Fill f = part(10, &extra);
            hipLaunchKernelGGL(count_kernel, dim3((unsigned)(p.tiles + extra)), dim3(SORT_THREADS), 0, s, a, f);
            f = part(6, &extra);
            hipLaunchKernelGGL(scan_kernel, dim3((unsigned)(ceil_div64(1 << p.bits, 4) + extra)), dim3(256), 0, s, a, f);
            f = part(14, &extra);
            if (p.per_tile == 1024) hipLaunchKernelGGL(scatter_kernel<4>, dim3((unsigned)(p.tiles + extra)), dim3(SORT_THREADS), 0, s, a, f);
            else hipLaunchKernelGGL(scatter_kernel<16>, dim3((unsigned)(p.tiles + extra)), dim3(SORT_THREADS), 0, s, a, f);
            RECO_CHECK_LAUNCH();
            a.ids = nullptr;
            a.key_in = a.key_out;
            a.pos_in = a.pos_out;
        }
        key = a.key_out;
        pos = a.pos_out;
    }
    return reco_with_type(dtype, [&](auto zero) -> int {
        typedef decltype(zero) T;
        const int bytes = access_bytes(grad, ldg, dim, sizeof(T)), ob = access_bytes(out, dim, dim, sizeof(T));
        return with_access<T>(bytes < ob ? bytes : ob, [&](auto width) -> int {
            constexpr int N = decltype(width)::value;
            SumArgs b{key, pos, n, rows, p.chunk, p.chunks, dim / N, dim, ldg, scale, (float*)(w + p.part)};
            const int sh = lanes_shift(b.packs, 6);
            const unsigned cols = (unsigned)ceil_div64(b.packs, 1 << sh);
            ProfScope prof(s, RECO_PROF_EMBEDDING);
            hipLaunchKernelGGL((sum_kernel<T, N>), dim3((unsigned)ceil_div64(p.chunks, 256 >> sh), cols), dim3(256), 0, s, b, (const T*)grad, (T*)out, sh);
            hipLaunchKernelGGL((join_kernel<T, N>), dim3((unsigned)ceil_div64(p.chunks, p.join), cols), dim3(256), 0, s, b, p.join, (T*)out, sh);
            RECO_CHECK_LAUNCH();
            return RECO_OK;
        });
    });
}

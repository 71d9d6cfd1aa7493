// K-g: softmax cross entropy of x W^T + bias over a whole catalogue, and its gradients, gfx950.
//
//   z[t, v] = sum_d x[t, d] W[v, d] + bias[v]             never stored whole: the vocabulary is walked in pieces
//   others_t = log sum over v != y_t of exp(z[t, v]),     d_t = others_t - z[t, y_t]
//   loss_t = log(1 + exp(d_t)),   q_t = 1 - p_t = 1 / (1 + exp(-d_t)),   lse_t = z[t, y_t] + loss_t
//   G[t, v] = g_t exp(z[t, v] - lse_t),  G[t, y_t] = -g_t q_t
//   dx = G W,   dW = G^T x,   dbias = column sums of G
//
// The target's own term is kept out of the sum: loss and q keep their digits where the model is sure of the target (p near one),
// which 1 - p would lose.  Ignored rows have no loss and no gradient, whatever their x holds.
//
// Everything but the operands of the matrix instructions is 32 bits wide: logits, running maxima and sums, losses, accumulators.  G is
// rounded to the operands' type to be multiplied: half a step of each term of dx and dW, where the result takes one such rounding too; more
// than that only where the terms cancel, and the matrix instructions take 16-bit operands in 16 bits.  dbias multiplies nothing and adds
// the terms as they are.  Half-precision G is held times 2^14, so that probabilities down to 2^-28 are normal numbers.
//
// This file: the forms for every width and for few rows.  A piece of G, [T, piece] in the operands' type, is written and read by two matrix
// products.  Bound by the matrix instructions: bf16 4096 x 131,072 x 1024 statistics 1.0 ms (1.1 PFLOP/s), G 0.16 ms and the products 0.12
// ms each per piece of 16,384 columns (0.84, 1.14, 1.08 PFLOP/s; a large library product reaches 1.34); f32 3706 x 6040 x 500 0.24 ms and
// 0.21 ms each, matrix instructions busy for 0.81 to 0.85 of the cycles.
//
// xent_narrow.h: rows of up to 128 values in 32 bits, 256 in 16 (4097 x 50,021 x 250 f16 with gradients 0.81 ms, 1.89 by this file's form).
#include "xent_plan.h"
#include "xent_shared.h"

namespace {

using namespace xent;

// ---------------------------------------------------------------------------------------------
// a B x B tile of a matrix product, B = 256 (8 waves, 128 x 64 each) or 128 (4 waves, 64 x 64 each): operands staged through LDS, two
// steps of k in it; the next one arrives in registers while this one is multiplied; one barrier per step
// ---------------------------------------------------------------------------------------------
// A matrix of which B rows r take part: KC: element (r, k) at p[r * ld + k], else at p[k * ld + r].  Row starts are 16-byte aligned;
// `rows` (the limit of r) and k_end count whole VEC groups along the contiguous side.
template <typename T> struct Operand {
    const T* p;
    int64_t ld;
    int64_t rows;
};

template <int B> struct Shape {
    static constexpr int THREADS = B * 2, WAVES_N = B / 64, WM = B == 256 ? 128 : 64, WN = 64, MB = WM / 32, NB = 2;
    static __device__ __forceinline__ int wm() { return (threadIdx.x >> 6) / WAVES_N * WM; }
    static __device__ __forceinline__ int wn() { return (threadIdx.x >> 6) % WAVES_N * WN; }
};

// 64 (32-bit: 32) of k for B rows, on their way from memory to LDS and from there to fragments.  In LDS without padding: the 16-byte
// chunks of a stored row change places with the row, so that 16 rows at one chunk, or 4 rows at 64 bytes (the transposed reads), spread
// over the 64 banks.  Memory to LDS without registers: a wave's load fills 1 KB in lane order, so the lanes choose what they fetch.
template <typename T, bool KC, int B> struct Stage {
    typedef typename Traits<T>::frag frag;
    static constexpr int VEC = Traits<T>::VEC, BK = Traits<T>::BK;
    static constexpr int ROW = KC ? BK : B, CH = ROW / VEC, ROWS = KC ? B : BK, WAVES = Shape<B>::THREADS / 64;
    static constexpr int SIZE = ROWS * ROW, PIECES = SIZE / VEC / Shape<B>::THREADS, ROW_STEP = ROWS / PIECES;
    static constexpr uint32_t NOWHERE = 0x80000000u;       // an offset behind every buffer: reads as zeros
    const T* base;
    int64_t step;
    uint32_t offset[PIECES];
    int k_of;               // KC: this lane's k inside the step; else the k of its first piece

    static __device__ __forceinline__ int twist(int row) { return KC ? (row >> 1) & 7 : ((row >> 2) & 3) | (row & 3) << 2; }

    __device__ __forceinline__ void init(const Operand<T>& o, int64_t r0, int64_t k0)
    {
        const int row = threadIdx.x / CH;
        base = o.p + (KC ? r0 * o.ld + k0 : k0 * o.ld + r0);
        step = KC ? BK : BK * o.ld;
        static_assert(!KC || ROW_STEP % 16 == 0, "every piece of a lane has the same k");
        k_of = KC ? ((threadIdx.x % CH) ^ twist(row)) * VEC : row;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int at = row + i * ROW_STEP, col = ((threadIdx.x % CH) ^ twist(at)) * VEC;
            offset[i] = r0 + (KC ? at : col) < o.rows ? (uint32_t)((at * o.ld + col) * (int64_t)sizeof(T)) : NOWHERE;
        }
    }
    // the next step's values, `left` of k before its end, set out for `lds`
    __device__ __forceinline__ void load(T* lds, int64_t left)
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        base += step;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const bool in = k_of + (KC ? 0 : i * ROW_STEP) < left;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + (i * WAVES + wave) * (64 * VEC)), 16,
                                                     in ? offset[i] : NOWHERE, 0, 0, 0);
        }
    }
    // rows r .. r + 31 (r a multiple of 32) and one KSTEP of k (a multiple of KSTEP) from LDS
    static __device__ __forceinline__ frag fragment(const T* lds, int r, int k)
    {
        const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
        frag f;
        if constexpr (KC) {
            f = *reinterpret_cast<const frag*>(lds + (r + l31) * ROW + (((k / VEC + half) ^ twist(l31)) * VEC));
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = k + 4 * half + i;
                f[i] = lds[row * ROW + (((r + l31) / 4) ^ twist(row)) * 4 + (l31 & 3)];
            }
        } else {
            // 16 lanes read 4 k rows of 16 values and get them transposed: lane i value i of each row
            const int row = k + 8 * half + ((lane & 15) >> 2), c = r / 8 + ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), in = (lane & 1) * 4;
            typedef __attribute__((address_space(3))) s16x4* lds_ptr;
            union { s16x4 h[2]; frag f; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + row * ROW + (c ^ twist(row)) * 8 + in));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + (row + 4) * ROW + (c ^ twist(row + 4)) * 8 + in));
            f = u.f;
        }
        return f;
    }
};

// Workgroups with the same number modulo 8 run on the same XCD, which has a cache of its own: the n-th of `total` takes the place that
// gives every XCD a contiguous run of places.  Neighbouring places share panels.
__device__ __forceinline__ int64_t place_of(int64_t n, int64_t total)
{
    const int64_t q = total / 8, r = total % 8, xcd = n % 8;
    return xcd * q + (xcd < r ? xcd : r) + n / 8;
}

// Places as (a, b), a < na: runs of 4 a beside each other, so that 32 consecutive places hold 4 a times 8 b
__device__ __forceinline__ void pair_of(int64_t place, int64_t na, int64_t nb, int64_t& a, int64_t& b)
{
    const int64_t group = place / (4 * nb), in = place - group * 4 * nb, wide = na - group * 4 < 4 ? na - group * 4 : 4;
    a = group * 4 + in % wide;
    b = in / wide;
}

// Two steps of both operands: four arrays, so that the compiler sees that what is read is not what is on its way
#define TILE_LDS(T, AKC, BKC, B)                                                                              \
    __shared__ __attribute__((aligned(1024))) T lds_a0[Stage<T, AKC, B>::SIZE], lds_a1[Stage<T, AKC, B>::SIZE]; \
    __shared__ __attribute__((aligned(1024))) T lds_b0[Stage<T, BKC, B>::SIZE], lds_b1[Stage<T, BKC, B>::SIZE]
#define TILE_LDS_ARGS lds_a0, lds_a1, lds_b0, lds_b1

template <int B> using Acc = f32x16[Shape<B>::MB][Shape<B>::NB];

// Whether the logits of the statistics may be kept for G: in 32 bits a product costs 2 D / 125 TFLOP/s per logit and its 8 bytes of traffic
// 2 ps (f32 4096 x 20,000 x 768, with gradients: 3.18 ms, 4.01 with a second product; 3706 x 6040 x 500 0.70 ms, 0.87).  In 16 bits the two
// are alike up to some 1000 values (bf16 4096 x 20,000 x 768: 0.86 both; 1000 x 60,000 x 2048: 1.34, 1.46), not worth the memory.
template <typename T> constexpr bool KEEPS = sizeof(T) == 4;

// A tile's logits as its lanes hold them (kept from the statistics for G): tile (token, vocabulary), then wave, register group, lane
template <int B> __device__ __forceinline__ int64_t kept_at(int64_t token_tile, int64_t tiles_v, int64_t v_tile)
{
    return (token_tile * tiles_v + v_tile) * (B * B) + (threadIdx.x >> 6) * (B * B / (Shape<B>::THREADS / 64)) + (threadIdx.x & 63) * 4;
}

template <int B, typename F> __device__ __forceinline__ void each_kept(F&& fn)          // fn(i, j, first register, offset)
{
#pragma unroll
    for (int i = 0; i < Shape<B>::MB; ++i)
#pragma unroll
        for (int j = 0; j < Shape<B>::NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4) fn(i, j, r, ((i * Shape<B>::NB + j) * 4 + r / 4) * 256);
}

// All of this wave's loads and LDS accesses are done, then the workgroup's.  The fences are for the compiler, to which neither the wait nor
// the barrier is an access to memory; the wait is for the loads from memory to LDS, which the fences leave under way.
__device__ __forceinline__ void drain_and_meet()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// acc += A (rows m0 ..) times B (rows n0 ..) over k in [k0, k_end).  Fragments are read one KSTEP before they are multiplied.  The barrier
// stands before the last quarter of a step, whose fragments are in registers already: behind it nobody reads this half of LDS any
// more, the step after next sets out for it, and the other half has arrived.
// DIRECT: whose tiles these are (product_kernel); the same work either way
template <typename T, bool AKC, bool BKC, int B, bool DIRECT = false>
__device__ __forceinline__ void tile_product(Acc<B>& acc, const Operand<T>& A, const Operand<T>& Bm, int64_t m0, int64_t n0, int64_t k0, int64_t k_end, T* a0, T* a1,
                                             T* b0, T* b1)
{
    typedef Shape<B> S;
    typedef Stage<T, AKC, B> SA;
    typedef Stage<T, BKC, B> SB;
    constexpr int BK = Traits<T>::BK, KSTEP = Traits<T>::KSTEP;
    static_assert(BK == 4 * KSTEP, "a step is four products deep");
    const int wm = S::wm(), wn = S::wn();
    SA sa;
    SB sb;
    typename Traits<T>::frag a[2][S::MB], b[2][S::NB];
    auto read = [&](const T* la, const T* lb, int s) {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) b[s & 1][j] = SB::fragment(lb, wn + 32 * j, s * KSTEP);
#pragma unroll
        for (int i = 0; i < S::MB; ++i) a[s & 1][i] = SA::fragment(la, wm + 32 * i, s * KSTEP);
    };
    auto multiply = [&](int s) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (sizeof(T) == 4) {
            // the four products of a fragment pair add to one accumulator: those of the other pairs stand between them
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < S::MB; ++i)
#pragma unroll
                    for (int j = 0; j < S::NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s & 1][i][u], b[s & 1][j][u], acc[i][j], 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < S::MB; ++i)
#pragma unroll
                for (int j = 0; j < S::NB; ++j) mma(acc[i][j], a[s & 1][i], b[s & 1][j]);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // Without a branch, which would part the accumulators' registers: behind the end of k the loads are told to fetch nothing (zeros), an
    // odd number of steps is rounded up by one of zeros.  left: k from the present step's beginning to the end.
    int64_t left = k_end - k0;
    auto step = [&](T* la, T* lb, T* next_a, T* next_b) {
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            read(la, lb, s + 1);
            multiply(s);
        }
        drain_and_meet();
        sa.load(la, left - 2 * BK);
        sb.load(lb, left - 2 * BK);
        read(next_a, next_b, 0);
        multiply(3);
        left -= BK;
    };
    sa.init(A, m0, k0);
    sb.init(Bm, n0, k0);
    drain_and_meet();                                    // the last product's LDS is free
    sa.load(a0, left);
    sb.load(b0, left);
    drain_and_meet();
    sa.load(a1, left - BK);
    sb.load(b1, left - BK);
    read(a0, b0, 0);
#pragma unroll 1
    do {
        step(a0, b0, a1, b1);
        step(a1, b1, a0, b0);
    } while (left > 0);
}

// The rows of a block's registers: row_of(i, r) behind this half's first, so that one number is compared with constants
__device__ __forceinline__ constexpr int row_of(int i, int r) { return 32 * i + acc_row(r, 0); }
__device__ __forceinline__ int rows_behind(int64_t v, int64_t V, int most) { return V - v < most ? (int)(V - v) : most; }

// acc: logits of vocabulary rows v0 .. (32 per i) and 32 tokens per j, plus the rows' bias
template <typename T, int MB, int NB> __device__ __forceinline__ void add_bias(const Problem& p, f32x16 (&acc)[MB][NB], int64_t v0)
{
    if (!p.bias) return;
    const int64_t first = v0 + 4 * (threadIdx.x >> 5 & 1);
    const int left = rows_behind(first, p.V, 32 * MB), last = left > 0 ? left - 1 : 0;
    const T* bias = (const T*)p.bias + (left > 0 ? first : 0);
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float z = (float)bias[row_of(i, r) < last ? row_of(i, r) : last];           // behind the vocabulary: any, it is cleared later
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j][r] += z;
        }
}

// The block's logits go into this lane's running maxima and sums (over: as in Sum), the targets' into z_target.  t0: this lane's first token
template <int MB, int NB>
__device__ __forceinline__ void fold(const Problem& p, f32x16 (&acc)[MB][NB], int64_t v0, int64_t t0, const int64_t (&y)[NB], Running (&run)[NB],
                                     float (&over)[NB], float* __restrict__ z_target)
{
    const int64_t first = v0 + 4 * (threadIdx.x >> 5 & 1);
    const int left = rows_behind(first, p.V, 32 * MB);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int64_t off = y[j] - first;
        const int here = off >= 0 && off < 32 * MB ? (int)off : -1;
        if (__any(here >= 0 || left < 32 * MB)) {
            float mine = 0.f;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    mine = row_of(i, r) == here ? acc[i][j][r] : mine;
                    acc[i][j][r] = row_of(i, r) == here || row_of(i, r) >= left ? -INFINITY : acc[i][j][r];
                }
            if (here >= 0 && !(here & 4) && here < left) z_target[t0 + 32 * j] = mine;         // & 4: the other half's row
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
        const float m = fmaxf(run[j].m, top), base = m == -INFINITY ? 0.f : m;
        float block = 0.f;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) block += __builtin_amdgcn_exp2f((acc[i][j][r] - base) * LOG2E);
        Sum sum{run[j].s, over[j]};
        sum.scale(exp2f((run[j].m - base) * LOG2E));
        sum.add<false>(block);
        run[j] = Running{m, sum.s};
        over[j] = sum.over;
    }
}

// Both halves of a wave hold sums of the same 32 columns
__device__ __forceinline__ Running halves_joined(const Running& mine)
{
    const Running o{__shfl_xor(mine.m, 32, 64), __shfl_xor(mine.s, 32, 64)};
    return threadIdx.x & 32 ? joined(o, mine) : joined(mine, o);
}

template <typename T, int B>
__global__ __launch_bounds__(Shape<B>::THREADS, 2) void stats_kernel(Problem p, int64_t splits, int64_t tiles_per_split, Running* __restrict__ part,
                                                                     float* __restrict__ z_target, float* __restrict__ kept)
{
    typedef Shape<B> S;
    int64_t token_tile, split;
    pair_of(place_of(blockIdx.x, gridDim.x), (p.T + B - 1) / B, splits, token_tile, split);
    TILE_LDS(T, true, true, B);
    const Operand<T> W{(const T*)p.w, p.ldw, p.V}, X{(const T*)p.x, p.ldx, p.T};
    const int64_t n0 = token_tile * B;
    const int lane = threadIdx.x & 63, half = lane >> 5, wm = S::wm(), wn = S::wn();
    int64_t y[S::NB];
    Running run[S::NB];
    float over[S::NB] = {};
#pragma unroll
    for (int j = 0; j < S::NB; ++j) {
        const int64_t t = n0 + wn + 32 * j + (lane & 31);
        y[j] = -1;
        if (t < p.T && p.target[t] != p.ignore) y[j] = clamp_target(p.target[t], p.V);
        run[j] = Running{-INFINITY, 0.f};
    }
    const int64_t first = split * tiles_per_split * B;
    const int64_t end = first + tiles_per_split * B < p.V ? first + tiles_per_split * B : p.V;
#pragma unroll 1
    for (int64_t m0 = first; m0 < end; m0 += B) {
        Acc<B> acc = {};
        tile_product<T, true, true, B>(acc, W, X, m0, n0, 0, p.D, TILE_LDS_ARGS);
        add_bias<T>(p, acc, m0 + wm);
        if (KEEPS<T> && kept) {
            float* to = kept + kept_at<B>(token_tile, (p.V + B - 1) / B, m0 / B);
            each_kept<B>([&](int i, int j, int r, int at) {
                *reinterpret_cast<f32x4*>(to + at) = f32x4{acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
            });
        }
        fold(p, acc, m0 + wm, n0 + wn + (lane & 31), y, run, over, z_target);
    }
    __syncthreads();
    Running* sh = reinterpret_cast<Running*>(lds_a0);              // [2 waves along the vocabulary][B tokens]
#pragma unroll
    for (int j = 0; j < S::NB; ++j) {
        const Running both = halves_joined(run[j]);
        if (half == 0) sh[(wm ? B : 0) + wn + 32 * j + lane] = both;
    }
    __syncthreads();
    const int64_t t = n0 + threadIdx.x;
    if (threadIdx.x < B && t < p.T) part[split * p.T + t] = joined(sh[threadIdx.x], sh[B + threadIdx.x]);
}

// The statistics of up to 64 rows (tokens): a tile of 128 would multiply mostly padding, and the one large operand is read once whatever is
// done.  A wave takes 64 vocabulary rows at a time, its operands straight from memory, two chunks of 128 bytes a row under way: lane l
// reads 64 consecutive bytes of row l % 32, the first or the second half of the chunk, for either operand -- the order of k is free --
// so every line is read whole.  No alignment is asked for and nothing is copied: the last pieces of a row are read from where the row
// ends, and what the piece before has had of them is cleared, in both operands.
template <typename T, int NB, int MB, int BYTES, int WAVES>
__global__ __launch_bounds__(64, WAVES) void few_kernel(Problem p, int64_t per, Running* __restrict__ part, float* __restrict__ z_target, float* __restrict__ kept)
{
    constexpr int ROWS = 32 * MB, VEC = Traits<T>::VEC, KC = BYTES / (int)sizeof(T), PIECES = KC / 2 / VEC;
    typedef typename Traits<T>::frag frag;
    typedef frag loose __attribute__((aligned(sizeof(T))));
    const int lane = threadIdx.x, l31 = lane & 31, half = lane >> 5, D = (int)p.D;
    const int64_t blocks = (p.V + ROWS - 1) / ROWS, b0 = blockIdx.x * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    const int last = D - VEC, chunks = (D + 2 * KC - 1) / (2 * KC) * 2;
    const T *wp[MB], *xp[NB];
    int64_t y[NB];
    Running run[NB];
    float over[NB] = {};
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int64_t t = 32 * j + l31;
        xp[j] = (const T*)p.x + (t < p.T ? t : p.T - 1) * p.ldx;
        y[j] = t < p.T && p.target[t] != p.ignore ? clamp_target(p.target[t], p.V) : -1;
        run[j] = Running{-INFINITY, 0.f};
    }
    struct Chunk { frag w[MB][PIECES], x[NB][PIECES]; } a, b;
    auto rows = [&](int64_t block) {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int64_t v = block * ROWS + 32 * i + l31;
            wp[i] = (const T*)p.w + (v < p.V ? v : p.V - 1) * p.ldw;
        }
    };
    auto load = [&](Chunk& c, int chunk) {
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            const int k = chunk * KC + half * (KC / 2) + n * VEC, at = k < last ? k : last;
#pragma unroll
            for (int i = 0; i < MB; ++i) c.w[i][n] = *reinterpret_cast<const loose*>(wp[i] + at);
#pragma unroll
            for (int j = 0; j < NB; ++j) c.x[j][n] = *reinterpret_cast<const loose*>(xp[j] + at);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x16 acc[MB][NB];
    auto multiply = [&](Chunk& c, int chunk) {
        if ((chunk + 1) * KC > D)
#pragma unroll
            for (int n = 0; n < PIECES; ++n) {
                const int k = chunk * KC + half * (KC / 2) + n * VEC, had = k - (k < last ? k : last);
#pragma unroll
                for (int u = 0; u < VEC; ++u) {
#pragma unroll
                    for (int i = 0; i < MB; ++i) c.w[i][n][u] = u < had ? (T)0.f : c.w[i][n][u];
#pragma unroll
                    for (int j = 0; j < NB; ++j) c.x[j][n][u] = u < had ? (T)0.f : c.x[j][n][u];
                }
            }
#pragma unroll
        for (int n = 0; n < PIECES; ++n)
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(c.w[i][n][u], c.x[j][n][u], acc[i][j], 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) mma(acc[i][j], c.w[i][n], c.x[j][n]);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    rows(b0);
    load(a, 0);
#pragma unroll 1
    for (int64_t block = b0; block < b1; ++block) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = f32x16{};
#pragma unroll 1
        for (int c = 0; c < chunks; c += 2) {
            load(b, c + 1);
            multiply(a, c);
            if (c + 2 == chunks) rows(block + 1);              // behind the last block: the last row, read for nothing
            load(a, c + 2 == chunks ? 0 : c + 2);
            multiply(b, c + 1);
        }
        add_bias<T>(p, acc, block * ROWS);
        if (KEEPS<T> && kept) {                                // as kept_at lays out tiles of 128
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int64_t v = block * ROWS + 32 * i;
                float* to = kept + v / 64 * (2 * 64 * 64) + (v & 32) / 32 * (2 * 4 * 256) + lane * 4;
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        *reinterpret_cast<f32x4*>(to + (j * 4 + r / 4) * 256) = f32x4{acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
            }
        }
        fold(p, acc, block * ROWS, l31, y, run, over, z_target);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const Running both = halves_joined(run[j]);
        if (half == 0 && 32 * j + l31 < p.T) part[blockIdx.x * p.T + 32 * j + l31] = both;
    }
}

// The statistics of up to four rows (tokens): nothing to multiply but the memory's stream.  A wave takes eight vocabulary rows at a time, 64
// lanes beside each other in a row, so that whole lines are read whatever the alignment is (32 rows at 128 bytes, as above, reach 2.6
// TB/s with rows off the lines); each lane adds its products of the rows, and the lanes' sums are added so that the number of values halves
// with each of the first three exchanges: lane l ends with row l % 8.
template <typename T, int NT>
__global__ __launch_bounds__(64, (NT == 1 && sizeof(T) == 4 ? 4 : NT <= 2 ? 3 : 2)) void dot_kernel(Problem p, int64_t per, Running* __restrict__ part, float* __restrict__ z_target,
                                                                 float* __restrict__ kept)
{
    constexpr int ROWS = 8, VEC = Traits<T>::VEC, STEP = 64 * VEC;
    typedef typename Traits<T>::frag frag;
    typedef frag loose __attribute__((aligned(sizeof(T))));
    const int lane = threadIdx.x, D = (int)p.D, last = D - VEC, steps = (D + STEP - 1) / STEP;
    const int64_t blocks = (p.V + ROWS - 1) / ROWS, b0 = blockIdx.x * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    const T* bias = (const T*)p.bias;
    const T *wp[ROWS], *xp[NT];
    int64_t y[NT];
    Running run[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t t = j < p.T ? j : p.T - 1;
        xp[j] = (const T*)p.x + t * p.ldx;
        y[j] = p.target[t] != p.ignore ? clamp_target(p.target[t], p.V) : -1;
        run[j] = Running{-INFINITY, 0.f};
    }
    frag a[ROWS], b[ROWS];
    auto rows = [&](int64_t block) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t v = block * ROWS + i;
            wp[i] = (const T*)p.w + (v < p.V ? v : p.V - 1) * p.ldw;
        }
    };
    auto load = [&](frag (&c)[ROWS], int step) {
        const int k = step * STEP + lane * VEC, at = k < last ? k : last;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) c[i] = *reinterpret_cast<const loose*>(wp[i] + at);
        __builtin_amdgcn_sched_barrier(0);
    };
    float acc[NT][ROWS];
    auto multiply = [&](frag (&c)[ROWS], int step) {
        // the last pieces of a row are read from where it ends: what the piece before has had of them is cleared, in both operands
        const int k = step * STEP + lane * VEC, at = k < last ? k : last, had = k - at;
        frag x[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j] = *reinterpret_cast<const loose*>(xp[j] + at);
        if ((step + 1) * STEP > D)
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i) c[i][u] = u < had ? (T)0.f : c[i][u];
#pragma unroll
                for (int j = 0; j < NT; ++j) x[j][u] = u < had ? (T)0.f : x[j][u];
            }
#pragma unroll
        for (int u = 0; u < VEC; ++u)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < ROWS; ++i) acc[j][i] = fmaf((float)c[i][u], (float)x[j][u], acc[j][i]);
        __builtin_amdgcn_sched_barrier(0);
    };
    rows(b0);
    load(a, 0);
#pragma unroll 1
    for (int64_t block = b0; block < b1; ++block) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) acc[j][i] = 0.f;
        auto step = [&](frag (&now)[ROWS], frag (&next)[ROWS], int s) {
            if (s + 1 == steps) rows(block + 1);               // behind the last block: the last row, read for nothing
            load(next, s + 1 == steps ? 0 : s + 1);
            multiply(now, s);
        };
        int s = 0;
#pragma unroll 1
        for (; s + 2 <= steps; s += 2) {
            step(a, b, s);
            step(b, a, s + 1);
        }
        if (s < steps) {
            step(a, b, s);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) a[i] = b[i];
        }
        const int64_t v = block * ROWS + (lane & 7);
        const float more = bias && v < p.V ? (float)bias[v] : 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float mine = lane & 4 ? acc[j][i + 4] : acc[j][i], other = lane & 4 ? acc[j][i] : acc[j][i + 4];
                f[i] = mine + __shfl_xor(other, 4, 64);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float mine = lane & 2 ? f[i + 2] : f[i], other = lane & 2 ? f[i] : f[i + 2];
                f[i] = mine + __shfl_xor(other, 2, 64);
            }
            const float mine = lane & 1 ? f[1] : f[0], other = lane & 1 ? f[0] : f[1];
            float z = mine + __shfl_xor(other, 1, 64);
#pragma unroll
            for (int d = 8; d < 64; d <<= 1) z += __shfl_xor(z, d, 64);
            z += more;
            if (lane < ROWS && j < p.T && v < p.V) {
                if (KEEPS<T> && kept) {                        // as kept_at lays out tiles of 128
                    const int in = (int)(v & 31);
                    kept[v / 64 * (2 * 64 * 64) + (v & 32) / 32 * (2 * 4 * 256) + in / 8 * 256 + ((in & 4) * 8 + j) * 4 + (in & 3)] = z;
                }
                if (v == y[j]) z_target[j] = z;
                else run[j] = joined(run[j], Running{z, 1.f});
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int d = 1; d < ROWS; d <<= 1) {
            const Running o{__shfl_xor(run[j].m, d, 64), __shfl_xor(run[j].s, d, 64)};
            run[j] = lane & d ? joined(o, run[j]) : joined(run[j], o);
        }
        if (lane == 0 && j < p.T) part[blockIdx.x * p.T + j] = run[j];
    }
}

// a + b as 32 bits round it, and exactly what that leaves (finite values)
struct Parts {
    float sum, rest;
};
__device__ __forceinline__ Parts exact_sum(float a, float b)
{
    const float sum = a + b, of_b = sum - a;
    return Parts{sum, (a - (sum - of_b)) + (b - of_b)};
}

// WAVES waves per row: the splits' sums joined, the row's loss, lse and q.  T, dx_part: with the parts of the narrow form's weighted
// sums of W [splits][T][D_out], D_out <= 256, also dx for an incoming gradient of one, in 32 bits.  A wave takes 64 splits at a time, and
// what it waits for is memory: with one wave to a row, 505 splits of 16 rows x 128 took 40 to 72 us, with eight 15; up to 64 splits the
// further waves only cost (6038 rows x 32: 11 us with one, 25 with four; 8192 x 128: 15, 34).
template <typename T, int WAVES>
__device__ __forceinline__ void one_row(const Problem& p, int64_t t, const Running* __restrict__ part, int64_t splits, const float* __restrict__ z_target,
                                        float* __restrict__ loss, float* __restrict__ lse, float* __restrict__ rest, int32_t* oob,
                                        const float* __restrict__ dx_part, int64_t D_out, float* __restrict__ dx_unit)
{
    __shared__ Running runs[WAVES];
    __shared__ float sums[WAVES > 1 ? WAVES : 1][WAVES > 1 ? 256 : 1];
    const int lane = threadIdx.x & 63, wave = WAVES > 1 ? threadIdx.x >> 6 : 0;
    const int64_t y = p.target[t];
    if (y == p.ignore) {
        if (wave) return;
        if (lane == 0) loss[t] = lse[t] = lse[p.T + t] = rest[t] = 0.f;
        if (dx_unit)
            for (int64_t d = lane; d < D_out; d += 64) dx_unit[t * D_out + d] = 0.f;
        return;
    }
    Running r{-INFINITY, 0.f};
    for (int64_t s = wave * 64 + lane; s < splits; s += 64 * WAVES) r = joined(r, part[s * p.T + t]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const Running o{__shfl_xor(r.m, d, 64), __shfl_xor(r.s, d, 64)};
        r = (lane & d) ? joined(o, r) : joined(r, o);
    }
    if constexpr (WAVES > 1) {
        if (lane == 0) runs[wave] = r;
        __syncthreads();
        r = runs[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) r = joined(r, runs[i]);
    }
    const float zt = z_target[t], ls = logf(r.s), d = (r.m - zt) + ls;
    // log(1 + e^d) from the smaller of e^d and e^-d; a target at -inf leaves the others' sum, a row of -inf alone is NaN
    const float e = expf(-fabsf(d)), l = log1pf(e);
    const bool none = d != d || zt == INFINITY, target_less = d > 0.f;
    const float q = none ? NAN : target_less ? 1.f / (1.f + e) : e / (1.f + e);
    if (wave == 0 && lane == 0) {
        if (oob && (y < 0 || y >= p.V)) atomicAdd(oob, 1);
        loss[t] = none ? NAN : target_less ? d + l : l;
        // lse in two parts: as 32 bits round it, and what that leaves.  Its summands are exact (the maximum or the target's logit, and k log 2
        // to 12 bits of it) or below 1.1, so that lse is within 2^-23 whatever its size is.
        int k;
        float f = frexpf(r.s, &k);
        if (f < 0.70710678f) {
            f *= 2.f;
            --k;
        }
        constexpr float LN2_HIGH = 0x1.62ep-1f, LN2_LOW = 3.19461832987e-05f;
        const Parts a = exact_sum(target_less ? r.m : zt, target_less ? k * LN2_HIGH : 0.f);
        const Parts b = exact_sum(a.sum, target_less ? fmaf(k, LN2_LOW, logf(f)) + l : l);
        lse[t] = none ? NAN : b.sum;
        lse[p.T + t] = none ? NAN : a.rest + b.rest;
        rest[t] = q;
    }
    if (!dx_unit) return;
    // p of a part's term = exp(m - M) / sum, all of them and the target's against one M
    const float M = fmaxf(r.m, zt), sum = r.s * exp2f((r.m - M) * LOG2E) + exp2f((zt - M) * LOG2E);
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t s0 = wave * 64; s0 < splits; s0 += 64 * WAVES) {
        // each lane has one split's factor: 0 for a split of nothing but -inf, whose sums are not looked at
        const float mine = s0 + lane < splits ? part[(s0 + lane) * p.T + t].m : -INFINITY, f = mine != -INFINITY ? exp2f((mine - M) * LOG2E) : 0.f;
        const int n = splits - s0 < 64 ? (int)(splits - s0) : 64;
        const float* src = dx_part + (s0 * p.T + t) * D_out;
        for (int i = 0; i < n; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (64 * k >= D_out) break;
                const int c = 64 * k + lane < D_out ? 64 * k + lane : (int)D_out - 1;        // eight loads on their way, none of them behind a branch
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = src[(int64_t)(i + j < n ? i + j : n - 1) * p.T * D_out + c];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float fj = __shfl(f, i + j, 64);
                    total[k] += fj != 0.f ? fj * v[j] : 0.f;
                }
            }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[wave][64 * k + lane] = total[k];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 1; i < WAVES; ++i) total[k] += sums[i][64 * k + lane];
    }
    const T* w = (const T*)p.w + clamp_target(y, p.V) * p.ldw;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int c = 64 * k + lane;
        if (c < D_out) dx_unit[t * D_out + c] = none ? NAN : fmaf(-q, (float)w[c], total[k] / sum);
    }
}

template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * 64 : 256) void rows_kernel(Problem p, const Running* __restrict__ part, int64_t splits,
                                                                            const float* __restrict__ z_target, float* __restrict__ loss,
                                                                            float* __restrict__ lse, float* __restrict__ rest, int32_t* oob,
                                                                            const float* __restrict__ dx_part, int64_t D_out, float* __restrict__ dx_unit)
{
    if constexpr (WAVES > 1) {
        one_row<T, WAVES>(p, blockIdx.x, part, splits, z_target, loss, lse, rest, oob, dx_part, D_out, dx_unit);
    } else {
#pragma unroll 1
        for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < p.T; t += (int64_t)gridDim.x * 4)
            one_row<T, 1>(p, t, part, splits, z_target, loss, lse, rest, oob, dx_part, D_out, dx_unit);
    }
}

// Number of rows that count, and the reduced loss (mean: NaN when none counts, as 0 / 0 is): partial sums per workgroup, joined in
// their order; one workgroup alone finishes by itself.
constexpr int REDUCE_NONE = RECO_XENT_NONE, REDUCE_MEAN = RECO_XENT_MEAN, REDUCE_SUM = RECO_XENT_SUM;

__device__ __forceinline__ float block_sum(float v, float* sh)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = 0.f;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) r += sh[w];
    __syncthreads();
    return r;
}

// rows: the rows' losses (of Problem p); or, where `parts` is given, those (sum, count) that an earlier launch left are joined
__global__ __launch_bounds__(1024) void reduce_kernel(Problem p, const float* __restrict__ rows, const float2* __restrict__ parts, int n_parts, int reduction,
                                                      float* __restrict__ loss, float* __restrict__ count_out, float2* __restrict__ part_out)
{
    __shared__ float sh[16];
    float sum = 0.f, count = 0.f;
    if (parts) {
        for (int i = threadIdx.x; i < n_parts; i += 1024) {
            sum += parts[i].x;
            count += parts[i].y;
        }
    } else {
        for (int64_t t = (int64_t)blockIdx.x * 1024 + threadIdx.x; t < p.T; t += (int64_t)gridDim.x * 1024) {
            sum += rows[t];
            count += p.target[t] != p.ignore ? 1.f : 0.f;
        }
    }
    sum = block_sum(sum, sh);
    count = block_sum(count, sh);
    if (threadIdx.x) return;
    if (gridDim.x > 1) {
        part_out[blockIdx.x] = float2{sum, count};
    } else {
        *loss = reduction == REDUCE_MEAN ? sum / count : sum;
        *count_out = count;
    }
}

// Rows' weights in two factors, gn[t] * scale[0]: |gn| < 2 and scale a power of two where every row has a weight of its own, so that G
// keeps its digits in 16 bits whatever the size of those weights is that are numbers; gn = 1 (NULL) and scale the incoming gradient, over
// the count for the mean, where it is the same for all.  scale[0] = scale[1] * scale[2]: a finite factor of the finished sums, and one of
// G's terms, 1 or what is no number: a row that does not count keeps its zeros.
__global__ __launch_bounds__(256) void top_kernel(Problem p, const float* __restrict__ dloss, float* __restrict__ tops)
{
    __shared__ float sh[4];
    float top = 0.f;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < p.T; t += (int64_t)gridDim.x * 256)
        if (p.target[t] != p.ignore && fabsf(dloss[t]) < INFINITY) top = fmaxf(top, fabsf(dloss[t]));
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) tops[blockIdx.x] = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}

// Also what the gradient kernels read per row: the target as 32 bits (-1: the row does not count), and for the narrow form the constant
// of its exponentials (see narrow_cols_kernel).
__global__ __launch_bounds__(256) void weights_kernel(Problem p, int reduction, const float* __restrict__ dloss, const float* __restrict__ count,
                                                      const float* __restrict__ tops, int n_tops, const float* __restrict__ lse, int whole_lse, float g_log2,
                                                      float* __restrict__ gn, float* __restrict__ scale, int* __restrict__ y, float* __restrict__ expo)
{
    float unit = 1.f;
    if (reduction == REDUCE_NONE) {
        float top = 0.f;
        for (int i = threadIdx.x & 63; i < n_tops; i += 64) top = fmaxf(top, tops[i]);
#pragma unroll
        for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        if (top > 0.f) {
            int e;
            (void)frexpf(top, &e);                       // top = f 2^e with f in [0.5, 1)
            unit = ldexpf(1.f, e < -120 ? -120 : e > 127 ? 127 : e);
        }
    } else if (reduction == REDUCE_MEAN) {
        unit = *count > 0.f ? *dloss / *count : 0.f;
    } else {
        unit = *count > 0.f ? *dloss : 0.f;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const bool number = fabsf(unit) < INFINITY;
        scale[0] = unit;
        scale[1] = number ? unit : 1.f;
        scale[2] = number ? 1.f : unit;
    }
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < p.T; t += (int64_t)gridDim.x * 256) {
        const int64_t target = p.target[t];
        const bool in = target != p.ignore;
        y[t] = in ? (int)clamp_target(target, p.V) : -1;
        if (reduction == REDUCE_NONE) gn[t] = in ? dloss[t] / unit : 0.f;
        if (p.bias || whole_lse) {
            expo[t] = in ? lse[t] : INFINITY;
            expo[p.T + t] = in ? -LOG2E * lse[p.T + t] : 0.f;
        } else expo[t] = in ? fmaf(-LOG2E, lse[t], g_log2) : -INFINITY;
    }
}

// dx = gn * scale * dx_unit, and 0 for rows that do not count (y < 0) whatever the scale is
template <typename T>
__global__ __launch_bounds__(256) void dx_kernel(const float* __restrict__ unit, int64_t rows, int64_t D, const float* __restrict__ gn,
                                                 const int* __restrict__ y, const float* __restrict__ scale, T* __restrict__ dx)
{
    const float f = *scale;
    const bool number = fabsf(f) < INFINITY;
    const int64_t n = rows * D;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        dx[i] = !number && y[i / D] < 0 ? (T)0.f : (T)(unit[i] * (gn ? gn[i / D] * f : f));
}

// N values of each lane (a multiple of 32), added over the 32 lanes of its half: the number of values halves with each exchange, and lane l
// ends with the sums of values PER l .. PER l + PER - 1, PER = N / 32, in v[0 .. PER)
template <int N, int FAR = 16> __device__ __forceinline__ void lanes_added(float* v)
{
    const bool up = threadIdx.x & FAR;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        const float mine = up ? v[k + N / 2] : v[k], other = up ? v[k] : v[k + N / 2];
        v[k] = mine + __shfl_xor(other, FAR, 64);
    }
    if constexpr (FAR > 1) lanes_added<N / 2, FAR / 2>(v);
}

// G of the vocabulary rows [v0, v0 + width): [T, ldg], columns behind the vocabulary zero.  KEPT: from the logits of the statistics.  gn: the
// rows' weights, or *unit where it is the same for all.  sums (nullable): dbias takes the terms before they are rounded -- they cancel
// where an item is the target as often as the model expects -- column sums of 64 tokens each, [tokens / 64, whole tiles][ldg] in 32 bits.
template <typename T, int B, bool KEPT>
__global__ __launch_bounds__(Shape<B>::THREADS, 2) void g_kernel(Problem p, int64_t v0, const float* __restrict__ kept, const float* __restrict__ lse,
                                                                 const float* __restrict__ rest, const float* __restrict__ gn, const float* __restrict__ unit,
                                                                 T* __restrict__ G, int64_t ldg, float* __restrict__ sums)
{
    typedef Shape<B> S;
    int64_t token_tile, panel;
    pair_of(place_of(blockIdx.x, gridDim.x), (p.T + B - 1) / B, ldg / B, token_tile, panel);
    TILE_LDS(T, true, true, B);
    const Operand<T> W{(const T*)p.w, p.ldw, p.V}, X{(const T*)p.x, p.ldx, p.T};
    const int64_t n0 = token_tile * B, m0 = v0 + panel * B;
    const int lane = threadIdx.x & 63, half = lane >> 5, wm = S::wm(), wn = S::wn();
    Acc<B> acc = {};
    if constexpr (KEPT) {
        if (m0 < p.V) {
            const float* from = kept + kept_at<B>(token_tile, (p.V + B - 1) / B, m0 / B);
            each_kept<B>([&](int i, int j, int r, int at) {
                const f32x4 z = *reinterpret_cast<const f32x4*>(from + at);
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[i][j][r + u] = z[u];
            });
        }
    } else {
        tile_product<T, true, true, B>(acc, W, X, m0, n0, 0, p.D, TILE_LDS_ARGS);
        add_bias<T>(p, acc, m0 + wm);
    }
    // through LDS, so that a row's values leave 16 bytes a lane: a wave's 64 rows (tokens) of WM values, chunks changing places by the row
    drain_and_meet();
    constexpr int ROW = S::WM, CH = ROW * (int)sizeof(T) / 16, VEC = Traits<T>::VEC, PER_ARRAY = Stage<T, true, B>::SIZE / (S::WN * ROW);
    const int wave = threadIdx.x >> 6;
    const int array = wave / PER_ARRAY;
    T* const mine = (array == 0 ? lds_a0 : array == 1 ? lds_a1 : array == 2 ? lds_b0 : lds_b1) + wave % PER_ARRAY * (S::WN * ROW);
    const int64_t first = m0 + wm + 4 * half;
    const int left = rows_behind(first, p.V, S::WM);
#pragma unroll
    for (int j = 0; j < S::NB; ++j) {
        const int row = 32 * j + (lane & 31);
        const int64_t t = n0 + wn + row;
        const int64_t y0 = t < p.T ? p.target[t] : p.ignore;
        const bool in = y0 != p.ignore;
        const int64_t off = in ? clamp_target(y0, p.V) - first : -1;
        const int here = off >= 0 && off < S::WM ? (int)off : -1;
        const float l = in ? lse[t] : 0.f, low = in ? -LOG2E * lse[p.T + t] : 0.f, q = in ? rest[t] : 0.f, g = in ? (gn ? gn[t] : *unit) * Traits<T>::G_SCALE : 0.f;
#pragma unroll
        for (int i = 0; i < S::MB; ++i)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int c = 32 * i + 8 * r4 + 4 * half;
                Pack<T, 4> o;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int v = row_of(i, 4 * r4 + u);
                    const float e = v == here ? -q : __builtin_amdgcn_exp2f(fmaf(acc[i][j][4 * r4 + u] - l, LOG2E, low));
                    const float term = in && v < left ? e * g : 0.f;
                    o.v[u] = (T)term;
                    acc[i][0][4 * r4 + u] = j ? acc[i][0][4 * r4 + u] + term : term;
                }
                *reinterpret_cast<Pack<T, 4>*>(mine + row * ROW + ((c / VEC) ^ (row & (CH - 1))) * VEC + c % VEC) = o;
            }
    }
    if (sums) {
        constexpr int PER = S::MB / 2;                              // of the 16 MB rows in a lane's registers
        float v[16 * S::MB];
#pragma unroll
        for (int i = 0; i < S::MB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) v[16 * i + r] = acc[i][0][r];
        lanes_added<16 * S::MB>(v);
        const int k = (lane & 31) * PER;
        float* const to = sums + (n0 + wn) / 64 * ldg + (m0 - v0 + wm) + 32 * (k / 16) + acc_row(k % 16, half);
        Pack<float, PER> own;
#pragma unroll
        for (int i = 0; i < PER; ++i) own.v[i] = v[i];
        *reinterpret_cast<Pack<float, PER>*>(to) = own;
    }
    drain_and_meet();
    for (int at = lane; at < S::WN * CH; at += 64) {
        const int row = at / CH, c = at % CH;
        const int64_t t = n0 + wn + row;
        if (t < p.T)
            *reinterpret_cast<Pack<T, VEC>*>(G + t * ldg + (m0 - v0 + wm) + c * VEC) =
                *reinterpret_cast<const Pack<T, VEC>*>(mine + row * ROW + (c ^ (row & (CH - 1))) * VEC);
    }
}

// A B in equal shares (xent_plan.h), tiles of one row of tiles beside each other.  A tile that lies in one share is finished here: `sum`
// [M, N], what earlier pieces left, is added to it (first: there is nothing yet), and it goes to `sum`, or with `out` [M, N], times
// scale / G_SCALE and rounded to T, there; in 16 bits through LDS, in whole lines (2 bytes a lane took 366 us for 131,072 x 1024 values
// of 8 tokens, and 174 instead of 130 per 16,384 x 1024 of 4096).  The 32-bit sums of a part of a tile go to one of the workgroup's two
// places, and join_kernel adds those in order.  DIRECT: no `sum`, all of it goes to `out`.
template <typename T, bool AKC, bool BKC, int B, bool DIRECT>
__global__ __launch_bounds__(Shape<B>::THREADS, 2) void product_kernel(Operand<T> A, Operand<T> Bm, int64_t tiles_n, int64_t M, int64_t N, int64_t K, int64_t steps,
                                                                       int64_t units, int64_t share, const float* __restrict__ scale, float* __restrict__ part,
                                                                       int first, float* __restrict__ sum, T* __restrict__ out)
{
    typedef Shape<B> S;
    TILE_LDS(T, AKC, BKC, B);
    const int64_t worker = place_of(blockIdx.x, gridDim.x);
    const int lane = threadIdx.x & 63, half = lane >> 5, wm = S::wm(), wn = S::wn();
    const int64_t end = (worker + 1) * share < units ? (worker + 1) * share : units;
    const bool whole16 = N * sizeof(T) % 16 == 0 && (uintptr_t)out % 16 == 0;
#pragma unroll 1
    for (int64_t u = worker * share; u < end;) {
        const TilePart q = tile_part(u, end, steps);
        const int64_t k0 = q.step * TB, k1 = (q.step + q.count) * TB < K ? (q.step + q.count) * TB : K;
        u += q.count;
        Acc<B> acc = {};
        const int64_t m0 = q.tile / tiles_n * B, n0 = q.tile % tiles_n * B;
        tile_product<T, AKC, BKC, B, DIRECT>(acc, A, Bm, m0, n0, k0, k1, TILE_LDS_ARGS);
        // fn(block i, j and register r of a value, its place in m): the values inside a matrix m [M, N], 32 of a row beside each other
        const auto each_value = [&](auto* m, auto&& fn) {
            const int left = rows_behind(m0 + wm + 4 * half, M, S::WM), at = (wm + 4 * half) * (int)N + wn + (lane & 31);
#pragma unroll
            for (int j = 0; j < S::NB; ++j) {
                const bool in = n0 + wn + 32 * j + (lane & 31) < N;
#pragma unroll
                for (int i = 0; i < S::MB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (in && row_of(i, r) < left) fn(i, j, r, (m + (m0 + row_of(i, r)) * N + n0 + 32 * j)[at]);
            }
        };
        if (q.count == steps) {
            if constexpr (!DIRECT) {
                if (!first) each_value(sum, [&](int i, int j, int r, const float& s) { acc[i][j][r] += s; });
                if (!out) {
                    each_value(sum, [&](int i, int j, int r, float& s) { s = acc[i][j][r]; });
                    continue;
                }
            }
            const float f = *scale / Traits<T>::G_SCALE;
            if constexpr (sizeof(T) == 2) {
                // a wave's WM rows of 64 values, chunks changing places by the row
                drain_and_meet();
                constexpr int VEC = Traits<T>::VEC, CH = S::WN / VEC, PER_ARRAY = Stage<T, AKC, B>::SIZE / (S::WM * S::WN);
                static_assert(PER_ARRAY * 4 >= S::THREADS / 64, "the waves' blocks fit the four arrays");
                const int wave = threadIdx.x >> 6, array = wave / PER_ARRAY;
                T* const mine = (array == 0 ? lds_a0 : array == 1 ? lds_a1 : array == 2 ? lds_b0 : lds_b1) + wave % PER_ARRAY * (S::WM * S::WN);
                static_assert(CH == 8, "a row's place among the chunks goes by its number modulo 8");
                int spot[4][S::NB];                        // of rows 4 half + u, columns 32 j + lane % 32
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int j = 0; j < S::NB; ++j) {
                        const int row = 4 * half + u, c = 32 * j + (lane & 31);
                        spot[u][j] = row * S::WN + ((c / VEC) ^ row) * VEC + c % VEC;
                    }
#pragma unroll
                for (int i = 0; i < S::MB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
#pragma unroll
                        for (int j = 0; j < S::NB; ++j) mine[spot[r & 3][j] + (32 * i + 8 * (r >> 2)) * S::WN] = (T)(acc[i][j][r] * f);
                drain_and_meet();
                for (int at = lane; at < S::WM * CH; at += 64) {
                    const int row = at / CH, c = at % CH;
                    const int64_t m = m0 + wm + row, col = n0 + wn + c * VEC;
                    if (m >= M) break;
                    const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(mine + row * S::WN + (c ^ (row & (CH - 1))) * VEC);
                    if (whole16) {
                        if (col < N) *reinterpret_cast<Pack<T, VEC>*>(out + m * N + col) = v;
                    } else {
#pragma unroll
                        for (int k = 0; k < VEC; ++k)
                            if (col + k < N) out[m * N + col + k] = v.v[k];
                    }
                }
            } else {
                each_value(out, [&](int i, int j, int r, T& o) { o = acc[i][j][r] * f; });
            }
            continue;
        }
        float* to = part + place_of_part(worker, q.step == 0) * (B * B);
        const int mine = (wm + 4 * half) * B + wn + (lane & 31);
#pragma unroll
        for (int i = 0; i < S::MB; ++i)
#pragma unroll
            for (int j = 0; j < S::NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) (to + (row_of(i, r) * B + 32 * j))[mine] = acc[i][j][r];
    }
}

// The parts of every tile that several workgroups shared, added; to `sum` [M, N] and `out` as the whole tiles of product_kernel go
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int B, int64_t tiles_n, int64_t steps, int64_t share, int64_t M, int64_t N,
                                                   const float* __restrict__ scale, int first, float* __restrict__ sum, T* __restrict__ out)
{
    const int64_t tile = blockIdx.x;
    const Workers from = workers_of(tile, steps, share);
    if (from.first == from.last) return;
    const int64_t m0 = tile / tiles_n * B, n0 = tile % tiles_n * B;
    const float f = out ? *scale / Traits<T>::G_SCALE : 1.f;
    const bool fours = N % 4 == 0 && (uintptr_t)out % sizeof(Pack<T, 4>) == 0;
    for (int i = (blockIdx.y * 256 + threadIdx.x) * 4; i < B * B; i += gridDim.y * 1024) {
        const int64_t m = m0 + i / B, n = n0 + i % B;
        if (m >= M || n >= N) continue;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int64_t w = from.first; w <= from.last; ++w) s += *reinterpret_cast<const f32x4*>(part + place_of_part(w, w == from.first) * (B * B) + i);
        const int64_t at = m * N + n;
        const int left = N - n < 4 ? (int)(N - n) : 4;
        if (sum && !first)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < left) s[j] += sum[at + j];
        if (!out) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < left) sum[at + j] = s[j];
            continue;
        }
        Pack<T, 4> o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[j] = (T)(s[j] * f);
        if (fours) *reinterpret_cast<Pack<T, 4>*>(out + at) = o;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < left) out[at + j] = o.v[j];
    }
}

// out[i] = scale / G_SCALE * sum over slices, `ld` values apart, rounded to T
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ part, int slices, int64_t ld, int64_t n, const float* __restrict__ scale, T* __restrict__ out)
{
    const float f = *scale / Traits<T>::G_SCALE;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < slices; ++k) s += part[k * ld + i];
        out[i] = (T)(s * f);
    }
}

// sums of `rows` rows of in [rows, ld], [slices][ld]: slice blockIdx.y takes rows [y * rows_per, ...); 16 bytes of a row per thread
__global__ __launch_bounds__(256) void column_sum_kernel(const float* __restrict__ in, int64_t ld, int64_t rows, int64_t rows_per, float* __restrict__ out)
{
    const int64_t v = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    const int64_t t0 = blockIdx.y * rows_per, t1 = t0 + rows_per < rows ? t0 + rows_per : rows;
    if (v >= ld) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int64_t t = t0; t < t1; ++t) s += *reinterpret_cast<const f32x4*>(in + t * ld + v);
    *reinterpret_cast<f32x4*>(out + blockIdx.y * ld + v) = s;
}

// rows with their width filled up to `ldo` with zeros; rows whose target (nullable) is `ignore` as zeros
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ in, int64_t rows, int64_t ld, int64_t D, T* __restrict__ out, int64_t ldo,
                                                   const int64_t* __restrict__ target, int64_t ignore)
{
    constexpr int VEC = Traits<T>::VEC;
    typedef typename Traits<T>::frag frag;
    typedef frag loose __attribute__((aligned(sizeof(T))));
    const int64_t per_row = ldo / VEC, n = rows * per_row;
#pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = n < (int64_t)1 << 32 ? (uint32_t)i / (uint32_t)per_row : i / per_row, c = (i - r * per_row) * VEC;
        const T* src = in + r * ld + c;
        const bool drop = target && target[r] == ignore;
        frag v;
        if (c + VEC <= D) {
            v = *reinterpret_cast<const loose*>(src);
            if (drop) v = frag{};
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = c + j < D && !drop ? src[j] : (T)0.f;
        }
        *reinterpret_cast<frag*>(out + r * ldo + c) = v;
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct Carve {
    char* base;
    size_t used = 0;
    void* take(size_t bytes)
    {
        void* p = base ? base + used : nullptr;
        used += align_up(bytes, 256);
        return p;
    }
};

unsigned stream_blocks(int64_t n)
{
    const int64_t b = ceil_div64(n, 256);
    return (unsigned)(b < 1 ? 1 : b > 4096 ? 4096 : b);
}

int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

struct Args {
    const void* x; int64_t ldx;
    const void* w; int64_t ldw;
    const void* bias;
    int dtype;
    int64_t T, V, D;
    const int64_t* target;
    int64_t ignore;
};

// Rows as the kernels read them: as they are, or copied with their width filled up, where a row does not start on 16 bytes or its
// width is no whole number of 16-byte groups (or a row lies 4 MB from the next: 256 rows are reached with 32-bit offsets).
bool must_pack(const void* p, int64_t ld, int64_t D, int size)
{
    return (uintptr_t)p % 16 || ld * size % 16 || D * size % 16 || ld * size >= (int64_t)1 << 22;
}

struct ForwardPlan {
    int64_t splits, tiles_per_split;
};

// The split of the vocabulary with the fewest rounds of tiles; the longest runs of tiles among equals
ForwardPlan forward_plan(int64_t T, int64_t V, int tile)
{
    const int64_t tiles = ceil_div64(V, tile), rows = ceil_div64(T, tile);
    int64_t best = 1, cost = INT64_MAX;
    for (int64_t per = 1; per <= tiles && per <= 256; ++per) {
        const int64_t c = ceil_div64(rows * ceil_div64(tiles, per), places_of(tile)) * per;
        if (c <= cost) {
            cost = c;
            best = per;
        }
    }
    // more splits than the sums of a row are worth: at most 2048
    if (ceil_div64(tiles, best) > 2048) best = ceil_div64(tiles, 2048);
    return ForwardPlan{ceil_div64(tiles, best), best};
}

struct BackwardPlan {
    int64_t width;                    // vocabulary rows per piece, a multiple of 256
    int64_t b_sums;                   // rows of 64 tokens' column sums of G
    int64_t b_slices, b_per;          // more than 64 of them are added in slices first (0: they are not)
};

constexpr size_t PIECE_BYTES = (size_t)128 << 20;

BackwardPlan backward_plan(int64_t T, int64_t V, int64_t D, int size)
{
    BackwardPlan b{};
    const int64_t tiles = ceil_div64(V, 256), by_g = (int64_t)(PIECE_BYTES / ((size_t)T * size)) / 256;
    b.width = clamp64(by_g, 1, tiles < 16384 ? tiles : 16384) * 256;
    const int tile = tile_of(size, T, V);
    b.b_sums = ceil_div64(T, tile) * (tile / 64);
    if (b.b_sums > 64) {
        b.b_per = ceil_div64(b.b_sums, 64);
        b.b_slices = ceil_div64(b.b_sums, b.b_per);
    }
    return b;
}

// `clean`: x copied in any case, rows that do not count as zeros (they are multiplied by zeros, and may hold anything)
template <typename T> int pack_rows(const Args& a, Problem& p, bool clean, Carve& c, bool launch, hipStream_t s)
{
    const int64_t padded = ceil_div64(a.D, Traits<T>::VEC) * Traits<T>::VEC;
    p = Problem{a.T, a.V, padded, a.ldx, a.ldw, a.x, a.w, a.bias, a.target, a.ignore};
    struct { const void** p; int64_t* ld; int64_t rows; } in[2] = {{&p.x, &p.ldx, a.T}, {&p.w, &p.ldw, a.V}};
    for (auto& m : in) {
        const bool is_x = m.p == &p.x;
        if (!(clean && is_x) && !must_pack(*m.p, *m.ld, a.D, sizeof(T))) continue;
        T* to = (T*)c.take((size_t)m.rows * padded * sizeof(T));
        if (launch) {
            hipLaunchKernelGGL(pack_kernel<T>, dim3(stream_blocks(m.rows * (padded / Traits<T>::VEC))), dim3(256), 0, s, (const T*)*m.p, m.rows, *m.ld, a.D, to, padded,
                               clean && is_x ? a.target : nullptr, a.ignore);
            RECO_CHECK_LAUNCH();
            *m.p = to;
            *m.ld = padded;
        }
    }
    return RECO_OK;
}

template <typename T, typename F> int with_tile(int tile, F&& fn)
{
    if constexpr (sizeof(T) == 2)
        if (tile == 256) return fn(std::integral_constant<int, 256>());
    return fn(std::integral_constant<int, 128>());
}

// sum (+)= A B, or with `out` its (and sum's) total times *scale, rounded to T
template <typename T, bool AKC, bool BKC>
int launch_product(const Operand<T>& A, const Operand<T>& B, int64_t M, int64_t N, int64_t K, const float* scale, bool first, float* part, float* sum, T* out,
                   hipStream_t s)
{
    const ProductPlan q = product_plan(sizeof(T), M, N, K);
    return with_tile<T>(q.tile, [&](auto t) -> int {
        constexpr int W = decltype(t)::value;
        const bool direct = out && !sum;
        const dim3 grid((unsigned)q.workers), block(Shape<W>::THREADS);
        if (direct)
            hipLaunchKernelGGL((product_kernel<T, AKC, BKC, W, true>), grid, block, 0, s, A, B, q.tiles_n, M, N, K, q.steps, q.units, q.share, scale, part, first, sum, out);
        else if constexpr (AKC)                      // dx; dw has no sum of earlier pieces
            hipLaunchKernelGGL((product_kernel<T, AKC, BKC, W, false>), grid, block, 0, s, A, B, q.tiles_n, M, N, K, q.steps, q.units, q.share, scale, part, first, sum, out);
        if (q.share % q.steps)
            hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)(q.tiles_m * q.tiles_n), (unsigned)(W * W / (q.tiles_m * q.tiles_n <= 64 ? 1024 : 4096))), dim3(256), 0, s, part, W, q.tiles_n, q.steps, q.share, M, N,
                           scale, first, sum, out);
        RECO_CHECK_LAUNCH();
        return RECO_OK;
    });
}

// The most logits that are kept for the gradient: 512 MB of them
constexpr int64_t KEPT_FLOATS = (int64_t)1 << 27;

// The forms for few rows (dot_kernel, few_kernel): vocabulary rows a wave takes at a time, how often, and the waves
struct FewPlan {
    int64_t rows, per, splits;
};

FewPlan few_plan(int64_t T, int64_t V, int64_t D, int size)
{
    // dot_kernel where a row keeps enough of the lanes beside each other at work.  With 33 tokens or more, 128 vocabulary rows read x half
    // as often as 64, once there are enough of them for the chip's 1024 places (64 x 131,071 x 1024 f32: 205 us, 256 with 64; at 65,536
    // 142, 97)
    const int64_t pieces = D * size / 16;
    const bool dot = T == 1 ? pieces >= 32 || size == 4 : T <= 4 && pieces >= (size == 4 ? 48 : 96);
    const int64_t rows = dot ? 8 : T <= 32 || V < 128 * 960 ? 64 : 128;
    const int64_t waves = 1024 * (rows == 128 ? 1 : rows == 64 ? 3 : T == 1 && size == 4 ? 4 : T <= 2 ? 3 : 2);
    const int64_t blocks = ceil_div64(V, rows), per = ceil_div64(blocks, waves);
    return FewPlan{rows, per, ceil_div64(blocks, per)};
}

// Where rows are wide.  Narrow ones that leave nothing for the gradient: where the narrow form would copy W first; in 32 bits a single
// token (1 x 1 M: x 64 84 us instead of 102, x 128 130 instead of 160) and 33 to 64, of which the narrow form keeps half its waves at
// work (64 x 1 M x 100: 255 us instead of 338; 64 x 50,000 x 128 35 both).
bool is_few(const Args& a, bool narrow, bool keep)
{
    const int size = a.dtype == RECO_DT_F32 ? 4 : 2;
    if (a.T > 64 || a.D * size < 16) return false;
    return !narrow || (!keep && (must_pack(a.w, a.ldw, a.D, size) || (size == 4 && a.D > 32 && (a.T == 1 || a.T > 32))));
}

constexpr int REDUCE_ROWS = 16384;            // rows that one workgroup reduces by itself

template <typename T>
int forward(const Args& a, int reduction, float* loss, float* state, float* kept, bool keep, int32_t* oob, char* ws, size_t* need, hipStream_t s)
{
    Carve c{ws};
    Problem p;
    const bool launch = ws != nullptr, narrow = narrow_fits(a.dtype, a.D);
    const int tile = tile_of(sizeof(T), a.T, a.V);
    const ForwardPlan f = forward_plan(a.T, a.V, tile);
    const NarrowPlan n = narrow ? narrow_plan_of<T>(a.T, a.V, a.D, keep) : NarrowPlan{};
    const bool few = is_few(a, narrow, keep);
    const FewPlan fp = few_plan(a.T, a.V, a.D, sizeof(T));
    const int64_t splits = few ? fp.splits : narrow ? n.x_splits : f.splits;
    Running* part = (Running*)c.take((size_t)splits * a.T * sizeof(Running));
    float* z_target = (float*)c.take((size_t)a.T * 4);
    float* rows = (float*)c.take((size_t)a.T * 4);
    float2* sums = (float2*)c.take(256 * sizeof(float2));
    float* dx_part = narrow && keep ? (float*)c.take((size_t)splits * a.T * a.D * 4) : nullptr;
    if (few) {
        p = Problem{a.T, a.V, a.D, a.ldx, a.ldw, a.x, a.w, a.bias, a.target, a.ignore};
    } else {
        const int rc = pack_rows<T>(a, p, false, c, launch, s);
        if (rc) return rc;
    }
    *need = c.used;
    if (!launch) return RECO_OK;
    if (reduction == REDUCE_NONE) rows = loss;
    if (few) {
        const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)splits), dim3(64), 0, s, p, fp.per, part, z_target, kept); };
        if (fp.rows == 8) {
            if (a.T == 1) launch(dot_kernel<T, 1>);
            else if (a.T == 2) launch(dot_kernel<T, 2>);
            else launch(dot_kernel<T, 4>);
        } else if (a.T <= 32) launch(few_kernel<T, 1, 2, 64, 3>);
        else if (fp.rows == 64) launch(few_kernel<T, 2, 2, 64, 3>);
        else launch(few_kernel<T, 2, 4, 128, 1>);
    } else if (narrow) {
        const int rn = narrow_rows_of<T>(p, n, a.D, part, z_target, dx_part, s);
        if (rn) return rn;
    } else {
        const int rs = with_tile<T>(tile, [&](auto t) -> int {
            constexpr int B = decltype(t)::value;
            hipLaunchKernelGGL((stats_kernel<T, B>), dim3((unsigned)(ceil_div64(a.T, B) * splits)), dim3(Shape<B>::THREADS), 0, s, p, splits, f.tiles_per_split,
                               part, z_target, kept);
            return RECO_OK;
        });
        if (rs) return rs;
    }
    const auto join = [&](auto waves) {
        constexpr int WAVES = decltype(waves)::value;
        hipLaunchKernelGGL((rows_kernel<T, WAVES>), dim3((unsigned)(WAVES > 1 ? a.T : clamp64(ceil_div64(a.T, 4), 1, 1 << 20))), dim3(WAVES > 4 ? WAVES * 64 : 256), 0, s, p, part,
                           splits, z_target, rows, state, state + 2 * a.T, oob, dx_part, a.D, dx_part ? kept : nullptr);
    };
    if (splits > 64) join(std::integral_constant<int, 8>());
    else join(std::integral_constant<int, 1>());
    if (reduction != REDUCE_NONE) {
        int blocks = (int)clamp64(ceil_div64(a.T, REDUCE_ROWS), 1, 256);
        hipLaunchKernelGGL(reduce_kernel, dim3(blocks), dim3(1024), 0, s, p, rows, nullptr, 0, reduction, loss, state + 3 * a.T, sums);
        if (blocks > 1)
            hipLaunchKernelGGL(reduce_kernel, dim3(1), dim3(1024), 0, s, p, rows, sums, blocks, reduction, loss, state + 3 * a.T, nullptr);
    }
    RECO_CHECK_LAUNCH();
    return RECO_OK;
}

template <typename T>
int backward(const Args& a, int reduction, const float* state, const float* kept, const float* dloss, void* dx, void* dw, void* db, char* ws, size_t* need,
             hipStream_t s)
{
    Carve c{ws};
    Problem p;
    const bool launch = ws != nullptr, narrow = narrow_fits(a.dtype, a.D);
    float* gn = (float*)c.take((size_t)a.T * 4);
    float* scale = (float*)c.take(3 * 4);
    float* tops = (float*)c.take(256 * 4);
    int* y = (int*)c.take((size_t)a.T * 4);
    float* expo = (float*)c.take((size_t)a.T * 8);
    const NarrowPlan n = narrow ? narrow_plan_of<T>(a.T, a.V, a.D, true) : NarrowPlan{};
    const BackwardPlan b = narrow ? BackwardPlan{} : backward_plan(a.T, a.V, a.D, sizeof(T));
    T* G = nullptr;
    float *x_part = nullptr, *w_part = nullptr, *b_part = nullptr;
    if (narrow) {
        if (n.w_shared) {
            w_part = (float*)c.take((size_t)n.w_shares * 2 * 128 * a.D * 4);
            b_part = (float*)c.take((size_t)n.w_shares * 2 * 128 * 4);
        }
    } else {
        G = (T*)c.take((size_t)a.T * b.width * sizeof(T));
        // the last piece may be narrower, and fewer units can mean shorter shares and more workgroups
        size_t places = 0;
        for (const int64_t width : {b.width < a.V ? b.width : a.V, (a.V - 1) % b.width + 1})
            for (const ProductPlan& q : {product_plan(sizeof(T), a.T, a.D, width), product_plan(sizeof(T), width, a.D, a.T)})
                if (q.floats > places) places = q.floats;
        w_part = (float*)c.take(places * 4);
        if (b.width < a.V) x_part = (float*)c.take((size_t)a.T * a.D * 4);
        b_part = (float*)c.take((size_t)(b.b_sums + b.b_slices) * b.width * 4);
    }
    const int rc = pack_rows<T>(a, p, !narrow, c, launch, s);
    if (rc) return rc;
    *need = c.used;
    if (!launch) return RECO_OK;
    const float *lse = state, *rest = state + 2 * a.T;
    const int row_blocks = (int)clamp64(ceil_div64(a.T, 256), 1, 256);
    if (reduction == REDUCE_NONE)
        hipLaunchKernelGGL(top_kernel, dim3(row_blocks), dim3(256), 0, s, p, dloss, tops);
    else
        gn = nullptr;
    hipLaunchKernelGGL(weights_kernel, dim3(row_blocks), dim3(256), 0, s, p, reduction, dloss, state + 3 * a.T, tops, row_blocks, lse, (int)(sizeof(T) == 4 || db),
                       log2f(Traits<T>::G_SCALE), gn, scale, y, expo);
    if (narrow) {
        if (dw || db) {
            const int rn = narrow_cols_of<T>(p, n, a.D, expo, y, rest, gn, scale, dw, db, w_part, b_part, s);
            if (rn) return rn;
        }
        if (dx) hipLaunchKernelGGL(dx_kernel<T>, dim3(stream_blocks(a.T * a.D)), dim3(256), 0, s, kept, a.T, a.D, gn, y, scale, (T*)dx);
        RECO_CHECK_LAUNCH();
        return RECO_OK;
    }
    for (int64_t v0 = 0; v0 < a.V; v0 += b.width) {
        const int64_t width = a.V - v0 < b.width ? a.V - v0 : b.width, ldg = ceil_div64(width, 256) * 256;
        int rl = with_tile<T>(tile_of(sizeof(T), a.T, a.V), [&](auto t) -> int {
            constexpr int B = decltype(t)::value;
            const dim3 grid((unsigned)(ceil_div64(a.T, B) * (ldg / B))), block(Shape<B>::THREADS);
            if constexpr (KEEPS<T>)
                if (kept) {
                    hipLaunchKernelGGL((g_kernel<T, B, true>), grid, block, 0, s, p, v0, kept, lse, rest, gn, scale + 2, G, ldg,
                                       db ? b_part : nullptr);
                    RECO_CHECK_LAUNCH();
                    return RECO_OK;
                }
            hipLaunchKernelGGL((g_kernel<T, B, false>), grid, block, 0, s, p, v0, nullptr, lse, rest, gn, scale + 2, G, ldg,
                               db ? b_part : nullptr);
            RECO_CHECK_LAUNCH();
            return RECO_OK;
        });
        if (!rl && dx)
            rl = launch_product<T, true, false>({G, ldg, a.T}, {(const T*)p.w + v0 * p.ldw, p.ldw, p.D}, a.T, a.D, width, scale + 1, v0 == 0, w_part, x_part,
                                                v0 + width == a.V ? (T*)dx : nullptr, s);
        if (!rl && dw) rl = launch_product<T, false, false>({G, ldg, ldg}, {(const T*)p.x, p.ldx, p.D}, width, a.D, a.T, scale + 1, true, w_part, nullptr, (T*)dw + v0 * a.D, s);
        if (rl) return rl;
        if (db) {
            const float* from = b_part;
            if (b.b_slices) {
                hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)ceil_div64(ldg, 1024), (unsigned)b.b_slices), dim3(256), 0, s, b_part, ldg, b.b_sums, b.b_per,
                                   b_part + b.b_sums * ldg);
                from += b.b_sums * ldg;
            }
            hipLaunchKernelGGL(finish_kernel<T>, dim3(stream_blocks(width)), dim3(256), 0, s, from, (int)(b.b_slices ? b.b_slices : b.b_sums), ldg, width, scale + 1,
                               (T*)db + v0);
        }
        RECO_CHECK_LAUNCH();
    }
    return RECO_OK;
}

int check_args(const char* what, const Args& a, int reduction)
{
    RECO_REQUIRE(a.dtype >= RECO_DT_F32 && a.dtype <= RECO_DT_F16, "%s: unknown element type %d", what, a.dtype);
    RECO_REQUIRE(a.T > 0 && a.T < (int64_t)1 << 31 && a.V > 0 && a.V < (int64_t)1 << 31 && a.D > 0 && a.D <= 1 << 20,
                 "%s: bad sizes: %lld rows, %lld columns, width %lld", what, (long long)a.T, (long long)a.V, (long long)a.D);
    RECO_REQUIRE(a.x && a.w && a.target, "%s: null pointer", what);
    RECO_REQUIRE(a.ldx >= a.D && a.ldw >= a.D, "%s: row strides %lld / %lld below the width %lld", what, (long long)a.ldx, (long long)a.ldw, (long long)a.D);
    RECO_REQUIRE(reduction >= REDUCE_NONE && reduction <= REDUCE_SUM, "%s: unknown reduction %d", what, reduction);
    return RECO_OK;
}

}  // namespace

extern "C" size_t reco_linear_xent_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int64_t T, int64_t V, int64_t D,
                                                   int keep)
{
    if (T <= 0 || V <= 0 || D <= 0) return 0;
    const Args a{x, ldx, w, ldw, nullptr, dtype, T, V, D, nullptr, 0};
    size_t need = 0;
    (void)reco_with_type(dtype, [&](auto z) -> int {
        return forward<decltype(z)>(a, 0, nullptr, nullptr, nullptr, keep != 0, nullptr, nullptr, &need, nullptr);
    });
    return need;
}

extern "C" int64_t reco_linear_xent_kept_floats(int dtype, int64_t T, int64_t V, int64_t D, int with_dx)
{
    if (dtype < RECO_DT_F32 || dtype > RECO_DT_F16 || T <= 0 || T >= (int64_t)1 << 31 || V <= 0 || V >= (int64_t)1 << 31 || D <= 0) return 0;
    if (narrow_fits(dtype, D)) return with_dx ? T * D : 0;
    if (dtype != RECO_DT_F32) return 0;                  // KEEPS
    const int64_t tile = tile_of(4, T, V);
    if (ceil_div64(T, tile) > KEPT_FLOATS / (tile * tile)) return 0;
    const int64_t n = ceil_div64(T, tile) * ceil_div64(V, tile) * tile * tile;
    return n <= KEPT_FLOATS ? n : 0;
}

extern "C" int reco_linear_xent(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int dtype, int64_t T, int64_t V, int64_t D,
                                const int64_t* target, int64_t ignore, int reduction, float* loss, float* state, float* kept, int32_t* oob,
                                void* ws, size_t ws_bytes, void* stream)
{
    const Args a{x, ldx, w, ldw, bias, dtype, T, V, D, target, ignore};
    const int rc = check_args("linear_xent", a, reduction);
    if (rc) return rc;
    RECO_REQUIRE(loss && state && ws && (uintptr_t)ws % 16 == 0, "linear_xent: null or misaligned loss, state or workspace");
    RECO_REQUIRE((uintptr_t)kept % 16 == 0, "linear_xent: misaligned room for what is kept");
    if (reco_linear_xent_kept_floats(dtype, T, V, D, 1) == 0) kept = nullptr;
    const size_t need = reco_linear_xent_workspace_bytes(x, ldx, w, ldw, dtype, T, V, D, kept != nullptr);
    if (ws_bytes < need) {
        reco_set_error("linear_xent: workspace of %zu bytes, %zu needed", ws_bytes, need);
        return RECO_ENOMEM;
    }
    ProfScope prof((hipStream_t)stream, RECO_PROF_XENT);
    size_t used = 0;
    return reco_with_type(dtype, [&](auto z) -> int {
        return forward<decltype(z)>(a, reduction, loss, state, kept, kept != nullptr, oob, (char*)ws, &used, (hipStream_t)stream);
    });
}

extern "C" size_t reco_linear_xent_grad_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int64_t T, int64_t V, int64_t D)
{
    if (T <= 0 || V <= 0 || D <= 0) return 0;
    const Args a{x, ldx, w, ldw, nullptr, dtype, T, V, D, nullptr, 0};
    size_t need = 0;
    (void)reco_with_type(dtype, [&](auto z) -> int {
        return backward<decltype(z)>(a, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, &need, nullptr);
    });
    return need;
}

extern "C" int reco_linear_xent_grad(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int dtype, int64_t T, int64_t V, int64_t D,
                                     const int64_t* target, int64_t ignore, int reduction, const float* state, const float* kept, const float* dloss,
                                     void* dx, void* dw, void* db, void* ws, size_t ws_bytes, void* stream)
{
    const Args a{x, ldx, w, ldw, bias, dtype, T, V, D, target, ignore};
    const int rc = check_args("linear_xent_grad", a, reduction);
    if (rc) return rc;
    RECO_REQUIRE(state && dloss && ws && (uintptr_t)ws % 16 == 0, "linear_xent_grad: null or misaligned state, gradient or workspace");
    const size_t need = reco_linear_xent_grad_workspace_bytes(x, ldx, w, ldw, dtype, T, V, D);
    if (ws_bytes < need) {
        reco_set_error("linear_xent_grad: workspace of %zu bytes, %zu needed", ws_bytes, need);
        return RECO_ENOMEM;
    }
    RECO_REQUIRE((uintptr_t)kept % 16 == 0, "linear_xent_grad: what was kept is misaligned");
    if (reco_linear_xent_kept_floats(dtype, T, V, D, 1) == 0) kept = nullptr;
    RECO_REQUIRE(!dx || kept || !narrow_fits(dtype, D), "linear_xent_grad: dx needs what the forward call kept");
    if (!dx && !dw && !db) return RECO_OK;
    ProfScope prof((hipStream_t)stream, RECO_PROF_XENT);
    size_t used = 0;
    return reco_with_type(dtype, [&](auto z) -> int {
        return backward<decltype(z)>(a, reduction, state, kept, dloss, dx, dw, db, (char*)ws, &used, (hipStream_t)stream);
    });
}

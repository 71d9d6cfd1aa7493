// K-g, the form for narrow rows (up to 256 values in 16 bits, 128 in 32): the logits never leave the registers.
//
// Both kernels hold rows of one operand ("held": 32 per wave) as matrix fragments for the whole launch and stream the rows of the
// other one through LDS, 32 at a time:
//   acc[streamed, held] = C R^T       one 32 x 32 block: lane l holds column l % 32, i.e. one held row, and 16 of the 32 streamed ones
//   e = exp(acc - ...)                in the registers the products left
//   O^T[d, held] += C^T e             e, rounded to the type, is a B operand as it lies: the order of k (streamed rows) inside a matrix
//                                     instruction is free, so A takes the order that the accumulator's rows have (LDS reads that
//                                     transpose 16-bit values 4 x 16 at a time; plain reads in 32 bits)
// rows: held x, streamed W, running maximum and sum per held row.  O / sum is the row's softmax-weighted mean of W, its gradient but for
//       the target's term, so one pass gives loss and dx.  The reference value of the exponentials follows the maximum only when that
//       grows by more than LAG (a power of e): then O and the sum are rescaled, which is rare after the first blocks.
// cols: held W, streamed x with the finished lse: O is dW, the sum of e over the streamed rows is dbias.
// A launch splits the streamed rows where there are few held ones; the parts are joined in order of the splits.
//
// What bounds it: a wave issues matrix instructions and exponentials in turn; an exponential per logit and two products of the row's width
// share a SIMD's issue.  bf16 8192 x 100,003 x 128: rows 0.47 ms, cols 0.50 (0.90, 0.84 PFLOP/s); f16 4097 x 50,021 x 250: 0.43 and 0.37 (0.48,
// 0.55); f32 6038 x 3533 x 32: 43 us each.  115 x 1 M x 128 without gradient: 64 us, 4.0 TB/s.  At rows of 256 bytes three waves a SIMD spilled;
// 64 held rows a wave halved the waves and were slower; so was a ring unrolled over six blocks.
#pragma once
#include "xent_shared.h"

namespace {

using namespace xent;

typedef int i32x4 __attribute__((ext_vector_type(4)));

template <typename T> constexpr float lag() { return 5.5f; }                         // e^5.5 = 2^7.9
template <> constexpr float lag<_Float16>() { return 2.75f; }                        // 2^10 x 2^4: G_SCALE as in the other direction
template <typename T> constexpr float G_LOG2 = sizeof(T) == 2 && Traits<T>::G_SCALE > 1.f ? 14.f : 0.f;
template <typename T> constexpr float e_shift() { return 0.f; }
template <> constexpr float e_shift<_Float16>() { return 10.f; }

// A tile of SB streamed rows of DP values in LDS.  The 64 banks take 256 bytes a cycle, i.e. 16 chunks of 16 bytes: the order of the
// chunks of a row is changed by the row (exclusive or with twist), so that both ways of reading spread over all of them: 16 rows at
// one chunk (logits), and 4 rows at 64 bytes each (the transposed reads).  CH: chunks per row.
template <int CH> __device__ __forceinline__ int twist(int row)
{
    constexpr int C = CH < 16 ? CH : 16;                        // chunks of a row that share 256 bytes, with those of 16 / C - 1 others
    return ((row >> 2) & 3) | ((row / (16 / C)) & (C / 4 - 1)) << 2;
}

template <typename T, int DP, int SB, int THREADS = 256> struct Tile {
    static constexpr int VEC = Traits<T>::VEC, ROWB = DP * (int)sizeof(T), CH = ROWB / 16, BYTES = SB * ROWB;
    static constexpr int PIECES = SB * CH / THREADS, ROW_STEP = THREADS / CH;
    static_assert(SB * CH % THREADS == 0 && THREADS % CH == 0 && (CH == 4 || CH % 8 == 0) && (CH & (CH - 1)) == 0, "tile shape");
    Pack<T, VEC> reg[PIECES];

    // rows r0 .. of m [rows, ld], `width` values each
    __device__ __forceinline__ void load(const T* m, int64_t ld, int64_t rows, int width, int64_t r0)
    {
        const int c = threadIdx.x % CH, row = threadIdx.x / CH;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int64_t r = r0 + row + i * ROW_STEP;
            if (r < rows && c * VEC < width) reg[i] = *reinterpret_cast<const Pack<T, VEC>*>(m + r * ld + c * VEC);
            else clear(i);
        }
    }
    __device__ __forceinline__ void clear(int i)
    {
#pragma unroll
        for (int j = 0; j < VEC; ++j) reg[i].v[j] = (T)0.f;
    }
    // drops (in LDS, nullable): rows of the tile with a negative entry are stored as zeros
    __device__ __forceinline__ void store(char* lds, const int* drops)
    {
        const int c = threadIdx.x % CH, row = threadIdx.x / CH;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = row + i * ROW_STEP;
            if (drops && drops[r] < 0) clear(i);
            *reinterpret_cast<Pack<T, VEC>*>(lds + r * ROWB + ((c ^ twist<CH>(r)) << 4)) = reg[i];
        }
    }
};

// A wave's view of the streamed rows and its 32 held ones
template <typename T, int DP> struct Wave {
    typedef typename Traits<T>::frag frag;
    static constexpr int STEPS = DP / Traits<T>::KSTEP, BLOCKS = DP / 32, ROWB = DP * (int)sizeof(T), CH = ROWB / 16;
    static constexpr bool WIDE = sizeof(T) == 4;
    static constexpr int C = CH < 16 ? CH : 16, ROW_KINDS = C / 2, COL_KINDS = C / 4;
    frag held[STEPS];
    int by_row[ROW_KINDS];          // byte of this lane's chunk of step j of a row: the steps repeat every 256 bytes
    int by_col[2][COL_KINDS];       // byte of this lane's value(s) for the transposed reading

    __device__ __forceinline__ void init(const T* m, int64_t ld, int64_t rows, int width, int64_t h0)
    {
        const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int64_t r = h0 + l31;
            const int k = i * Traits<T>::KSTEP + half * Traits<T>::VEC;
            if (r < rows && k < width) {
                held[i] = *reinterpret_cast<const frag*>(m + r * ld + k);
            } else {
#pragma unroll
                for (int j = 0; j < Traits<T>::VEC; ++j) held[i][j] = (T)0.f;
            }
        }
        const int t = twist<CH>(l31);
#pragma unroll
        for (int j = 0; j < ROW_KINDS; ++j) by_row[j] = l31 * ROWB + (((2 * j + half) ^ t) << 4);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < COL_KINDS; ++j) {
                if constexpr (WIDE) {       // row 8 (2 i + u) + 4 half + (0 .. 3): what twist adds above its low two bits is j
                    by_col[u][j] = 4 * half * ROWB + (((l31 >> 2) ^ (2 * u + half) ^ ((j & 1) << 2)) << 4) + (l31 & 3) * 4;
                } else {                    // rows 16 i + 8 u + 4 half + (0 .. 3), columns 32 j + ..
                    const int i16 = lane & 15, row = 8 * u + 4 * half + (i16 >> 2);
                    by_col[u][j] = row * ROWB + (((4 * j + ((lane >> 4) & 1) * 2 + ((i16 >> 1) & 1)) ^ twist<CH>(row)) << 4) + (i16 & 1) * 8;
                }
            }
    }

    __device__ __forceinline__ frag streamed(const char* lds, int i) const
    {
        return *reinterpret_cast<const frag*>(lds + by_row[i % ROW_KINDS] + i / ROW_KINDS * (C * 16));
    }
    // columns 32 d .. of streamed rows 16 j .., transposed
    __device__ __forceinline__ frag turned(const char* lds, int j, int d) const
    {
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const char* src = lds + d / COL_KINDS * (C * 16) + 16 * j * ROWB;
        union { s16x4 h[2]; frag f; } a;
        a.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(src + by_col[0][d % COL_KINDS]));
        a.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(src + by_col[1][d % COL_KINDS]));
        return a.f;
    }

    // s += the 32 streamed rows at `lds` times the held ones
    __device__ __forceinline__ void logits(const char* lds, f32x16& s) const
    {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) mma(s, streamed(lds, i), held[i]);
    }

    // The first streamed fragments of a block's logits are read while the block before it is worked on
    static constexpr int AHEAD = STEPS < 3 ? STEPS : 3;
    frag a[AHEAD];
    __device__ __forceinline__ void read_ahead(const char* lds)
    {
        if constexpr (!WIDE)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) a[i] = streamed(lds, i);
    }

    // next += the logits of the block at `ahead` (its first fragments are in a), while weight(r) turns s[r] of this block (at `lds`) into
    // its weight; then, after between(), o += (this block)^T times the weights, with beside(k, n) called as part k of n.  Leaves the
    // first fragments of the block at `then` in a.
    // A wave issues in order and a product waits for the one before it: the vector work stands between the products, in this order.
    // READ_THEN: that block is in LDS already (tiles of more than one block); else the caller reads the fragments when it is.
    template <bool SUMS, bool READ_THEN, typename Weight, typename Between, typename Beside>
    __device__ __forceinline__ void block(const char* ahead, const char* then, const char* lds, f32x16& next, f32x16& s, f32x16 (&o)[SUMS ? BLOCKS : 1],
                                          Weight&& weight, Between&& between, Beside&& beside)
    {
        if constexpr (WIDE) {
            logits(ahead, next);
#pragma unroll
            for (int r = 0; r < 16; ++r) weight(r);
            between();
            beside(0, 1);
            if constexpr (SUMS)
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int d = 0; d < BLOCKS; ++d) {
                        // the row's number in its 256 bytes is known here: twist's upper bits pick one of the two kinds, and the 128 bytes
                        const int up = (r & 3) / (16 / C) & (C / 4 - 1);
                        const float a =
                            *reinterpret_cast<const float*>(lds + by_col[(r >> 2) & 1][up & 1] + (8 * (r >> 2) + (r & 3)) * ROWB + ((d ^ (up >> 1)) * 128));
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[r], o[d], 0, 0, 0);
                    }
        } else {
            constexpr int EACH_STEP = (16 + STEPS - 1) / STEPS, PARTS = 2 * BLOCKS, TURN = PARTS < 2 ? PARTS : 2;
            frag c[TURN];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                mma(next, a[i % AHEAD], held[i]);
                if (i + AHEAD < STEPS) a[i % AHEAD] = streamed(ahead, i + AHEAD);
                if constexpr (SUMS)
                    if (i == (STEPS > 2 ? STEPS - 2 : 0))
#pragma unroll
                        for (int k = 0; k < TURN; ++k) c[k] = turned(lds, k / BLOCKS, k % BLOCKS);
#pragma unroll
                for (int r = i * EACH_STEP; r < (i + 1) * EACH_STEP && r < 16; ++r) weight(r);
                __builtin_amdgcn_sched_barrier(0);
            }
            between();
            if constexpr (SUMS) {
                frag p[2];
#pragma unroll
                for (int i = 0; i < 8; ++i) p[0][i] = (T)s[i];
#pragma unroll
                for (int k = 0; k < PARTS; ++k) {
                    mma(o[k % BLOCKS], c[k % TURN], p[k / BLOCKS]);
                    if (k + TURN < PARTS) c[k % TURN] = turned(lds, (k + TURN) / BLOCKS, (k + TURN) % BLOCKS);
                    if (k == 0)
#pragma unroll
                        for (int i = 0; i < 8; ++i) p[1][i] = (T)s[8 + i];
                    if (READ_THEN && k == PARTS - 2) read_ahead(then);
                    beside(k, PARTS);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                if (READ_THEN) read_ahead(then);
                beside(0, 1);
            }
        }
    }
};

template <typename T, int DP> constexpr int stream_rows() { return DP * (int)sizeof(T) >= 512 ? 32 : 64; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }        // below 2^-126: 0

// Four values of a row from column c on; fours: rows are whole aligned groups of four
template <typename U> __device__ __forceinline__ void store4(U* row, int c, int width, bool fours, float v0, float v1, float v2, float v3)
{
    if (fours) {
        if (c < width) *reinterpret_cast<Pack<U, 4>*>(row + c) = Pack<U, 4>{{(U)v0, (U)v1, (U)v2, (U)v3}};
        return;
    }
    if (c < width) row[c] = (U)v0;
    if (c + 1 < width) row[c + 1] = (U)v1;
    if (c + 2 < width) row[c + 2] = (U)v2;
    if (c + 3 < width) row[c + 3] = (U)v3;
}

// Waves per SIMD that the registers are cut for.  8192 x 100,003 in bf16 with gradients: x 32 462 us with two, 408 with three, 399 with
// four; x 64 593, 570, 1206 (spills); f32 2000 x 50,000 x 32 282, 280, 309 and 6038 x 3533 x 32 109, 113, 130.
template <typename T, int DP> constexpr int waves_per_simd()
{
    if (sizeof(T) == 4) return DP == 128 ? 1 : 2;
    return DP == 32 ? 4 : DP == 64 ? 3 : DP == 128 ? 2 : 1;
}

// of the rows kernel: one more without dx, whose sums are half of the registers (8192 x 100,003 x 128 bf16 311 -> 289 us, 4097 x 50,021 x 256
// f16 225 -> 154, 115 x 1 M x 128 f32 336 -> 295; f32 2000 x 50,000 x 64 137 both, and below that there are enough)
template <typename T, int DP, bool DX> constexpr int rows_waves() { return waves_per_simd<T, DP>() + (!DX && DP >= 128 ? 1 : 0); }

// ---------------------------------------------------------------------------------------------
// rows: loss statistics, and with DX the softmax-weighted sums of W
// ---------------------------------------------------------------------------------------------
template <typename T, int DP, bool BIAS, bool DX, int WAVES>
__global__ __launch_bounds__(WAVES * 64, (WAVES == 1 ? 1 : rows_waves<T, DP, DX>())) void narrow_rows_kernel(Problem p, int splits, int64_t rows_per_split, int width_out,
                                                                                   Running* __restrict__ part, float* __restrict__ z_target,
                                                                                   float* __restrict__ dx_part)
{
    constexpr int SB = stream_rows<T, DP>(), NS = SB / 32;
    typedef Tile<T, DP, SB, WAVES * 64> Streamed;
    typedef Wave<T, DP> W;
    __shared__ __attribute__((aligned(16))) char tiles[3][Streamed::BYTES];
    __shared__ __attribute__((aligned(16))) float biases[3][SB];
    const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t split = blockIdx.x % splits, h0 = (blockIdx.x / splits * WAVES + wave) * 32, t = h0 + l31;
    const bool active = h0 < p.T;
    const T* w = (const T*)p.w;
    const T* bias = (const T*)p.bias;
    const int64_t first = split * rows_per_split, end = first + rows_per_split < p.V ? first + rows_per_split : p.V;
    const int n_tiles = (int)((end - first + SB - 1) / SB);

    W me;
    me.init((const T*)p.x, p.ldx, p.T, (int)p.D, h0);
    int y = -1;
    if (t < p.T && p.target[t] != p.ignore) y = (int)clamp_target(p.target[t], p.V);
    float m = -INFINITY;
    Sum sum;
    f32x16 o[DX ? W::BLOCKS : 1];
    if constexpr (DX)
#pragma unroll
        for (int d = 0; d < W::BLOCKS; ++d) o[d] = f32x16{};

    Streamed st;
    float bias_reg = 0.f;
    auto fetch = [&](int tile) {
        const int64_t v0 = first + (int64_t)tile * SB;
        st.load(w, p.ldw, end, (int)p.D, v0);
        if (threadIdx.x < SB) {
            const int64_t v = v0 + threadIdx.x;
            bias_reg = v >= end ? -INFINITY : BIAS ? (float)bias[v] : 0.f;        // rows behind the split have no weight
        }
    };
    auto put = [&](int at) {
        st.store(tiles[at], nullptr);
        if (threadIdx.x < SB) biases[at][threadIdx.x] = bias_reg;
    };
    auto init = [&](const float* biases32, f32x16& z) {
        if (BIAS) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 c = *reinterpret_cast<const f32x4*>(biases32 + 8 * q + 4 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) z[4 * q + i] = c[i];
            }
        } else {
            z = f32x16{};
        }
    };
    // a finished block's rows v0 ..: those behind the split and the target's logit out, and the reference value of the exponentials;
    // top: this lane's largest
    auto settle = [&](int64_t v0, f32x16& z, float top) {
        const int here = y - (int)v0;                                           // the target's place in this block, if it is in it
        const bool tail = !BIAS && v0 + 32 > end, mine = __any((unsigned)here < 32u);
        if (tail || mine) {
            const int left = (int)(end - v0), at = here - 4 * half, stop = left - 4 * half;      // registers are compared with constants
            float own = 0.f;
            top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = acc_row(r, 0);
                own = row == at ? z[r] : own;
                z[r] = row == at || row >= stop ? -INFINITY : z[r];
                top = fmaxf(top, z[r]);
            }
            if ((unsigned)here < 32u && (here & 4) == 4 * half && here < left) z_target[t] = own;
        }
        if (__any(top > m + lag<T>())) {
            top = fmaxf(top, __shfl_xor(top, 32, 64));                          // both halves of a column keep one reference
            if (top > m + lag<T>()) {
                const float f = m == -INFINITY ? 0.f : exp2_fast((m - top) * LOG2E);
                m = top;
                sum.scale(f);
                if constexpr (DX)
#pragma unroll
                    for (int d = 0; d < W::BLOCKS; ++d) o[d] *= f;
            }
        }
    };
    auto largest = [](const f32x16& z) {
        float top = z[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, z[r]);
        return top;
    };

    // Three tiles in LDS: tile i is weighed and the logits of tile i + 1's first block are taken while tile i + 2 arrives; one barrier
    // per tile
    fetch(0);
    put(0);
    if (n_tiles > 1) {
        fetch(1);
        put(1);
    }
    __syncthreads();
    constexpr int BLOCK_BYTES = 32 * W::ROWB, RING = 3 * NS;
    char* const ring = &tiles[0][0];
    const int n_blocks = (int)((end - first + 31) / 32);
    f32x16 s0, s1;
    if (active) {
        init(&biases[0][0], s0);
        me.logits(ring, s0);
        settle(first, s0, largest(s0));
        if (NS > 1) me.read_ahead(ring + BLOCK_BYTES);
    }
    int at = 0;
    // block i: s holds its logits, next gets those of block i + 1
    auto work = [&](int i, f32x16& s, f32x16& next) {
        const int after = at + 1 == RING ? 0 : at + 1, then = after + 1 == RING ? 0 : after + 1;
        const int tile = i / NS;
        if (i % NS == 0 && tile + 2 < n_tiles) fetch(tile + 2);
        if (active) {
            // nothing above -inf yet: any finite reference leaves the sum at 0
            const float base = m == -INFINITY ? 0.f : m, shift = e_shift<T>() - base * LOG2E;
            float top = -INFINITY, here = 0.f;
            init(&biases[0][0] + after * 32, next);
            if (NS == 1) me.read_ahead(ring + after * BLOCK_BYTES);
            me.template block<DX, (NS > 1)>(
                ring + after * BLOCK_BYTES, ring + then * BLOCK_BYTES, ring + at * BLOCK_BYTES, next, s, o,
                [&](int r) {
                    // the difference first in 32 bits, for its digits, and with a bias, whose logits may be the type's lowest
                    s[r] = BIAS || W::WIDE ? exp2_fast(fmaf(s[r] - base, LOG2E, e_shift<T>())) : exp2_fast(fmaf(s[r], LOG2E, shift));
                },
                [] {},
                [&](int k, int n) {
#pragma unroll
                    for (int r = k * 16 / n; r < (k + 1) * 16 / n; ++r) here += s[r];
                    if (k == n / 2) top = largest(next);
                });
            sum.add<false>(here);
            if (i + 1 < n_blocks) settle(first + 32 * (int64_t)(i + 1), next, top);
        }
        if (i % NS == NS - 1) {
            if (tile + 2 < n_tiles) put((tile + 2) % 3);
            __syncthreads();
        }
        at = after;
    };
#pragma unroll 1
    for (int i = 0; i < n_blocks; i += 2) {
        work(i, s0, s1);
        if (i + 1 < n_blocks) work(i + 1, s1, s0);
    }
    if (!active) return;
    const float total = sum.s + __shfl_xor(sum.s, 32, 64);
    if (t >= p.T) return;
    if (half == 0) part[split * p.T + t] = Running{m, total * exp2f(-e_shift<T>())};
    if constexpr (DX) {
        float* dst = dx_part + (split * p.T + t) * width_out;
        const float f = exp2f(-e_shift<T>());
#pragma unroll
        for (int d = 0; d < W::BLOCKS; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                store4(dst, 32 * d + 8 * q + 4 * half, width_out, width_out % 4 == 0, o[d][4 * q] * f, o[d][4 * q + 1] * f, o[d][4 * q + 2] * f, o[d][4 * q + 3] * f);
    }
}

// ---------------------------------------------------------------------------------------------
// cols: dW and dbias
// ---------------------------------------------------------------------------------------------
// expo[t]: -lse_t log2(e) + log2(G_SCALE), -inf for rows that do not count.  In 32 bits, and with BIAS, as such logits may be the type's
// lowest: lse_t itself (+inf), and in 32 bits expo[T + t] minus what rounding left of lse_t, times log2(e).  y[t]: the target, -1 for
// rows that do not count.  BIAS: there is one, or its gradient is asked for.  EACH: rows have weights gn[t].
// The work is groups of 128 held rows times tiles of streamed ones, in that order; every workgroup takes an equal share of consecutive
// (group, tile) units, so that the groups need not be a multiple of what the chip holds at once (782 groups over 512 places: 0.72 ms
// with a group to a workgroup).  A group inside one share is finished there; else its parts are written in 32 bits (place 1 of a
// workgroup: a part that begins its group, place 0: one that does not) and added by narrow_join_kernel in order.
template <typename T, int DP, bool BIAS, bool EACH>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP>())) void narrow_cols_kernel(Problem p, int64_t units, int64_t share, int tiles_in_all, int width_out,
                                                                                   const float* __restrict__ expo, const int* __restrict__ y,
                                                                                   const float* __restrict__ rest, const float* __restrict__ gn,
                                                                                   const float* __restrict__ scale, T* __restrict__ dw, T* __restrict__ db,
                                                                                   float* __restrict__ dw_part, float* __restrict__ db_part)
{
    constexpr int SB = stream_rows<T, DP>(), NS = SB / 32;
    typedef Tile<T, DP, SB> Streamed;
    typedef Wave<T, DP> W;
    __shared__ __attribute__((aligned(16))) char tiles[3][Streamed::BYTES];
    __shared__ __attribute__((aligned(16))) float expos[3][SB];
    __shared__ __attribute__((aligned(16))) float lows[W::WIDE ? 3 : 1][SB];
    __shared__ __attribute__((aligned(16))) float gns[EACH ? 3 : 1][SB];
    __shared__ __attribute__((aligned(16))) float minus_q[3][SB];
    __shared__ __attribute__((aligned(16))) int ys[4][SB];
    const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    char* const ring = &tiles[0][0];
    constexpr int BLOCK_BYTES = 32 * W::ROWB, RING = 3 * NS;
    const bool fours = width_out % 4 == 0 && (uintptr_t)dw % sizeof(Pack<T, 4>) == 0;
    const int64_t u0 = blockIdx.x * share, u1 = u0 + share < units ? u0 + share : units;
    W me;
    me.init((const T*)p.w, p.ldw, p.V, (int)p.D, (u0 / tiles_in_all * 4 + wave) * 32);
#pragma unroll 1
    for (int64_t u = u0; u < u1;) {
    const int64_t group = u / tiles_in_all;
    const int tile0 = (int)(u - group * tiles_in_all), n_tiles = u1 - u < tiles_in_all - tile0 ? (int)(u1 - u) : tiles_in_all - tile0;
    const int64_t h0 = (group * 4 + wave) * 32, v = h0 + l31;
    const bool active = h0 < p.V;
    const int64_t first = (int64_t)tile0 * SB, end = first + (int64_t)n_tiles * SB < p.T ? first + (int64_t)n_tiles * SB : p.T;
    const bool whole = n_tiles == tiles_in_all, stage = u == u0 || tiles_in_all > 1;     // a single tile stays for every group
    u += n_tiles;

    const float bias = BIAS && p.bias && v < p.V ? (float)((const T*)p.bias)[v] : 0.f;
    Sum sum;
    f32x16 o[W::BLOCKS];
#pragma unroll
    for (int d = 0; d < W::BLOCKS; ++d) o[d] = f32x16{};

    // In 32 bits the products are added to the bias, as in the rows' pass: the same bits, or p of a sure row would be off by a rounding of its
    // logit.  In 16 bits p is rounded to more than that, and the bias is added afterwards (8192 x 100,003 x 32 bf16 483 us, 505 this way).
    auto begin = [&](f32x16& z) {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = W::WIDE ? bias : 0.f;
    };
    Streamed st;
    float expo_reg = 0.f, low_reg = 0.f, gn_reg = 0.f, q_reg = 0.f;
    int y_reg = -1;
    auto fetch = [&](int tile) {
        const int64_t t0 = first + (int64_t)tile * SB;
        st.load((const T*)p.x, p.ldx, end, (int)p.D, t0);
        if (threadIdx.x < SB) {
            const int64_t t = t0 + threadIdx.x;
            expo_reg = t < end ? expo[t] : BIAS || W::WIDE ? INFINITY : -INFINITY;
            if (W::WIDE) low_reg = t < end ? expo[p.T + t] : 0.f;
            y_reg = t + SB < end ? y[t + SB] : -1;
            q_reg = t < end ? rest[t] : 0.f;
            if (EACH) gn_reg = t < end ? gn[t] : 0.f;
        }
    };
    // the targets run one tile ahead of the rows: storing a tile looks at those of its rows that do not count
    auto put = [&](int tile) {
        const int at = tile % 3;
        st.store(tiles[at], ys[tile & 3]);
        if (threadIdx.x < SB) {
            expos[at][threadIdx.x] = expo_reg;
            if (W::WIDE) lows[W::WIDE ? at : 0][threadIdx.x] = low_reg;
            minus_q[at][threadIdx.x] = -Traits<T>::G_SCALE * (EACH ? q_reg * gn_reg : q_reg);
            ys[(tile + 1) & 3][threadIdx.x] = y_reg;
            if (EACH) gns[at][threadIdx.x] = gn_reg;
        }
    };
    if (stage) {
        if (threadIdx.x < 2 * SB) ys[threadIdx.x / SB][threadIdx.x % SB] = first + threadIdx.x < end ? y[first + threadIdx.x] : -1;
        __syncthreads();
        fetch(0);
        put(0);
        if (n_tiles > 1) {
            fetch(1);
            put(1);
        }
        __syncthreads();
    }
    const int n_blocks = (int)((end - first + 31) / 32);
    f32x16 s0, s1;
    f32x4 x4, g4, low4, x_next = {}, g_next = {};
    if (active) {
        x_next = *reinterpret_cast<const f32x4*>(&expos[0][4 * half]);
        if (EACH) g_next = *reinterpret_cast<const f32x4*>(&gns[0][4 * half]);
        begin(s0);
        me.logits(ring, s0);
        if (NS > 1) me.read_ahead(ring + BLOCK_BYTES);
    }
    int at = 0;
    auto work = [&](int i, f32x16& s, f32x16& next) {
        const int after = at + 1 == RING ? 0 : at + 1, then = after + 1 == RING ? 0 : after + 1;
        const int tile = i / NS;
        if (i % NS == 0 && tile + 2 < n_tiles) fetch(tile + 2);
        if (active) {
            const float *expo32 = &expos[0][0] + 4 * half, *gn32 = &gns[0][0] + 4 * half;
            const int* y32 = &ys[tile & 3][i % NS * 32];
            const int mine = y32[l31];
            float here = 0.f;
            begin(next);
            if (NS == 1) me.read_ahead(ring + after * BLOCK_BYTES);
            me.template block<true, (NS > 1)>(
                ring + after * BLOCK_BYTES, ring + then * BLOCK_BYTES, ring + at * BLOCK_BYTES, next, s, o,
                [&](int r) {
                    if (r % 4 == 0) {                               // the rows' constants are read four ahead
                        const int ahead = r < 12 ? at * 32 + 8 * (r / 4 + 1) : after * 32;
                        x4 = x_next;
                        x_next = *reinterpret_cast<const f32x4*>(expo32 + ahead);
                        if (W::WIDE) low4 = *reinterpret_cast<const f32x4*>(&lows[0][0] + at * 32 + 2 * r + 4 * half);
                        if (EACH) {
                            g4 = g_next;
                            g_next = *reinterpret_cast<const f32x4*>(gn32 + ahead);
                        }
                    }
                    const float e = W::WIDE ? exp2_fast(fmaf(s[r] - x4[r % 4], LOG2E, low4[r % 4]))
                                    : BIAS ? exp2_fast(fmaf(s[r] + bias - x4[r % 4], LOG2E, G_LOG2<T>)) : exp2_fast(fmaf(s[r], LOG2E, x4[r % 4]));
                    s[r] = EACH ? e * g4[r % 4] : e;
                },
                [&] {
                    // A target of these 32 rows that lies in this wave's part of the vocabulary.  Without memory loads or branches per
                    // value: with a popular item among its 32, a wave comes here for most blocks.
                    if (__any((unsigned)(mine - (int)h0) < 32u))
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const i32x4 y4 = *reinterpret_cast<const i32x4*>(y32 + 8 * q + 4 * half);
                            const f32x4 q4 = *reinterpret_cast<const f32x4*>(&minus_q[0][0] + at * 32 + 8 * q + 4 * half);
#pragma unroll
                            for (int j = 0; j < 4; ++j) s[4 * q + j] = y4[j] == (int)v ? q4[j] : s[4 * q + j];
                        }
                },
                [&](int k, int n) {
#pragma unroll
                    for (int r = k * 16 / n; BIAS && r < (k + 1) * 16 / n; ++r) here += s[r];
                });
            if (BIAS) sum.add<EACH>(here);                         // rows' weights may be infinite
        }
        if (i % NS == NS - 1 && tile + 1 < n_tiles) {
            if (tile + 2 < n_tiles) put(tile + 2);
            __syncthreads();
        }
        at = after;
    };
#pragma unroll 1
    for (int i = 0; i < n_blocks; i += 2) {
        work(i, s0, s1);
        if (i + 1 < n_blocks) work(i + 1, s1, s0);
    }
    if (tiles_in_all > 1) __syncthreads();                      // the next group's tiles overwrite these
    if (u < u1) me.init((const T*)p.w, p.ldw, p.V, (int)p.D, ((group + 1) * 4 + wave) * 32);      // on its way during the stores
    if (!active) continue;
    const float f = whole ? *scale / Traits<T>::G_SCALE : 1.f;
    const float total = (sum.s + __shfl_xor(sum.s, 32, 64)) * f;
    if (v >= p.V) continue;
    const int64_t row = ((int64_t)blockIdx.x * 2 + (tile0 ? 0 : 1)) * 128 + wave * 32 + l31;
    if (BIAS && half == 0) {
        if (!whole) db_part[row] = total;
        else if (db) db[v] = (T)total;
    }
    if (!whole || dw)
#pragma unroll
        for (int d = 0; d < W::BLOCKS; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = 32 * d + 8 * q + 4 * half;
                if (!whole) store4(dw_part + row * width_out, c, width_out, width_out % 4 == 0, o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]);
                else store4(dw + v * width_out, c, width_out, fours, o[d][4 * q] * f, o[d][4 * q + 1] * f, o[d][4 * q + 2] * f, o[d][4 * q + 3] * f);
            }
    }
}

// The groups that several workgroups shared: blockIdx.x is the group, the threads take its 128 x (width, then 1) sums
template <typename T>
__global__ __launch_bounds__(256) void narrow_join_kernel(int64_t V, int64_t share, int tiles_in_all, int width, const float* __restrict__ scale,
                                                          const float* __restrict__ dw_part, const float* __restrict__ db_part, T* __restrict__ dw, T* __restrict__ db)
{
    const int64_t group = blockIdx.x, a = group * tiles_in_all / share, b = ((group + 1) * tiles_in_all - 1) / share;
    if (a == b) return;
    const float f = *scale / Traits<T>::G_SCALE;
    const int n = 128 * width;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < n + 128; i += gridDim.y * 256) {
        const bool bias = i >= n;
        const int64_t v = group * 128 + (bias ? i - n : i / width);
        if (v >= V || !(bias ? db : dw)) continue;
        float s = 0.f;
#pragma unroll 4
        for (int64_t g = a; g <= b; ++g) {
            const int64_t place = g * 2 + (g == a ? 1 : 0);
            s += bias ? db_part[place * 128 + (i - n)] : dw_part[place * n + i];
        }
        if (bias) db[v] = (T)(s * f);
        else dw[group * n + i] = (T)(s * f);
    }
}

template <typename T, typename F> int with_width(int64_t D, F&& fn)
{
    if (D <= 32) return fn(std::integral_constant<int, 32>());
    if (D <= 64) return fn(std::integral_constant<int, 64>());
    if constexpr (sizeof(T) == 2)
        if (D > 128) return fn(std::integral_constant<int, 256>());
    return fn(std::integral_constant<int, 128>());
}

template <typename F> int with_flag(bool v, F&& fn) { return v ? fn(std::true_type()) : fn(std::false_type()); }

constexpr int64_t HELD = 128;                  // held rows per workgroup: 4 waves of 32

// Up to 32 rows keep one wave of a workgroup busy.  In 32 bits at 65 to 128 values a compute unit holds one workgroup of four waves but
// three of one wave, and the matrix instructions bound the launch: 1 row x 1 M x 128 164 us instead of 326, with dx 255 instead of 551.
// In 16 bits, and with shorter rows, memory does, which four waves ask more of at once (bf16 1 x 1 M x 128: 47 us, 59 with one wave).
template <typename T, int DP> constexpr bool ONE_WAVE = sizeof(T) == 4 && DP == 128;

template <typename T, typename F> int shape_of(int64_t D, F&& fn)
{
    return with_width<T>(D, [&](auto dp) -> int {
        constexpr int DP = decltype(dp)::value;
        return fn(dp, (int64_t)stream_rows<T, DP>(), 256 * waves_per_simd<T, DP>());
    });
}

// Splits of the streamed rows, whole tiles each: the fewest microseconds out of rounds of workgroups (at the rate that the kernels reach,
// 0.8 PFLOP/s in 16 bits and 0.12 in 32, and 4 us to begin and end one) and of the parts of dx, written and read at 4 TB/s
inline void split_plan(int64_t T, int64_t D, int64_t groups, int64_t streamed, int64_t tile, int64_t places, double rate, int64_t* splits, int64_t* per)
{
    const int64_t tiles = ceil_div64(streamed, tile);
    const double tile_us = 4.0 * tile * HELD * D * places / rate * 1e6;
    double best = 1e30;
    int64_t most = 4 * places / groups + 1;
    if (most > tiles) most = tiles;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t run = ceil_div64(tiles, s), n = ceil_div64(tiles, run);
        const double us = ceil_div64(groups * n, places) * (run * tile_us + 4.0) + n * T * D * 8.0 / 4e12 * 1e6;
        if (us < best) {
            best = us;
            *splits = n;
            *per = run * tile;
        }
    }
}

}  // namespace

namespace xent {

template <typename T> NarrowPlan narrow_plan_of(int64_t T_rows, int64_t V, int64_t D, bool dx)
{
    NarrowPlan n{};
    (void)shape_of<T>(D, [&](auto dp, int64_t tile, int64_t places) -> int {
        constexpr int DP = decltype(dp)::value;
        n.x_waves = ONE_WAVE<T, DP> && T_rows <= 32 ? 1 : 4;
        n.x_groups = ceil_div64(T_rows, 32 * n.x_waves);
        const int64_t x_places = n.x_waves == 4 ? 256 * (dx ? rows_waves<T, DP, true>() : rows_waves<T, DP, false>()) : 256 * (160 * 1024 / (3 * tile * (DP * (int)sizeof(T) + 4)));
        split_plan(T_rows, DP, n.x_groups, V, tile, x_places, sizeof(T) == 2 ? 0.8e15 : 0.12e15, &n.x_splits, &n.x_per);
        n.w_groups = ceil_div64(V, HELD);
        n.w_tiles = ceil_div64(T_rows, tile);
        const int64_t units = n.w_groups * n.w_tiles;
        // a share of less than four tiles is mostly beginning and end
        n.w_share = ceil_div64(units, places);
        if (n.w_share < 4) n.w_share = n.w_tiles < 4 ? n.w_tiles : 4;
        n.w_shares = ceil_div64(units, n.w_share);
        n.w_shared = n.w_share % n.w_tiles != 0;
        return RECO_OK;
    });
    return n;
}

template <typename T> int narrow_rows_of(const Problem& p, const NarrowPlan& n, int64_t width_out, Running* part, float* z_target, float* dx_part, hipStream_t s)
{
    return shape_of<T>(p.D, [&](auto dp, int64_t, int64_t) -> int {
        return with_flag(p.bias != nullptr, [&](auto bias) -> int {
            return with_flag(dx_part != nullptr, [&](auto dx) -> int {
                const auto launch = [&](auto waves) {
                    constexpr int WAVES = decltype(waves)::value;
                    hipLaunchKernelGGL((narrow_rows_kernel<T, decltype(dp)::value, decltype(bias)::value, decltype(dx)::value, WAVES>),
                                       dim3((unsigned)(n.x_groups * n.x_splits)), dim3(WAVES * 64), 0, s, p, (int)n.x_splits, n.x_per, (int)width_out, part,
                                       z_target, dx_part);
                };
                if constexpr (ONE_WAVE<T, decltype(dp)::value>)
                    if (n.x_waves == 1) {
                        launch(std::integral_constant<int, 1>());
                        RECO_CHECK_LAUNCH();
                        return RECO_OK;
                    }
                launch(std::integral_constant<int, 4>());
                RECO_CHECK_LAUNCH();
                return RECO_OK;
            });
        });
    });
}

template <typename T>
int narrow_cols_of(const Problem& p, const NarrowPlan& n, int64_t width_out, const float* expo, const int* y, const float* rest, const float* gn,
                   const float* scale, void* dw, void* db, float* dw_part, float* db_part, hipStream_t s)
{
    return shape_of<T>(p.D, [&](auto dp, int64_t, int64_t) -> int {
        return with_flag(p.bias || db, [&](auto bias) -> int {
            return with_flag(gn != nullptr, [&](auto each) -> int {
                hipLaunchKernelGGL((narrow_cols_kernel<T, decltype(dp)::value, decltype(bias)::value, decltype(each)::value>), dim3((unsigned)n.w_shares), dim3(256),
                                   0, s, p, n.w_groups * n.w_tiles, n.w_share, (int)n.w_tiles, (int)width_out, expo, y, rest, gn, scale, (T*)dw, (T*)db, dw_part,
                                   db_part);
                if (n.w_shared)
                    hipLaunchKernelGGL(narrow_join_kernel<T>, dim3((unsigned)n.w_groups, (unsigned)ceil_div64(HELD * (width_out + 1), 1024)), dim3(256), 0, s, p.V,
                                       n.w_share, (int)n.w_tiles, (int)width_out, scale, dw_part, db_part, (T*)dw, (T*)db);
                RECO_CHECK_LAUNCH();
                return RECO_OK;
            });
        });
    });
}

}  // namespace xent

// One source file per element type instantiates these
#define XENT_NARROW(T)                                                                                                                             \
    template xent::NarrowPlan xent::narrow_plan_of<T>(int64_t, int64_t, int64_t, bool);                                                             \
    template int xent::narrow_rows_of<T>(const xent::Problem&, const xent::NarrowPlan&, int64_t, xent::Running*, float*, float*, hipStream_t);      \
    template int xent::narrow_cols_of<T>(const xent::Problem&, const xent::NarrowPlan&, int64_t, const float*, const int*, const float*,            \
                                         const float*, const float*, void*, void*, float*, float*, hipStream_t)

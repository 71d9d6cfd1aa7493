// K-g, the form for narrow rows (up to 256 values in 16 bits, 128 in 32): the logits never leave the registers.
//
// Both kernels hold rows of one operand ("held": 32 NB per wave) as matrix fragments for the whole launch and stream the rows of the
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
#include "xent_shared.h"

namespace {

using namespace xent;

typedef int i32x4 __attribute__((ext_vector_type(4)));

template <typename T> constexpr float lag() { return 5.5f; }                         // e^5.5 = 2^7.9
template <> constexpr float lag<_Float16>() { return 2.75f; }                        // 2^10 x 2^4: G_SCALE as in the other direction
template <typename T> constexpr float G_LOG2 = sizeof(T) == 2 && Traits<T>::G_SCALE > 1.f ? 14.f : 0.f;
template <typename T> constexpr float e_shift() { return 0.f; }
template <> constexpr float e_shift<_Float16>() { return 10.f; }

// A tile of SB streamed rows of DP values in LDS: 16-byte chunks, their order within a row changed by the row so that both ways of
// reading (32 rows at one chunk; 4 rows at 32 bytes) touch every bank equally.  CH: chunks per row.
template <int CH> __device__ __forceinline__ int twist(int row)
{
    return CH == 4 ? (((row >> 1) & 1) << 1) | ((row >> 2) & 1) : ((row & 3) << 1) | ((row >> 2) & 1);
}

template <typename T, int DP, int SB> struct Tile {
    static constexpr int VEC = Traits<T>::VEC, ROWB = DP * (int)sizeof(T), CH = ROWB / 16, BYTES = SB * ROWB;
    static constexpr int PIECES = SB * CH / 256, ROW_STEP = 256 / CH;
    static_assert(SB * CH % 256 == 0 && (CH == 4 || CH % 8 == 0) && (CH & (CH - 1)) == 0, "tile shape");
    Pack<T, VEC> reg[PIECES];

    // rows r0 .. of m [rows, ld], `width` values each; rows with drop[row] < 0 (nullable) are read as zeros
    __device__ __forceinline__ void load(const T* m, int64_t ld, int64_t rows, int width, int64_t r0, const int* drop)
    {
        const int c = threadIdx.x % CH, row = threadIdx.x / CH;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int64_t r = r0 + row + i * ROW_STEP;
            bool ok = r < rows && c * VEC < width;
            if (drop && ok) ok = drop[r] >= 0;
            if (ok) {
                reg[i] = *reinterpret_cast<const Pack<T, VEC>*>(m + r * ld + c * VEC);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) reg[i].v[j] = (T)0.f;
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) const
    {
        const int c = threadIdx.x % CH, row = threadIdx.x / CH;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = row + i * ROW_STEP;
            *reinterpret_cast<Pack<T, VEC>*>(lds + r * ROWB + ((c ^ twist<CH>(r)) << 4)) = reg[i];
        }
    }
};

// A wave's view of the streamed tile and its held rows
template <typename T, int DP, int NB> struct Wave {
    typedef typename Traits<T>::frag frag;
    static constexpr int STEPS = DP / Traits<T>::KSTEP, BLOCKS = DP / 32, ROWB = DP * (int)sizeof(T), CH = ROWB / 16;
    static constexpr bool WIDE = sizeof(T) == 4;
    frag held[NB][STEPS];
    f32x16 s[NB];
    int by_row[4];         // byte of this lane's chunk of step j of a row: the steps repeat every 128 bytes
    int by_col[4];         // byte of this lane's value(s) for the transposed reading

    __device__ __forceinline__ void init(const T* m, int64_t ld, int64_t rows, int width, int64_t h0)
    {
        const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int64_t r = h0 + 32 * b + l31;
                const int k = i * Traits<T>::KSTEP + half * Traits<T>::VEC;
                if (r < rows && k < width) {
                    held[b][i] = *reinterpret_cast<const frag*>(m + r * ld + k);
                } else {
#pragma unroll
                    for (int j = 0; j < Traits<T>::VEC; ++j) held[b][i][j] = (T)0.f;
                }
            }
        const int t = twist<CH>(l31);
#pragma unroll
        for (int j = 0; j < 4; ++j) by_row[j] = l31 * ROWB + (((2 * j + half) ^ t) << 4);
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < 4; ++j) by_col[j] = (4 * half + j) * ROWB + (((l31 >> 2) ^ ((j << 1) | half)) << 4) + (l31 & 3) * 4;
        } else {
            const int i16 = lane & 15, row = 4 * half + (i16 >> 2), tr = twist<CH>(row);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                by_col[j] = row * ROWB + ((((j & 1) * 4 + ((lane >> 4) & 1) * 2 + ((i16 >> 1) & 1)) ^ tr) << 4) + (i16 & 1) * 8;
        }
    }

    // s += the 32 streamed rows at `lds` times the held ones
    __device__ __forceinline__ void logits(const char* lds)
    {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const frag a = *reinterpret_cast<const frag*>(lds + by_row[i & 3] + (i >> 2) * 128);
#pragma unroll
            for (int b = 0; b < NB; ++b) mma(s[b], a, held[b][i]);
        }
    }

    // o += (the 32 streamed rows)^T times s, which holds weights now
    __device__ __forceinline__ void weigh(const char* lds, f32x16 (&o)[NB][BLOCKS]) const
    {
        if constexpr (WIDE) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int d = 0; d < BLOCKS; ++d) {
                    const float a = *reinterpret_cast<const float*>(lds + by_col[r & 3] + 8 * (r >> 2) * ROWB + d * 128);
#pragma unroll
                    for (int b = 0; b < NB; ++b) o[b][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[b][r], o[b][d], 0, 0, 0);
                }
        } else {
            frag p[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) p[b][i >> 3][i & 7] = (T)s[b][i];
            typedef __attribute__((address_space(3))) s16x4* lds_ptr;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 0; d < BLOCKS; ++d) {
                    const char* src = lds + by_col[d & 1] + (d >> 1) * 128 + 16 * j * ROWB;
                    union { s16x4 h[2]; frag f; } a;
                    a.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)src);
                    a.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(src + 8 * ROWB));
#pragma unroll
                    for (int b = 0; b < NB; ++b) mma(o[b][d], a.f, p[b][j]);
                }
        }
    }
};

template <typename T, int DP> constexpr int stream_rows() { return DP * (int)sizeof(T) >= 512 ? 32 : 64; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }        // below 2^-126: 0

// ---------------------------------------------------------------------------------------------
// rows: loss statistics, and with DX the softmax-weighted sums of W
// ---------------------------------------------------------------------------------------------
template <typename T, int DP, int NB, bool BIAS, bool DX>
__global__ __launch_bounds__(256) void narrow_rows_kernel(Problem p, int splits, int64_t rows_per_split, int width_out, Running* __restrict__ part,
                                                          float* __restrict__ z_target, float* __restrict__ dx_part)
{
    constexpr int SB = stream_rows<T, DP>();
    typedef Tile<T, DP, SB> Streamed;
    typedef Wave<T, DP, NB> W;
    __shared__ __attribute__((aligned(16))) char tiles[2][Streamed::BYTES];
    __shared__ __attribute__((aligned(16))) float biases[2][SB];
    const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t split = blockIdx.x % splits, h0 = (blockIdx.x / splits * 4 + wave) * (32 * NB);
    const bool active = h0 < p.T;
    const T* w = (const T*)p.w;
    const T* bias = (const T*)p.bias;
    const int64_t first = split * rows_per_split, end = first + rows_per_split < p.V ? first + rows_per_split : p.V;

    W me;
    me.init((const T*)p.x, p.ldx, p.T, (int)p.D, h0);
    int y[NB];
    float m[NB], sum[NB];
    f32x16 o[NB][DX ? W::BLOCKS : 1];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t t = h0 + 32 * b + l31;
        y[b] = -1;
        if (t < p.T && p.target[t] != p.ignore) y[b] = (int)clamp_target(p.target[t], p.V);
        m[b] = -INFINITY;
        sum[b] = 0.f;
        if constexpr (DX)
#pragma unroll
            for (int d = 0; d < W::BLOCKS; ++d) o[b][d] = f32x16{};
    }

    Streamed st;
    float bias_reg = 0.f;
    auto fetch = [&](int64_t v0) {
        st.load(w, p.ldw, end, (int)p.D, v0, nullptr);
        if (threadIdx.x < SB) {
            const int64_t v = v0 + threadIdx.x;
            bias_reg = v >= end ? -INFINITY : BIAS ? (float)bias[v] : 0.f;        // rows behind the split have no weight
        }
    };
    auto put = [&](int at) {
        st.store(tiles[at]);
        if (threadIdx.x < SB) biases[at][threadIdx.x] = bias_reg;
    };
    fetch(first);
    put(0);
    __syncthreads();
    int at = 0;
    for (int64_t v0 = first; v0 < end; v0 += SB, at ^= 1) {
        const bool more = v0 + SB < end;
        if (more) fetch(v0 + SB);
        if (active) {
            const bool tail = v0 + SB > end;
#pragma unroll 1
            for (int sub = 0; sub < SB / 32; ++sub) {
                const char* rows = tiles[at] + sub * 32 * W::ROWB;
                if (BIAS || tail) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 c = *reinterpret_cast<const f32x4*>(&biases[at][sub * 32 + 8 * q + 4 * half]);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i) me.s[b][4 * q + i] = c[i];
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < NB; ++b) me.s[b] = f32x16{};
                }
                me.logits(rows);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int here = y[b] - (int)(v0 + 32 * sub);               // the target's place in this block, if it is in it
                    if (__any((unsigned)here < 32u)) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (here == acc_row(r, half)) {
                                z_target[h0 + 32 * b + l31] = me.s[b][r];
                                me.s[b][r] = -INFINITY;
                            }
                    }
                    float top = me.s[b][0];
#pragma unroll
                    for (int r = 1; r < 16; ++r) top = fmaxf(top, me.s[b][r]);
                    if (__any(top > m[b] + lag<T>())) {
                        top = fmaxf(top, __shfl_xor(top, 32, 64));              // both halves of a column keep one reference
                        if (top > m[b] + lag<T>()) {
                            const float f = m[b] == -INFINITY ? 0.f : exp2_fast((m[b] - top) * LOG2E);
                            m[b] = top;
                            sum[b] *= f;
                            if constexpr (DX)
#pragma unroll
                                for (int d = 0; d < W::BLOCKS; ++d) o[b][d] *= f;
                        }
                    }
                    // nothing above -inf yet: any finite reference leaves the sum at 0
                    const float base = m[b] == -INFINITY ? 0.f : m[b];
                    if (BIAS) {                                                 // logits up to the type's lowest: their difference first
#pragma unroll
                        for (int r = 0; r < 16; ++r) me.s[b][r] = exp2_fast(fmaf(me.s[b][r] - base, LOG2E, e_shift<T>()));
                    } else {
                        const float shift = e_shift<T>() - base * LOG2E;
#pragma unroll
                        for (int r = 0; r < 16; ++r) me.s[b][r] = exp2_fast(fmaf(me.s[b][r], LOG2E, shift));
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[b] += me.s[b][r];
                }
                if constexpr (DX) me.weigh(rows, o);
            }
        }
        if (more) put(at ^ 1);
        __syncthreads();
    }
    if (!active) return;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t t = h0 + 32 * b + l31;
        const float total = sum[b] + __shfl_xor(sum[b], 32, 64);
        if (t >= p.T) continue;
        if (half == 0) part[split * p.T + t] = Running{m[b], total * exp2f(-e_shift<T>())};
        if constexpr (DX) {
            float* dst = dx_part + (split * p.T + t) * width_out;
#pragma unroll
            for (int d = 0; d < W::BLOCKS; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = 32 * d + 8 * q + 4 * half + i;
                        if (c < width_out) dst[c] = o[b][d][4 * q + i] * exp2f(-e_shift<T>());
                    }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// cols: dW and dbias
// ---------------------------------------------------------------------------------------------
// expo[t]: -lse_t log2(e) + log2(G_SCALE), -inf for rows that do not count; with a bias, whose logits may be the type's lowest, lse_t
// itself and +inf.  y[t]: the target, -1 for rows that do not count.  EACH: rows have weights gn[t]
template <typename T, int DP, int NB, bool BIAS, bool EACH>
__global__ __launch_bounds__(256) void narrow_cols_kernel(Problem p, int splits, int64_t rows_per_split, int width_out, const float* __restrict__ expo,
                                                          const int* __restrict__ y, const float* __restrict__ rest, const float* __restrict__ gn,
                                                          const float* __restrict__ scale, T* __restrict__ dw, T* __restrict__ db,
                                                          float* __restrict__ dw_part, float* __restrict__ db_part)
{
    constexpr int SB = stream_rows<T, DP>();
    typedef Tile<T, DP, SB> Streamed;
    typedef Wave<T, DP, NB> W;
    __shared__ __attribute__((aligned(16))) char tiles[2][Streamed::BYTES];
    __shared__ __attribute__((aligned(16))) float expos[2][SB];
    __shared__ __attribute__((aligned(16))) float gns[2][SB];
    __shared__ __attribute__((aligned(16))) int ys[2][SB];
    const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t split = blockIdx.x % splits, h0 = (blockIdx.x / splits * 4 + wave) * (32 * NB);
    const bool active = h0 < p.V;
    const int64_t first = split * rows_per_split, end = first + rows_per_split < p.T ? first + rows_per_split : p.T;

    W me;
    me.init((const T*)p.w, p.ldw, p.V, (int)p.D, h0);
    float bias[NB], sum[NB];
    f32x16 o[NB][W::BLOCKS];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t v = h0 + 32 * b + l31;
        bias[b] = BIAS && v < p.V ? (float)((const T*)p.bias)[v] : 0.f;
        sum[b] = 0.f;
#pragma unroll
        for (int d = 0; d < W::BLOCKS; ++d) o[b][d] = f32x16{};
    }

    Streamed st;
    float expo_reg = 0.f, gn_reg = 0.f;
    int y_reg = -1;
    auto fetch = [&](int64_t t0) {
        st.load((const T*)p.x, p.ldx, end, (int)p.D, t0, y);
        if (threadIdx.x < SB) {
            const int64_t t = t0 + threadIdx.x;
            expo_reg = t < end ? expo[t] : BIAS ? INFINITY : -INFINITY;
            y_reg = t < end ? y[t] : -1;
            if (EACH) gn_reg = t < end ? gn[t] : 0.f;
        }
    };
    auto put = [&](int at) {
        st.store(tiles[at]);
        if (threadIdx.x < SB) {
            expos[at][threadIdx.x] = expo_reg;
            ys[at][threadIdx.x] = y_reg;
            if (EACH) gns[at][threadIdx.x] = gn_reg;
        }
    };
    fetch(first);
    put(0);
    __syncthreads();
    int at = 0;
    for (int64_t t0 = first; t0 < end; t0 += SB, at ^= 1) {
        const bool more = t0 + SB < end;
        if (more) fetch(t0 + SB);
        if (active) {
#pragma unroll 1
            for (int sub = 0; sub < SB / 32; ++sub) {
                const char* rows = tiles[at] + sub * 32 * W::ROWB;
#pragma unroll
                for (int b = 0; b < NB; ++b) me.s[b] = f32x16{};
                me.logits(rows);
                // targets of these 32 rows that lie in this wave's part of the vocabulary
                const int64_t away = (int64_t)ys[at][sub * 32 + l31] - h0;
                const bool hit = __any(away >= 0 && away < 32 * NB);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 x4 = *reinterpret_cast<const f32x4*>(&expos[at][sub * 32 + 8 * q + 4 * half]);
                    f32x4 g4;
                    if (EACH) g4 = *reinterpret_cast<const f32x4*>(&gns[at][sub * 32 + 8 * q + 4 * half]);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float z = me.s[b][4 * q + i];
                            float e = BIAS ? exp2_fast(fmaf(z + bias[b] - x4[i], LOG2E, G_LOG2<T>)) : exp2_fast(fmaf(z, LOG2E, x4[i]));
                            if (EACH) e *= g4[i];
                            me.s[b][4 * q + i] = e;
                        }
                }
                if (hit) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int row = sub * 32 + acc_row(r, half);
                            if ((int64_t)ys[at][row] == h0 + 32 * b + l31) {
                                const float q = rest[t0 + row] * Traits<T>::G_SCALE;
                                me.s[b][r] = EACH ? -q * gns[at][row] : -q;
                            }
                        }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[b] += me.s[b][r];
                me.weigh(rows, o);
            }
        }
        if (more) put(at ^ 1);
        __syncthreads();
    }
    if (!active) return;
    const float f = splits == 1 ? *scale / Traits<T>::G_SCALE : 1.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t v = h0 + 32 * b + l31;
        const float total = (sum[b] + __shfl_xor(sum[b], 32, 64)) * f;
        if (v >= p.V) continue;
        if (half == 0) {
            if (splits == 1) {
                if (db) db[v] = (T)total;
            } else {
                db_part[split * p.V + v] = total;
            }
        }
#pragma unroll
        for (int d = 0; d < W::BLOCKS; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 32 * d + 8 * q + 4 * half + i;
                    if (c < width_out) {
                        if (splits == 1) {
                            if (dw) dw[v * width_out + c] = (T)(o[b][d][4 * q + i] * f);
                        } else {
                            dw_part[(split * p.V + v) * width_out + c] = o[b][d][4 * q + i];
                        }
                    }
                }
    }
}

// held rows per wave, in blocks of 32
template <typename T, int DP> constexpr int held_blocks() { return sizeof(T) == 2 && DP <= 128 ? 2 : 1; }

template <typename F> int with_width(int64_t D, int size, F&& fn)
{
    if (D <= 32) return fn(std::integral_constant<int, 32>());
    if (D <= 64) return fn(std::integral_constant<int, 64>());
    if (D <= 128 || size == 4) return fn(std::integral_constant<int, 128>());
    return fn(std::integral_constant<int, 256>());
}

template <typename F> int with_flag(bool v, F&& fn) { return v ? fn(std::true_type()) : fn(std::false_type()); }

}  // namespace

namespace xent {

bool narrow_fits(int dtype, int64_t D) { return D <= (dtype == RECO_DT_F32 ? 128 : 256); }

// Splits of the streamed rows: about two workgroups per compute unit, whole tiles each
static void split_plan(int64_t held_groups, int64_t streamed, int64_t tile, int64_t* splits, int64_t* per)
{
    const int64_t tiles = ceil_div64(streamed, tile);
    int64_t s = 512 / held_groups;
    s = s < 1 ? 1 : s > tiles ? tiles : s;
    *per = ceil_div64(tiles, s) * tile;
    *splits = ceil_div64(streamed, *per);
}

template <typename T, typename F> static int shape_of(int64_t D, F&& fn)
{
    return with_width(D, sizeof(T), [&](auto dp) -> int {
        constexpr int DP = decltype(dp)::value;
        return fn(dp, std::integral_constant<int, held_blocks<T, DP>()>(), (int64_t)stream_rows<T, DP>());
    });
}

NarrowPlan narrow_plan(int dtype, int64_t T, int64_t V, int64_t D)
{
    NarrowPlan n{};
    (void)reco_with_type(dtype, [&](auto z) -> int {
        return shape_of<decltype(z)>(D, [&](auto, auto nb, int64_t tile) -> int {
            const int64_t per = 128 * decltype(nb)::value;
            n.x_groups = ceil_div64(T, per);
            n.w_groups = ceil_div64(V, per);
            split_plan(n.x_groups, V, tile, &n.x_splits, &n.x_per);
            split_plan(n.w_groups, T, tile, &n.w_splits, &n.w_per);
            return RECO_OK;
        });
    });
    return n;
}

int narrow_rows(int dtype, const Problem& p, const NarrowPlan& n, int64_t width_out, Running* part, float* z_target, float* dx_part, hipStream_t s)
{
    return reco_with_type(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        return shape_of<T>(p.D, [&](auto dp, auto nb, int64_t) -> int {
            return with_flag(p.bias != nullptr, [&](auto bias) -> int {
                return with_flag(dx_part != nullptr, [&](auto dx) -> int {
                    hipLaunchKernelGGL((narrow_rows_kernel<T, decltype(dp)::value, decltype(nb)::value, decltype(bias)::value, decltype(dx)::value>),
                                       dim3((unsigned)(n.x_groups * n.x_splits)), dim3(256), 0, s, p, (int)n.x_splits, n.x_per, (int)width_out, part, z_target,
                                       dx_part);
                    RECO_CHECK_LAUNCH();
                    return RECO_OK;
                });
            });
        });
    });
}

int narrow_cols(int dtype, const Problem& p, const NarrowPlan& n, int64_t width_out, const float* expo, const int* y, const float* rest, const float* gn,
                const float* scale, void* dw, void* db, float* dw_part, float* db_part, hipStream_t s)
{
    return reco_with_type(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        return shape_of<T>(p.D, [&](auto dp, auto nb, int64_t) -> int {
            return with_flag(p.bias != nullptr, [&](auto bias) -> int {
                return with_flag(gn != nullptr, [&](auto each) -> int {
                    hipLaunchKernelGGL((narrow_cols_kernel<T, decltype(dp)::value, decltype(nb)::value, decltype(bias)::value, decltype(each)::value>),
                                       dim3((unsigned)(n.w_groups * n.w_splits)), dim3(256), 0, s, p, (int)n.w_splits, n.w_per, (int)width_out, expo, y, rest, gn,
                                       scale, (T*)dw, (T*)db, dw_part, db_part);
                    RECO_CHECK_LAUNCH();
                    return RECO_OK;
                });
            });
        });
    });
}

}  // namespace xent

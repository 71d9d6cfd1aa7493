// K-g: what the forms of the catalogue cross entropy share (internal).
#pragma once
#include "types16.h"

#include <type_traits>

namespace xent {

constexpr float LOG2E = 1.44269504088896340736f;

template <typename T> struct Traits;
template <> struct Traits<float> {
    static constexpr int VEC = 4, KSTEP = 8, BK = 32;
    static constexpr float G_SCALE = 1.f;
    typedef f32x4 frag;
};
template <> struct Traits<__bf16> {
    static constexpr int VEC = 8, KSTEP = 16, BK = 64;
    static constexpr float G_SCALE = 1.f;
    typedef bf16x8 frag;
};
template <> struct Traits<_Float16> {
    static constexpr int VEC = 8, KSTEP = 16, BK = 64;
    static constexpr float G_SCALE = 16384.f;
    typedef f16x8 frag;
};

// acc[m, n] += sum over KSTEP k of a[m, k] b[n, k].  Lane l holds m (n) = l % 32; its k are 8 (l / 32) + 0 .. 7 of 16, in 32 bits
// 4 (l / 32) + 0 .. 3 of 8 -- the order of k is free as long as both operands have the same.  The result: n = l % 32, m of
// register r is 8 (r / 4) + 4 (l / 32) + r % 4.
__device__ __forceinline__ void mma(f32x16& acc, const f32x4& a, const f32x4& b)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const bf16x8& a, const bf16x8& b) { acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void mma(f32x16& acc, const f16x8& a, const f16x8& b) { acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0); }

struct Problem {
    int64_t T, V, D;            // D: values per row as read (whole VEC groups, zeros behind the caller's width)
    int64_t ldx, ldw;
    const void* x;
    const void* w;
    const void* bias;           // nullable
    const int64_t* target;
    int64_t ignore;
};

__device__ __forceinline__ int64_t clamp_target(int64_t y, int64_t V) { return y < 0 ? 0 : y >= V ? V - 1 : y; }

// (m, s): running maximum and sum of exp(z - m) of the logits that are not the target's.  A lane adds the terms of a block one after the
// other and the blocks' sums as a Sum: hundreds of thousands of equal terms, as of items that have no vector yet, round the same way each
// time (16384 x 600,007 x 24: a loss 2e-4 off), and dbias has thousands of small terms of one sign before the targets' of the other (11127 x
// 43,808 x 32: 7e-6 off, now 4e-8).
struct Running { float m, s; };

__device__ __forceinline__ Running joined(Running a, Running b)
{
    Running r;
    r.m = fmaxf(a.m, b.m);
    const float base = r.m == -INFINITY ? 0.f : r.m;            // nothing but -inf so far: the sum stays 0
    r.s = a.s * exp2f((a.m - base) * LOG2E) + b.s * exp2f((b.m - base) * LOG2E);
    return r;
}

__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// The form for narrow rows (xent_narrow.h).  x: groups of held rows, times splits of `per` vocabulary rows.  w: groups of held
// vocabulary rows, times tiles of x rows, in shares of consecutive (group, tile) units; shared: some group has parts in several.
struct NarrowPlan {
    int64_t x_waves, x_groups, x_splits, x_per, w_groups, w_tiles, w_share, w_shares;
    bool w_shared;
};
template <typename T> NarrowPlan narrow_plan_of(int64_t T_rows, int64_t V, int64_t D, bool dx);
template <typename T> int narrow_rows_of(const Problem& p, const NarrowPlan& n, int64_t width_out, Running* part, float* z_target, float* dx_part, hipStream_t s);
template <typename T>
int narrow_cols_of(const Problem& p, const NarrowPlan& n, int64_t width_out, const float* expo, const int* y, const float* rest, const float* gn,
                   const float* scale, void* dw, void* db, float* dw_part, float* db_part, hipStream_t s);

// widths of the narrow form: what fits the registers of a wave beside its sums
inline bool narrow_fits(int dtype, int64_t D) { return D <= (dtype == RECO_DT_F32 ? 128 : 256); }

}  // namespace xent

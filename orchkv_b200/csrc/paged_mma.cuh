// paged_mma.cuh — warp-level matrix products and asynchronous row loads for
// the kernels with few query rows (paged_rows.cu).
#pragma once

#include <type_traits>

#include "paged_split.cuh"

namespace okv {

__device__ __forceinline__ uint32_t smem_addr(const void *p)
{
    return (uint32_t)__cvta_generic_to_shared(p);
}
// 16 bytes to shared memory, zeros when !ok (nothing is read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool ok)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0));
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t *r)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t *r)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums
template <class T> __device__ __forceinline__ void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}
// 2^x by the special function unit (relative error under 2^-22)
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// Log2 of what the weights of the second product are multiplied with.  They
// are rounded to the pages' type, half a step each; of fp16 that holds down to
// 2^-14 only, so the largest weight (2^grow times the reference) is 2^15
// there: weights down to 2^(grow - 29) of the largest keep their 11 bits, and
// smaller ones are off by 2^(grow - 40) of it at most.  The maximum and the sum
// that go with the weights are taken with it, so results do not see it.
template <class T> __host__ __device__ constexpr float weight_bias(float grow)
{
    return std::is_same<T, __half>::value ? 15.f - grow : 0.f;
}

// Whether 16-bit values are all finite, a pair at a time: x * 0 is 0 for a finite
// x and NaN for the others, and stays NaN in a sum.
template <class T> struct Finite;
template <> struct Finite<__nv_bfloat16> {
    __nv_bfloat162 a = __floats2bfloat162_rn(0.f, 0.f);
    __device__ __forceinline__ void see(uint32_t w)
    {
        a = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&w), __floats2bfloat162_rn(0.f, 0.f), a);
    }
    __device__ __forceinline__ bool none() const { return __low2float(a) == 0.f && __high2float(a) == 0.f; }
};
template <> struct Finite<__half> {
    __half2 a = __floats2half2_rn(0.f, 0.f);
    __device__ __forceinline__ void see(uint32_t w)
    {
        a = __hfma2(*reinterpret_cast<__half2 *>(&w), __floats2half2_rn(0.f, 0.f), a);
    }
    __device__ __forceinline__ bool none() const { return __low2float(a) == 0.f && __high2float(a) == 0.f; }
};
template <class T> __device__ __forceinline__ bool infinite(uint32_t w, int half)
{
    const uint32_t m = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    return ((half ? w >> 16 : w) & m) == m;
}

// Offset of 16-byte column c of row r in a tile of rows of DP elements: the
// column is exchanged within its row so that 8 rows of one column fall on
// different banks.
template <int DP> __device__ __forceinline__ uint32_t swz(uint32_t r, uint32_t c)
{
    return r * (DP * 2) + ((c ^ (r & 7)) << 4);
}

// Query rows of a unit as A fragments: rows lane/4 and lane/4 + 8.
template <class T, int DP>
__device__ __forceinline__ void load_q_frag(const RowsDev &q, const RowInfo &r0, const RowInfo &r1,
                                            uint32_t D, uint32_t (*qf)[4])
{
    const uint32_t lane = threadIdx.x & 31, c = (lane & 3) * 2;
    const char *p0 = q.p + (long long)r0.row * q.row_b + (long long)r0.head * q.head_b;
    const char *p1 = q.p + (long long)r1.row * q.row_b + (long long)r1.head * q.head_b;
#pragma unroll
    for (int k = 0; k < DP / 16; k++) {
        const uint32_t d = k * 16 + c;
        qf[k][0] = r0.row >= 0 && d < D ? *(const uint32_t *)(p0 + d * 2) : 0;
        qf[k][1] = r1.row >= 0 && d < D ? *(const uint32_t *)(p1 + d * 2) : 0;
        qf[k][2] = r0.row >= 0 && d + 8 < D ? *(const uint32_t *)(p0 + (d + 8) * 2) : 0;
        qf[k][3] = r1.row >= 0 && d + 8 < D ? *(const uint32_t *)(p1 + (d + 8) * 2) : 0;
    }
}

// One 16-key tile of rows from the pages to shared memory by one warp.  `off`
// (lanes 0..15): byte offset of key `lane`'s row, negative if it has none.
template <int DP>
__device__ __forceinline__ void load_rows16(uint32_t dst, const char *base, long long off, uint32_t D)
{
    const uint32_t lane = threadIdx.x & 31;
    constexpr int LPR = DP / 8;          // lanes of a row
    constexpr int RPI = 32 / LPR;        // rows an instruction
#pragma unroll
    for (int j = 0; j < 16 / RPI; j++) {
        const uint32_t r = j * RPI + lane / LPR, c = lane % LPR;
        const long long o = __shfl_sync(0xFFFFFFFFu, off, r);
        const bool ok = o >= 0 && c * 8 < D;
        cp16(dst + swz<DP>(r, c), base + (ok ? o + c * 16 : 0), ok);
    }
}

// The same when the 16 rows lie in one page, tok_b apart from `off` on (the
// whole warp's; negative: no page); rows outside `have` become zeros.
template <int DP>
__device__ __forceinline__ void load_run16(uint32_t dst, const char *base, long long off, long long tok_b,
                                           uint32_t have, uint32_t D)
{
    const uint32_t lane = threadIdx.x & 31;
    constexpr int LPR = DP / 8, RPI = 32 / LPR;
    const uint32_t r0 = lane / LPR, c = lane % LPR;
    const bool col = c * 8 < D;
    const char *src = base + (have ? off : 0) + c * 16 + r0 * tok_b;
#pragma unroll
    for (int j = 0; j < 16 / RPI; j++) {
        const uint32_t r = j * RPI + r0;
        const bool ok = col && (have >> r & 1);
        cp16(dst + swz<DP>(r, c), ok ? src : base, ok);
        src += RPI * tok_b;
    }
}
// Bits [lo, hi] of 16.
__device__ __forceinline__ uint32_t bits16(int lo, int hi)
{
    lo = lo < 0 ? 0 : lo;
    hi = hi > 15 ? 15 : hi;
    return hi < lo ? 0u : ((2u << hi) - 1) & ~((1u << lo) - 1);
}

// s[2][4] = scores of 16 keys (tiles of 8) against the 16 rows.
template <class T, int DP>
__device__ __forceinline__ void scores16(uint32_t kt, const uint32_t (*qf)[4], float (*s)[4])
{
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; j++) s[0][j] = s[1][j] = 0.f;
    // matrices: keys 0-7 | 0-7 | 8-15 | 8-15, columns lo | hi | lo | hi
    const uint32_t r = (lane & 7) + ((lane >> 4) << 3), cx = (lane >> 3) & 1;
#pragma unroll
    for (int k = 0; k < DP / 16; k++) {
        uint32_t f[4];
        ldsm4(kt + swz<DP>(r, 2 * k + cx), f);
        mma16816<T>(s[0], qf[k], f[0], f[1]);
        mma16816<T>(s[1], qf[k], f[2], f[3]);
    }
}

}  // namespace okv

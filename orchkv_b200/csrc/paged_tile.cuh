// paged_tile.cuh — tensor-core and copy-engine primitives of the tile kernels:
// mbarriers with bounded waits, TMA page loads, tcgen05 products and their
// descriptors.
#pragma once

#include <cuda.h>

#include "paged_mma.cuh"

namespace okv {

// ---- mbarriers -------------------------------------------------------------------

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\n"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                 "selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long global_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
constexpr unsigned long long kWaitNs = 2000000000ull;

// Waits for the phase; gives up after kWaitNs, or when another role has: then
// *dead is set and every role leaves its loop.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *dead)
{
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = global_ns();
    for (;;) {
#pragma unroll 1
        for (int k = 0; k < 64; k++)
            if (mbar_try(bar, parity)) return true;
        if (*dead || global_ns() - t0 > kWaitNs) {
            *dead = 1;
            return false;
        }
    }
}
// The same for a role that is leaving: what is still in flight, at most 0.1 s.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity)
{
    const unsigned long long t0 = global_ns();
    while (!mbar_try(bar, parity) && global_ns() - t0 < 100000000ull) {}
}

// ---- TMA ---------------------------------------------------------------------------

__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w,
                                     uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void fence_async()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- tcgen05 -------------------------------------------------------------------------

__device__ __forceinline__ void tm_alloc(uint32_t where, uint32_t cols)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tm_free(uint32_t base, uint32_t cols)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 columns of this thread's lane
#define OKV_R32(M) M(0) M(1) M(2) M(3) M(4) M(5) M(6) M(7) M(8) M(9) M(10) M(11) M(12) M(13) M(14) M(15) \
    M(16) M(17) M(18) M(19) M(20) M(21) M(22) M(23) M(24) M(25) M(26) M(27) M(28) M(29) M(30) M(31)

__device__ __forceinline__ void tm_ld32(uint32_t a, float *v)
{
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
          "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
}
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
          "r"(a)
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(a)
        : "memory");
}

// Shared-memory operand, 128-byte swizzle: start address and byte strides.  For
// an operand whose k runs along the 128-byte rows, 8-row groups are 1024 bytes
// apart; for one whose n runs along them, `lbo` is the distance of its
// 64-element column groups and 8-row (k) groups are 1024 bytes apart.  The low
// word varies (addresses stay below 2^18: no carry), the high one is kDescHi.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return addr >> 4 | (lbo >> 4) << 16; }
constexpr uint32_t kDescHi = 1024 >> 4 | 1u << 14 | 2u << 29;
// kind::f16, fp32 sums: fmt 0 fp16, 1 bf16 (both operands); b_mn: B's n runs
// along its rows.
__host__ __device__ constexpr uint32_t inst_desc(uint32_t fmt, uint32_t M, uint32_t N, uint32_t b_mn)
{
    return 1u << 4 | fmt << 7 | fmt << 10 | b_mn << 16 | (N >> 3) << 17 | (M >> 4) << 24;
}
// One thread of a warp issues; every operand is the same for the whole warp.
// A single thread's instructions are what limits the rate of products, so the
// descriptors are one 32-bit add each.
__device__ __forceinline__ bool elect_one()
{
    uint32_t y;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(y));
    return y != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool add)
{
    asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.u32 p, %4, 0;\n"
                 "mov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(id), "r"((uint32_t)add), "n"(kDescHi) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool add)
{
    asm volatile("{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.u32 p, %4, 0;\n"
                 "mov.b64 b, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(id), "r"((uint32_t)add), "n"(kDescHi) : "memory");
}

// ---- pairs of fp32 ---------------------------------------------------------------------

__device__ __forceinline__ ull f2(float x, float y)
{
    ull r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unf2(ull v, float *x, float *y)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(*x), "=f"(*y) : "l"(v));
}
__device__ __forceinline__ ull fma2(ull a, ull b, ull c)
{
    ull r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ ull add2(ull a, ull b)
{
    ull r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ ull mul2(ull a, ull b)
{
    ull r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b)
{
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Two powers of two without the special function unit: x = n + f with |f| <=
// 1/2 (adding 1.5 * 2^23 rounds x to n and leaves n in the low bits), 2^f by a
// polynomial, times 2^n.  Arguments are held to [-127, 128], where the bits of
// 2^n are those of 0 and of infinity; NaN stays NaN.  The polynomial of degree
// 5 minimises the largest relative error over [-1/2, 1/2] (Remez exchange in
// double, coefficients rounded): 2.1e-7 when evaluated in fp32, 5e-8 on
// average, about what a sum of many is off by.
__device__ __forceinline__ ull ex2_poly(ull x)
{
    float a, b;
    unf2(x, &a, &b);
    x = f2(min_nan(max_nan(a, -127.f), 128.f), min_nan(max_nan(b, -127.f), 128.f));
    const ull t = add2(x, f2(12582912.f, 12582912.f));
    const ull f = fma2(add2(t, f2(-12582912.f, -12582912.f)), f2(-1.f, -1.f), x);
    constexpr float c[6] = {0x1.000002p+0f, 0x1.62e428p-1f, 0x1.ebf918p-3f, 0x1.c6b6e4p-5f, 0x1.3d0c52p-7f,
                            0x1.5c08e6p-10f};
    ull p = f2(c[5], c[5]);
#pragma unroll
    for (int k = 4; k >= 0; k--) p = fma2(p, f, f2(c[k], c[k]));
    unf2(t, &a, &b);
    return mul2(p, f2(__uint_as_float((__float_as_uint(a) << 23) + 0x3F800000u),
                      __uint_as_float((__float_as_uint(b) << 23) + 0x3F800000u)));
}

__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A tensor map over query rows: (element, head, row), boxes of 64 elements by
// the G heads of a KV head by `toks` rows.
bool rows_map(CUtensorMap *m, const RowsDev &q, uint32_t D, uint32_t Hq, uint32_t rows, uint32_t G,
              uint32_t toks, int dtype);
// A tensor map over pages: (element, token, head, page), boxes of 64 elements
// by min(page, 128) tokens, 128-byte swizzle.  False if the driver has none.
bool page_map(CUtensorMap *m, const PagesDev &p, const char *base, int dtype);
// Whether pages can be loaded so: a page is a whole number of 128-key tiles
// or divides one into boxes of whole 8-row groups.
inline bool pages_tile(const PagesDev &p)
{
    const uint32_t t = p.bs.d;
    return p.D <= 128 && (t % 128 == 0 || t == 8 || t == 16 || t == 32 || t == 64);
}

// The units of one CTA's share, in order; every role walks them alike.
struct Walk {
    const Geo &g;
    const BatchDev &b;
    uint32_t bs;
    Pos at, end;
    // the unit at hand: key tiles [first + t0, first + t1) of nt
    SeqDev s;
    uint32_t RT, first, nt, t0, t1;
    bool stop;

    // moves `at` to a unit with work; false at the end
    __device__ bool settle()
    {
        while (at.i < b.n) {
            s = load_seq(b, bs, at.i);
            RT = row_tiles(g, s);
            if (RT == 0) { at = Pos{at.i + 1, 0, 0, 0}; continue; }
            if (at.i > end.i) return false;            // the end was a sequence without units
            stop = same_unit(at, end);
            key_tiles(g, s, at.rt, &first, &nt);
            t0 = at.t;
            t1 = stop ? end.t : nt;
            if (t0 < t1) return true;
            if (stop) return false;
            advance();
        }
        return false;
    }
    __device__ void advance()
    {
        at.t = 0;
        if (++at.rt == RT) {
            at.rt = 0;
            if (++at.h == g.H) { at.h = 0; at.i++; }
        }
    }
    __device__ bool next()
    {
        if (stop) return false;
        advance();
        return settle();
    }
    __device__ uint32_t live() const { return min(g.R, (uint32_t)s.m * g.G - at.rt * g.R); }
};

}  // namespace okv

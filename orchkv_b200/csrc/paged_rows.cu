// paged_rows.cu — attention over pages and block masses for few query rows a
// sequence (decode), and for every shape the tile kernels do not take.
//
// A decode step reads each cached key and value once and does 4 G products
// with it, so HBM bounds it; what the kernel has to do is keep enough loads in
// flight on every SM.  A CTA is 4 warps that never wait for each other inside
// a unit: each takes every fourth group of 16 keys, brings its rows of K and V
// by 16-byte asynchronous copies through its own ring of groups (an SM holds 2
// CTAs x 4 warps x 2 groups x 8 KB of loads in flight, more than the 45 KB
// that bandwidth x latency asks for), and runs its own online softmax in
// registers.  The 16-row matrix instruction holds all G query
// heads of a KV head (rows past G idle: the products are free under the
// loads).  The warps' parts are joined in shared memory once a unit, the
// CTAs' as paged_split.cuh describes.  Places outside the range of every row,
// past the length or in no page are filled with zeros and never read.
//
// 32 requests x 1 token over 8192, 28/4 heads of 128, bf16: 96 to 101 us over the
// devices measured, 0.81 to 0.85 of the measured copy rate, 6 us of them the join;
// 61 requests over 1 to 16000 tokens, window 6000: 208 to 215 us, 0.9.  Chunks
// that come here reread K and V for every 16 rows: 1024 tokens over 7168, 32/8
// heads, take 865 us at 128 elements and 24-token pages, 2.60 ms at 256 elements
// (their products: 78 and 156 us).
#include <algorithm>

#include "kernels.h"
#include "paged_mma.cuh"

namespace okv {
namespace {

constexpr int kW = 4;
constexpr uint32_t kR = 16, kKeys = 16 * kW;

template <int DP> struct RowsCfg {
    static constexpr int stages = DP == 256 ? 3 : DP == 128 ? 3 : 5;
    static constexpr int ctas = DP == 256 ? 1 : 2;     // resident an SM
    static constexpr uint32_t tile = 16 * DP * 2;      // bytes of 16 rows
    static constexpr size_t ring = (size_t)stages * 2 * tile;
    // a warp's joined part: 16 x DP fp32, in its ring
    static_assert(ring >= 16 * DP * 4, "the part does not fit the ring");
    static constexpr size_t smem = kW * ring;
};

// One value of another CTA of the cluster's shared memory, at the address that
// `p` has in this one.
__device__ __forceinline__ float4 peer4(const float *p, uint32_t rank)
{
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ float peer1(const float *p, uint32_t rank)
{
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void cluster_meet()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Before a product with 16 keys that only some rows attend to: a weight of 0
// times an infinite or NaN value would reach the rows that do not, so such
// values become 0 and the results of the rows that do attend NaN.  Only groups
// on a chunk's diagonal or a window's edge come here (1.5 % of a decode step
// that never does, by its registers).
template <class T, int DP>
__device__ __forceinline__ void drop_infinite(uint32_t vt, const RowInfo &r0, const RowInfo &r1, int k0,
                                              uint32_t have, float (*acc)[4])
{
    const uint32_t lane = threadIdx.x & 31;
    Finite<T> fin;
#pragma unroll
    for (int k = 0; k < DP / 16; k++) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vt + (k * 32 + lane) * 16));
#pragma unroll
        for (int j = 0; j < 4; j++) fin.see(w[j]);
    }
    if (__all_sync(0xFFFFFFFFu, fin.none())) return;
#pragma unroll
    for (int n = 0; n < DP / 8; n++)
#pragma unroll 1
        for (uint32_t c = 0; c < 16; c++) {
            const int key = k0 + (int)c;
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vt + swz<DP>(c, n) + (lane & 3) * 4));
            if (!(have >> c & 1)) continue;
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (infinite<T>(w, j)) {
                    if (key <= r0.hi && key >= r0.lo) acc[n][j] = NAN;
                    if (key <= r1.hi && key >= r1.lo) acc[n][2 + j] = NAN;
                }
        }
    __syncwarp();
#pragma unroll 1
    for (uint32_t e = lane; e < 16 * DP / 2; e += 32) {
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vt + e * 4));
        if (infinite<T>(w, 0)) w &= 0xFFFF0000u;
        if (infinite<T>(w, 1)) w &= 0xFFFFu;
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(vt + e * 4), "r"(w) : "memory");
    }
    __syncwarp();
}

// CL: a unit is one cluster of `split` CTAs, which share its keys equally and
// join their parts over each other's shared memory; else the CTAs share the
// whole call's work and join_kernel adds cut units.
// AL: pages of whole 16-key groups, so a group's rows lie side by side.
template <class T, int DP, bool CL, bool AL>
__global__ void __launch_bounds__(kW * 32, RowsCfg<DP>::ctas)
attend_rows_kernel(Geo g, PagesDev p, BatchDev b, AttendDev a, SplitDev sp, uint32_t split, uint32_t tiles_max)
{
    using Cfg = RowsCfg<DP>;
    constexpr int ST = Cfg::stages;
    extern __shared__ __align__(128) char smem[];
    __shared__ SplitShared sh;
    __shared__ uint32_t have_s[kW][ST];                // keys of a group that lie in a page
    __shared__ float m_s[kW][kR], l_s[kW][kR];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5, D = p.D;
    char *ring = smem + wid * Cfg::ring;
    const uint32_t ring_a = smem_addr(ring);

    Pos at, end;
    uint32_t rank = 0;
    if (CL) {
        const uint32_t u = blockIdx.x / split, ih = u / tiles_max;
        rank = blockIdx.x - u * split;
        at = Pos{ih / g.H, ih % g.H, u - ih * tiles_max, 0};
        end = Pos{b.n, 0, 0, 0};
        if (at.rt >= row_tiles(g, load_seq(b, p.bs.d, at.i))) return;   // the whole cluster
    } else {
        ull W;
        find_share<kW * 32>(g, b, p.bs.d, blockIdx.x, sp.ctas, &sh, &at, &end, &W);
        // the join behind this launch may be scheduled now; it waits for our end
        cudaTriggerProgrammaticLaunchCompletion();
        if (W == 0) return;
    }
    while (at.i < b.n) {
        const SeqDev s = load_seq(b, p.bs.d, at.i);
        const uint32_t RT = row_tiles(g, s);
        if (RT == 0) { at = Pos{at.i + 1, 0, 0, 0}; continue; }
        if (at.i > end.i) break;                           // the end was a sequence without units
        const bool stop = same_unit(at, end);
        if (stop && end.t == 0) break;
        uint32_t first, nt;
        key_tiles(g, s, at.rt, &first, &nt);
        const uint32_t t0 = CL ? rank * nt / split : at.t;
        const uint32_t t1 = CL ? (rank + 1) * nt / split : stop ? end.t : nt;
        if (CL || t0 < t1) {
            const uint32_t rows = (uint32_t)s.m * g.G, pr0 = at.rt * kR;
            const RowInfo r0 = row_info(g, s, at.h, pr0 + (lane >> 2));
            const RowInfo r1 = row_info(g, s, at.h, pr0 + (lane >> 2) + 8);
            // keys any row attends to, and keys that every row does
            const RowInfo rf = row_info(g, s, at.h, pr0);
            const RowInfo rl = row_info(g, s, at.h, min(pr0 + kR, rows) - 1);
            const int any_lo = rf.lo, any_hi = rl.hi, all_lo = rl.lo, all_hi = rf.hi;

            uint32_t qf[DP / 16][4];
            load_q_frag<T, DP>(a.q, r0, r1, D, qf);

            // page of this lane's key (lanes 0..15; AL: of the group) of group t,
            // asked for one group ahead
            auto key_of = [&](uint32_t t) {
                return (int)((first + t) * kKeys + wid * 16 + (AL ? 0 : (lane & 15)));
            };
            auto page = [&](uint32_t t) {
                const int key = key_of(t);
                if (t >= t1 || key + (AL ? 15 : 0) < any_lo || key > any_hi) return -1;
                return page_of(b, p.n_pages, at.i, at.h, (uint32_t)key / p.bs);
            };
            auto issue = [&](uint32_t t, int pg, uint32_t st) {
                if (t < t1) {
                    const int key = key_of(t);
                    long long off = -1;
                    if (pg >= 0)
                        off = pg * p.page_b + at.h * p.head_b +
                              (long long)((uint32_t)key - (uint32_t)key / p.bs * p.bs.d) * p.tok_b;
                    const uint32_t have = AL ? (pg >= 0 ? bits16(any_lo - key, any_hi - key) : 0u)
                                             : __ballot_sync(0xFFFFFFFFu, pg >= 0) & 0xFFFFu;
                    if (lane == 0) have_s[wid][st] = have;
                    const uint32_t kt = ring_a + st * 2 * Cfg::tile;
                    if (AL) {
                        load_run16<DP>(kt, p.k, off, p.tok_b, have, D);
                        load_run16<DP>(kt + Cfg::tile, p.v, off, p.tok_b, have, D);
                    } else {
                        load_rows16<DP>(kt, p.k, off, D);
                        load_rows16<DP>(kt + Cfg::tile, p.v, off, D);
                    }
                }
                cp_commit();
            };

            float acc[DP / 8][4];
#pragma unroll
            for (int n = 0; n < DP / 8; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[n][j] = 0.f;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

            int pg = page(t0);
#pragma unroll
            for (int k = 0; k < ST - 1; k++) {
                issue(t0 + k, pg, k);
                pg = page(t0 + k + 1);
            }
            uint32_t st = 0, st_in = ST - 1;
            for (uint32_t t = t0; t < t1; t++) {
                issue(t + ST - 1, pg, st_in);
                pg = page(t + ST);
                st_in = st_in + 1 == ST ? 0 : st_in + 1;
                cp_wait<ST - 1>();
                __syncwarp();
                const uint32_t have = have_s[wid][st];
                const uint32_t kt = ring_a + st * 2 * Cfg::tile, vt = kt + Cfg::tile;
                st = st + 1 == ST ? 0 : st + 1;
                if (have) {
                    const int k0 = (int)((first + t) * kKeys + wid * 16);
                    float sc[2][4];
                    scores16<T, DP>(kt, qf, sc);
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) sc[n][j] *= a.sl2;
                    if (have != 0xFFFFu || k0 < all_lo || k0 + 15 > all_hi) {
#pragma unroll
                        for (int n = 0; n < 2; n++)
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const uint32_t c = n * 8 + (lane & 3) * 2 + (j & 1);
                                const int key = k0 + (int)c;
                                const RowInfo &r = j < 2 ? r0 : r1;
                                if (!(have >> c & 1) || key > r.hi || key < r.lo) sc[n][j] = -INFINITY;
                            }
                    }
                    uint32_t pf[4];
                    float f[2];
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        float mx = fmaxf(fmaxf(sc[0][2 * x], sc[0][2 * x + 1]),
                                         fmaxf(sc[1][2 * x], sc[1][2 * x + 1]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                        mx = fmaxf(mx - weight_bias<T>(0.f), m[x]);
                        const float ms = mx == -INFINITY ? 0.f : mx;
                        f[x] = ex2(m[x] - ms);
                        m[x] = mx;
                        float q[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) q[j] = ex2(sc[j >> 1][2 * x + (j & 1)] - ms);
                        l[x] = l[x] * f[x] + ((q[0] + q[1]) + (q[2] + q[3]));
                        // the weights are rounded to the pages' type: half a
                        // step each, as the result's own (see weight_bias)
                        pf[x] = pack2<T>(q[0], q[1]);
                        pf[2 + x] = pack2<T>(q[2], q[3]);
                    }
                    if (__any_sync(0xFFFFFFFFu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                        for (int n = 0; n < DP / 8; n++) {
                            acc[n][0] *= f[0];
                            acc[n][1] *= f[0];
                            acc[n][2] *= f[1];
                            acc[n][3] *= f[1];
                        }
                    }
                    if (k0 < all_lo || k0 + 15 > all_hi) drop_infinite<T, DP>(vt, r0, r1, k0, have, acc);
                    // matrices: keys lo | hi | lo | hi, columns 0-7 | 0-7 | 8-15 | 8-15
                    const uint32_t r = lane & 15, cx = lane >> 4;
#pragma unroll
                    for (int n = 0; n < DP / 16; n++) {
                        uint32_t vf[4];
                        ldsm4t(vt + swz<DP>(r, 2 * n + cx), vf);
                        mma16816<T>(acc[2 * n], pf, vf[0], vf[1]);
                        mma16816<T>(acc[2 * n + 1], pf, vf[2], vf[3]);
                    }
                }
                __syncwarp();
            }
            cp_wait<0>();

            // the warps' parts, then the rows
            float *part = (float *)ring;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                l[x] += __shfl_xor_sync(0xFFFFFFFFu, l[x], 1);
                l[x] += __shfl_xor_sync(0xFFFFFFFFu, l[x], 2);
                const uint32_t r = (lane >> 2) + 8 * x;
                if ((lane & 3) == 0) { m_s[wid][r] = m[x]; l_s[wid][r] = l[x]; }
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
                    *(float2 *)(part + r * DP + n * 8 + (lane & 3) * 2) =
                        make_float2(acc[n][2 * x], acc[n][2 * x + 1]);
            }
            __syncthreads();
            const bool whole = CL ? split == 1 : t0 == 0 && t1 == nt;
            // (a cluster's parts lie as a slot does)
            float *sl = CL ? (float *)(smem + Cfg::smem) : whole ? nullptr : slot_of(sp.ws, 2 * blockIdx.x + (t0 == 0 ? 1 : 0), kR, D);
            const uint32_t live = min(kR, rows - pr0), d8 = D / 8;
            for (uint32_t e = threadIdx.x; e < live * d8; e += kW * 32) {
                const uint32_t r = e / d8, d = (e - r * d8) * 8;
                float M = -INFINITY;
#pragma unroll
                for (int k = 0; k < kW; k++) M = fmaxf(M, m_s[k][r]);
                const float Ms = M == -INFINITY ? 0.f : M;
                float L = 0.f, o[8] = {};
#pragma unroll
                for (int k = 0; k < kW; k++) {
                    const float w = ex2(m_s[k][r] - Ms);
                    L += w * l_s[k][r];
                    const float *x = (const float *)(smem + k * Cfg::ring) + r * DP + d;
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] += w * x[j];
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 8; j++) sl[2 * kR + r * D + d + j] = o[j];
                    if (d == 0) { sl[r] = M; sl[kR + r] = L; }
                } else {
                    const RowInfo ri = row_info(g, s, at.h, pr0 + r);
                    const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] *= inv;
                    *(uint4 *)(a.out.p + (long long)ri.row * a.out.row_b +
                               (long long)ri.head * a.out.head_b + d * 2) = Vec<T>::down(o);
                    if (a.lse && d == 0)
                        a.lse[(size_t)ri.row * a.Hq + ri.head] =
                            L > 0.f ? (Ms + log2f(L)) * kLn2 : L == 0.f ? -INFINITY : L;
                }
            }
            if (CL) {
                if (!whole) {
                    cluster_meet();
                    const uint32_t d4 = D / 4;
                    for (uint32_t e = rank * (kW * 32) + threadIdx.x; e < live * d4; e += split * (kW * 32)) {
                        const uint32_t r = e / d4, d = (e - r * d4) * 4;
                        float M = -INFINITY, L = 0.f, o[4] = {};
#pragma unroll 1
                        for (uint32_t k0 = 0; k0 < split; k0 += 4) {
                            float m[4], l[4];
                            float4 v[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint32_t c = min(k0 + k, split - 1);
                                m[k] = peer1(sl + r, c);
                                l[k] = peer1(sl + kR + r, c);
                                v[k] = peer4(sl + 2 * kR + r * D + d, c);
                            }
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                if (k0 + k >= split) break;
                                const float nm = fmaxf(M, m[k]), ms = nm == -INFINITY ? 0.f : nm;
                                const float f = ex2(M - ms), w = ex2(m[k] - ms);
                                M = nm;
                                L = L * f + w * l[k];
                                o[0] = o[0] * f + w * v[k].x;
                                o[1] = o[1] * f + w * v[k].y;
                                o[2] = o[2] * f + w * v[k].z;
                                o[3] = o[3] * f + w * v[k].w;
                            }
                        }
                        const RowInfo ri = row_info(g, s, at.h, pr0 + r);
                        const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
                        *(uint2 *)(a.out.p + (long long)ri.row * a.out.row_b + (long long)ri.head * a.out.head_b +
                                   d * 2) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv),
                                                       pack2<T>(o[2] * inv, o[3] * inv));
                        if (a.lse && d == 0)
                            a.lse[(size_t)ri.row * a.Hq + ri.head] =
                                L > 0.f ? ((M == -INFINITY ? 0.f : M) + log2f(L)) * kLn2
                                        : L == 0.f ? -INFINITY : L;
                    }
                    cluster_meet();                    // nobody leaves while its part is read
                }
                return;
            }
            __syncthreads();
        }
        if (stop) break;
        at.t = 0;
        if (++at.rt == RT) {
            at.rt = 0;
            if (++at.h == g.H) { at.h = 0; at.i++; }
        }
    }
}

// ---- masses ----------------------------------------------------------------------
//
// Only K is read.  A warp owns runs of whole blocks (an item: one block, or as
// many as fit 16 keys) and brings their keys 16 at a time through a ring; the
// column sums of exp(s - lse) over the 16 rows are three shuffles.  The masses
// of the run stay in shared memory over the row tiles, so each is written
// once, in one order of sums.  32 requests x 1 token over 8192, 28/4 heads: 46 to
// 51 us over the devices measured, 0.81 to 0.90 of the measured copy rate; a chunk
// of 1024 over 7168 of 256 elements, which the tile kernel does not take: 3.09 ms.
constexpr int kMassStages = 3;
constexpr uint32_t kMaxRun = 64;                       // blocks of a warp's run

// Pages of whole 16-key groups: a group lies in one block, so its 16 x 16
// weights add up to one number; a thread keeps its share of a block until the
// block ends.
template <class T, int DP>
__global__ void __launch_bounds__(kW * 32)
mass_runs_kernel(Geo g, PagesDev p, BatchDev b, MassDev a, uint32_t run, uint32_t groups)
{
    constexpr int ST = kMassStages;
    constexpr uint32_t tile = 16 * DP * 2;
    extern __shared__ __align__(128) char smem[];
    __shared__ float mass_s[kW][kMaxRun];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5, D = p.D;
    const uint32_t ring_a = smem_addr(smem + wid * ST * tile);
    const uint32_t x = blockIdx.x % groups, ih = blockIdx.x / groups;
    const uint32_t h = ih % p.H, i = ih / p.H;
    const SeqDev s = load_seq(b, p.bs.d, i);
    const uint32_t rows = (uint32_t)s.m * g.G;
    if ((rows <= g.min_rows && g.min_rows) || rows > g.max_rows) return;

    const uint32_t b0 = (x * kW + wid) * run;
    if (b0 >= b.width) return;
    const uint32_t n_blk = min(run, b.width - b0), per = p.bs.d / 16;    // groups of a block
    for (uint32_t k = lane; k < n_blk; k += 32) mass_s[wid][k] = 0.f;
    __syncwarp();
    const int key0 = (int)(b0 * p.bs.d);

    for (uint32_t rt = 0; rt * kR < rows; rt++) {
        const RowInfo r0 = row_info(g, s, h, rt * kR + (lane >> 2));
        const RowInfo r1 = row_info(g, s, h, rt * kR + (lane >> 2) + 8);
        const RowInfo rf = row_info(g, s, h, rt * kR);
        const RowInfo rl = row_info(g, s, h, min((rt + 1) * kR, rows) - 1);
        const int any_lo = rf.lo, any_hi = rl.hi, all_lo = rl.lo, all_hi = rf.hi;
        // the blocks of the run that hold a key of this row tile
        if (any_hi < key0 || any_lo >= key0 + (int)(n_blk * p.bs.d)) continue;
        const uint32_t first = any_lo > key0 ? (uint32_t)(any_lo - key0) / p.bs : 0;
        const uint32_t last = min((uint32_t)(any_hi - key0) / p.bs, n_blk - 1);

        uint32_t qf[DP / 16][4];
        load_q_frag<T, DP>(a.q, r0, r1, D, qf);
        // a row behind the last weighs nothing, whatever its zeros make of a key
        const bool on0 = r0.row >= 0, on1 = r1.row >= 0;
        float ls[2];
        ls[0] = on0 ? a.lse[(size_t)r0.row * a.Hq + r0.head] * kLog2e : 0.f;
        ls[1] = on1 ? a.lse[(size_t)r1.row * a.Hq + r1.head] * kLog2e : 0.f;

        // the next group to load (block, group in it) and to weigh; a lane
        // holds the pages of two blocks of the run (of at most 64)
        uint32_t lb = first, lg = 0, wb = first, wg = 0;
        auto page = [&](uint32_t blk) { return blk <= last ? page_of(b, p.n_pages, i, h, b0 + blk) : -1; };
        const int pa = page(first + lane), pb = page(first + 32 + lane);
        auto page_at = [&](uint32_t blk) {
            const uint32_t k = blk - first;
            const int x = __shfl_sync(0xFFFFFFFFu, pa, k & 31), y = __shfl_sync(0xFFFFFFFFu, pb, k & 31);
            return k < 32 ? x : y;
        };
        int pg = page_at(first);
        auto have_of = [&](uint32_t blk, uint32_t gr) {
            const int k = key0 + (int)(blk * p.bs.d + gr * 16);
            return bits16(any_lo - k, any_hi - k);
        };
        auto issue = [&](uint32_t st) {
            if (lb <= last) {
                const uint32_t have = pg >= 0 ? have_of(lb, lg) : 0;
                if (have)
                    load_run16<DP>(ring_a + st * tile, p.k,
                                   pg * p.page_b + h * p.head_b + (long long)(lg * 16) * p.tok_b, p.tok_b, have, D);
                if (++lg == per) {
                    lg = 0;
                    lb++;
                    pg = page_at(min(lb, last));
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int k = 0; k < ST - 1; k++) issue(k);
        uint32_t st = 0, st_in = ST - 1;
        int pw = page_at(first);                           // of the block being weighed
        float part = 0.f;
        while (wb <= last) {
            issue(st_in);
            st_in = st_in + 1 == ST ? 0 : st_in + 1;
            cp_wait<ST - 1>();
            __syncwarp();
            const uint32_t have = pw >= 0 ? have_of(wb, wg) : 0, kt = ring_a + st * tile;
            st = st + 1 == ST ? 0 : st + 1;
            if (have) {
                const int k0 = key0 + (int)(wb * p.bs.d + wg * 16);
                float sc[2][4];
                scores16<T, DP>(kt, qf, sc);
                if (have == 0xFFFFu && k0 >= all_lo && k0 + 15 <= all_hi) {
                    float e[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) e[j] = ex2(sc[j >> 2][j & 3] * a.sl2 - ls[j >> 1 & 1]);
                    const float w0 = on0 ? e[0] + e[1] : 0.f, w1 = on1 ? e[2] + e[3] : 0.f;
                    const float w2 = on0 ? e[4] + e[5] : 0.f, w3 = on1 ? e[6] + e[7] : 0.f;
                    part += (w0 + w1) + (w2 + w3);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t col = (j >> 2) * 8 + (lane & 3) * 2 + (j & 1);
                        const RowInfo &r = j & 2 ? r1 : r0;
                        const int key = k0 + (int)col;
                        if ((have >> col & 1) && key <= r.hi && key >= r.lo)
                            part += ex2(sc[j >> 2][j & 3] * a.sl2 - ls[j >> 1 & 1]);
                    }
                }
            }
            if (++wg == per) {
#pragma unroll
                for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xFFFFFFFFu, part, o);
                if (lane == 0) mass_s[wid][wb] += part;
                part = 0.f;
                wg = 0;
                wb++;
                pw = page_at(min(wb, last));
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncwarp();
    }
    __syncwarp();
    float *out = a.mass + ((size_t)i * p.H + h) * b.width + b0;
    for (uint32_t k = lane; k < n_blk; k += 32) out[k] = mass_s[wid][k];
}

template <class T, int DP>
__global__ void __launch_bounds__(kW * 32)
mass_rows_kernel(Geo g, PagesDev p, BatchDev b, MassDev a, uint32_t per_item, uint32_t items_per_warp,
                 uint32_t groups)
{
    constexpr int ST = kMassStages;
    constexpr uint32_t tile = 16 * DP * 2;
    extern __shared__ __align__(128) char smem[];
    __shared__ float mass_s[kW][kMaxRun];
    __shared__ uint32_t have_s[kW][ST];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5, D = p.D;
    const uint32_t ring_a = smem_addr(smem + wid * ST * tile);
    const uint32_t x = blockIdx.x % groups, ih = blockIdx.x / groups;
    const uint32_t h = ih % p.H, i = ih / p.H;
    const SeqDev s = load_seq(b, p.bs.d, i);
    const uint32_t rows = (uint32_t)s.m * g.G;
    if ((rows <= g.min_rows && g.min_rows) || rows > g.max_rows) return;

    const uint32_t run = per_item * items_per_warp;    // blocks
    const uint32_t b0 = (x * kW + wid) * run;
    if (b0 >= b.width) return;
    const uint32_t n_blk = min(run, b.width - b0);
    for (uint32_t k = lane; k < n_blk; k += 32) mass_s[wid][k] = 0.f;
    __syncwarp();

    const uint32_t ikeys = per_item * p.bs.d, steps = (ikeys + 15) / 16;   // of an item
    for (uint32_t rt = 0; rt * kR < rows; rt++) {
        const RowInfo r0 = row_info(g, s, h, rt * kR + (lane >> 2));
        const RowInfo r1 = row_info(g, s, h, rt * kR + (lane >> 2) + 8);
        const RowInfo rf = row_info(g, s, h, rt * kR);
        const RowInfo rl = row_info(g, s, h, min((rt + 1) * kR, rows) - 1);
        // steps of the run that hold a key of this row tile
        const long long run_key = (long long)b0 * p.bs.d;
        if (rl.hi < run_key || rf.lo >= run_key + (long long)n_blk * p.bs.d) continue;
        const uint32_t last_it = min((uint32_t)((rl.hi - run_key) / ikeys), (n_blk - 1) / per_item);
        const uint32_t first_it = rf.lo > run_key ? (uint32_t)((rf.lo - run_key) / ikeys) : 0;
        const uint32_t u0 = first_it * steps, u1 = (last_it + 1) * steps;

        uint32_t qf[DP / 16][4];
        load_q_frag<T, DP>(a.q, r0, r1, D, qf);
        float ls[2];
        ls[0] = r0.row >= 0 ? a.lse[(size_t)r0.row * a.Hq + r0.head] * kLog2e : 0.f;
        ls[1] = r1.row >= 0 ? a.lse[(size_t)r1.row * a.Hq + r1.head] * kLog2e : 0.f;

        // key c of step u: item u / steps, its 16 keys from (u % steps) * 16
        auto where = [&](uint32_t u, uint32_t c, uint32_t *blk, uint32_t *in) {
            const uint32_t it = u / steps, kk = (u - it * steps) * 16 + c;
            const uint32_t q = kk / p.bs;
            *blk = it * per_item + q;
            *in = kk - q * p.bs.d;
            return kk < ikeys && *blk < n_blk ? (int)((b0 + *blk) * p.bs.d + *in) : 0x7FFFFFFF;
        };
        auto page = [&](uint32_t u) {
            uint32_t blk, in;
            const int key = where(u, lane & 15, &blk, &in);
            if (u >= u1 || key > rl.hi || key < rf.lo) return -1;
            return page_of(b, p.n_pages, i, h, b0 + blk);
        };
        auto issue = [&](uint32_t u, int pg, uint32_t st) {
            if (u < u1) {
                uint32_t blk, in;
                where(u, lane & 15, &blk, &in);
                const long long off = pg >= 0 ? pg * p.page_b + h * p.head_b + (long long)in * p.tok_b : -1;
                const uint32_t have = __ballot_sync(0xFFFFFFFFu, pg >= 0) & 0xFFFFu;
                if (lane == 0) have_s[wid][st] = have;
                load_rows16<DP>(ring_a + st * tile, p.k, off, D);
            }
            cp_commit();
        };
        int pg = page(u0);
#pragma unroll
        for (int k = 0; k < ST - 1; k++) {
            issue(u0 + k, pg, k);
            pg = page(u0 + k + 1);
        }
        uint32_t st = 0, st_in = ST - 1;
        for (uint32_t u = u0; u < u1; u++) {
            issue(u + ST - 1, pg, st_in);
            pg = page(u + ST);
            st_in = st_in + 1 == ST ? 0 : st_in + 1;
            cp_wait<ST - 1>();
            __syncwarp();
            const uint32_t have = have_s[wid][st], kt = ring_a + st * tile;
            st = st + 1 == ST ? 0 : st + 1;
            if (have) {
                float sc[2][4], sum[4];
                scores16<T, DP>(kt, qf, sc);
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint32_t col = n * 8 + (lane & 3) * 2 + c;
                        uint32_t blk, in;
                        const int key = where(u, col, &blk, &in);
                        const bool ok = have >> col & 1;
                        float y = 0.f;
                        if (ok && key <= r0.hi && key >= r0.lo) y = ex2(sc[n][c] * a.sl2 - ls[0]);
                        if (ok && key <= r1.hi && key >= r1.lo) y += ex2(sc[n][2 + c] * a.sl2 - ls[1]);
                        sum[n * 2 + c] = y;
                    }
#pragma unroll
                for (int o = 4; o <= 16; o <<= 1)
#pragma unroll
                    for (int j = 0; j < 4; j++) sum[j] += __shfl_xor_sync(0xFFFFFFFFu, sum[j], o);
                // a lane of each quad column holds keys 2q, 2q+1, 8+2q, 9+2q
                uint32_t bl, in;
                where(u, 0, &bl, &in);
                if (per_item == 1) {
                    float y = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    y += __shfl_xor_sync(0xFFFFFFFFu, y, 1);
                    y += __shfl_xor_sync(0xFFFFFFFFu, y, 2);
                    if (lane == 0) mass_s[wid][bl] += y;
                } else {
                    for (uint32_t j = 0; j < per_item; j++) {
                        float y = 0.f;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const uint32_t col = (q >> 1) * 8 + (lane & 3) * 2 + (q & 1);
                            if (col / p.bs == j && col < ikeys) y += sum[q];
                        }
                        y += __shfl_xor_sync(0xFFFFFFFFu, y, 1);
                        y += __shfl_xor_sync(0xFFFFFFFFu, y, 2);
                        if (lane == 0 && bl + j < n_blk) mass_s[wid][bl + j] += y;
                    }
                }
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncwarp();
    }
    __syncwarp();
    float *out = a.mass + ((size_t)i * p.H + h) * b.width + b0;
    for (uint32_t k = lane; k < n_blk; k += 32) out[k] = mass_s[wid][k];
}

// CTAs of a unit's cluster, 0: the equal shares.  A cluster needs no join
// launch (5 us of a call), but its CTAs are one unit's for the whole launch;
// so it is taken when the units and their splits are one wave of two CTAs an
// SM, or need none, and no CTA has more than 8 key tiles to do.  A CTA gets two
// tiles at least (one request over 900 tokens: 8.2 us with 8 CTAs a unit, 9.5
// with 15).
uint32_t cluster_split(unsigned long long units, unsigned long long keys)
{
    const unsigned long long tiles = (keys + kKeys - 1) / kKeys;
    uint32_t s = 1;
    while (s < 16 && 2 * s < tiles && units * s * 2 <= 148 * 2) s *= 2;
    return tiles <= 8ull * s && units * s < (1u << 30) ? s : 0;
}

template <class T, int DP, bool AL>
int attend_a(const PagesDev &p, const BatchDev &b, const AttendDev &a, const ClassDev &cl,
             const SplitDev &sp, cudaStream_t s)
{
    const Geo g = {kR, kKeys, a.G, p.H, a.window, cl.min_rows, cl.max_rows, 0};
    if (sp.split) {
        auto k = attend_rows_kernel<T, DP, true, AL>;
        constexpr size_t smem = RowsCfg<DP>::smem + (size_t)kR * (DP + 2) * sizeof(float);
        static std::atomic<uint64_t> done, wide;
        OKV_CUDA_TRY(allow_smem(k, smem, done));
        if (sp.split > 8) OKV_CUDA_TRY(allow_wide_cluster(k, wide));
        cudaLaunchConfig_t c = {};
        c.gridDim = dim3(b.n * p.H * sp.tiles_max * sp.split);
        c.blockDim = dim3(kW * 32);
        c.dynamicSmemBytes = smem;
        c.stream = s;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = sp.split;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        c.attrs = &at;
        c.numAttrs = 1;
        OKV_CUDA_TRY(cudaLaunchKernelEx(&c, k, g, p, b, a, sp, sp.split, sp.tiles_max));
        note_launches(1);
        return ORCHKV_OK;
    }
    auto k = attend_rows_kernel<T, DP, false, AL>;
    static std::atomic<uint64_t> done;
    OKV_CUDA_TRY(allow_smem(k, RowsCfg<DP>::smem, done));
    k<<<sp.ctas, kW * 32, RowsCfg<DP>::smem, s>>>(g, p, b, a, sp, 1, 1);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    if (sp.ctas > 1) {
        OKV_CUDA_TRY(launch_after(join_kernel<T, 128>, sp.ctas - 1, 128, 0, s, g, p, b, a, sp, 1u));
        note_launches(1);
    }
    return ORCHKV_OK;
}

template <class T, int DP>
int attend_d(const PagesDev &p, const BatchDev &b, const AttendDev &a, const ClassDev &cl,
             const SplitDev &sp, cudaStream_t s)
{
    return p.bs.d % 16 == 0 ? attend_a<T, DP, true>(p, b, a, cl, sp, s) : attend_a<T, DP, false>(p, b, a, cl, sp, s);
}

template <class T, int DP>
int mass_d(const PagesDev &p, const BatchDev &b, const MassDev &a, const ClassDev &cl, cudaStream_t s)
{
    const Geo g = {kR, 0, a.G, p.H, a.window, cl.min_rows, cl.max_rows, 0};
    const uint32_t per_item = p.bs.d >= 16 ? 1 : 16 / p.bs.d;
    const uint32_t items = (b.width + per_item - 1) / per_item;
    // A CTA takes 4 us to its first product (rows, queries, table, keys one
    // after the other), as long as 30 blocks take: as few and as long runs as
    // leave no place (3 an SM) of the device empty.  32 requests over 8192
    // tokens: 101 us with 16 CTAs a place, 77 with 8, 61 with 4.
    const uint32_t most = kMaxRun / per_item;
    unsigned long long groups64 = 148ull * 3 / ((unsigned long long)b.n * p.H);
    groups64 = std::max<unsigned long long>(groups64, (items + most * kW - 1) / (most * kW));
    groups64 = std::max<unsigned long long>(groups64, 1);
    const uint32_t run = (uint32_t)((items + groups64 * kW - 1) / (groups64 * kW));
    const uint32_t groups = (items + run * kW - 1) / (run * kW);
    const unsigned long long grid = (unsigned long long)b.n * p.H * groups;
    if (grid > 0x7FFFFFFFull) return ORCHKV_ERR_INVALID;
    const size_t smem = (size_t)kW * kMassStages * 16 * DP * 2;
    static std::atomic<uint64_t> done, done_al;
    if (p.bs.d % 16 == 0) {
        auto k = mass_runs_kernel<T, DP>;
        OKV_CUDA_TRY(allow_smem(k, smem, done_al));
        k<<<(unsigned)grid, kW * 32, smem, s>>>(g, p, b, a, run, groups);
    } else {
        auto k = mass_rows_kernel<T, DP>;
        OKV_CUDA_TRY(allow_smem(k, smem, done));
        k<<<(unsigned)grid, kW * 32, smem, s>>>(g, p, b, a, per_item, run, groups);
    }
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    return ORCHKV_OK;
}

}  // namespace

SplitDev attend_rows_split(uint32_t D, uint32_t n, uint32_t H, uint32_t tiles_max, unsigned long long units,
                           unsigned long long keys)
{
    SplitDev sp = {};
    sp.tiles_max = tiles_max;
    sp.split = cluster_split((unsigned long long)n * H * tiles_max, keys);
    if (sp.split) return sp;
    const unsigned long long tiles = units * ((keys + kKeys - 1) / kKeys);
    const unsigned long long most = 148ull * (D > 128 ? 1 : 2);
    sp.ctas = (uint32_t)(tiles < most ? tiles : most);
    return sp;
}

int launch_attend_rows(int dtype, const PagesDev &p, const BatchDev &b, const AttendDev &a,
                       const ClassDev &cl, const SplitDev &sp, cudaStream_t s)
{
    if (dtype == DTYPE_BF16) {
        if (p.D <= 64) return attend_d<__nv_bfloat16, 64>(p, b, a, cl, sp, s);
        if (p.D <= 128) return attend_d<__nv_bfloat16, 128>(p, b, a, cl, sp, s);
        return attend_d<__nv_bfloat16, 256>(p, b, a, cl, sp, s);
    }
    if (p.D <= 64) return attend_d<__half, 64>(p, b, a, cl, sp, s);
    if (p.D <= 128) return attend_d<__half, 128>(p, b, a, cl, sp, s);
    return attend_d<__half, 256>(p, b, a, cl, sp, s);
}

int launch_mass_rows(int dtype, const PagesDev &p, const BatchDev &b, const MassDev &a,
                     const ClassDev &cl, cudaStream_t s)
{
    if (dtype == DTYPE_BF16) {
        if (p.D <= 64) return mass_d<__nv_bfloat16, 64>(p, b, a, cl, s);
        if (p.D <= 128) return mass_d<__nv_bfloat16, 128>(p, b, a, cl, s);
        return mass_d<__nv_bfloat16, 256>(p, b, a, cl, s);
    }
    if (p.D <= 64) return mass_d<__half, 64>(p, b, a, cl, s);
    if (p.D <= 128) return mass_d<__half, 128>(p, b, a, cl, s);
    return mass_d<__half, 256>(p, b, a, cl, s);
}

}  // namespace okv

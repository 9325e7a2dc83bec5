// paged_tile.cu — attention of longer chunks over pages on the fifth-generation
// tensor cores (tcgen05, accumulators in tensor memory, pages by TMA).
//
// A unit is 256 packed rows (new tokens times the query heads of one KV head,
// so K and V are read once for the whole group) against its keys, 128 at a
// time: S = Q K^T, P = 2^(S - m), O += P V.  4 D products a score against one
// power of two: at D = 128 the tensor core needs 2048 clocks for 256 x 128
// scores and the special function unit as many for their powers, so both have
// to run all the time.  Roles (384 threads, one CTA an SM):
//   warp 0     loads: pages of K and V into a ring of 128-key tiles
//   warp 1     products: one thread issues them all
//   warps 4-7  softmax of rows 0..127, warps 8-11 of rows 128..255: a thread
//              owns a row, whose scores it reads from its lane of tensor memory
// While one half's softmax runs, the tensor core works for the other half.
// P goes back to tensor memory over the columns of its S (16 bits a weight)
// and is the A operand of the second product, so weights never touch shared
// memory.  O stays in tensor memory; it is scaled only when a row's maximum
// has grown by more than 2^8 (weights then reach 256, which neither type nor
// the fp32 sums mind), which after the first tiles is rare.
#include <type_traits>

#include "kernels.h"
#include "paged_tile.cuh"

namespace okv {

namespace {

// Set when a wait ran out (orchkv_paged_status).
__device__ int g_paged_dead;

constexpr int kThreads = 384;
constexpr uint32_t kR = 256, kK = 128;
constexpr float kGrow = 8.f;               // log2 of the growth that O is scaled at
constexpr int kMeta = 8;                   // tiles whose column masks are kept

template <int DP> struct TileCfg {
    static constexpr uint32_t tile = kK * DP * 2;          // bytes of a K or V tile
    static constexpr int stages = DP == 128 ? 5 : 8;
    static constexpr uint32_t q = kR * DP * 2;
    static constexpr size_t smem = 1024 + q + (size_t)stages * tile;
};

struct TileShared {
    ull full[8], empty[8], s_full[2], p_full[2], q_full[2], o_full[2], fix, drain;
    uint32_t tmem;
    int dead;
    alignas(16) uint32_t mask[kMeta][4];   // columns of a tile that hold a token
    SplitShared split;
};

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
attend_tile_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, Geo g,
                   PagesDev p, BatchDev b, AttendDev a, SplitDev sp, int by_head)
{
    using Cfg = TileCfg<DP>;
    constexpr int ST = Cfg::stages;
    extern __shared__ char raw[];
    __shared__ TileShared sh;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    const uint32_t q_s = base, ring = base + Cfg::q;
    const uint32_t wid = threadIdx.x >> 5, lane = threadIdx.x & 31;

    Walk w{g, b, p.bs.d};
    ull W;
    find_share<kThreads>(g, b, p.bs.d, blockIdx.x, sp.ctas, &sh.split, &w.at, &w.end, &W);
    cudaTriggerProgrammaticLaunchCompletion();
    if (W == 0) return;
    if (!w.settle()) return;                               // an empty share (the same for all threads)

    if (threadIdx.x == 0) {
        for (int k = 0; k < ST; k++) {
            mbar_init(smem_addr(&sh.full[k]), 1);
            mbar_init(smem_addr(&sh.empty[k]), 1);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(smem_addr(&sh.s_full[k]), 1);
            mbar_init(smem_addr(&sh.p_full[k]), 4);
            mbar_init(smem_addr(&sh.q_full[k]), 4);
            mbar_init(smem_addr(&sh.o_full[k]), 1);
        }
        mbar_init(smem_addr(&sh.fix), 1);
        mbar_init(smem_addr(&sh.drain), 1);
        sh.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (wid == 1) tm_alloc(smem_addr(&sh.tmem), 512);
    tm_before();
    __syncthreads();
    tm_after();
    const uint32_t tm = sh.tmem;
    volatile int *dead = &sh.dead;

    // 4 x 88 + 8 x 208 registers a lane are the 12 x 168 of the launch
    if (wid < 4) {
      regs_down<88>();
      if (wid == 0) {
        // ---- loads ----
        const uint32_t bs = p.bs.d, per = bs < kK ? kK / bs : 1, box = bs < kK ? bs : kK;
        constexpr uint32_t halves = DP / 64;
        uint32_t st = 0, ph = 0, fix_ph = 0, tile_no = 0, issued = 0;
        bool ok = true;
        do {
            const uint32_t h = w.at.h, i = w.at.i;
            const int zh = by_head ? 0 : (int)h;
            auto page = [&](uint32_t t) {                  // lane q: page q of tile t
                if (t >= w.t1 || lane >= per) return -1;
                const uint32_t k0 = (w.first + t) * kK + lane * bs;
                if ((int)k0 >= w.s.len) return -1;
                return page_of(b, p.n_pages, i, h, k0 / p.bs);
            };
            int pg = page(w.t0);
            for (uint32_t t = w.t0; ok && t < w.t1; t++) {
                const uint32_t k0 = (w.first + t) * kK;
                const int nxt = page(t + 1);
                const uint32_t have = __ballot_sync(0xFFFFFFFFu, pg >= 0);
                // column masks of the tile, one word a lane
                uint32_t word = 0;
                const uint32_t c0 = (lane & 3) * 32;
                for (uint32_t q = c0 / bs; q * bs < c0 + 32 && q < per; q++)
                    if (have >> q & 1) {
                        const uint32_t lo = max(q * bs, c0) - c0;
                        const uint32_t hi = min((bs < kK ? (q + 1) * bs : kK), c0 + 32) - c0;
                        word |= (hi == 32 ? 0xFFFFFFFFu : (1u << hi) - 1) & ~((1u << lo) - 1);
                    }
                const int lim = w.s.len - (int)(k0 + c0);
                if (lim <= 0) word = 0;
                else if (lim < 32) word &= (1u << lim) - 1;
                const bool part = __any_sync(0xFFFFFFFFu, word != 0xFFFFFFFFu);
                const uint32_t bytes = __popc(have) * box * 128 * halves;
                const int y = bs < kK ? 0 : (int)(k0 % bs);
#pragma unroll 1
                for (int kv = 0; ok && kv < 2; kv++) {
                    ok = mbar_wait(smem_addr(&sh.empty[st]), ph ^ 1, dead);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    if (kv == 0 && lane < 4) sh.mask[tile_no % kMeta][lane] = word;
                    const uint32_t full = smem_addr(&sh.full[st]);
                    const bool fix = kv == 1 && part;
                    const uint32_t bar = fix ? smem_addr(&sh.fix) : full;
                    const uint32_t dst = ring + st * Cfg::tile;
                    __syncwarp();
                    if (lane == 0) mbar_expect(bar, bytes);
                    __syncwarp();
                    if (pg >= 0)
#pragma unroll
                        for (uint32_t x = 0; x < halves; x++)
                            tma4(dst + x * kK * 128 + lane * box * 128, kv ? &vmap : &kmap, (int)x * 64, y, zh,
                                 pg, bar);
                    if (fix) {
                        // rows of V without a token become zeros: their weights
                        // are 0, and 0 times a stale NaN would not be
                        ok = mbar_wait(bar, fix_ph, dead);
                        ok = __all_sync(0xFFFFFFFFu, ok);
                        fix_ph ^= 1;
                        for (uint32_t r = lane; r < kK; r += 32) {
                            const uint32_t wd = __shfl_sync(0xFFFFFFFFu, word, r >> 5);
                            if (!(wd >> (r & 31) & 1))
#pragma unroll
                                for (uint32_t x = 0; x < halves; x++)
#pragma unroll
                                    for (uint32_t c = 0; c < 8; c++)
                                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                                         dst + x * kK * 128 + r * 128 + c * 16), "r"(0) : "memory");
                        }
                        fence_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(full);
                    }
                    issued++;
                    if (++st == ST) { st = 0; ph ^= 1; }
                }
                pg = nxt;
                tile_no++;
            }
        } while (ok && w.next());
        if (!ok) {
            // leave no copy in flight behind
            if (lane == 0)
                for (uint32_t k = 0; k < ST && k < issued; k++) {
                    st = st == 0 ? ST - 1 : st - 1;
                    if (st == ST - 1) ph ^= 1;
                    mbar_drain(smem_addr(&sh.full[st]), ph);
                }
            __syncwarp();
        }
      } else if (wid == 1) {
        // ---- products ----
        if (lane == 0) {
            const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
            const uint32_t id_qk = inst_desc(f, 128, kK, 0), id_pv = inst_desc(f, 128, DP, 1);
            uint32_t st = 0, ph = 0, q_ph[2] = {0, 0}, p_ph[2] = {0, 0};
            bool ok = true;
            auto qk = [&](int x, uint32_t stage) {
                const uint32_t qa = q_s + x * 128 * DP * 2, ka = ring + stage * Cfg::tile;
#pragma unroll
                for (int k = 0; k < DP / 16; k++) {
                    const uint32_t o = (k >> 2) * kK * 128 + (k & 3) * 32;
                    mma_ss(tm + x * 128, smem_desc(qa + o, 16, 1024), smem_desc(ka + o, 16, 1024), id_qk, k > 0);
                }
                tm_commit(smem_addr(&sh.s_full[x]));
            };
            do {
                const int nx = w.live() > 128 ? 2 : 1;
                uint32_t ks = st;
                ok = mbar_wait(smem_addr(&sh.full[ks]), ph, dead);
                if (!ok) break;
                for (int x = 0; ok && x < nx; x++) {
                    ok = mbar_wait(smem_addr(&sh.q_full[x]), q_ph[x], dead);
                    q_ph[x] ^= 1;
                    tm_after();
                    if (ok) qk(x, ks);
                }
                if (!ok) break;
                tm_commit(smem_addr(&sh.empty[ks]));
                if (++st == ST) { st = 0; ph ^= 1; }
                for (uint32_t t = w.t0; ok && t < w.t1; t++) {
                    const bool more = t + 1 < w.t1;
                    const uint32_t vs = st;
                    ok = mbar_wait(smem_addr(&sh.full[vs]), ph, dead);
                    if (++st == ST) { st = 0; ph ^= 1; }
                    if (ok && more) {
                        ks = st;
                        ok = mbar_wait(smem_addr(&sh.full[ks]), ph, dead);
                        if (++st == ST) { st = 0; ph ^= 1; }
                    }
                    for (int x = 0; ok && x < nx; x++) {
                        ok = mbar_wait(smem_addr(&sh.p_full[x]), p_ph[x], dead);
                        p_ph[x] ^= 1;
                        if (!ok) break;
                        tm_after();
                        const uint32_t va = ring + vs * Cfg::tile;
#pragma unroll
                        for (int k = 0; k < kK / 16; k++)
                            mma_ts(tm + 256 + x * 128, tm + x * 128 + k * 8,
                                   smem_desc(va + k * 2048, kK * 128, 1024), id_pv, t > w.t0 || k > 0);
                        if (more) qk(x, ks);
                        else tm_commit(smem_addr(&sh.o_full[x]));
                    }
                    if (!ok) break;
                    tm_commit(smem_addr(&sh.empty[vs]));
                    if (more) tm_commit(smem_addr(&sh.empty[ks]));
                }
            } while (ok && w.next());
            if (!ok) {
                tm_commit(smem_addr(&sh.drain));
                mbar_drain(smem_addr(&sh.drain), 0);
            }
        }
        __syncwarp();
      }
    } else {
        regs_up<208>();
        // ---- softmax of one half ----
        const int x = (wid - 4) >> 2;
        const uint32_t r = threadIdx.x - 128 - x * 128;    // row of the half
        const uint32_t lanes = (wid & 3) << 21;            // first lane of this warp, in a TMEM address
        const uint32_t S = tm + x * 128 + lanes, O = tm + 256 + x * 128 + lanes;
        uint32_t s_ph = 0, o_ph = 0, tile_no = 0;
        const ull sl2 = f2(a.sl2, a.sl2);

        auto load_q = [&](const Walk &u) {
            const RowInfo ri = row_info(g, u.s, u.at.h, u.at.rt * kR + x * 128 + r);
            const char *src = a.q.p + (long long)ri.row * a.q.row_b + (long long)ri.head * a.q.head_b;
            const uint32_t dst = q_s + x * 128 * DP * 2 + r * 128;
#pragma unroll
            for (uint32_t c = 0; c < DP / 8; c++) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (ri.row >= 0 && c * 8 < p.D) v = *(const uint4 *)(src + c * 16);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                 dst + (c >> 3) * kK * 128 + (((c & 7) ^ (r & 7)) << 4)),
                             "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&sh.q_full[x]));
        };
        bool live = true;
        while (live && x == 1 && w.live() <= 128) {
            tile_no += w.t1 - w.t0;
            live = w.next();
        }
        if (live) load_q(w);
        bool ok = true;
        while (live && ok) {
            const uint32_t pr0 = w.at.rt * kR + x * 128, rows = (uint32_t)w.s.m * g.G;
            const RowInfo ri = row_info(g, w.s, w.at.h, pr0 + r);
            // keys that every row of the half attends to
            const int all_hi = row_info(g, w.s, w.at.h, pr0).hi;
            const int all_lo = row_info(g, w.s, w.at.h, min(pr0 + 128, rows) - 1).lo;
            float m = -INFINITY;
            ull l2[2] = {0, 0};
            for (uint32_t t = w.t0; t < w.t1; t++, tile_no++) {
                ok = mbar_wait(smem_addr(&sh.s_full[x]), s_ph, dead);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                s_ph ^= 1;
                tm_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; c++) tm_ld32(S + c * 32, s + c * 32);
                tm_wait_ld();
                const int k0 = (int)((w.first + t) * kK);
                const uint4 mk = *(const uint4 *)sh.mask[tile_no % kMeta];
                if (k0 < all_lo || k0 + (int)kK - 1 > all_hi || (mk.x & mk.y & mk.z & mk.w) != 0xFFFFFFFFu) {
                    const uint32_t mw[4] = {mk.x, mk.y, mk.z, mk.w};
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int lo = ri.lo - k0 - c * 32, hi = ri.hi - k0 - c * 32;
                        uint32_t bits = mw[c];
                        bits &= hi < 0 ? 0u : hi >= 31 ? 0xFFFFFFFFu : (2u << hi) - 1;
                        bits &= lo > 31 ? 0u : lo <= 0 ? 0xFFFFFFFFu : ~((1u << lo) - 1);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!(bits >> j & 1)) s[c * 32 + j] = -INFINITY;
                    }
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int j = 4; j < 128; j += 4)
#pragma unroll
                    for (int k = 0; k < 4; k++) mx[k] = fmaxf(mx[k], s[j + k]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const float ms = top * a.sl2;          // the scale is positive here
                if (t == w.t0) {
                    m = ms;
                } else {
                    const bool grow = ms > m + kGrow || (m == -INFINITY && ms > m);
                    if (__any_sync(0xFFFFFFFFu, grow)) {
                        const float nm = grow ? ms : m;
                        const float f = nm == -INFINITY ? 1.f : ex2(m - nm);
                        m = nm;
                        const ull ff = f2(f, f);
                        l2[0] = mul2(l2[0], ff);
                        l2[1] = mul2(l2[1], ff);
#pragma unroll 1
                        for (int c = 0; c < DP / 32; c++) {
                            float o[32];
                            tm_ld32(O + c * 32, o);
                            tm_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; j++) o[j] *= f;
                            tm_st32(O + c * 32, (const uint32_t *)o);
                        }
                        tm_wait_st();
                    }
                }
                const float mm = m == -INFINITY ? 0.f : m;
                const ull nm2 = f2(-mm, -mm);
                // weights: rounded to the pages' type for the product (half a
                // step each, as the result's own rounding); their sum is taken
                // before that
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t pk[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        float *e = s + c * 32 + 2 * j;
                        float u, v;
                        unf2(fma2(f2(e[0], e[1]), sl2, nm2), &u, &v);
                        u = ex2(u);
                        v = ex2(v);
                        l2[j & 1] = add2(l2[j & 1], f2(u, v));
                        pk[j] = pack2<T>(u, v);
                    }
                    tm_st16(S + c * 16, pk);
                }
                tm_wait_st();
                tm_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.p_full[x]));
            }
            if (!ok) break;
            // the next unit's queries while the last products run, then the rows
            Walk u = w;
            live = u.next();
            uint32_t skipped = 0;
            while (live && x == 1 && u.live() <= 128) {
                skipped += u.t1 - u.t0;
                live = u.next();
            }
            if (live) load_q(u);
            ok = mbar_wait(smem_addr(&sh.o_full[x]), o_ph, dead);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            o_ph ^= 1;
            tm_after();
            float la, lb, lc, ld;
            unf2(l2[0], &la, &lb);
            unf2(l2[1], &lc, &ld);
            const float L = (la + lb) + (lc + ld);
            const bool whole = w.t0 == 0 && w.t1 == w.nt;
            const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
            float *sl = slot_of(sp.ws, 2 * blockIdx.x + (w.t0 == 0 ? 1 : 0), kR, p.D);
            char *dst = a.out.p + (long long)ri.row * a.out.row_b + (long long)ri.head * a.out.head_b;
#pragma unroll 1
            for (int c = 0; c < DP / 32; c++) {
                float o[32];
                tm_ld32(O + c * 32, o);
                tm_wait_ld();
                if (ri.row >= 0 && whole) {
#pragma unroll
                    for (int j = 0; j < 32; j++) o[j] *= inv;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if ((uint32_t)(c * 32 + j * 8) < p.D)
                            *(uint4 *)(dst + c * 64 + j * 16) = Vec<T>::down(o + j * 8);
                } else if (ri.row >= 0) {
                    float *d = sl + 2 * kR + (size_t)(x * 128 + r) * p.D + c * 32;
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if ((uint32_t)(c * 32 + j * 4) < p.D)
                            *(float4 *)(d + j * 4) = make_float4(o[j * 4], o[j * 4 + 1], o[j * 4 + 2], o[j * 4 + 3]);
                }
                __syncwarp();
            }
            if (ri.row >= 0) {
                const float mm = m == -INFINITY ? 0.f : m;
                if (!whole) {
                    sl[x * 128 + r] = m;
                    sl[kR + x * 128 + r] = L;
                } else if (a.lse) {
                    a.lse[(size_t)ri.row * a.Hq + ri.head] =
                        L > 0.f ? (mm + log2f(L)) * kLn2 : L == 0.f ? -INFINITY : L;
                }
            }
            tm_before();
            tile_no += skipped;
            w.at = u.at;
            w.s = u.s;
            w.RT = u.RT;
            w.first = u.first;
            w.nt = u.nt;
            w.t0 = u.t0;
            w.t1 = u.t1;
            w.stop = u.stop;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && sh.dead) g_paged_dead = 1;
    if (wid == 1) tm_free(tm, 512);
}

template <class T, int DP>
int go(const CUtensorMap &km, const CUtensorMap &vm, const PagesDev &p, const BatchDev &b, const AttendDev &a,
       const ClassDev &cl, const SplitDev &sp, cudaStream_t s)
{
    const Geo g = {kR, kK, a.G, p.H, a.window, cl.min_rows, cl.max_rows};
    auto k = attend_tile_kernel<T, DP>;
    OKV_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TileCfg<DP>::smem));
    k<<<sp.ctas, kThreads, TileCfg<DP>::smem, s>>>(km, vm, g, p, b, a, sp, p.head_b == 0);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    if (sp.ctas > 1) {
        OKV_CUDA_TRY(launch_after(join_kernel<T, 512>, sp.ctas - 1, 512, 0, s, g, p, b, a, sp));
        note_launches(1);
    }
    return ORCHKV_OK;
}

}  // namespace

bool page_map(CUtensorMap *m, const PagesDev &p, const char *base, int dtype)
{
    typedef CUresult (*encode_t)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);
    static encode_t encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (encode_t)f;
    }();
    if (!encode) return false;
    // pages of one head: a head axis of one entry
    const bool by_head = p.head_b == 0;
    const cuuint64_t dims[4] = {p.D, p.bs.d, by_head ? 1 : p.H, p.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)p.tok_b, (cuuint64_t)(by_head ? p.tok_b : p.head_b),
                                   (cuuint64_t)p.page_b};
    const cuuint32_t box[4] = {64, p.bs.d < 128 ? p.bs.d : 128, 1, 1};
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return encode(m, dtype == DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  4, (void *)base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 16-bit pages whose tokens fill whole boxes; a scale that keeps the order of
// the scores (the mask is applied before it).
bool attend_tile_takes(const PagesDev &p, int dtype, float sl2)
{
    return dtype != DTYPE_FP32 && pages_tile(p) && sl2 > 0.f && p.page_b >= 0 && p.head_b >= 0 && p.tok_b > 0 &&
           p.page_b < (1ll << 40) && p.head_b < (1ll << 40) && p.tok_b < (1ll << 40);
}

uint32_t attend_tile_ctas(unsigned long long units, unsigned long long keys)
{
    const unsigned long long tiles = units * ((keys + kK - 1) / kK);
    return (uint32_t)(tiles < 148 ? tiles : 148);
}

int launch_attend_tile(int dtype, const PagesDev &p, const BatchDev &b, const AttendDev &a, const ClassDev &cl,
                       const SplitDev &sp, cudaStream_t s)
{
    CUtensorMap km, vm;
    if (!page_map(&km, p, p.k, dtype) || !page_map(&vm, p, p.v, dtype)) return ORCHKV_ERR_CUDA;
    if (dtype == DTYPE_BF16)
        return p.D <= 64 ? go<__nv_bfloat16, 64>(km, vm, p, b, a, cl, sp, s)
                         : go<__nv_bfloat16, 128>(km, vm, p, b, a, cl, sp, s);
    return p.D <= 64 ? go<__half, 64>(km, vm, p, b, a, cl, sp, s) : go<__half, 128>(km, vm, p, b, a, cl, sp, s);
}

}  // namespace okv

extern "C" int orchkv_paged_status(void)
{
    int dead = 0;
    OKV_CUDA_TRY(cudaMemcpyFromSymbol(&dead, okv::g_paged_dead, sizeof(dead)));
    return dead ? ORCHKV_ERR_CUDA : ORCHKV_OK;
}

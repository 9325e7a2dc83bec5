// paged_tile.cu — attention of longer chunks over pages on the fifth-generation
// tensor cores (tcgen05, accumulators in tensor memory, pages by TMA).
//
// A unit is 256 packed rows (new tokens times the query heads of one KV head,
// so K and V are read once for the whole group) against its keys, 128 at a
// time: S = Q K^T, P = 2^(S - m), O += P V.  4 D products a score against one
// power of two: at D = 128 the tensor core needs 2048 clocks for 256 x 128
// scores and the special function unit as many for their powers, so both have
// to run all the time.  Roles (384 threads, one CTA an SM):
//   warps 0, 2 loads: pages of K, pages of V, into a ring of 128-key tiles
//   warp 1     products: one thread issues them all
//   warps 4-7  softmax of rows 0..127, warps 8-11 of rows 128..255: a thread
//              owns a row, whose scores it reads from its lane of tensor memory
// Tensor memory is full at D = 128: O of both halves (256 columns), the weights
// P of both (64 each, 16 bits a weight: the A operand of the second product, so
// weights never touch shared memory) and one S of 128 that the halves fill and
// read in turn: a half's next scores are computed while it still weighs its
// last ones.  O stays there; it is scaled only when a row's maximum has grown
// by more than 2^8 (fp16: 2^4; the weights in between are larger than 1, which
// neither type nor the fp32 sums mind), which after the first tiles is rare.
//
// 4096 new tokens over 28672, 32/8 heads of 128, bf16: 1.77 to 2.01 ms over the
// devices measured, 1030 to 1170 TFLOP/s, 0.62 to 0.71 of the measured matrix rate
// (1654.6).  ncu on 2048 over 6144: tensor pipe 56 % active, special functions
// 57 %, instruction issue 38 %: what is
// left is the latency of the chain scores -> maximum -> powers -> weights with
// two warps a scheduler.  Measured and not kept: a quarter of the powers as
// polynomials (+3 % at 128 elements; not measured at 64), weights handed over in
// two parts (+5 %).  A warp whose lanes each issue their page's copy took 4000
// clocks a tile for the loads alone; one thread in a loop hides them.  An S of
// its own for each half, with P over it, has been measured with such loads only
// (2220 us together), not by itself.
#include <type_traits>

#include "kernels.h"
#include "paged_tile.cuh"

namespace okv {

namespace {

// Set when a wait ran out (orchkv_paged_status).
__device__ int g_paged_dead;

constexpr int kThreads = 384;
constexpr uint32_t kR = 256, kK = 128;
// Columns of tensor memory: the weights of half 0, the scores, the weights of
// half 1 (64, 128 and 64 columns), then O of either half.
constexpr uint32_t kP0 = 0, kS = 64, kP1 = 192;
// Log2 of the growth that O is scaled at: less for fp16, whose weights have
// less room above and below.
template <class T> constexpr float kGrow = std::is_same<T, __half>::value ? 4.f : 8.f;
// A join costs 20 to 30 us (every cut unit's partials are 128 KB written and read),
// as long as 10 tiles of keys: 512 tokens over 1000, 32/8 heads: 68 us with every
// boundary cut, 48 with none.
constexpr uint32_t kJoinKeys = 10 * kK;
constexpr int kMeta = 8;                   // tiles whose column masks are kept

template <int DP> struct TileCfg {
    static constexpr uint32_t tile = kK * DP * 2;          // bytes of a K or V tile
    static constexpr int stages = DP == 128 ? 5 : 8;
    static constexpr uint32_t q = kR * DP * 2;
    static constexpr size_t smem = 1024 + q + (size_t)stages * tile;
};

struct TileShared {
    ull full[8], empty[8], s_full[2], p_full[2], q_full[2], o_full[2], s_free, fix, drain;
    uint32_t tmem;
    int dead;
    // the last unit (counted from 1) of every kMeta with values that are not
    // finite behind some row's mask; never reset, since a half may look at a
    // unit long after the loads have left it
    uint32_t odd[kMeta];
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
        mbar_init(smem_addr(&sh.s_free), 4);
        mbar_init(smem_addr(&sh.fix), 1);
        mbar_init(smem_addr(&sh.drain), 1);
        for (int k = 0; k < kMeta; k++) sh.odd[k] = 0;
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
      if (wid == 0 || wid == 2) {
        // ---- loads: K by one warp, V by another, into every other place of the ring ----
        const bool is_v = wid == 2;
        const CUtensorMap *map = is_v ? &vmap : &kmap;
        const uint32_t bs = p.bs.d, per = bs < kK ? kK / bs : 1, box = bs < kK ? bs : kK;
        const uint32_t page_bytes = box * 128, all_pages = per == 32 ? 0xFFFFFFFFu : (1u << per) - 1;
        constexpr uint32_t halves = DP / 64;
        uint32_t st = is_v ? 1 : 0, ph = 0, fix_ph = 0, tile_no = 0, u_no = 0;
        const bool one = elect_one();
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            if (ok) ok = mbar_wait(bar, parity, dead);
            ok = __all_sync(0xFFFFFFFFu, ok);
        };
        do {
            const uint32_t h = w.at.h, i = w.at.i;
            const int zh = by_head ? 0 : (int)h;
            // keys that every row of the unit attends to
            const int all_hi = row_info(g, w.s, h, w.at.rt * kR).hi;
            const int all_lo = row_info(g, w.s, h, w.at.rt * kR + w.live() - 1).lo;
            auto page = [&](uint32_t t) {                  // lane q: page q of tile t
                if (t >= w.t1 || lane >= per) return -1;
                const uint32_t k0 = (w.first + t) * kK + lane * bs;
                if ((int)k0 >= w.s.len) return -1;
                return page_of(b, p.n_pages, i, h, k0 / p.bs);
            };
            int pg = page(w.t0);
            for (uint32_t t = w.t0; ok && t < w.t1; t++, tile_no++) {
                const uint32_t k0 = (w.first + t) * kK;
                const int nxt = page(t + 1);
                const uint32_t have = __ballot_sync(0xFFFFFFFFu, pg >= 0);
                // columns that hold a token, one word a lane
                const bool part = have != all_pages || (int)(k0 + kK) > w.s.len;
                uint32_t word = 0xFFFFFFFFu;
                if (part) {
                    word = 0;
                    const uint32_t c0 = (lane & 3) * 32;
                    for (uint32_t q = c0 / p.bs; q * bs < c0 + 32 && q < per; q++)
                        if (have >> q & 1) {
                            const uint32_t lo = max(q * bs, c0) - c0;
                            const uint32_t hi = min((bs < kK ? (q + 1) * bs : kK), c0 + 32) - c0;
                            word |= (hi == 32 ? 0xFFFFFFFFu : (1u << hi) - 1) & ~((1u << lo) - 1);
                        }
                    const int lim = w.s.len - (int)(k0 + c0);
                    if (lim <= 0) word = 0;
                    else if (lim < 32) word &= (1u << lim) - 1;
                }
                const uint32_t full = smem_addr(&sh.full[st]), dst = ring + st * Cfg::tile;
                const bool some = (int)k0 < all_lo || (int)(k0 + kK) - 1 > all_hi;
                const bool fix = is_v && (part || some);
                const uint32_t bar = fix ? smem_addr(&sh.fix) : full;
                wait(smem_addr(&sh.empty[st]), ph ^ 1);
                if (!ok) break;
                if (!is_v && lane < 4) sh.mask[tile_no % kMeta][lane] = word;
                __syncwarp();
                if (one) mbar_expect(bar, __popc(have) * page_bytes * halves);
                __syncwarp();
                const int y = bs < kK ? 0 : (int)(k0 - k0 / p.bs * bs);
                // one thread, one page after another: a warp whose lanes issue
                // copies of their own takes four times as long for each
                for (uint32_t q = 0; q < per; q++) {
                    const int pq = __shfl_sync(0xFFFFFFFFu, pg, q);
                    if (one && pq >= 0)
#pragma unroll
                        for (uint32_t x = 0; x < halves; x++)
                            tma4(dst + x * kK * 128 + q * page_bytes, map, (int)x * 64, y, zh, pq, bar);
                }
                __syncwarp();
                if (fix) {
                    // rows of V without a token become zeros: their weights are
                    // 0, and 0 times a stale NaN would not be
                    wait(bar, fix_ph);
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
                    __syncwarp();
                    // nor would 0 times an infinite value of a token that only
                    // some rows attend to: it becomes 0 here, and the results of
                    // the rows that do attend to it NaN at the unit's end
                    if (ok && some) {
                        Finite<T> fin;
#pragma unroll 8
                        for (uint32_t e = lane; e < Cfg::tile / 16; e += 32) {
                            uint32_t v[4];
                            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(dst + e * 16));
#pragma unroll
                            for (int j = 0; j < 4; j++) fin.see(v[j]);
                        }
                        if (!__all_sync(0xFFFFFFFFu, fin.none())) {
#pragma unroll 1
                            for (uint32_t e = lane; e < Cfg::tile / 4; e += 32) {
                                uint32_t v;
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(dst + e * 4));
                                if (infinite<T>(v, 0)) v &= 0xFFFF0000u;
                                if (infinite<T>(v, 1)) v &= 0xFFFFu;
                                asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + e * 4), "r"(v) : "memory");
                            }
                            if (lane == 0) sh.odd[u_no % kMeta] = u_no + 1;
                        }
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full);
                }
                st += 2;
                if (st >= ST) { st -= ST; ph ^= 1; }
                pg = nxt;
            }
            u_no++;
        } while (ok && w.next());
        if (!ok) {
            // leave no copy in flight behind
            if (lane == 0)
                for (uint32_t k = 0; k < (ST + 1) / 2 && k < tile_no; k++) {
                    if (st < 2) { st += ST; ph ^= 1; }
                    st -= 2;
                    mbar_drain(smem_addr(&sh.full[st]), ph);
                }
            __syncwarp();
        }
      } else if (wid == 1) {
        // ---- products ----
        const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        const uint32_t id_qk = inst_desc(f, 128, kK, 0), id_pv = inst_desc(f, 128, DP, 1);
        const uint32_t q_lo = desc_lo(q_s, 16), k_lo = desc_lo(ring, 16), v_lo = desc_lo(ring, kK * 128);
        uint32_t st = 0, ph = 0, q_ph[2] = {0, 0}, p_ph[2] = {0, 0}, s_no = 0;
        bool ok = true;
        const bool one = elect_one();
        auto wait = [&](ull &bar, uint32_t parity) {
            if (ok) ok = mbar_wait(smem_addr(&bar), parity, dead);
            ok = __all_sync(0xFFFFFFFFu, ok);
        };
        // scores of half x into the one buffer, once its last ones are read
        auto qk = [&](int x, uint32_t stage) {
            wait(sh.s_free, (s_no & 1) ^ 1);
            s_no++;
            if (!ok) return;
            tm_after();
            if (one) {
                const uint32_t qa = q_lo + x * (128 * DP * 2 >> 4), ka = k_lo + stage * (Cfg::tile >> 4);
#pragma unroll
                for (int k = 0; k < DP / 16; k++) {
                    const uint32_t o = ((k >> 2) * kK * 128 + (k & 3) * 32) >> 4;
                    mma_ss(tm + kS, qa + o, ka + o, id_qk, k > 0);
                }
                tm_commit(smem_addr(&sh.s_full[x]));
            }
            __syncwarp();
        };
        auto release = [&](uint32_t stage) {
            if (one) tm_commit(smem_addr(&sh.empty[stage]));
            __syncwarp();
        };
        do {
            const int nx = w.live() > 128 ? 2 : 1;
            uint32_t ks = st;
            wait(sh.full[ks], ph);
            for (int x = 0; ok && x < nx; x++) {
                wait(sh.q_full[x], q_ph[x]);
                q_ph[x] ^= 1;
                if (ok) qk(x, ks);
            }
            if (!ok) break;
            release(ks);
            if (++st == ST) { st = 0; ph ^= 1; }
            for (uint32_t t = w.t0; ok && t < w.t1; t++) {
                const bool more = t + 1 < w.t1;
                const uint32_t vs = st;
                wait(sh.full[vs], ph);
                if (++st == ST) { st = 0; ph ^= 1; }
                if (more) {
                    ks = st;
                    wait(sh.full[ks], ph);
                    if (++st == ST) { st = 0; ph ^= 1; }
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    if (!ok || x >= nx) break;
                    // the next scores first: their half reads them as soon as
                    // its weights are out
                    if (more) qk(x, ks);
                    wait(sh.p_full[x], p_ph[x]);
                    p_ph[x] ^= 1;
                    if (!ok) break;
                    tm_after();
                    if (one) {
                        const uint32_t va = v_lo + vs * (Cfg::tile >> 4);
#pragma unroll
                        for (int k = 0; k < kK / 16; k++)
                            mma_ts(tm + 256 + x * 128, tm + (x ? kP1 : kP0) + k * 8, va + k * (2048 >> 4), id_pv,
                                   k > 0 || t > w.t0);
                        tm_commit(smem_addr(&sh.o_full[x]));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                release(vs);
                if (more) release(ks);
            }
        } while (ok && w.next());
        if (!ok) {
            if (one) {
                tm_commit(smem_addr(&sh.drain));
                mbar_drain(smem_addr(&sh.drain), 0);
            }
            __syncwarp();
        }
      }
    } else {
        regs_up<208>();
        // ---- softmax of one half ----
        const int x = (wid - 4) >> 2;
        const uint32_t r = threadIdx.x - 128 - x * 128;    // row of the half
        const uint32_t lanes = (wid & 3) << 21;            // first lane of this warp, in a TMEM address
        const uint32_t S = tm + kS + lanes, P = tm + (x ? kP1 : kP0) + lanes, O = tm + 256 + x * 128 + lanes;
        uint32_t s_ph = 0, o_ph = 0, tile_no = 0, u_no = 0;
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
            u_no++;
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
                tm_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.s_free));
                const int k0 = (int)((w.first + t) * kK);
                const uint4 mk = *(const uint4 *)sh.mask[tile_no % kMeta];
                const bool masked = k0 < all_lo || k0 + (int)kK - 1 > all_hi ||
                                    (mk.x & mk.y & mk.z & mk.w) != 0xFFFFFFFFu;
                if (masked) {
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
                float mx[4];
#pragma unroll
                for (int k = 0; k < 4; k++) mx[k] = fmaxf(s[k], s[k + 4]);
#pragma unroll
                for (int j = 8; j < 128; j += 8)
#pragma unroll
                    for (int k = 0; k < 4; k++) mx[k] = max3(mx[k], s[j + k], s[j + k + 4]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                // the scale is positive here
                const float ms = fmaf(top, a.sl2, -weight_bias<T>(kGrow<T>));
                if (t == w.t0) {
                    m = ms;
                } else {
                    // the last product has read P and written O
                    ok = mbar_wait(smem_addr(&sh.o_full[x]), o_ph, dead);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    o_ph ^= 1;
                    tm_after();
                    const bool grow = ms > m + kGrow<T> || (m == -INFINITY && ms > m);
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
                        const float *e = s + c * 32 + 2 * j;
                        float u, v;
                        unf2(fma2(f2(e[0], e[1]), sl2, nm2), &u, &v);
                        u = ex2(u);
                        v = ex2(v);
                        l2[j & 1] = add2(l2[j & 1], f2(u, v));
                        pk[j] = pack2<T>(u, v);
                    }
                    tm_st16(P + c * 16, pk);
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
            uint32_t skipped = 0, units = 1;
            while (live && x == 1 && u.live() <= 128) {
                skipped += u.t1 - u.t0;
                units++;
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
            // (a later unit of the same place asks for a look that finds nothing)
            const bool whole = w.t0 == 0 && w.t1 == w.nt, odd = sh.odd[u_no % kMeta] > u_no;
            const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
            float *sl = slot_of(sp.ws, 2 * blockIdx.x + (w.t0 == 0 ? 1 : 0), kR, p.D);
            char *dst = a.out.p + (long long)ri.row * a.out.row_b + (long long)ri.head * a.out.head_b;
#pragma unroll 1
            for (int c = 0; c < DP / 32; c++) {
                float o[32];
                tm_ld32(O + c * 32, o);
                tm_wait_ld();
                if (odd && ri.row >= 0) {
                    // rare: look the tokens over that only some rows attend to
                    const int u_hi = row_info(g, w.s, w.at.h, w.at.rt * kR).hi;
                    const int u_lo = row_info(g, w.s, w.at.h, w.at.rt * kR + w.live() - 1).lo;
                    const int key_a = max((int)((w.first + w.t0) * kK), ri.lo);
                    const int key_e = min((int)((w.first + w.t1) * kK) - 1, ri.hi);
                    for (int key = key_a; key <= key_e; key++) {
                        const int tile0 = key / (int)kK * (int)kK;
                        if (tile0 >= u_lo && tile0 + (int)kK - 1 <= u_hi) continue;
                        const uint32_t blk = (uint32_t)key / p.bs;
                        const int pg = page_of(b, p.n_pages, w.at.i, w.at.h, blk);
                        if (pg < 0) continue;
                        const T *v = (const T *)(p.v + pg * p.page_b + w.at.h * p.head_b +
                                                 (long long)((uint32_t)key - blk * p.bs.d) * p.tok_b) + c * 32;
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if ((uint32_t)(c * 32 + j) < p.D && !isfinite(to_f(v[j]))) o[j] = NAN;
                    }
                }
                __syncwarp();
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
            u_no += units;
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
    const Geo g = {kR, kK, a.G, p.H, a.window, cl.min_rows, cl.max_rows, kJoinKeys};
    auto k = attend_tile_kernel<T, DP>;
    static std::atomic<uint64_t> done;
    OKV_CUDA_TRY(allow_smem(k, TileCfg<DP>::smem, done));
    k<<<sp.ctas, kThreads, TileCfg<DP>::smem, s>>>(km, vm, g, p, b, a, sp, p.head_b == 0);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    if (sp.ctas > 1 && may_cut(g, (ull)b.width * p.bs.d)) {
        OKV_CUDA_TRY(launch_after(join_kernel<T, 256>, (sp.ctas - 1) * 8, 256, 0, s, g, p, b, a, sp, 8u));
        note_launches(1);
    }
    return ORCHKV_OK;
}

// ---- masses of chunks --------------------------------------------------------------
//
// The product is turned round: the 128 keys of a tile are the rows of the
// accumulator, so a thread owns a key and its sum over all query rows is a sum
// of its own lane's columns, with no exchange between threads.  Nothing but the
// sums leaves the CTA: 2 D products a score against one power of two, so the
// special function unit (16 a clock) would take twice the tensor core's time; a
// quarter of the powers go to the FMA units as polynomials (ex2_poly), where a
// pair costs what it costs the other unit.  A unit is 256 keys (two tiles)
// against the rows that may attend to them; the K tiles stay, the query rows
// stream through a ring (by TMA: a box of G heads by 128/G tokens is 128 packed
// rows).  Two groups of four warps work on each K tile, on every other query
// tile, so four warps a scheduler hide each other's latencies.  CTAs cut the
// list of units as the attention does; pieces of one unit are added by
// mass_join_kernel in row order.
//
// 2048 new tokens over 14336, 32/8 heads of 128, bf16: 276 to 324 us over the
// devices and loads measured, 795 to 935 TFLOP/s, 0.48 to 0.57 of the measured
// matrix rate; of them 5 us keep NaN and infinities in the polynomials.  Before
// those: 363 us with one group a K tile, 308, 281, 275 and 294 us with 1/2, 3/8,
// 1/4 and none of the powers as polynomials.

constexpr int kMassThreads = 640;
constexpr int kMassPoly = 2;                           // of 8 pairs of powers, those on the FMA units
constexpr uint32_t kMK = 256;                          // keys of a unit

constexpr int kMassRing = 3;                           // query tiles

template <int DP> struct MassCfg {
    static constexpr uint32_t tile = 128 * DP * 2;
    static constexpr size_t tiles = (size_t)(4 + kMassRing) * tile;    // two units' keys, the ring
};

struct MassGeo {
    uint32_t G, H, window, min_rows, toks;             // toks: tokens of a query tile
};

// Key tiles of a sequence, and the tokens that may attend to one.
struct MassSeq {
    uint32_t kf, kn;                                   // unit k covers keys (kf + k) * 256, k < kn
};
__device__ __forceinline__ MassSeq mass_seq(const MassGeo &g, const SeqDev &s)
{
    MassSeq q = {0, 0};
    if ((uint32_t)s.m * g.G <= g.min_rows) return q;
    const int hi = s.len;
    int lo = g.window ? s.c0 - (int)g.window + 1 : 0;
    lo = lo < 0 ? 0 : lo;
    q.kf = (uint32_t)lo / kMK;
    const uint32_t kl = ((uint32_t)hi + kMK - 1) / kMK;
    q.kn = kl > q.kf ? kl - q.kf : 1;                  // one unit at least: it writes the zeros
    return q;
}
// Tokens [a, e) of the sequence's rows that may attend to keys [k0, k0 + 256).
__device__ __forceinline__ void mass_tokens(const MassGeo &g, const SeqDev &s, uint32_t k0, int *a, int *e)
{
    *a = max(0, (int)k0 - s.c0);
    *e = s.m;
    if (g.window) *e = min(s.m, (int)k0 + (int)kMK - 1 - s.c0 + (int)g.window);
    if (*e < *a) *e = *a;
}
// Weight of unit k: its tokens and 16 for the unit itself; without a window the
// tokens fall by 256 a unit from the sequence's first new key on.
__device__ __forceinline__ ull mass_before(const MassGeo &g, const SeqDev &s, const MassSeq &q, ull k)
{
    const ull m = s.m;
    if (g.window) return k * (min(m, (ull)g.window + kMK) + 16);
    const ull c0 = s.c0 > 0 ? s.c0 : 0, f = c0 / kMK;  // unit f still has every token
    ull v = k * (m + 16);
    if (k > f + 1) {
        const ull n = k - 1 - f;                       // units f+1 .. k-1
        v -= kMK * ((f + 1 + k - 1) * n / 2) - c0 * n;
    }
    return v;
}
__device__ __forceinline__ ull mass_weight(const MassGeo &g, const BatchDev &b, uint32_t bs, uint32_t i)
{
    const SeqDev s = load_seq(b, bs, i);
    const MassSeq q = mass_seq(g, s);
    return q.kn ? g.H * mass_before(g, s, q, q.kn) : 0;
}
// Query tiles of unit k, at least one.
__device__ __forceinline__ uint32_t mass_tiles(const MassGeo &g, const SeqDev &s, const MassSeq &q, uint32_t k)
{
    int a, e;
    mass_tokens(g, s, (q.kf + k) * kMK, &a, &e);
    const uint32_t n = ((uint32_t)(e - a) + g.toks - 1) / g.toks;
    return n ? n : 1;
}
__device__ __forceinline__ Pos mass_inside(const MassGeo &g, const SeqDev &s, uint32_t i, ull x)
{
    const MassSeq q = mass_seq(g, s);
    const ull U = mass_before(g, s, q, q.kn);
    Pos p;
    p.i = i;
    p.h = (uint32_t)quot(x, U);
    const ull y = x - (ull)p.h * U;
    uint32_t lo = 0, hi = q.kn;                        // the last k with before(k) <= y
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (mass_before(g, s, q, mid) <= y) lo = mid;
        else hi = mid;
    }
    p.rt = lo;
    const ull z = y - mass_before(g, s, q, lo), w = mass_before(g, s, q, lo + 1) - mass_before(g, s, q, lo);
    p.t = (uint32_t)quot(z * mass_tiles(g, s, q, lo), w);
    return p;
}

struct MassWalk {
    const MassGeo &g;
    const BatchDev &b;
    uint32_t bs;
    Pos at, end;
    SeqDev s;
    MassSeq q;
    uint32_t nt, t0, t1;
    int a, e;                                          // tokens of the unit
    bool stop;

    __device__ bool settle()
    {
        while (at.i < b.n) {
            s = load_seq(b, bs, at.i);
            q = mass_seq(g, s);
            if (q.kn == 0) { at = Pos{at.i + 1, 0, 0, 0}; continue; }
            stop = same_unit(at, end);
            mass_tokens(g, s, key0(), &a, &e);
            nt = mass_tiles(g, s, q, at.rt);
            t0 = at.t;
            t1 = stop ? end.t : nt;
            if (t0 < t1) return true;
            if (stop) return false;
            advance();
        }
        return false;
    }
    __device__ uint32_t key0() const { return (q.kf + at.rt) * kMK; }
    __device__ void advance()
    {
        at.t = 0;
        if (++at.rt == q.kn) {
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
};

struct MassShared {
    ull k_full[2], k_empty[2], q_full[kMassRing], q_empty[kMassRing], s_full[4], s_empty[4], drain, sums[3];
    uint32_t tmem;
    int dead;
    alignas(16) float lse[kMassRing][128];                     // of a query tile's rows, times -log2(e)
    alignas(16) float key[kMK];
    SplitShared split;
};

static_assert(MassCfg<128>::tiles + sizeof(MassShared) <= 232448, "over an SM's 227 KB");

// The zeros in front of a sequence's first unit and behind its last.
__device__ __forceinline__ void mass_zero_rest(const MassWalk &w, const BatchDev &b, const PagesDev &p, float *mass,
                                               uint32_t tid, uint32_t nt)
{
    float *out = mass + ((size_t)w.at.i * w.g.H + w.at.h) * b.width;
    const uint32_t per = kMK / p.bs.d;
    if (w.at.rt == 0)
        for (uint32_t k = tid; k < min(w.q.kf * per, b.width); k += nt) out[k] = 0.f;
    if (w.at.rt + 1 == w.q.kn)
        for (uint32_t k = (w.q.kf + w.q.kn) * per + tid; k < b.width; k += nt) out[k] = 0.f;
}

template <class T, int DP>
__global__ void __launch_bounds__(kMassThreads, 1)
mass_tile_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap qmap, MassGeo g,
                 PagesDev p, BatchDev b, MassDev a, SplitDev sp, int by_head)
{
    using Cfg = MassCfg<DP>;
    constexpr int RQ = kMassRing;
    constexpr uint32_t halves = DP / 64;
    // no static part, so the tiles start on the 1024 bytes their swizzle needs
    extern __shared__ __align__(1024) char raw[];
    MassShared &sh = *(MassShared *)(raw + Cfg::tiles);
    const uint32_t base = smem_addr(raw);
    if (base & 1023) {
        if (threadIdx.x == 0) g_paged_dead = 1;
        return;
    }
    const uint32_t keys_s = base, ring = base + 4 * Cfg::tile;
    const uint32_t wid = threadIdx.x >> 5, lane = threadIdx.x & 31;

    MassWalk w{g, b, p.bs.d};
    ull W;
    find_share<kMassThreads>(b, p.bs.d, blockIdx.x, sp.ctas, &sh.split, &w.at, &w.end, &W,
                             [&](uint32_t i) { return mass_weight(g, b, p.bs.d, i); },
                             [&](const SeqDev &s, uint32_t i, ull x, ull) { return mass_inside(g, s, i, x); });
    cudaTriggerProgrammaticLaunchCompletion();
    if (W == 0) return;
    if (!w.settle()) return;

    const uint32_t cols = g.toks * g.G;                    // of a query tile
    if (threadIdx.x == 0) {
        for (int k = 0; k < 2; k++) {
            mbar_init(smem_addr(&sh.k_full[k]), 1);
            mbar_init(smem_addr(&sh.k_empty[k]), 1);
        }
        for (int k = 0; k < RQ; k++) {
            mbar_init(smem_addr(&sh.q_full[k]), 2);
            mbar_init(smem_addr(&sh.q_empty[k]), 9);
        }
        for (int k = 0; k < 3; k++) mbar_init(smem_addr(&sh.sums[k]), k < 2 ? 8 : 16);
        for (int k = 0; k < 4; k++) {
            mbar_init(smem_addr(&sh.s_full[k]), 1);
            mbar_init(smem_addr(&sh.s_empty[k]), 4);
        }
        mbar_init(smem_addr(&sh.drain), 1);
        sh.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // rows of the query tiles that no box covers: zeros, not stale bits
    for (uint32_t e = threadIdx.x; e < RQ * (128 - cols) * halves * 8; e += kMassThreads) {
        const uint32_t c = e & 7, x = (e >> 3) % halves, r = (e >> 3) / halves;
        const uint32_t st = r / (128 - cols), row = cols + r - st * (128 - cols);
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                         ring + st * Cfg::tile + x * 128 * 128 + row * 128 + c * 16), "r"(0) : "memory");
    }
    for (uint32_t e = threadIdx.x; e < RQ * 128; e += kMassThreads) sh.lse[e >> 7][e & 127] = 0.f;
    for (uint32_t e = threadIdx.x; e < kMK; e += kMassThreads) sh.key[e] = 0.f;
    fence_async();
    if (wid == 1) tm_alloc(smem_addr(&sh.tmem), 512);
    tm_before();
    __syncthreads();
    tm_after();
    const uint32_t tm = sh.tmem;
    volatile int *dead = &sh.dead;

    if (wid < 4) {
      if (wid == 0) {
        // ---- loads ----
        const uint32_t bs = p.bs.d, per = bs < 128 ? 128 / bs : 1, box = bs < 128 ? bs : 128;
        uint32_t u_no = 0, st = 0, ph = 0, issued = 0;
        bool ok = true;
        do {
            const uint32_t kb = u_no & 1, k0 = w.key0();
            int pg[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t key = k0 + x * 128 + lane * bs;
                pg[x] = lane < per && (int)key < w.s.len ? page_of(b, p.n_pages, w.at.i, w.at.h, key / p.bs) : -1;
            }
            const uint32_t n = __popc(__ballot_sync(0xFFFFFFFFu, pg[0] >= 0)) +
                               __popc(__ballot_sync(0xFFFFFFFFu, pg[1] >= 0));
            ok = mbar_wait(smem_addr(&sh.k_empty[kb]), (u_no >> 1 & 1) ^ 1, dead);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            const uint32_t kbar = smem_addr(&sh.k_full[kb]);
            if (lane == 0) mbar_expect(kbar, n * box * 128 * halves);
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 2; x++)
                if (pg[x] >= 0)
#pragma unroll
                    for (uint32_t c = 0; c < halves; c++)
                        tma4(keys_s + (kb * 2 + x) * Cfg::tile + c * 128 * 128 + lane * box * 128, &kmap,
                             (int)c * 64, bs < 128 ? 0 : (int)((k0 + x * 128) % bs), by_head ? 0 : (int)w.at.h,
                             pg[x], kbar);
            u_no++;
            for (uint32_t t = w.t0; t < w.t1; t++) {
                ok = mbar_wait(smem_addr(&sh.q_empty[st]), ph ^ 1, dead);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t bar = smem_addr(&sh.q_full[st]);
                    mbar_expect(bar, cols * 128 * halves);
                    const int row = w.s.start + w.a + (int)(t * g.toks);
#pragma unroll
                    for (uint32_t c = 0; c < halves; c++)
                        tma3(ring + st * Cfg::tile + c * 128 * 128, &qmap, (int)c * 64, (int)(w.at.h * g.G), row, bar);
                }
                __syncwarp();
                issued++;
                if (++st == RQ) { st = 0; ph ^= 1; }
            }
        } while (ok && w.next());
        if (!ok) {
            // leave no copy in flight behind
            if (lane == 0) {
                for (uint32_t k = 0; k < (uint32_t)RQ && k < issued; k++) {
                    st = st == 0 ? RQ - 1 : st - 1;
                    if (st == RQ - 1) ph ^= 1;
                    mbar_drain(smem_addr(&sh.q_full[st]), ph);
                }
                for (uint32_t k = 0; k < 2 && k < u_no; k++)
                    mbar_drain(smem_addr(&sh.k_full[(u_no - 1 - k) & 1]), (u_no - 1 - k) >> 1 & 1);
            }
            __syncwarp();
        }
      } else if (wid == 1) {
        // ---- products ----
        const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        const uint32_t id = inst_desc(f, 128, 128, 0);
        const uint32_t k_lo = desc_lo(keys_s, 16), q_lo = desc_lo(ring, 16);
        uint32_t u_no = 0, st = 0, ph = 0, tile = 0;
        bool ok = true;
        const bool one = elect_one();
        auto wait = [&](ull &bar, uint32_t parity) {
            if (ok) ok = mbar_wait(smem_addr(&bar), parity, dead);
            ok = __all_sync(0xFFFFFFFFu, ok);
        };
        do {
            const uint32_t kb = u_no & 1;
            wait(sh.k_full[kb], u_no >> 1 & 1);
            for (uint32_t t = w.t0; ok && t < w.t1; t++, tile++) {
                wait(sh.q_full[st], ph);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t sb = x * 2 + (tile & 1);
                    wait(sh.s_empty[sb], (tile >> 1 & 1) ^ 1);
                    if (!ok) break;
                    tm_after();
                    if (one) {
                        const uint32_t ka = k_lo + (kb * 2 + x) * (Cfg::tile >> 4), qa = q_lo + st * (Cfg::tile >> 4);
#pragma unroll
                        for (int k = 0; k < DP / 16; k++) {
                            const uint32_t o = ((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4;
                            mma_ss(tm + sb * 128, ka + o, qa + o, id, k > 0);
                        }
                        tm_commit(smem_addr(&sh.s_full[sb]));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (one) tm_commit(smem_addr(&sh.q_empty[st]));
                __syncwarp();
                if (++st == RQ) { st = 0; ph ^= 1; }
            }
            if (ok && one) tm_commit(smem_addr(&sh.k_empty[kb]));
            __syncwarp();
            u_no++;
        } while (ok && w.next());
        if (!ok) {
            if (one) {
                tm_commit(smem_addr(&sh.drain));
                mbar_drain(smem_addr(&sh.drain), 0);
            }
            __syncwarp();
        }
      } else if (wid == 2) {
        // ---- the rows' lse ----
        uint32_t st = 0, ph = 0;
        bool ok = true;
        do {
            for (uint32_t t = w.t0; t < w.t1; t++) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t c = lane + 32 * k, j = c / g.G;
                    const int tok = w.a + (int)(t * g.toks + j);
                    v[k] = c < cols ? 0.f : -INFINITY; // a column of no row weighs nothing
                    if (c < cols && tok < w.e)
                        v[k] = a.lse[(size_t)(w.s.start + tok) * a.Hq + w.at.h * g.G + (c - j * g.G)] * -kLog2e;
                }
                ok = mbar_wait(smem_addr(&sh.q_empty[st]), ph ^ 1, dead);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < 4; k++) sh.lse[st][lane + 32 * k] = v[k];
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.q_full[st]));
                if (++st == RQ) { st = 0; ph ^= 1; }
            }
        } while (ok && w.next());
      }
    } else {
        // ---- sums of one half's keys, over every other query tile ----
        const int x = (wid - 4) >> 2 & 1;
        const uint32_t y = (wid - 4) >> 3;                 // the tiles of this parity
        const uint32_t r = (threadIdx.x - 128) & 127;
        const uint32_t lanes = (wid & 3) << 21;
        const ull sl2 = f2(a.sl2, a.sl2);
        uint32_t st = 0, ph = 0, tile = 0, sum_ph = 0;
        bool ok = true, live = true;
        while (live && ok) {
            const int key = (int)(w.key0() + x * 128 + r);
            const uint32_t blk = (uint32_t)key / p.bs;
            const bool there = key < w.s.len && page_of(b, p.n_pages, w.at.i, w.at.h, blk) >= 0;
            // tokens [ja, je) of the rows attend to this key
            const int ja = max(0, key - w.s.c0);
            int je = w.s.m;
            if (g.window) je = min(je, key - w.s.c0 + (int)g.window);
            ull sum[2] = {0, 0};
            for (uint32_t t = w.t0; t < w.t1; t++, tile++) {
                if ((tile & 1) != y) {
                    if (++st == RQ) { st = 0; ph ^= 1; }
                    continue;
                }
                const uint32_t sb = x * 2 + y;
                ok = mbar_wait(smem_addr(&sh.s_full[sb]), tile >> 1 & 1, dead) &&
                     mbar_wait(smem_addr(&sh.q_full[st]), ph, dead);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tm_after();
                const uint32_t S = tm + sb * 128 + lanes;
                const int j0 = w.a + (int)(t * g.toks);
                int lo = (ja - j0) * (int)g.G, hi = (min(je, w.e) - j0) * (int)g.G;
                lo = lo < 0 ? 0 : lo;
                hi = hi > (int)cols ? (int)cols : hi;
                if (!there) hi = 0;
                const bool all = __all_sync(0xFFFFFFFFu, lo == 0 && hi == (int)cols);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float s[32];
                    tm_ld32(S + c * 32, s);
                    tm_wait_ld();
                    if (c == 3) {                      // the scores are all read
                        tm_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_addr(&sh.s_empty[sb]));
                    }
                    const float4 *ls = (const float4 *)&sh.lse[st][c * 32];
                    // (columns of no row are masked: their zeros times an
                    // infinite key are not 0)
                    if (all && cols >= c * 32 + 32) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float4 l4 = ls[j];
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const ull z = fma2(f2(s[4 * j + 2 * k], s[4 * j + 2 * k + 1]), sl2,
                                                   k ? f2(l4.z, l4.w) : f2(l4.x, l4.y));
                                if ((2 * j + k) * kMassPoly % 8 < kMassPoly) {
                                    sum[k] = add2(sum[k], ex2_poly(z));
                                } else {
                                    float e0, e1;
                                    unf2(z, &e0, &e1);
                                    sum[k] = add2(sum[k], f2(ex2(e0), ex2(e1)));
                                }
                            }
                        }
                    } else {
                        const int l0 = lo - c * 32, h0 = hi - c * 32;
                        uint32_t bits = h0 <= 0 ? 0u : h0 >= 32 ? 0xFFFFFFFFu : (1u << h0) - 1;
                        bits &= l0 > 31 ? 0u : l0 <= 0 ? 0xFFFFFFFFu : ~((1u << l0) - 1);
                        if (__any_sync(0xFFFFFFFFu, bits != 0)) {
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                const float4 l4 = ls[j];
                                const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
                                float e[4];
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    e[k] = bits >> (4 * j + k) & 1 ? ex2(s[4 * j + k] * a.sl2 + lv[k]) : 0.f;
                                sum[0] = add2(sum[0], f2(e[0], e[1]));
                                sum[1] = add2(sum[1], f2(e[2], e[3]));
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.q_empty[st]));
                if (++st == RQ) { st = 0; ph ^= 1; }
            }
            if (!ok) break;
            float s0, s1, s2, s3;
            unf2(sum[0], &s0, &s1);
            unf2(sum[1], &s2, &s3);
            // two terms onto zero: the same whichever comes first
            atomicAdd(&sh.key[x * 128 + r], (s0 + s1) + (s2 + s3));
            const bool whole = w.t0 == 0 && w.t1 == w.nt;
            const uint32_t bs = p.bs.d;
            // blocks of at most 128 keys belong to one group, larger ones to both
            const bool both = bs > 128;
            const uint32_t bar = smem_addr(&sh.sums[both ? 2 : x]);
            auto meet = [&] {                          // of the threads that add a block's keys
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
                ok = mbar_wait(bar, sum_ph, dead);
                ok = __all_sync(0xFFFFFFFFu, ok);
                sum_ph ^= 1;
            };
            meet();
            if (!ok) break;
            const uint32_t nb = both ? 1 : 128 / bs;
            if (y == 0 && r < nb && !(both && x == 1)) {
                float v = 0.f;
                for (uint32_t k = 0; k < bs; k++) {
                    v += sh.key[x * 128 + r * bs + k];
                    sh.key[x * 128 + r * bs + k] = 0.f;
                }
                const uint32_t lb = (both ? 0 : x * nb) + r;          // block of the unit
                const uint32_t gb = w.key0() / bs + lb;
                if (!whole) sp.ws[(size_t)(2 * blockIdx.x + (w.t0 == 0 ? 1 : 0)) * kMassSlot + lb] = v;
                else if (gb < b.width) a.mass[((size_t)w.at.i * g.H + w.at.h) * b.width + gb] = v;
            }
            if (w.t0 == 0 && y == 0) mass_zero_rest(w, b, p, a.mass, x * 128 + r, 256);
            meet();
            live = w.next();
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && sh.dead) g_paged_dead = 1;
    if (wid == 1) tm_free(tm, 512);
}

// Pieces of cut units: slots as join_kernel finds them.
__global__ void __launch_bounds__(128)
mass_join_kernel(MassGeo g, PagesDev p, BatchDev b, MassDev a, SplitDev sp)
{
    __shared__ SplitShared sh;
    __shared__ uint32_t slots[kMaxPieces];
    const uint32_t c = blockIdx.x + 1;
    Pos prev, at;
    ull W;
    find_share<128>(b, p.bs.d, c - 1, sp.ctas, &sh, &prev, &at, &W,
                    [&](uint32_t i) { return mass_weight(g, b, p.bs.d, i); },
                    [&](const SeqDev &s, uint32_t i, ull x, ull) { return mass_inside(g, s, i, x); });
    // (no block ends before the kernel in front: the next launch counts on that)
    if (W == 0 || at.i >= b.n || at.t == 0 || (same_unit(prev, at) && prev.t > 0)) {
        cudaGridDependencySynchronize();
        return;
    }
    __syncthreads();
    const SeqDev s = load_seq(b, p.bs.d, at.i);
    const MassSeq q = mass_seq(g, s);
    const uint32_t K = find_pieces<128>(b, c, sp.ctas, at, sh.off[1], quot(W + sp.ctas - 1, sp.ctas),
                                        at.h * mass_before(g, s, q, q.kn) + mass_before(g, s, q, at.rt + 1),
                                        mass_tiles(g, s, q, at.rt), slots,
                                        [&](ull x) { return mass_inside(g, s, at.i, x); });
    const uint32_t nb = kMK / p.bs.d, lb = threadIdx.x, gb = (q.kf + at.rt) * nb + lb;
    cudaGridDependencySynchronize();
    if (lb >= nb || gb >= b.width) return;
    float y = 0.f;
#pragma unroll 4
    for (uint32_t k = 0; k < K; k++)
        y += sp.ws[(size_t)slots[k] * kMassSlot + lb];
    a.mass[((size_t)at.i * g.H + at.h) * b.width + gb] = y;
}

template <class T, int DP>
int go_mass(const CUtensorMap &km, const CUtensorMap &qm, const MassGeo &g, const PagesDev &p, const BatchDev &b,
            const MassDev &a, const SplitDev &sp, cudaStream_t s)
{
    auto k = mass_tile_kernel<T, DP>;
    const size_t smem = MassCfg<DP>::tiles + sizeof(MassShared);
    static std::atomic<uint64_t> done;
    OKV_CUDA_TRY(allow_smem(k, smem, done));
    k<<<sp.ctas, kMassThreads, smem, s>>>(km, qm, g, p, b, a, sp, p.head_b == 0);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    if (sp.ctas > 1) {
        OKV_CUDA_TRY(launch_after(mass_join_kernel, sp.ctas - 1, 128, 0, s, g, p, b, a, sp));
        note_launches(1);
    }
    return ORCHKV_OK;
}

}  // namespace

namespace {

CUresult encode_map(CUtensorMap *m, int dtype, int rank, const char *base, const cuuint64_t *dims,
                    const cuuint64_t *strides, const cuuint32_t *box)
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
    if (!encode) return CUDA_ERROR_NOT_SUPPORTED;
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return encode(m, dtype == DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  rank, (void *)base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

}  // namespace

bool page_map(CUtensorMap *m, const PagesDev &p, const char *base, int dtype)
{
    // pages of one head: a head axis of one entry
    const bool by_head = p.head_b == 0;
    const cuuint64_t dims[4] = {p.D, p.bs.d, by_head ? 1 : p.H, p.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)p.tok_b, (cuuint64_t)(by_head ? p.tok_b : p.head_b),
                                   (cuuint64_t)p.page_b};
    const cuuint32_t box[4] = {64, p.bs.d < 128 ? p.bs.d : 128, 1, 1};
    return encode_map(m, dtype, 4, base, dims, strides, box) == CUDA_SUCCESS;
}

bool rows_map(CUtensorMap *m, const RowsDev &q, uint32_t D, uint32_t Hq, uint32_t rows, uint32_t G,
              uint32_t toks, int dtype)
{
    const cuuint64_t dims[3] = {D, Hq, rows};
    const cuuint64_t strides[2] = {(cuuint64_t)q.head_b, (cuuint64_t)q.row_b};
    const cuuint32_t box[3] = {64, G, toks};
    return encode_map(m, dtype, 3, q.p, dims, strides, box) == CUDA_SUCCESS;
}

// 16-bit pages whose tokens fill whole boxes; a scale that keeps the order of
// the scores (the mask is applied before it).
bool attend_tile_takes(const PagesDev &p, int dtype, float sl2)
{
    return dtype != DTYPE_FP32 && pages_tile(p) && sl2 > 0.f && p.page_b > 0 && p.tok_b > 0 &&
           p.page_b < (1ll << 40) && p.head_b < (1ll << 40) && p.tok_b < (1ll << 40);
}

// Besides: whole blocks in a unit's 256 keys, a group of at most 128 heads,
// row strides that a tensor map takes.
bool mass_tile_takes(const PagesDev &p, int dtype, float sl2, const RowsDev &q, uint32_t G)
{
    return attend_tile_takes(p, dtype, sl2) && kMK % p.bs.d == 0 && G <= 128 && q.head_b > 0 && q.row_b > 0 &&
           q.head_b < (1ll << 40) && q.row_b < (1ll << 40);
}

uint32_t mass_tile_ctas(unsigned long long units, unsigned long long rows)
{
    const unsigned long long tiles = units * ((rows + 63) / 64);
    return (uint32_t)(tiles < 148 ? tiles : 148);
}

int launch_mass_tile(int dtype, const PagesDev &p, const BatchDev &b, const MassDev &a, const ClassDev &cl,
                     const SplitDev &sp, cudaStream_t s)
{
    const MassGeo g = {a.G, p.H, a.window, cl.min_rows, 128 / a.G};
    CUtensorMap km, qm;
    if (!page_map(&km, p, p.k, dtype) || !rows_map(&qm, a.q, p.D, a.Hq, b.rows, a.G, g.toks, dtype))
        return ORCHKV_ERR_CUDA;
    if (dtype == DTYPE_BF16)
        return p.D <= 64 ? go_mass<__nv_bfloat16, 64>(km, qm, g, p, b, a, sp, s)
                         : go_mass<__nv_bfloat16, 128>(km, qm, g, p, b, a, sp, s);
    return p.D <= 64 ? go_mass<__half, 64>(km, qm, g, p, b, a, sp, s)
                     : go_mass<__half, 128>(km, qm, g, p, b, a, sp, s);
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

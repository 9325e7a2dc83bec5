// paged_simt.cu — attention over pages and block masses on the CUDA cores,
// for fp32 pages: the tensor cores have no 24-bit product, so these run the
// formula in plain fp32.
//
// A warp takes 32 keys at a time.  For the scores a lane owns a key (its row
// of K comes 16 bytes at a time, eight query rows broadcast from shared
// memory), so the maximum and the sum of a softmax step are one warp reduction
// each for 32 keys; for the values a lane owns dimensions and the rows of V
// come whole.  A score that the mask drops adds nothing (its value is not
// multiplied by 0), so nothing stored there reaches a row.  1 request x 1 token
// over 901, 32/8 heads of 128: 30 us (bytes: 1.1); 32 x 1 over 4000: 805 us (160),
// masses 202 (80); 512 over 3584: 3.95 ms, masses 2.69 ms.  A unit computes 8 rows
// whatever the group is, and loads no value before its scores are ready.
#include "kernels.h"
#include "paged_split.cuh"

namespace okv {
namespace {

constexpr int kW = 4;                              // warps of a CTA
constexpr int R = kSimtRows;
constexpr int kD = 256;

// Scores of this lane's key against the R rows in q_s (already scaled).
__device__ __forceinline__ void dots(const char *krow, const float (*q_s)[kD], uint32_t D, float *sc)
{
#pragma unroll
    for (int r = 0; r < R; r++) sc[r] = 0.f;
#pragma unroll 4
    for (uint32_t d = 0; d < D; d += 4) {
        const float4 k = __ldg((const float4 *)(krow + (size_t)d * 4));
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float4 q = *(const float4 *)&q_s[r][d];
            sc[r] += q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
        }
    }
}

__device__ __forceinline__ void load_q(const RowsDev &q, const RowInfo *ri, float sl2, uint32_t D,
                                       float (*q_s)[kD], int tid, int nt)
{
    for (uint32_t e = tid; e < R * D; e += nt) {
        const uint32_t r = e / D, d = e - r * D;
        float x = 0.f;
        if (ri[r].row >= 0)
            x = ((const float *)(q.p + (long long)ri[r].row * q.row_b +
                                 (long long)ri[r].head * q.head_b))[d] * sl2;
        q_s[r][d] = x;
    }
}

__global__ void __launch_bounds__(kW * 32)
attend_simt_kernel(Geo g, PagesDev p, BatchDev b, AttendDev a, SplitDev sp)
{
    __shared__ __align__(16) float q_s[R][kD];
    __shared__ __align__(16) float acc_s[kW][R][kD];
    __shared__ float m_s[kW][R], l_s[kW][R];
    __shared__ RowInfo ri[R];
    __shared__ SplitShared sh;
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5, D = p.D;
    Pos at, end;
    ull W;
    find_share<kW * 32>(g, b, p.bs.d, blockIdx.x, sp.ctas, &sh, &at, &end, &W);
    if (W == 0) return;
    while (at.i < b.n) {
        const SeqDev s = load_seq(b, p.bs.d, at.i);
        const uint32_t RT = row_tiles(g, s);
        if (RT == 0) { at = Pos{at.i + 1, 0, 0, 0}; continue; }
        if (at.i > end.i) break;                           // the end was a sequence without units
        if (same_unit(at, end) && end.t == 0) break;
        uint32_t first, nt;
        key_tiles(g, s, at.rt, &first, &nt);
        const bool stop = same_unit(at, end);
        const uint32_t t0 = at.t, t1 = stop ? end.t : nt;
        if (t0 < t1) {
            __syncthreads();
            if (threadIdx.x < R) ri[threadIdx.x] = row_info(g, s, at.h, at.rt * R + threadIdx.x);
            __syncthreads();
            load_q(a.q, ri, a.sl2, D, q_s, threadIdx.x, kW * 32);
            __syncthreads();
            float m[R], l[R], acc[R][2][4];
#pragma unroll
            for (int r = 0; r < R; r++) {
                m[r] = -INFINITY;
                l[r] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) acc[r][j / 4][j % 4] = 0.f;
            }
            for (uint32_t t = t0; t < t1; t++) {
                const int key = (int)((first + t) * kSimtKeys + wid * 32 + lane);
                int pg = -1;
                uint32_t blk = 0;
                if (key < s.len) {
                    blk = (uint32_t)key / p.bs;
                    pg = page_of(b, p.n_pages, at.i, at.h, blk);
                }
                bool any = false;
#pragma unroll
                for (int r = 0; r < R; r++) any |= pg >= 0 && key <= ri[r].hi && key >= ri[r].lo;
                if (!__any_sync(0xFFFFFFFFu, any)) continue;
                const long long off = pg * p.page_b + at.h * p.head_b +
                                      (long long)(key - (int)(blk * p.bs.d)) * p.tok_b;
                float sc[R];
#pragma unroll
                for (int r = 0; r < R; r++) sc[r] = -INFINITY;
                if (any) {
                    dots(p.k + off, q_s, D, sc);
#pragma unroll
                    for (int r = 0; r < R; r++)
                        if (!(key <= ri[r].hi && key >= ri[r].lo)) sc[r] = -INFINITY;
                }
                uint32_t hit = 0;
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const bool on = any && key <= ri[r].hi && key >= ri[r].lo;
                    float mx = sc[r];
#pragma unroll
                    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
                    mx = fmaxf(mx, m[r]);
                    const float ms = mx == -INFINITY ? 0.f : mx;
                    const float f = exp2f(m[r] - ms);
                    m[r] = mx;
                    float e = on ? exp2f(sc[r] - ms) : 0.f;
                    sc[r] = e;
                    hit |= on ? 1u << r : 0u;
#pragma unroll
                    for (int o = 16; o; o >>= 1) e += __shfl_xor_sync(0xFFFFFFFFu, e, o);
                    l[r] = l[r] * f + e;
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[r][j / 4][j % 4] *= f;
                }
#pragma unroll 4
                for (int kk = 0; kk < 32; kk++) {
                    const uint32_t hk = __shfl_sync(0xFFFFFFFFu, hit, kk);
                    const long long vo = __shfl_sync(0xFFFFFFFFu, off, kk);
                    float v[2][4] = {};
                    if (hk) {
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t d = j * 128 + lane * 4;
                            if (d < D) {
                                const float4 x = __ldg((const float4 *)((const float *)(p.v + vo) + d));
                                v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const float pr = __shfl_sync(0xFFFFFFFFu, sc[r], kk);
                        if (hk >> r & 1)
#pragma unroll
                            for (int j = 0; j < 8; j++) acc[r][j / 4][j % 4] += pr * v[j / 4][j % 4];
                    }
                }
            }
            // the warps' parts of every row, then the rows out
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (lane == 0) { m_s[wid][r] = m[r]; l_s[wid][r] = l[r]; }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t d = (j / 4) * 128 + lane * 4 + j % 4;
                    if (d < D) acc_s[wid][r][d] = acc[r][j / 4][j % 4];
                }
            }
            __syncthreads();
            const bool whole = t0 == 0 && t1 == nt;
            float *sl = whole ? nullptr
                              : slot_of(sp.ws, 2 * blockIdx.x + (t0 == 0 ? 1 : 0), R, D);
            for (uint32_t e = threadIdx.x; e < R * D; e += kW * 32) {
                const uint32_t r = e / D, d = e - r * D;
                float M = -INFINITY;
#pragma unroll
                for (int k = 0; k < kW; k++) M = fmaxf(M, m_s[k][r]);
                const float Ms = M == -INFINITY ? 0.f : M;
                float L = 0.f, o = 0.f;
#pragma unroll
                for (int k = 0; k < kW; k++) {
                    const float w = exp2f(m_s[k][r] - Ms);
                    L += w * l_s[k][r];
                    o += w * acc_s[k][r][d];
                }
                if (!whole) {
                    sl[2 * R + r * D + d] = o;
                    if (d == 0) { sl[r] = M; sl[R + r] = L; }
                } else if (ri[r].row >= 0) {
                    const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
                    ((float *)(a.out.p + (long long)ri[r].row * a.out.row_b +
                               (long long)ri[r].head * a.out.head_b))[d] = o * inv;
                    if (a.lse && d == 0)
                        a.lse[(size_t)ri[r].row * a.Hq + ri[r].head] =
                            L > 0.f ? (Ms + log2f(L)) * 0.69314718055994531f
                                    : L == 0.f ? -INFINITY : L;
                }
            }
        }
        if (stop) break;
        at.t = 0;
        if (++at.rt == RT) {
            at.rt = 0;
            if (++at.h == g.H) { at.h = 0; at.i++; }
        }
    }
}

// Masses: a warp takes whole blocks of one (sequence, head), as many as fit 32
// keys, and walks over all the rows that may attend to them.
__global__ void __launch_bounds__(kW * 32)
mass_simt_kernel(Geo g, PagesDev p, BatchDev b, MassDev a, uint32_t per_warp, uint32_t groups)
{
    __shared__ __align__(16) float q_s[R][kD];
    __shared__ RowInfo ri[R];
    __shared__ float lse_s[R];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint32_t per_cta = kW * per_warp;
    const uint32_t x = blockIdx.x % groups, ih = blockIdx.x / groups;
    const uint32_t h = ih % p.H, i = ih / p.H;
    const SeqDev s = load_seq(b, p.bs.d, i);
    const uint32_t rows = (uint32_t)s.m * g.G;
    if (rows <= g.min_rows && g.min_rows) return;
    if (rows > g.max_rows) return;
    const uint32_t b0 = x * per_cta + wid * per_warp;
    const uint32_t keys = per_warp * p.bs.d;       // of one warp; over 32 only with one block
    float tot = 0.f;
    for (uint32_t k0 = 0; k0 < keys; k0 += 32) {
        const uint32_t kk = k0 + lane;
        const int key = kk < keys ? (int)(b0 * p.bs.d + kk) : 0x7FFFFFFF;
        const uint32_t blk = b0 + kk / p.bs;
        int pg = -1;
        if (key < s.len && blk < b.width) pg = page_of(b, p.n_pages, i, h, blk);
        const long long off = pg * p.page_b + h * p.head_b +
                              (long long)(kk - kk / p.bs * p.bs.d) * p.tok_b;
        float sum = 0.f;
        for (uint32_t r0 = 0; r0 < rows; r0 += R) {
            __syncthreads();
            if (threadIdx.x < R) {
                const RowInfo q = row_info(g, s, h, r0 + threadIdx.x);
                ri[threadIdx.x] = q;
                lse_s[threadIdx.x] = q.row < 0 ? 0.f : a.lse[(size_t)q.row * a.Hq + q.head];
            }
            __syncthreads();
            load_q(a.q, ri, a.sl2, p.D, q_s, threadIdx.x, kW * 32);
            __syncthreads();
            bool any = false;
#pragma unroll
            for (int r = 0; r < R; r++) any |= pg >= 0 && key <= ri[r].hi && key >= ri[r].lo;
            if (!any) continue;
            float sc[R];
            dots(p.k + off, q_s, p.D, sc);
#pragma unroll
            for (int r = 0; r < R; r++)
                if (key <= ri[r].hi && key >= ri[r].lo)
                    sum += exp2f(sc[r] - lse_s[r] * 1.4426950408889634f);
        }
        if (per_warp == 1) {
            tot += sum;
        } else {
            // key order within each block; one lane a block adds them
            for (uint32_t j = 0; j < per_warp; j++) {
                float y = kk < keys && blk == b0 + j ? sum : 0.f;
#pragma unroll
                for (int o = 16; o; o >>= 1) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
                if (lane == 0 && b0 + j < b.width)
                    a.mass[((size_t)i * p.H + h) * b.width + b0 + j] = y;
            }
        }
    }
    if (per_warp == 1) {
#pragma unroll
        for (int o = 16; o; o >>= 1) tot += __shfl_xor_sync(0xFFFFFFFFu, tot, o);
        if (lane == 0 && b0 < b.width) a.mass[((size_t)i * p.H + h) * b.width + b0] = tot;
    }
}

}  // namespace

uint32_t attend_simt_ctas(unsigned long long units, unsigned long long keys)
{
    const unsigned long long tiles = units * ((keys + kSimtKeys - 1) / kSimtKeys);
    return (uint32_t)(tiles < 148 * 4 ? tiles : 148 * 4);
}

int launch_attend_simt(const PagesDev &p, const BatchDev &b, const AttendDev &a,
                       const ClassDev &cl, const SplitDev &sp, cudaStream_t s)
{
    const Geo g = {kSimtRows, kSimtKeys, a.G, p.H, a.window, cl.min_rows, cl.max_rows, 0};
    attend_simt_kernel<<<sp.ctas, kW * 32, 0, s>>>(g, p, b, a, sp);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    if (sp.ctas > 1) {
        OKV_CUDA_TRY(launch_after(join_kernel<float, 128>, sp.ctas - 1, 128, 0, s, g, p, b, a, sp, 1u));
        note_launches(1);
    }
    return ORCHKV_OK;
}

int launch_mass_simt(const PagesDev &p, const BatchDev &b, const MassDev &a,
                     const ClassDev &cl, cudaStream_t s)
{
    const Geo g = {kSimtRows, kSimtKeys, a.G, p.H, a.window, cl.min_rows, cl.max_rows, 0};
    const uint32_t per_warp = p.bs.d >= 32 ? 1 : 32 / p.bs.d;
    const uint32_t groups = (b.width + kW * per_warp - 1) / (kW * per_warp);
    const unsigned long long grid = (unsigned long long)b.n * p.H * groups;
    if (grid > 0x7FFFFFFFull) return ORCHKV_ERR_INVALID;
    mass_simt_kernel<<<(unsigned)grid, kW * 32, 0, s>>>(g, p, b, a, per_warp, groups);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    return ORCHKV_OK;
}

}  // namespace okv

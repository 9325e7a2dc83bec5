// paged_append.cu — new tokens into a paged cache: per-head norm, position
// rotation, K and V to their pages, rotated Q to its rows, in one pass.
//
// Per head x of q and k: y = x * rsqrt(mean(x^2) + eps) * w (if a norm is
// given); pair (a, b) of y at rotation index p becomes
// (a cos - b sin, b cos + a sin) * scale with angle 2 pi frac(pos * turns[p]).
// The product and its fraction are taken in double (the angle of a position
// in the millions keeps 2^-24 of a turn), the rest in fp32, rounded once.
//
// Each element is read once and written once, so HBM bounds it.  A lane holds
// two 16-byte vectors whose elements are each other's pairs, so a head is
// 2..32 lanes and the rotation needs no exchange.  A warp walks over heads of
// ONE token: the angles (the costly part: 8 double products and sincospif a
// lane) are computed once and used for all of them, and few-token calls give
// each warp few heads so that there are enough warps to hide the latency.
#include "kernels.h"
#include "paged.cuh"

namespace okv {
namespace {

constexpr int kWarps = 4;

// VEC: elements of a vector (16 bytes, or 1 where the pairs do not fall on
// vectors); GL: lanes of one head (power of two); NU: units a lane holds.
// The v heads of a token run through the same loop as plain copies.
template <class T, int VEC, int GL, int NU, bool INTER>
__global__ void __launch_bounds__(kWarps * 32)
append_kernel(PagesDev p, BatchDev b, AppendDev a, uint32_t heads_per_warp, uint32_t chunks)
{
    const uint32_t w = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t r = w / chunks, ch = w - r * chunks;
    if (r >= b.rows) return;
    const uint32_t i = seq_of_row(b, (int)r);
    if (i >= b.n) return;                              // a padding row
    const SeqDev sq = load_seq(b, p.bs.d, i);
    const int at = sq.c0 + (int)r - sq.start;          // its place in the sequence
    const uint32_t blk = (uint32_t)at / p.bs, off = (uint32_t)at - blk * p.bs.d;
    const bool in_table = at >= 0 && at < sq.len;

    const uint32_t D = p.D, units = D / (2 * VEC);
    const uint32_t rot = a.rot, half = rot / 2, rest = (D - rot) / 2;
    const uint32_t gl = lane % GL, gh = lane / GL;
    constexpr int HPW = 32 / GL;

    uint32_t e0[NU], e1[NU];                           // first elements of the unit's vectors
    float cs[NU][VEC], sn[NU][VEC];
    long long pos = at;
    if (a.pos) pos = a.pos64 ? ((const long long *)a.pos)[r] : (long long)((const int *)a.pos)[r];
#pragma unroll
    for (int u = 0; u < NU; u++) {
        const uint32_t x = u * GL + gl;
        if (INTER && VEC > 1) {
            e0[u] = 2 * x * VEC;
            e1[u] = e0[u] + VEC;
        } else if (x * VEC < half) {
            e0[u] = INTER ? 2 * x : x * VEC;
            e1[u] = INTER ? 2 * x + 1 : half + x * VEC;
        } else {
            e0[u] = rot + x * VEC - half;
            e1[u] = e0[u] + rest;
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const uint32_t pr = x * VEC + j;
            cs[u][j] = 1.f;
            sn[u][j] = 0.f;
            if (x < units && pr < half) {
                double t = (double)pos * a.turns[pr];
                t -= rint(t);
                sincospif(2.f * (float)t, &sn[u][j], &cs[u][j]);
                cs[u][j] *= a.scale;
                sn[u][j] *= a.scale;
            }
        }
    }

    const uint32_t H = p.H, slots = a.Hq + 2 * H;
    const uint32_t first = ch * heads_per_warp, last = min(first + heads_per_warp, slots);
    constexpr int U = NU == 1 ? 4 : 1;                 // heads in flight a lane
    for (uint32_t s0 = first; s0 < last; s0 += U * HPW) {
        float x[U][2][NU][VEC];
        const char *src[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const uint32_t s = s0 + k * HPW + gh;
            if (s >= last) { src[k] = nullptr; continue; }
            const RowsDev &rw = s < a.Hq ? a.q : s < a.Hq + H ? a.k : a.v;
            const uint32_t h = s < a.Hq ? s : s < a.Hq + H ? s - a.Hq : s - a.Hq - H;
            src[k] = rw.p + (long long)r * rw.row_b + (long long)h * rw.head_b;
        }
        if constexpr (VEC > 1) {
            uint4 raw[U][2];
#pragma unroll
            for (int k = 0; k < U; k++)
                if (src[k] && gl < units) {
                    raw[k][0] = *(const uint4 *)(src[k] + (size_t)e0[0] * sizeof(T));
                    raw[k][1] = *(const uint4 *)(src[k] + (size_t)e1[0] * sizeof(T));
                } else {
                    raw[k][0] = raw[k][1] = make_uint4(0, 0, 0, 0);
                }
#pragma unroll
            for (int k = 0; k < U; k++) {
                Vec<T>::up(raw[k][0], x[k][0][0]);
                Vec<T>::up(raw[k][1], x[k][1][0]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int u = 0; u < NU; u++) {
                    const bool ok = src[k] && u * GL + gl < units;
                    x[k][0][u][0] = ok ? to_f(((const T *)src[k])[e0[u]]) : 0.f;
                    x[k][1][u][0] = ok ? to_f(((const T *)src[k])[e1[u]]) : 0.f;
                }
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            const uint32_t s = s0 + k * HPW + gh;
            const bool is_q = s < a.Hq, is_v = s >= a.Hq + H;
            const void *nw = is_v || !src[k] ? nullptr : is_q ? a.q_norm : a.k_norm;
            if (a.q_norm || a.k_norm) {                // the lanes of a warp reduce together
                float ss = 0.f;
#pragma unroll
                for (int u = 0; u < NU; u++)
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        ss += x[k][0][u][j] * x[k][0][u][j] + x[k][1][u][j] * x[k][1][u][j];
#pragma unroll
                for (int o = GL / 2; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                if (nw) {
                    const float inv = rsqrtf(ss / (float)D + a.eps);
#pragma unroll
                    for (int u = 0; u < NU; u++)
                        if (u * GL + gl < units) {
#pragma unroll
                            for (int j = 0; j < VEC; j++) {
                                x[k][0][u][j] *= inv * to_f(((const T *)nw)[e0[u] + j]);
                                x[k][1][u][j] *= inv * to_f(((const T *)nw)[e1[u] + j]);
                            }
                        }
                }
            }
            if (!src[k]) continue;
            char *dst;
            if (is_q) {
                dst = a.q_out.p + (long long)r * a.q_out.row_b + (long long)s * a.q_out.head_b;
            } else {
                const uint32_t h = is_v ? s - a.Hq - H : s - a.Hq;
                const int pg = in_table ? page_of(b, p.n_pages, i, h, blk) : -1;
                if (pg < 0) continue;
                dst = (is_v ? p.v : p.k) + pg * p.page_b + h * p.head_b + off * p.tok_b;
            }
#pragma unroll
            for (int u = 0; u < NU; u++) {
                if (u * GL + gl >= units) continue;
                float y0[VEC], y1[VEC];
#pragma unroll
                for (int j = 0; j < VEC; j++) { y0[j] = x[k][0][u][j]; y1[j] = x[k][1][u][j]; }
                if (!is_v) {
                    if constexpr (INTER && VEC > 1) {
#pragma unroll
                        for (int j = 0; j < VEC / 2; j++) {
                            const float c0 = cs[u][j], z0 = sn[u][j];
                            const float c1 = cs[u][VEC / 2 + j], z1 = sn[u][VEC / 2 + j];
                            const float *f = x[k][0][u], *g = x[k][1][u];
                            y0[2 * j] = f[2 * j] * c0 - f[2 * j + 1] * z0;
                            y0[2 * j + 1] = f[2 * j + 1] * c0 + f[2 * j] * z0;
                            y1[2 * j] = g[2 * j] * c1 - g[2 * j + 1] * z1;
                            y1[2 * j + 1] = g[2 * j + 1] * c1 + g[2 * j] * z1;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; j++) {
                            y0[j] = x[k][0][u][j] * cs[u][j] - x[k][1][u][j] * sn[u][j];
                            y1[j] = x[k][1][u][j] * cs[u][j] + x[k][0][u][j] * sn[u][j];
                        }
                    }
                }
                if constexpr (VEC > 1) {
                    *(uint4 *)(dst + (size_t)e0[u] * sizeof(T)) = Vec<T>::down(y0);
                    *(uint4 *)(dst + (size_t)e1[u] * sizeof(T)) = Vec<T>::down(y1);
                } else {
                    ((T *)dst)[e0[u]] = from_f<T>(y0[0]);
                    ((T *)dst)[e1[u]] = from_f<T>(y1[0]);
                }
            }
        }
    }
}

template <class T, int VEC, int GL, int NU>
int go(const PagesDev &p, const BatchDev &b, const AppendDev &a, cudaStream_t s)
{
    const uint32_t slots = a.Hq + 2 * p.H, step = 32 / GL;
    // heads a warp walks over: all of a token's when the tokens alone fill
    // the device (the angles are computed once a warp), else as few as give
    // about 8 warps an SM
    uint32_t per = slots;
    const unsigned long long want = 148ull * 8;
    if (b.rows < want) {
        const uint32_t ch = (uint32_t)((want + b.rows - 1) / b.rows);
        per = (slots + ch - 1) / ch;
    }
    per = (per + step - 1) / step * step;
    const uint32_t chunks = (slots + per - 1) / per;
    const unsigned long long warps = (unsigned long long)b.rows * chunks;
    const unsigned grid = (unsigned)((warps + kWarps - 1) / kWarps);
    if (a.inter) append_kernel<T, VEC, GL, NU, true><<<grid, kWarps * 32, 0, s>>>(p, b, a, per, chunks);
    else append_kernel<T, VEC, GL, NU, false><<<grid, kWarps * 32, 0, s>>>(p, b, a, per, chunks);
    note_launches(1);
    OKV_CUDA_TRY(cudaGetLastError());
    return ORCHKV_OK;
}

template <class T> int by_width(const PagesDev &p, const BatchDev &b, const AppendDev &a, cudaStream_t s)
{
    constexpr int N = Vec<T>::N;
    // whole vectors pair up: adjacent pairs need an even number of vectors a
    // head, half-apart pairs a whole number in each half
    const bool vec = a.inter ? p.D % (2 * N) == 0
                             : (a.rot / 2) % N == 0 && (p.D - a.rot) % (2 * N) == 0;
    if (!vec) return go<T, 1, 32, 4>(p, b, a, s);
    const uint32_t units = p.D / (2 * N);
    if (units <= 4) return go<T, N, 4, 1>(p, b, a, s);
    if (units <= 8) return go<T, N, 8, 1>(p, b, a, s);
    if (units <= 16) return go<T, N, 16, 1>(p, b, a, s);
    return go<T, N, 32, 1>(p, b, a, s);
}

}  // namespace

int launch_paged_append(int dtype, const PagesDev &p, const BatchDev &b, const AppendDev &a,
                        cudaStream_t s)
{
    if (dtype == DTYPE_BF16) return by_width<__nv_bfloat16>(p, b, a, s);
    if (dtype == DTYPE_FP16) return by_width<__half>(p, b, a, s);
    return by_width<float>(p, b, a, s);
}

}  // namespace okv

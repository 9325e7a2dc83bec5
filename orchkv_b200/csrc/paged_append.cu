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
// 2..32 lanes and the rotation needs no exchange.  A CTA works on heads of ONE
// token: its threads take a pair's angle each (a double product and a
// sincospif) and leave it in shared memory for all heads; the norm's weights
// are multiplied into the rotation's factors once a warp.  6449 tokens of 64/8
// heads of 128 with norms, bf16: 60.8 us, 4.3 TB/s, 0.66 of the measured copy
// rate (a warp a token: 78); one token: 2.5 us.  A lane has two loads in flight,
// 27 KB an SM with the 27 warps that run; bandwidth x latency asks for 45.
#include "kernels.h"
#include "paged.cuh"

namespace okv {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxPairs = kWarps * 32;                 // a thread each: heads of at most 256

// VEC: elements of a vector (16 bytes, or 1 where the pairs do not fall on
// vectors); GL: lanes of one head (power of two); NU: units a lane holds.
// The v heads of a token run through the same loop as plain copies.
template <class T, int VEC, int GL, int NU, bool INTER>
__global__ void __launch_bounds__(kWarps * 32, 8)
append_kernel(PagesDev p, BatchDev b, AppendDev a, uint32_t heads_per_warp, uint32_t ctas)
{
    __shared__ float cos_s[kMaxPairs], sin_s[kMaxPairs];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint32_t r = blockIdx.x / ctas, ch = (blockIdx.x - r * ctas) * kWarps + wid;
    const uint32_t D = p.D, units = D / (2 * VEC);
    const uint32_t rot = a.rot, half = rot / 2, rest = (D - rot) / 2;
    const double turns = threadIdx.x < half ? a.turns[threadIdx.x] : 0.;
    long long pos = 0;
    if (a.pos) pos = a.pos64 ? ((const long long *)a.pos)[r] : (long long)((const int *)a.pos)[r];
    const uint32_t i = seq_of_row(b, (int)r);
    if (i >= b.n) return;                              // a padding row
    const SeqDev sq = load_seq(b, p.bs.d, i);
    const int at = sq.c0 + (int)r - sq.start;          // its place in the sequence
    const uint32_t blk = (uint32_t)at / p.bs, off = (uint32_t)at - blk * p.bs.d;
    const bool in_table = at >= 0 && at < sq.len;
    if (threadIdx.x < half) {
        double t = (double)(a.pos ? pos : (long long)at) * turns;
        t -= rint(t);
        float c, z;
        sincospif(2.f * (float)t, &z, &c);
        cos_s[threadIdx.x] = c * a.scale;
        sin_s[threadIdx.x] = z * a.scale;
    }
    __syncthreads();

    const uint32_t gl = lane % GL, gh = lane / GL;
    constexpr int HPW = 32 / GL;
    uint32_t e0[NU], e1[NU];                           // first elements of the unit's vectors
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
    }
    // of pair j of a unit; elements behind the rotated ones turn by nothing, and
    // their partners, be they infinite, have no part in them (rests)
    auto cosine = [&](int u, int j) {
        const uint32_t pr = (u * GL + gl) * VEC + j;
        return pr < half ? cos_s[pr] : 1.f;
    };
    auto sine = [&](int u, int j) {
        const uint32_t pr = (u * GL + gl) * VEC + j;
        return pr < half ? sin_s[pr] : 0.f;
    };
    const bool some_rest = rot < D;
    auto rests = [&](int u, int j) { return some_rest && (u * GL + gl) * VEC + j >= half; };

    const uint32_t H = p.H, slots = a.Hq + 2 * H;
    const uint32_t first = ch * heads_per_warp, last = min(first + heads_per_warp, slots);
    // one page for all heads, or one each
    const int pg_all = in_table && b.ts_head == 0 ? page_of(b, p.n_pages, i, 0, blk) : -1;
    auto place = [&](char *base, uint32_t h) -> char * {
        const int pg = b.ts_head == 0 ? pg_all : in_table ? page_of(b, p.n_pages, i, h, blk) : -1;
        return pg < 0 ? nullptr : base + pg * p.page_b + h * p.head_b + off * p.tok_b;
    };
    auto load = [&](const char *src, float (*x)[NU][VEC]) {
        if constexpr (VEC > 1) {
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (src && gl < units) {
                lo = *(const uint4 *)(src + (size_t)e0[0] * sizeof(T));
                hi = *(const uint4 *)(src + (size_t)e1[0] * sizeof(T));
            }
            Vec<T>::up(lo, x[0][0]);
            Vec<T>::up(hi, x[1][0]);
        } else {
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const bool ok = src && u * GL + gl < units;
                x[0][u][0] = ok ? to_f(((const T *)src)[e0[u]]) : 0.f;
                x[1][u][0] = ok ? to_f(((const T *)src)[e1[u]]) : 0.f;
            }
        }
    };

    // q or k heads [lo, hi): the norm's weights go into the rotation's factors,
    //   a' = inv (a wa cos - b wb sin),  b' = inv (b wb cos + a wa sin)
    auto turn = [&](bool is_q, uint32_t lo, uint32_t hi) {
        if (lo >= hi) return;
        const T *nw = (const T *)(is_q ? a.q_norm : a.k_norm);
        float f[4][NU][VEC];                           // wa cos, wb sin, wb cos, wa sin
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                float wa = 1.f, wb = 1.f, wc = 1.f, wd = 1.f;   // of x0[j], x1[j] and their pairs
                const bool in = nw && u * GL + gl < units;
                if (INTER && VEC > 1) {                // pairs lie inside a vector
                    if (in) {
                        wa = to_f(nw[e0[u] + j]);
                        wb = to_f(nw[e0[u] + (j ^ 1)]);
                        wc = to_f(nw[e1[u] + j]);
                        wd = to_f(nw[e1[u] + (j ^ 1)]);
                    }
                    const int pr = j / 2;
                    const float c0 = cosine(u, pr), z0 = sine(u, pr);
                    const float c1 = cosine(u, VEC / 2 + pr), z1 = sine(u, VEC / 2 + pr);
                    // y[j] = x[j] w[j] cos -+ x[pair] w[pair] sin
                    f[0][u][j] = wa * c0;
                    f[1][u][j] = j & 1 ? wb * z0 : -wb * z0;
                    f[2][u][j] = wc * c1;
                    f[3][u][j] = j & 1 ? wd * z1 : -wd * z1;
                } else {
                    if (in) {
                        wa = to_f(nw[e0[u] + j]);
                        wb = to_f(nw[e1[u] + j]);
                    }
                    f[0][u][j] = wa * cosine(u, j);
                    f[1][u][j] = -wb * sine(u, j);
                    f[2][u][j] = wb * cosine(u, j);
                    f[3][u][j] = wa * sine(u, j);
                }
            }
        const RowsDev &rw = is_q ? a.q : a.k;
        const char *src0 = rw.p + (long long)r * rw.row_b;
        for (uint32_t h0 = lo; h0 < hi; h0 += HPW) {
            const uint32_t h = h0 + gh;
            float x[2][NU][VEC];
            load(h < hi ? src0 + (long long)h * rw.head_b : nullptr, x);
            float inv = 1.f;
            if (nw) {                              // the lanes of a head reduce together
                float ss = 0.f;
#pragma unroll
                for (int u = 0; u < NU; u++)
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        ss += x[0][u][j] * x[0][u][j] + x[1][u][j] * x[1][u][j];
#pragma unroll
                for (int o = GL / 2; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                inv = rsqrtf(ss / (float)D + a.eps);
            }
            if (h >= hi) continue;
            char *dst = is_q ? a.q_out.p + (long long)r * a.q_out.row_b + (long long)h * a.q_out.head_b
                             : place(p.k, h);
            if (!dst) continue;
#pragma unroll
            for (int u = 0; u < NU; u++) {
                if (u * GL + gl >= units) continue;
                float y0[VEC], y1[VEC];
                const float *xa = x[0][u], *xb = x[1][u];
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    y0[j] = xa[j] * f[0][u][j];
                    y1[j] = xb[j] * f[2][u][j];
                    if (INTER && VEC > 1) {
                        if (!rests(u, j / 2)) y0[j] += xa[j ^ 1] * f[1][u][j];
                        if (!rests(u, VEC / 2 + j / 2)) y1[j] += xb[j ^ 1] * f[3][u][j];
                    } else if (!rests(u, 0)) {     // a vector's pairs all turn or all rest
                        y0[j] += xb[j] * f[1][u][j];
                        y1[j] += xa[j] * f[3][u][j];
                    }
                    if (nw) {
                        y0[j] *= inv;
                        y1[j] *= inv;
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
    };
    turn(true, first, min(last, a.Hq));
    turn(false, first > a.Hq ? first - a.Hq : 0, last > a.Hq ? min(last - a.Hq, H) : 0);

    // v heads: copies
    const uint32_t v0 = a.Hq + H;
    const uint32_t v_lo = first > v0 ? first - v0 : 0, v_hi = last > v0 ? last - v0 : 0;
    for (uint32_t h = v_lo + gh; h < v_hi; h += HPW) {
        const char *src = a.v.p + (long long)r * a.v.row_b + (long long)h * a.v.head_b;
        char *dst = place(p.v, h);
        if (!dst) continue;
        if constexpr (VEC > 1) {
            if (gl < units) {
                *(uint4 *)(dst + (size_t)e0[0] * sizeof(T)) = *(const uint4 *)(src + (size_t)e0[0] * sizeof(T));
                *(uint4 *)(dst + (size_t)e1[0] * sizeof(T)) = *(const uint4 *)(src + (size_t)e1[0] * sizeof(T));
            }
        } else {
#pragma unroll
            for (int u = 0; u < NU; u++)
                if (u * GL + gl < units) {
                    ((T *)dst)[e0[u]] = ((const T *)src)[e0[u]];
                    ((T *)dst)[e1[u]] = ((const T *)src)[e1[u]];
                }
        }
    }
}

template <class T, int VEC, int GL, int NU>
int go(const PagesDev &p, const BatchDev &b, const AppendDev &a, cudaStream_t s)
{
    const uint32_t slots = a.Hq + 2 * p.H, step = 32 / GL;
    // one CTA a token when the tokens alone fill the device, else as many as
    // give about 8 warps an SM
    const unsigned long long want = 148ull * 2;
    uint32_t ctas = 1;
    if (b.rows < want) ctas = (uint32_t)((want + b.rows - 1) / b.rows);
    uint32_t per = (slots + ctas * kWarps - 1) / (ctas * kWarps);
    per = (per + step - 1) / step * step;
    ctas = (slots + per * kWarps - 1) / (per * kWarps);
    const unsigned grid = b.rows * ctas;
    if (a.inter) append_kernel<T, VEC, GL, NU, true><<<grid, kWarps * 32, 0, s>>>(p, b, a, per, ctas);
    else append_kernel<T, VEC, GL, NU, false><<<grid, kWarps * 32, 0, s>>>(p, b, a, per, ctas);
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

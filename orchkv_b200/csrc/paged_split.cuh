// paged_split.cuh — how the attention kernels divide a call among their CTAs,
// and how pieces of one row tile are joined.
//
// The work is a list of units (sequence, KV head, tile of R packed rows), each
// over a range of key tiles (KT keys).  Lengths differ from sequence to
// sequence and are known on the device alone, so a fixed number of CTAs cut
// the list into equal shares: every unit gets a weight proportional to the
// keys it reads (closed form: keys grow by R/G a row tile under the causal
// mask), CTA c takes [c, c+1) of C equal parts of the sum, and a boundary that
// falls inside a unit is mapped to a key tile of it.  A unit cut by boundaries
// leaves one partial (running maximum, sum, unnormalised output) a piece, at
// most two a CTA, and join_kernel adds the pieces in key order: no atomics,
// the same result for the same lengths every time.
#pragma once

#include <atomic>

#include "paged.cuh"

namespace okv {

typedef unsigned long long ull;

// 64-bit quotient; the values of small calls fit 32 bits, where a division
// takes a fraction of the time.
__device__ __forceinline__ ull quot(ull x, ull y)
{
    if (((x | y) >> 32) == 0) return (uint32_t)x / (uint32_t)y;
    return x / y;
}

struct Geo {                     // what the division depends on besides the lengths
    uint32_t R, KT, G, H, window;
    uint32_t min_rows, max_rows;
    uint32_t join;               // what a join costs, in keys of a unit
};

__device__ __forceinline__ uint32_t row_tiles(const Geo &g, const SeqDev &s)
{
    const uint32_t rows = (uint32_t)s.m * g.G;
    return rows > g.min_rows && rows <= g.max_rows ? (rows + g.R - 1) / g.R : 0;
}

// Weight of row tile rt: base + slope * rt, in keys * G; 64 keys' worth stand
// for a unit's fixed cost.  Where the rows' places are not those of the tokens
// in the table (lens says more tokens than the table holds, or fewer than the
// rows), every row tile counts as if it read them all.  So no unit weighs more
// than G * (keys of the table + 64) + R, which may_cut goes by.
__device__ __forceinline__ void weights(const Geo &g, const SeqDev &s, ull *base, ull *slope)
{
    const bool odd = s.c0 < 0 || s.c0 + s.m > s.len;
    const uint32_t keys = odd ? s.len : s.c0;
    if (g.window && g.window < keys + (odd ? 0 : s.m)) {
        *base = (ull)g.G * (g.window + 64) + g.R;
        *slope = 0;
    } else {
        *base = (ull)g.G * (keys + 64) + g.R;
        *slope = odd ? 0 : g.R;
    }
}
// Units over tables of at most so many keys are never cut: whole units leave a
// CTA less than the heaviest one over its share, so at most g.join keys over.
inline bool may_cut(const Geo &g, ull keys) { return keys + 64 + g.R > g.join; }
__device__ __forceinline__ ull weight_before(ull base, ull slope, ull rt)
{
    return rt * base + slope * (rt * (rt - 1) / 2 * (rt > 0));
}

// Key tiles [first, first + nt) of row tile rt; nt >= 1 (an empty row tile
// still has its rows to write).
__device__ __forceinline__ void key_tiles(const Geo &g, const SeqDev &s, uint32_t rt,
                                          uint32_t *first, uint32_t *nt)
{
    const uint32_t rows = (uint32_t)s.m * g.G;
    const uint32_t last_row = min((rt + 1) * g.R, rows) - 1;
    const int hi = min(s.len, s.c0 + (int)(last_row / g.G) + 1);
    int lo = 0;
    if (g.window) lo = max(0, s.c0 + (int)(rt * g.R / g.G) - (int)g.window + 1);
    *first = (uint32_t)lo / g.KT;
    *nt = hi > lo ? ((uint32_t)hi + g.KT - 1) / g.KT - *first : 1;
}

struct Pos {
    uint32_t i, h, rt, t;        // t counts from the unit's first key tile; i == n: the end
};

// Position of offset x inside sequence i's weight.  A unit is cut only if that
// gains more than the join costs: not when whole units leave a CTA (of `share`)
// at most g.join keys more to do; the boundary then goes to the unit's nearer
// end.
__device__ __forceinline__ Pos inside(const Geo &g, const SeqDev &s, uint32_t i, ull x, ull share)
{
    ull base, slope;
    weights(g, s, &base, &slope);
    const uint32_t RT = row_tiles(g, s);
    const ull U = weight_before(base, slope, RT);
    Pos p;
    p.i = i;
    p.h = (uint32_t)quot(x, U);
    const ull y = x - (ull)p.h * U;
    ull rt;
    if (RT == 1) {
        rt = 0;
    } else if (slope == 0) {
        rt = quot(y, base);
    } else {
        const double bb = (double)base - 0.5 * (double)slope;
        rt = (ull)((sqrt(bb * bb + 2.0 * (double)slope * (double)y) - bb) / (double)slope);
        if (rt >= RT) rt = RT - 1;
        while (rt > 0 && weight_before(base, slope, rt) > y) rt--;
        while (rt + 1 < RT && weight_before(base, slope, rt + 1) <= y) rt++;
    }
    p.rt = (uint32_t)rt;
    uint32_t first, nt;
    key_tiles(g, s, p.rt, &first, &nt);
    const ull z = y - weight_before(base, slope, rt), w = base + slope * rt;
    if (quot(share + w - 1, w) * w <= share + (ull)g.join * g.G) {
        p.t = 0;
        if (2 * z >= w && ++p.rt == RT) {
            p.rt = 0;
            if (++p.h == g.H) {
                p.h = 0;
                p.i++;                   // a sequence without units, or the end, perhaps
            }
        }
        return p;
    }
    p.t = (uint32_t)quot(z * nt, w);
    return p;
}

struct SplitShared {
    ull red[33];
    ull total;
    uint32_t seq[2];
    ull off[2];
    uint32_t end_seq;
};

__device__ __forceinline__ ull seq_weight(const Geo &g, const BatchDev &b, uint32_t bs, uint32_t i)
{
    if (i >= b.n) return 0;
    const SeqDev s = load_seq(b, bs, i);
    const uint32_t RT = row_tiles(g, s);
    if (RT == 0) return 0;
    ull base, slope;
    weights(g, s, &base, &slope);
    return g.H * weight_before(base, slope, RT);
}

// Inclusive sum over the block (NT threads) of v; *total the whole sum.
template <int NT> __device__ __forceinline__ ull block_scan(ull v, ull *red, ull *total)
{
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const ull u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) red[wid] = v;
    __syncthreads();
    ull before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < NT / 32; k++) {
        if (k < (int)wid) before += red[k];
        all += red[k];
    }
    *total = all;
    __syncthreads();
    return before + v;
}

// Boundaries c and c + 1 of C equal shares, by the whole block; *total 0: no
// work.  The end of the list is {n, 0, 0, 0}.  weight(i) is sequence i's part
// of the list, where(s, i, x, share) the position of offset x in it.
template <int NT, class Weight, class Where>
__device__ void find_share(const BatchDev &b, uint32_t bs, uint32_t c, uint32_t C, SplitShared *sh, Pos *from,
                           Pos *to, ull *W, Weight weight, Where where)
{
    if (b.n <= 32) {
        // every warp for itself, a lane a sequence: no barriers
        const uint32_t lane = threadIdx.x & 31;
        const ull w = lane < b.n ? weight(lane) : 0;
        ull inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const ull u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += u;
        }
        const ull total = __shfl_sync(0xFFFFFFFFu, inc, 31);
        *W = total;
        if (total == 0) return;
        const ull share = quot(total + C - 1, C);
        Pos *out[2] = {from, to};
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const ull x = min((c + k) * share, total);
            const uint32_t in = __ballot_sync(0xFFFFFFFFu, x >= inc - w && x < inc);
            const uint32_t i = in ? __ffs(in) - 1 : 0;
            const ull off = x - __shfl_sync(0xFFFFFFFFu, inc - w, i);
            if (k == 1 && threadIdx.x == 0) sh->off[1] = off;
            *out[k] = in ? where(load_seq(b, bs, i), i, off, share) : Pos{b.n, 0, 0, 0};
        }
        return;
    }
    ull sum = 0, one = 0;
    for (uint32_t i = threadIdx.x; i < b.n; i += NT) {
        one = weight(i);
        sum += one;
    }
    ull total;
    const ull inc0 = block_scan<NT>(sum, sh->red, &total);
    *W = total;
    if (total == 0) return;
    // shares of ceil(total / C): the last ones may be empty
    const ull share = quot(total + C - 1, C);
    const ull x[2] = {min(c * share, total), min((c + 1) * share, total)};
    if (threadIdx.x == 0) sh->seq[0] = sh->seq[1] = b.n;
    __syncthreads();
    ull carry = 0;
    for (uint32_t i0 = 0; i0 < b.n; i0 += NT) {
        const uint32_t i = i0 + threadIdx.x;
        ull w, inc, all;
        if (b.n <= NT) {
            w = one;
            inc = inc0;
            all = total;
        } else {
            w = i < b.n ? weight(i) : 0;
            inc = block_scan<NT>(w, sh->red, &all);
        }
        const ull ex = carry + inc - w;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (x[k] >= ex && x[k] < ex + w) {
                sh->seq[k] = i;
                sh->off[k] = x[k] - ex;
            }
        carry += all;
        if (carry > x[1]) break;
    }
    __syncthreads();
    Pos *out[2] = {from, to};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t i = sh->seq[k];
        if (i >= b.n) *out[k] = Pos{b.n, 0, 0, 0};
        else *out[k] = where(load_seq(b, bs, i), i, sh->off[k], share);
    }
    __syncthreads();
}
template <int NT>
__device__ void find_share(const Geo &g, const BatchDev &b, uint32_t bs, uint32_t c, uint32_t C,
                           SplitShared *sh, Pos *from, Pos *to, ull *W)
{
    find_share<NT>(b, bs, c, C, sh, from, to, W, [&](uint32_t i) { return seq_weight(g, b, bs, i); },
                   [&](const SeqDev &s, uint32_t i, ull x, ull share) { return inside(g, s, i, x, share); });
}

__device__ __forceinline__ bool same_unit(const Pos &a, const Pos &b)
{
    return a.i == b.i && a.h == b.h && a.rt == b.rt;
}

// A row of a unit.
struct RowInfo {
    int row;                     // row of the call's tensors, -1 behind the unit's last
    uint32_t head;               // query head
    int hi, lo;                  // it attends to tokens lo <= t <= hi
};
__device__ __forceinline__ RowInfo row_info(const Geo &g, const SeqDev &s, uint32_t h, uint32_t pr)
{
    RowInfo r;
    if (pr >= (uint32_t)s.m * g.G) {
        r.row = -1;
        r.head = 0;
        r.hi = -1;
        r.lo = 0;
        return r;
    }
    const uint32_t j = pr / g.G;
    r.row = s.start + (int)j;
    r.head = h * g.G + (pr - j * g.G);
    r.hi = min(s.c0 + (int)j, s.len - 1);
    r.lo = g.window ? max(0, s.c0 + (int)j - (int)g.window + 1) : 0;
    return r;
}

// A partial slot: m[R], l[R], then acc[R][D].
__device__ __forceinline__ float *slot_of(float *ws, uint32_t slot, uint32_t R, uint32_t D)
{
    return ws + (size_t)slot * R * (D + 2);
}
__host__ __device__ inline size_t slot_floats(uint32_t R, uint32_t D) { return (size_t)R * (D + 2); }

// The slots of the pieces of the unit (up to offset `unit_end` of its sequence)
// that boundary c (at position `at`, offset `off`) is the first to cut, in key order: slot 2(c-1)+1 for
// the unit's start, held by CTA c - 1, then 2c, 2(c+1), ... but for empty
// pieces.  A thread takes a boundary.  Returns their number.
constexpr uint32_t kMaxPieces = 600;
template <int NT, class Where>
__device__ uint32_t find_pieces(const BatchDev &b, uint32_t c, uint32_t C, const Pos &at, ull off, ull share,
                                ull unit_end, uint32_t nt, uint32_t *slots, Where where)
{
    constexpr uint32_t kOut = 0xFFFFFFFFu;
    __shared__ uint32_t t_s[NT + 1];
    __shared__ uint32_t n_w[NT / 32];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        t_s[0] = at.t;
        slots[0] = 2 * (c - 1) + 1;
    }
    uint32_t n = 1;
    for (uint32_t k0 = 0;; k0 += NT) {
        const uint32_t cc = c + k0 + threadIdx.x;          // a piece: boundaries cc and cc + 1
        const ull x = off + (ull)(k0 + threadIdx.x + 1) * share;
        uint32_t t = kOut;
        if (cc + 1 < C && x < unit_end) {
            const Pos nx = where(x);
            if (same_unit(nx, at)) t = nx.t;
        }
        t_s[threadIdx.x + 1] = t;
        __syncthreads();
        const uint32_t from = t_s[threadIdx.x], to = t == kOut ? nt : t;
        const bool piece = from != kOut && cc < C && to > from;
        const uint32_t in = __ballot_sync(0xFFFFFFFFu, piece);
        if (lane == 0) n_w[wid] = __popc(in);
        const bool more = t_s[NT] != kOut;
        __syncthreads();
        uint32_t before = n;
#pragma unroll
        for (int k = 0; k < NT / 32; k++) {
            if (k < (int)wid) before += n_w[k];
            n += n_w[k];
        }
        before += __popc(in & ((1u << lane) - 1));
        if (piece && before < kMaxPieces) slots[before] = 2 * cc;
        if (!more) break;
        if (threadIdx.x == 0) t_s[0] = t_s[NT];
        __syncthreads();
    }
    __syncthreads();
    return min(n, kMaxPieces);
}

// The pieces of every cut unit into its rows.  Block c looks at boundary c: it
// works if that is the first boundary inside a unit (`parts` blocks share the
// unit's rows).  All but the partials is known beforehand and found out while
// the kernel in front still runs.
template <class T, int NT>
__global__ void __launch_bounds__(NT)
join_kernel(Geo g, PagesDev p, BatchDev b, AttendDev a, SplitDev sp, uint32_t parts)
{
    __shared__ SplitShared sh;
    __shared__ uint32_t slots[kMaxPieces];
    const uint32_t c = blockIdx.x / parts + 1, part = blockIdx.x % parts;
    Pos prev, at;
    ull W;
    find_share<NT>(g, b, p.bs.d, c - 1, sp.ctas, &sh, &prev, &at, &W);
    // (no block ends before the kernel in front: the next launch counts on that)
    if (W == 0 || at.i >= b.n || at.t == 0 || (same_unit(prev, at) && prev.t > 0)) {
        cudaGridDependencySynchronize();
        return;
    }
    __syncthreads();
    const SeqDev s = load_seq(b, p.bs.d, at.i);
    uint32_t first, nt;
    key_tiles(g, s, at.rt, &first, &nt);
    ull base, slope;
    weights(g, s, &base, &slope);
    const ull unit_end = at.h * weight_before(base, slope, row_tiles(g, s)) + weight_before(base, slope, at.rt + 1);
    const ull share = quot(W + sp.ctas - 1, sp.ctas);
    const uint32_t K = find_pieces<NT>(b, c, sp.ctas, at, sh.off[1], share, unit_end, nt, slots,
                                       [&](ull x) { return inside(g, s, at.i, x, share); });
    const uint32_t D = p.D, R = g.R, d4 = D / 4;
    const uint32_t live = min(R, (uint32_t)s.m * g.G - at.rt * R);
    const uint32_t each = (live + parts - 1) / parts, r_end = min(live, (part + 1) * each);
    cudaGridDependencySynchronize();
    for (uint32_t e = part * each * d4 + threadIdx.x; e < r_end * d4; e += NT) {
        const uint32_t rr = e / d4, d = (e - rr * d4) * 4;
        float M = -INFINITY, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t k0 = 0; k0 < K; k0 += 8) {           // eight pieces' loads at once
            float m[8], l[8];
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const bool in = k0 + k < K;
                const float *sl = slot_of(sp.ws, slots[in ? k0 + k : 0], R, D);
                m[k] = in ? sl[rr] : -INFINITY;
                l[k] = sl[R + rr];
                v[k] = *(const float4 *)(sl + 2 * R + (size_t)rr * D + d);
            }
            float nm = M;
#pragma unroll
            for (int k = 0; k < 8; k++) nm = fmaxf(nm, m[k]);
            const float ms = nm == -INFINITY ? 0.f : nm, f = exp2f(M - ms);
            M = nm;
            L *= f;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] *= f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                // a piece without an attended token holds zeros, one past the
                // last weighs nothing
                const float w = exp2f(m[k] - ms);
                L += k0 + k < K ? w * l[k] : 0.f;
                o[0] += k0 + k < K ? w * v[k].x : 0.f;
                o[1] += k0 + k < K ? w * v[k].y : 0.f;
                o[2] += k0 + k < K ? w * v[k].z : 0.f;
                o[3] += k0 + k < K ? w * v[k].w : 0.f;
            }
        }
        const float Ms = M == -INFINITY ? 0.f : M;
        const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
        const RowInfo ri = row_info(g, s, at.h, at.rt * R + rr);
        T y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = from_f<T>(o[j] * inv);
        char *dst = a.out.p + (long long)ri.row * a.out.row_b + (long long)ri.head * a.out.head_b + d * sizeof(T);
        if (sizeof(T) == 4) *(uint4 *)dst = *(const uint4 *)y;
        else *(uint2 *)dst = *(const uint2 *)y;
        if (a.lse && d == 0)
            a.lse[(size_t)ri.row * a.Hq + ri.head] =
                L > 0.f ? (Ms + log2f(L)) * 0.69314718055994531f : L == 0.f ? -INFINITY : L;
    }
}

// Dynamic shared memory over 48 KB, once a kernel and device.
template <class K> cudaError_t allow_smem(K k, size_t bytes, std::atomic<uint64_t> &done)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.load() >> dev & 1)) return e;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) done |= 1ull << dev;
    return e;
}

// Clusters of more than 8 CTAs, once a kernel and device.
template <class K> cudaError_t allow_wide_cluster(K k, std::atomic<uint64_t> &done)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.load() >> dev & 1)) return e;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) done |= 1ull << dev;
    return e;
}

// A launch that may begin before the one in front of it in the stream has
// ended (the kernel waits itself with cudaGridDependencySynchronize).
template <class... P, class... A>
cudaError_t launch_after(void (*k)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                         A... args)
{
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(block);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, k, args...);
}

}  // namespace okv

// paged.cuh — device view of a paged cache and of one call's sequences,
// shared by the operators over them (paged_*.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "orchkv/paged_ops.h"

namespace okv {

// n / d by one multiply for n < 2^31, 1 <= d < 2^31: m = ceil(2^(31+s) / d)
// with s = ceil(log2 d) is exact there (the round-up method).
struct FastDiv {
    uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d)
{
    FastDiv f;
    f.d = d;
    f.s = 0;
    while ((1ull << f.s) < d) f.s++;
    f.m = (uint32_t)(((1ull << (31 + f.s)) + d - 1) / d);
    return f;
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const FastDiv &f)
{
    return (uint32_t)(((unsigned long long)n * f.m) >> (31 + f.s));
}

struct PagesDev {
    char *k, *v;
    long long page_b, head_b, tok_b;     // strides in bytes
    uint32_t n_pages, H, D;
    FastDiv bs;                          // tokens of a page
};

struct BatchDev {
    const int32_t *table;
    long long ts_seq, ts_head;
    uint32_t width, n, rows;
    const int32_t *lens, *starts;
};

struct RowsDev {
    char *p;
    long long row_b, head_b;             // strides in bytes
};

// One sequence of a call.  m rows from `start`; the first has cache position
// c0, which is negative when lens says fewer tokens than the rows.
struct SeqDev {
    int start, m, c0, len;
};
__device__ __forceinline__ SeqDev load_seq(const BatchDev &b, uint32_t bs, uint32_t i)
{
    SeqDev s;
    int a = b.starts[i], e = b.starts[i + 1];
    const int rows = (int)b.rows;
    a = a < 0 ? 0 : a > rows ? rows : a;
    e = e < a ? a : e > rows ? rows : e;
    const int len = max(b.lens[i], 0);
    s.start = a;
    s.m = e - a;
    s.c0 = len - s.m;
    // no token lies past the table
    const long long cap = (long long)b.width * bs;
    s.len = len > cap ? (int)cap : len;
    return s;
}

// The page of block `blk` (below the table's width) of head h, -1 if none.
__device__ __forceinline__ int page_of(const BatchDev &b, uint32_t n_pages, uint32_t i, uint32_t h,
                                       uint32_t blk)
{
    const int p = __ldg(b.table + (long long)i * b.ts_seq + (long long)h * b.ts_head + blk);
    return (uint32_t)p < n_pages ? p : -1;
}

// Sequence of row r by one warp: the last i with starts[i] <= r; n when the
// row lies behind the last sequence.  Each step takes one 32-way probe.
__device__ __forceinline__ uint32_t seq_of_row(const BatchDev &b, int r)
{
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = b.n + 1;       // first j in [0, n] with starts[j] > r, minus one
    while (hi - lo > 0) {
        const uint32_t step = (hi - lo + 31) / 32;
        const uint32_t j = lo + lane * step;
        const bool le = j < hi && __ldg(b.starts + j) <= r;
        const uint32_t c = __popc(__ballot_sync(0xFFFFFFFFu, le));
        if (c == 0) return b.n;          // row before the first sequence
        lo += (c - 1) * step;
        if (step == 1) break;
        hi = min(hi, lo + step);
    }
    return lo;
}

// 16-byte vectors of a type, to and from fp32.
template <class T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void up(const uint4 &r, float *f)
    {
        f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y);
        f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 down(const float *f)
    {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                          __float_as_uint(f[3]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void up(const uint4 &r, float *f)
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 down(const float *f)
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void up(const uint4 &r, float *f)
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 h = *reinterpret_cast<const __half2 *>(&w[i]);
            const float2 x = __half22float2(h);
            f[2 * i] = x.x;
            f[2 * i + 1] = x.y;
        }
    }
    static __device__ __forceinline__ uint4 down(const float *f)
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x)
{
    return __float2bfloat16_rn(x);
}

// ---- launchers ---------------------------------------------------------------------

struct AppendDev {
    RowsDev q, q_out, k, v;
    uint32_t Hq, rot;
    int inter, pos64;
    float scale, eps;
    const double *turns;
    const void *pos, *q_norm, *k_norm;
};
int launch_paged_append(int dtype, const PagesDev &p, const BatchDev &b, const AppendDev &a,
                        cudaStream_t s);

// The softmax runs in powers of two: sl2 = scale * log2(e).
struct AttendDev {
    RowsDev q, out;
    float *lse;
    uint32_t Hq, G, window;
    float sl2;
};
struct MassDev {
    RowsDev q;
    const float *lse;
    float *mass;
    uint32_t Hq, G, window;
    float sl2;
};

// One launch's share of the sequences: those with at most max_rows packed rows
// (new tokens times query heads of a KV head) and more than min_rows.
struct ClassDev {
    uint32_t min_rows, max_rows;
};
// ctas: persistent CTAs that divide the work; ws: 2 * ctas partial slots.
// split: instead, each unit (tiles_max row tiles a sequence and KV head) is a
// cluster of so many CTAs.
struct SplitDev {
    uint32_t ctas, split, tiles_max;
    float *ws;
};
constexpr uint32_t kSimtRows = 8, kSimtKeys = 128;
uint32_t attend_simt_ctas(unsigned long long units, unsigned long long keys);
int launch_attend_simt(const PagesDev &p, const BatchDev &b, const AttendDev &a,
                       const ClassDev &cl, const SplitDev &sp, cudaStream_t s);
int launch_mass_simt(const PagesDev &p, const BatchDev &b, const MassDev &a,
                     const ClassDev &cl, cudaStream_t s);

constexpr uint32_t kRowsRows = 16;
SplitDev attend_rows_split(uint32_t D, uint32_t n, uint32_t H, uint32_t tiles_max, unsigned long long units,
                           unsigned long long keys);
int launch_attend_rows(int dtype, const PagesDev &p, const BatchDev &b, const AttendDev &a,
                       const ClassDev &cl, const SplitDev &sp, cudaStream_t s);
int launch_mass_rows(int dtype, const PagesDev &p, const BatchDev &b, const MassDev &a,
                     const ClassDev &cl, cudaStream_t s);

constexpr uint32_t kTileRows = 256;
// Whether the tile kernel takes these pages (and a call with this scale).
bool attend_tile_takes(const PagesDev &p, int dtype, float sl2);
uint32_t attend_tile_ctas(unsigned long long units, unsigned long long keys);
bool mass_tile_takes(const PagesDev &p, int dtype, float sl2, const RowsDev &q, uint32_t G);
uint32_t mass_tile_ctas(unsigned long long units, unsigned long long rows);
constexpr uint32_t kMassSlot = 32;       // floats of a partial slot
int launch_mass_tile(int dtype, const PagesDev &p, const BatchDev &b, const MassDev &a,
                     const ClassDev &cl, const SplitDev &sp, cudaStream_t s);
int launch_attend_tile(int dtype, const PagesDev &p, const BatchDev &b, const AttendDev &a,
                       const ClassDev &cl, const SplitDev &sp, cudaStream_t s);

}  // namespace okv

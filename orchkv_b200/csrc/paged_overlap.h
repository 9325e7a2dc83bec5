// paged_overlap.h — whether row tensors of one call share memory (host).
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdlib>

#include "orchkv/paged_ops.h"

namespace okv {

// The bytes of a row tensor: rows x heads blocks of `block` bytes.
struct RowSpan {
    int64_t p, row, head, rows, heads, block;
    int64_t end() const { return p + (rows - 1) * row + (heads - 1) * head + block; }
};
inline RowSpan row_span(const orchkv_rows_t &r, int64_t rows, int64_t heads, int64_t block, int64_t elem)
{
    return RowSpan{(int64_t)(uintptr_t)r.p, rows > 1 ? r.row_stride * elem : 0, heads > 1 ? r.head_stride * elem : 0,
                   rows, heads, block};
}

// Whether some j in [lo, hi] brings x + j * step within less than `block` of 0.
inline bool meets(int64_t x, int64_t step, int64_t lo, int64_t hi, int64_t block)
{
    if (step == 0) return std::llabs(x) < block;
    for (int64_t j = -x / step - 1; j <= -x / step + 1; j++)
        if (std::llabs(x + std::min(std::max(j, lo), hi) * step) < block) return true;
    return false;
}

// Whether two tensors share a byte (exact for equal row strides, otherwise by
// their first and last bytes).
inline bool overlap(const RowSpan &a, const RowSpan &b)
{
    if (!a.rows || !b.rows || !a.heads || !b.heads || a.end() <= b.p || b.end() <= a.p) return false;
    if (a.rows > 1 && b.rows > 1 && a.row != b.row) return true;
    const int64_t step = a.rows > 1 ? a.row : b.row, d = b.p - a.p;
    if (a.heads == 1 || b.heads == 1 || a.head == b.head) {
        const int64_t hs = a.heads > 1 ? a.head : b.head;
        for (int64_t h = 1 - a.heads; h < b.heads; h++)
            if (meets(d + h * hs, step, 1 - a.rows, b.rows - 1, a.block)) return true;
        return false;
    }
    for (int64_t i = 0; i < a.heads; i++)
        for (int64_t j = 0; j < b.heads; j++)
            if (meets(d + j * b.head - i * a.head, step, 1 - a.rows, b.rows - 1, a.block)) return true;
    return false;
}

// Whether two blocks of one tensor share a byte.
inline bool overlaps_itself(const RowSpan &a)
{
    if (!a.rows) return false;
    if (a.rows > 1 && a.row < a.block) return true;
    for (int64_t h = 1; h < a.heads; h++)
        if (meets(h * a.head, a.row, 1 - a.rows, a.rows - 1, a.block)) return true;
    return false;
}

inline bool same_rows(const RowSpan &a, const RowSpan &b)
{
    return a.p == b.p && a.row == b.row && a.head == b.head;
}

// Whether the masses, which are written while q and lse are read, lie between
// the first and last byte of either (of q's rows and heads).
inline bool mass_overlaps(const float *mass, int64_t seqs, int64_t kv_heads, int64_t width, const RowSpan &q,
                          const float *lse)
{
    const int64_t p = (int64_t)(uintptr_t)mass, e = p + 4 * seqs * kv_heads * width;
    const int64_t l = (int64_t)(uintptr_t)lse, le = l + 4 * q.rows * q.heads;
    return q.rows && p < e && ((p < q.end() && q.p < e) || (p < le && l < e));
}

}  // namespace okv

// Causal 1-D neighbourhood attention of new tokens over a paged cache: the geometry that its kernels share, and how they divide
// the work.
//
// Dilation.  A query at position p sees p, p - d, p - 2d, ...: the positions of its residue modulo d.  So the new tokens of a
// sequence fall into d classes (i mod d), and with t = (position - residue) / d each class is attention without dilation: query
// u of the class stands at t = T0 + u and sees the keys t - K + 1 ... t.  Keys are fetched row by row through the page table
// anyway, so a class's keys are as dense a tile as consecutive ones.
//
// Rows.  The query heads of a group share their keys: a row is (query u of the class, head g of the group), numbered u * G + g,
// and a row tile is M consecutive rows, whatever G is.  A unit is (sequence, class, row tile, key/value head); its keys are the
// union of its rows' windows, cut into tiles of `keys` keys from the first one on.
//
// Division of work.  The lengths are on the device, and differ.  Every CTA computes the number of key tiles of all units (the same
// sums in every CTA), and takes the piece [c T / C, (c + 1) T / C) of their concatenation: equal shares, whatever the lengths are,
// with no host read and no atomics.  A unit that lies inside one piece is written out directly.  Of one that several CTAs share,
// each writes its unnormalised sum, maximum and row sum to the workspace (at most two units a CTA: one that its piece begins
// inside of, one that it ends inside of), and a second kernel joins them, in the CTAs' order: results do not depend on timing.
// Where windows or tables keep every unit short (`whole`), a CTA takes the units that begin in its piece, to their ends: the
// second kernel and the partial results would cost more than the unequal shares.
#pragma once
#include "fast_div.cuh"

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace natten {
namespace paged {

constexpr int kAllOfThePast = 1 << 30;        // tokens of a sequence at most; as a window: no limit

struct Args {
    const void *q, *kc, *vc;
    void* out;
    float* lse;                              // may be null
    unsigned char* ws;
    const int *table, *cache_lens, *seq_lens;
    int64_t table_stride, qs[3], ks[3], vs[3];
    int B, L, Hq, Hkv, G, D;
    int pages, page_size, table_width;
    int K, dil;                              // window, at most kAllOfThePast
    int M, keys, overhead, least;            // rows and keys (a power of two) of a tile; in key tiles: what beginning a unit costs, a CTA's least piece
    int keys_log, whole;                     // units are not shared (whole)
    int align;                               // tiles start at multiples of it: a power of two, 1 with a dilation
    int long_classes, tiles_long, tiles_short, per_seq, columns, ctas;
    FastDiv by_page, by_group, by_dil, by_seq, by_long, by_short, by_ctas;      // by page_size, G, dil, ...
    int capacity;                            // positions below it have a place in the page table
    float scale_log2;                        // scale * log2(e)
};

// What a CTA tells the joining kernel: the unit that it began and others go on with (-1: none), and how many CTAs share it.  Its
// own part of it is in its slot 2c + 1, the next ones' in 2(c + 1), 2(c + 2), ...
struct Shared { int unit, parts; };

__host__ __device__ inline size_t shared_bytes(int ctas) { return ((size_t)ctas * sizeof(Shared) + 15) & ~(size_t)15; }
__host__ __device__ inline size_t slot_bytes(int M, int D) { return (size_t)M * (D + 2) * sizeof(float); }
__device__ __forceinline__ float2* slot_sums(const Args& A, int slot)     // [M] maximum (of scale * log2(e) * score), row sum
{
    return reinterpret_cast<float2*>(A.ws + shared_bytes(A.ctas) + slot * slot_bytes(A.M, A.D));
}
__device__ __forceinline__ float* slot_out(const Args& A, int slot) { return reinterpret_cast<float*>(slot_sums(A, slot) + A.M); }

struct Tile {                                // a row tile of a class of a sequence; the same for every key/value head
    int b, cls, row0, rows;                  // rows: of the class, from row0 on, at most M
    int fresh, t0, residue;                  // new tokens of the sequence; t of the class's first query
    int lo, hi, base, n;                     // keys lo ... hi (t), in n tiles from base on
};

// Called several times in front of a unit's first load, one call behind the other: products and shifts instead of divisions (a
// step of one token against a window of 255 took 12.6 us with them).
__device__ __forceinline__ Tile tile_of(const Args& A, int column)
{
    Tile x;
    x.b = A.by_seq.div(column);
    const int fresh = A.seq_lens ? A.seq_lens[x.b] : A.L, held = A.cache_lens[x.b];
    int k = column - x.b * A.per_seq, queries = A.by_dil.div(A.L);
    if (k < A.long_classes * A.tiles_long) {
        x.cls = A.by_long.div(k);
        k -= x.cls * A.tiles_long;
        ++queries;
    } else {
        k -= A.long_classes * A.tiles_long;
        const int c = A.by_short.div(k);
        x.cls = A.long_classes + c;
        k -= c * A.tiles_short;
    }
    x.row0 = k * A.M;
    x.rows = min(A.M, queries * A.G - x.row0);
    x.fresh = min(max(fresh, 0), A.L);
    const int p = min(max(held, 0), kAllOfThePast) - x.fresh + x.cls;   // position of the class's first query
    x.t0 = p >= 0 ? A.by_dil.div(p) : -A.by_dil.div(-p + A.dil - 1);
    x.residue = p - x.t0 * A.dil;
    const int live = x.fresh > x.cls ? A.by_dil.div(x.fresh - x.cls + A.dil - 1) : 0;
    const int first = A.by_group.div(x.row0), last = min(A.by_group.div(x.row0 + x.rows - 1), live - 1);
    x.hi = A.capacity <= x.residue ? -1 : min(x.t0 + last, A.by_dil.div(A.capacity - 1 - x.residue));
    const int back = x.t0 + first - (A.K - 1);
    x.lo = x.t0 + first > 0 && back > 0 ? back : 0;
    x.base = x.lo & ~(A.align - 1);
    x.n = last >= first && x.hi >= x.lo ? ((x.hi - x.base) >> A.keys_log) + 1 : 0;
    return x;
}

// A CTA's piece, unit by unit.  `begin` is called by all `kThreads` threads; the rest is uniform arithmetic.
struct Piece {
    long long left, total;                   // of the piece; of all pieces
    long long share;                         // every CTA's share, and `rest` more among them; or pieces of A.least each (`few`)
    FastDiv by_ctas;
    int rest, pieces;
    bool few;
    int column, h, off;                      // where the piece goes on: unit (column, h), cost `off` into it
    Tile tile;

    // portion of the unit (column, h): key tiles [x0, x1).  n == 0: nothing to see, rows are to be cleared if `first`.
    struct Portion { int h, x0, x1; bool work, whole, first; };
    // What `begin` needs of shared memory
    struct Scratch { long long sums[32], at; int column; Tile tile; };

    template <int kThreads> __device__ void begin(const Args& A, int cta, Scratch* scratch)
    {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int each = A.columns <= kThreads ? 1 : (A.columns + kThreads - 1) / kThreads;
        const int c0 = min(A.columns, tid * each), c1 = min(A.columns, c0 + each);
        long long mine = 0;
        Tile t{};
        for (int c = c0; c < c1; ++c) {
            t = tile_of(A, c);
            mine += (long long)(t.n + A.overhead) * A.Hkv;
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) scratch->sums[warp] = upto;
        __syncthreads();
        long long before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += scratch->sums[w];
            total += scratch->sums[w];
        }
        const long long from = before + upto - mine;
        // No CTA gets less than A.least: every piece of a unit then has tiles, and a unit's CTAs are consecutive.
        few = total < (long long)A.ctas * A.least;
        pieces = few ? max((int)total / A.least, 1) : A.ctas;
        share = few ? A.least : total < 0x7fffffff ? A.by_ctas.div((int)total) : total / A.ctas;
        rest = few ? 0 : (int)(total - share * A.ctas);
        by_ctas = A.by_ctas;
        const long long start = start_of(cta), stop = start_of(cta + 1);
        if (start < stop && start >= from && start < from + mine) {
            long long at = start - from;
            int c = c0;
            if (each > 1)
                for (;; ++c) {
                    t = tile_of(A, c);
                    const long long w = (long long)(t.n + A.overhead) * A.Hkv;
                    if (at < w) break;
                    at -= w;
                }
            scratch->column = c;
            scratch->at = at;
            scratch->tile = t;
        }
        __syncthreads();
        left = stop - start;
        column = h = off = 0;
        if (left > 0) {
            column = scratch->column;
            tile = scratch->tile;
            const int w = tile.n + A.overhead;
            long long at = scratch->at;                      // less than w * Hkv, which may pass 31 bits
            for (; at >= w; at -= w) ++h;
            off = (int)at;
            if (A.whole && off > 0) advance(A);              // another CTA's
        }
    }
    // where CTA c's piece starts
    __device__ __forceinline__ long long start_of(int c) const
    {
        if (c >= pieces) return total;
        return share * c + (few ? 0 : by_ctas.div(rest * c));
    }
    // CTAs from `cta` on that share the unit that its piece ends inside of
    __device__ int parts(const Args& A, int cta) const
    {
        const long long end = start_of(cta + 1) + (tile.n + A.overhead - off - left);
        int c = cta + 1;
        c = max(c, (int)min((long long)pieces, end / (share + 1)));      // start_of(c) <= (share + 1) c
        while (c < pieces && start_of(c) < end) ++c;
        return c - cta;
    }
    __device__ __forceinline__ int take(const Args& A, int w) const { return A.whole || left >= w - off ? w - off : (int)left; }
    __device__ __forceinline__ bool more() const { return left > 0; }
    __device__ __forceinline__ Portion portion(const Args& A) const
    {
        Portion p;
        p.h = h;
        p.x0 = max(off - A.overhead, 0);
        p.x1 = max(off + take(A, tile.n + A.overhead) - A.overhead, 0);
        p.first = off == 0;
        p.work = p.x1 > p.x0;
        p.whole = p.work && p.x0 == 0 && p.x1 == tile.n;
        return p;
    }
    __device__ __forceinline__ void advance(const Args& A)
    {
        const int w = tile.n + A.overhead, t = take(A, w);
        left -= t;
        off += t;
        if (off == w) {
            off = 0;
            if (++h == A.Hkv) {
                h = 0;
                if (++column < A.columns) tile = tile_of(A, column);
                else left = 0;
            }
        }
    }
};

// index of row r (< rows) of a tile in [B, L, Hq], and t of its query; false where there is no such query (a padding row)
__device__ __forceinline__ bool row_of(const Args& A, const Tile& x, int h, int r, long long& index, int& t)
{
    const int row = x.row0 + r, u = A.by_group.div(row), g = row - u * A.G, i = x.cls + A.dil * u;
    index = ((long long)x.b * A.L + i) * A.Hq + (long long)h * A.G + g;
    t = x.t0 + u;
    return i < x.fresh;
}
// offset of a row of q (elements)
__device__ __forceinline__ long long query_offset(const Args& A, const Tile& x, int h, int r)
{
    const int row = x.row0 + r, u = A.by_group.div(row), g = row - u * A.G;
    return x.b * A.qs[0] + (long long)(x.cls + A.dil * u) * A.qs[1] + (long long)(h * A.G + g) * A.qs[2];
}
// page and slot of key t of the tile's class: false where it is not there
__device__ __forceinline__ bool locate(const Args& A, const Tile& x, int t, int& page, int& slot)
{
    if (t > x.hi) return false;              // hi is below the table's end
    const int pos = x.residue + A.dil * t, n = A.by_page.div(pos);
    slot = pos - n * A.page_size;
    page = A.table[x.b * A.table_stride + n];
    return page >= 0 && page < A.pages;
}

// Host side.  A kernel family says which tiles it would use (false: it does not cover the call); `divide` (paged.cu) divides the
// call by them.  `aligned`: every row of q and of the caches starts on a 16-byte boundary, or could.
// most: key tiles up to which a unit is not shared
struct Shape { int M, keys, overhead, least, most, ctas; };
bool general_shape(int dtype, const Args& A, Shape& shape);
int general_run(int dtype, const Args& A, bool aligned, cudaStream_t s);
bool warp_shape(int dtype, const Args& A, bool aligned, int warps, Shape& shape);
int warp_run(int dtype, const Args& A, int warps, cudaStream_t s);
bool tc_shape(int dtype, const Args& A, bool aligned, Shape& shape);
int tc_run(int dtype, const Args& A, cudaStream_t s);

// A kernel that others may start behind: its dependents' launch overlaps its end.
__device__ __forceinline__ void let_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Everything that the kernel in front wrote is there.
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

} // namespace paged

void note_path(int path);        // what natten_last_path reports

} // namespace natten

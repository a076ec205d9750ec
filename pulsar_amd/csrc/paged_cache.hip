// The paged cache's book-keeping and moves: taking pages for new tokens, storing
// their keys and values, forking and freeing rows, compacting and copying pages.
//
// Book-keeping (extend, fork, compact) is one workgroup of 1024 threads that
// scans the reference counts, 4096 or 16384 pages a step: the pages dealt
// out are the lowest-numbered free ones in order, so the result does not depend
// on timing, and the scan ends at the last page needed.  Its time is a few
// memory latencies (one or two steps), not bandwidth: a grid would have to wait
// for itself between counting and dealing, which costs more.  What is bulk --
// page contents, table rows -- is left to a second launch of many workgroups,
// which reads what the first decided from the workspace.
//
// (1000 pages dealt of 4000: 6.3 us.)
//
// Page moves are bound by HBM: each byte is read and written once, in 16 KB
// pieces of 64 bytes a thread, so a pool of any page size keeps every CU busy:
// compacting 1.1 GB of moves takes 214 us (5.0 TB/s, both ways counted; a copy of
// 4 GiB reaches 4.7), forking 48 rows of 32 planes 69 us.  Storing 65 MB of new
// keys and values takes 13.3 us.
#include "pulsar_paged.h"

#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged_common.h"

using namespace pw4;

namespace {

constexpr int kMetaThreads = 1024, kMetaWaves = kMetaThreads / 64;
constexpr int kMaxRows = 4096;  // rows (extend) or pairs (fork) of a call: their prefix sums lie in LDS

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t page_size) {
    return tokens == 0 ? 0 : (tokens - 1) / page_size + 1;
}

// First i in [0, n) with ends[i] > v (ends ascending); n if none.
__device__ __forceinline__ int first_above(const int* ends, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > v) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    return lo;
}

// Bit j: page p0 + j is free (in use, with USED), for a thread's PER pages.
template <bool USED, int PER>
__device__ __forceinline__ uint32_t page_mask(const int32_t* refs, int p0, int pages, bool vec) {
    uint32_t m = 0;
    if (vec && p0 + PER <= pages) {
#pragma unroll
        for (int v = 0; v < PER / 4; ++v) {
            const int4 r = *reinterpret_cast<const int4*>(refs + p0 + 4 * v);
            m |= ((r.x > 0) | (r.y > 0) << 1 | (r.z > 0) << 2 | (r.w > 0) << 3) << (4 * v);
        }
        return USED ? m : ~m & ((1u << PER) - 1);
    }
    for (int j = 0; j < PER && p0 + j < pages; ++j) m |= ((refs[p0 + j] > 0) == USED ? 1u : 0u) << j;
    return m;
}

// Deals the lowest-numbered free pages, in order: take(f, page) for the f-th, f <
// need.  Returns how many there were, up to need or a little past it.  Every
// thread of the workgroup calls it.
template <int PER, typename F>
__device__ __forceinline__ int deal_free_pages_by(const int32_t* refs, int pages, int need, int* lds, F take) {
    const bool vec = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
    int found = 0;
    for (int base = 0; base < pages && found < need; base += kMetaThreads * PER) {
        const int p0 = base + (int)threadIdx.x * PER;
        uint32_t m = p0 < pages ? page_mask<false, PER>(refs, p0, pages, vec) : 0;
        int total;
        const int count = __popc(m);
        int f = found + block_inclusive_scan<kMetaWaves>(count, lds, total) - count;
        for (; m != 0 && f < need; m &= m - 1, ++f) take(f, p0 + __ffs((int)m) - 1);
        found += total;
    }
    return found;
}
template <typename F>
__device__ __forceinline__ int deal_free_pages(const int32_t* refs, int pages, int need, int* lds, F take) {
    // 4 pages a thread where few steps do: the pages of a thread are dealt one after the other
    // (1000 pages of 4000: 16 a thread take 10.0 us, 4 a thread 6.3)
    return pages <= 4 * 4 * kMetaThreads ? deal_free_pages_by<4>(refs, pages, need, lds, take)
                                         : deal_free_pages_by<16>(refs, pages, need, lds, take);
}

// ---- extend -----------------------------------------------------------------

struct ExtendArgs {
    int32_t* refs;
    int32_t* tables;
    int32_t* lens;
    const int32_t* cu_q;
    int64_t* slots;
    int32_t* missing;
    int64_t table_stride, num_tokens;
    int32_t pages, width, rows, page_size;
};

// Tokens that row b gets.
__device__ __forceinline__ uint32_t new_tokens(const int32_t* cu, int b) {
    return cu[b + 1] > cu[b] ? min((uint32_t)cu[b + 1] - (uint32_t)cu[b], (uint32_t)INT_MAX) : 0;
}

__device__ __forceinline__ int64_t slot_of(const ExtendArgs& a, const int32_t* cu, int row, int t, int old_len) {
    const uint32_t pos = (uint32_t)(old_len + t - cu[row]);
    const uint32_t col = pos / (uint32_t)a.page_size;
    const int page = a.tables[(int64_t)row * a.table_stride + min(col, (uint32_t)a.width - 1)];
    return (int64_t)page * a.page_size + (pos - col * (uint32_t)a.page_size);
}

// `inline_slots`: the slots too, else slots_kernel follows.
__global__ __launch_bounds__(kMetaThreads) void extend_kernel(const ExtendArgs a, int inline_slots) {
    extern __shared__ int shared[];
    int* const need_end = shared;               // [rows] pages needed by rows up to this one
    int* const cu = shared + a.rows;            // [rows + 1]
    __shared__ int scratch[kMetaWaves];
    const int tid = threadIdx.x;
    int need = 0, over = 0;
    for (int b = tid; b <= a.rows; b += kMetaThreads) cu[b] = a.rows ? a.cu_q[b] : 0;
    __syncthreads();
    for (int b0 = 0; b0 < a.rows; b0 += kMetaThreads) {
        const int b = b0 + tid;
        int mine = 0;
        if (b < a.rows) {
            // counts below 2^31 each, so sums below 2^32, whatever lens and cu hold
            const uint32_t len = max(a.lens[b], 0), n = new_tokens(cu, b), width = a.width;
            const uint32_t want = pages_of(len + n, a.page_size);
            mine = (int)min(want - pages_of(len, a.page_size), (uint32_t)INT_MAX);
            over += want > width ? (int)min(want - width, 1u << 18) : 0;  // a sum that 4096 rows do not overflow
        }
        int total;
        const int upto = block_inclusive_scan<kMetaWaves>(mine, scratch, total);
        if (b < a.rows) need_end[b] = need + upto;
        need += total;
    }
    block_inclusive_scan<kMetaWaves>(over, scratch, over);
    const bool dealing = over == 0;
    auto place = [&](int f, int& row) -> int64_t {  // the table entry that takes the f-th page
        row = first_above(need_end, a.rows, f);
        const int col = (int)pages_of(max(a.lens[row], 0), a.page_size) + f - (row ? need_end[row - 1] : 0);
        return (int64_t)row * a.table_stride + col;
    };
    const int found = deal_free_pages(a.refs, a.pages, need, scratch, [&](int f, int page) {
        if (!dealing) return;
        int row;
        a.tables[place(f, row)] = page;
        a.refs[page] = 1;
    });
    const int missing = (int)min((int64_t)max(need - found, 0) + over, (int64_t)INT_MAX);
    __syncthreads();
    if (missing != 0 && dealing) {  // give back what was dealt
        for (int f = tid; f < found; f += kMetaThreads) {
            int row;
            const int64_t at = place(f, row);
            a.refs[a.tables[at]] = 0;
            a.tables[at] = -1;
        }
    }
    if (tid == 0) *a.missing = missing;
    if (inline_slots) {
        for (int t = tid; t < (int)a.num_tokens; t += kMetaThreads) {
            const int row = first_above(cu + 1, a.rows, t);
            const bool in = missing == 0 && row < a.rows && t >= cu[row];
            a.slots[t] = in ? slot_of(a, cu, row, t, max(a.lens[row], 0)) : -1;
        }
    }
    __syncthreads();
    if (missing == 0) {
        for (int b = tid; b < a.rows; b += kMetaThreads) a.lens[b] = max(a.lens[b], 0) + (int)new_tokens(cu, b);
    }
}

// The slots of many tokens, after extend_kernel without them: seq_lens has grown.
__global__ __launch_bounds__(256) void slots_kernel(const ExtendArgs a) {
    extern __shared__ int cu[];
    for (int b = threadIdx.x; b <= a.rows; b += 256) cu[b] = a.rows ? a.cu_q[b] : 0;
    __syncthreads();
    const bool ok = *a.missing == 0;
    const int t = (int)(blockIdx.x * 256 + threadIdx.x);
    if (t >= a.num_tokens) return;
    const int row = first_above(cu + 1, a.rows, t);
    const bool in = ok && row < a.rows && t >= cu[row];
    a.slots[t] = in ? slot_of(a, cu, row, t, a.lens[row] - (int)new_tokens(cu, row)) : -1;
}

// ---- write --------------------------------------------------------------------

struct WriteArgs {
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* k_cache;
    uint16_t* v_cache;
    const int64_t* slots;
    int64_t k_token, k_head, v_token, v_head, page_stride, row_stride, head_stride, num_slots;
    uint32_t units, page_size, dim_units, token_units;  // units of VEC elements: all, of a head, of a token
};

// One VEC of keys and one of values a thread; a token's units lie side by side.
template <int VEC>
__global__ __launch_bounds__(256) void write_kernel(const WriteArgs a) {
    using Unit = std::conditional_t<VEC == 8, u32x4, uint16_t>;
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;
    if (u >= a.units) return;
    const uint32_t t = u / a.token_units, in_token = u - t * a.token_units, h = in_token / a.dim_units;
    const int64_t d = (int64_t)(in_token - h * a.dim_units) * VEC;
    const int64_t at = a.slots[t];
    if (at < 0 || at >= a.num_slots) return;
    const uint32_t slot = (uint32_t)at, page = slot / a.page_size;
    const int64_t to = page * a.page_stride + (slot - page * a.page_size) * a.row_stride + h * a.head_stride + d;
    const Unit uk = *reinterpret_cast<const Unit*>(a.k + t * a.k_token + h * a.k_head + d);
    const Unit uv = *reinterpret_cast<const Unit*>(a.v + t * a.v_token + h * a.v_head + d);
    *reinterpret_cast<Unit*>(a.k_cache + to) = uk;
    *reinterpret_cast<Unit*>(a.v_cache + to) = uv;
}

// ---- moving whole pages ---------------------------------------------------------

constexpr int kPieceBytes = 16384;  // 256 threads, 64 bytes each

struct Pool {
    uint8_t* base;
    int64_t plane_stride, page_stride, page_bytes;
    int32_t planes, pages, pieces;  // pieces of a page
};

// Pieces (pair, plane, piece of the page) first, first + step, ... of n pairs.
template <typename V>
__device__ __forceinline__ void move_pages(const Pool& pool, const int32_t* src, const int32_t* dst, int n,
                                           int64_t first, int64_t step) {
    const int64_t per_pair = (int64_t)pool.planes * pool.pieces, units = n * per_pair;
    for (int64_t u = first; u < units; u += step) {
        const int pair = (int)(u / per_pair);
        const int rest = (int)(u - pair * per_pair), plane = rest / pool.pieces, piece = rest - plane * pool.pieces;
        const int s = src[pair], d = dst[pair];
        if (s < 0 || d < 0 || s >= pool.pages || d >= pool.pages || s == d) continue;
        uint8_t* const base = pool.base + plane * pool.plane_stride;
        const V* const from = reinterpret_cast<const V*>(base + s * pool.page_stride);
        V* const to = reinterpret_cast<V*>(base + d * pool.page_stride);
        const int64_t begin = (int64_t)piece * (kPieceBytes / sizeof(V));
        const int64_t end = min(begin + (int64_t)(kPieceBytes / sizeof(V)), pool.page_bytes / (int64_t)sizeof(V));
        int64_t at = begin + threadIdx.x;
        for (; at + 3 * 256 < end; at += 4 * 256) {
            const V r0 = from[at], r1 = from[at + 256], r2 = from[at + 512], r3 = from[at + 768];
            to[at] = r0;
            to[at + 256] = r1;
            to[at + 512] = r2;
            to[at + 768] = r3;
        }
        for (; at < end; at += 256) to[at] = from[at];
    }
}

template <typename V>
__global__ __launch_bounds__(256) void copy_kernel(const Pool pool, const int32_t* src, const int32_t* dst, int n) {
    move_pages<V>(pool, src, dst, n, blockIdx.x, gridDim.x);
}

// ---- fork ----------------------------------------------------------------------

struct ForkArgs {
    int32_t* refs;
    int32_t* tables;
    int32_t* lens;
    const int32_t* src_rows;
    const int32_t* dst_rows;
    int32_t* missing;
    int32_t* pair_src;  // workspace [n]: the page in part filled, and
    int32_t* pair_dst;  // [n] the fresh page it goes to; -1 for none
    int64_t table_stride;
    int32_t pages, width, rows, page_size, n;
};

// Tokens of pair i's source, -1 where the pair names no row.
__device__ __forceinline__ int fork_length(const ForkArgs& a, int i) {
    const int s = a.src_rows[i], d = a.dst_rows[i];
    if (s < 0 || s >= a.rows || d < 0 || d >= a.rows || s == d) return -1;
    return min(max(a.lens[s], 0), (int)min((int64_t)INT_MAX, (int64_t)a.width * a.page_size));
}

__global__ __launch_bounds__(kMetaThreads) void fork_pages_kernel(const ForkArgs a) {
    extern __shared__ int need_end[];
    __shared__ int scratch[kMetaWaves];
    const int tid = threadIdx.x;
    int need = 0;
    for (int i0 = 0; i0 < a.n; i0 += kMetaThreads) {
        const int i = i0 + tid;
        const int len = i < a.n ? fork_length(a, i) : -1;
        const int part = len > 0 && len % a.page_size != 0;
        if (i < a.n) {
            a.pair_src[i] = part ? a.tables[a.src_rows[i] * a.table_stride + len / a.page_size] : -1;
            a.pair_dst[i] = -1;
        }
        int total;
        const int upto = block_inclusive_scan<kMetaWaves>(part, scratch, total);
        if (i < a.n) need_end[i] = need + upto;
        need += total;
    }
    __syncthreads();
    const int found = deal_free_pages(a.refs, a.pages, need, scratch, [&](int f, int page) {
        a.pair_dst[first_above(need_end, a.n, f)] = page;
        a.refs[page] = 1;
    });
    const int missing = max(need - found, 0);
    __syncthreads();
    if (missing != 0) {
        for (int i = tid; i < a.n; i += kMetaThreads) {
            if (a.pair_dst[i] >= 0) a.refs[a.pair_dst[i]] = 0;
            a.pair_dst[i] = -1;
        }
    }
    if (tid == 0) *a.missing = missing;
}

// Workgroup i < n: row i's table and length, and the counts of the pages it
// shares; the others move the contents of the pages in part filled.
template <typename V>
__global__ __launch_bounds__(256) void fork_kernel(const ForkArgs a, const Pool pool) {
    if (*a.missing != 0) return;
    const int i = blockIdx.x;
    if (i >= a.n) {
        move_pages<V>(pool, a.pair_src, a.pair_dst, a.n, i - a.n, gridDim.x - a.n);
        return;
    }
    const int len = fork_length(a, i);
    if (len < 0) return;
    const int full = len / a.page_size;
    const int32_t* const from = a.tables + a.src_rows[i] * a.table_stride;
    int32_t* const to = a.tables + a.dst_rows[i] * a.table_stride;
    for (int c = threadIdx.x; c < a.width; c += 256) {
        int page = -1;
        if (c < full) {
            page = from[c];
            if (page >= 0 && page < a.pages) atomicAdd(a.refs + page, 1);
        } else if (c == full) {
            page = a.pair_dst[i];
        }
        to[c] = page;
    }
    if (threadIdx.x == 0) a.lens[a.dst_rows[i]] = len;
}

// ---- free ----------------------------------------------------------------------

__global__ __launch_bounds__(256) void free_kernel(int32_t* refs, int pages, int32_t* tables, int rows, int width,
                                                   int64_t table_stride, int32_t* lens, const int32_t* which) {
    const int row = which[blockIdx.x];
    if (row < 0 || row >= rows) return;
    int32_t* const table = tables + row * table_stride;
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c < width) {
        // the exchange lets one of two calls for the same row have the entry
        const int page = atomicExch(table + c, -1);
        if (page >= 0 && page < pages) atomicSub(refs + page, 1);
    }
    if (c == 0) lens[row] = 0;
}

// ---- compact -------------------------------------------------------------------

struct CompactArgs {
    int32_t* refs;
    int32_t* tables;
    int32_t* used;
    int32_t* moves;      // workspace [2]: how many pages move,
    int32_t* move_src;   // [most_moves(pages)] from where
    int32_t* move_dst;   // [most_moves(pages)] to where,
    int32_t* new_name;   // [pages] where each page that moves goes
    int64_t table_stride;
    int32_t pages, rows, width;
};

__global__ __launch_bounds__(kMetaThreads) void compact_pages_kernel(const CompactArgs a) {
    __shared__ int scratch[kMetaWaves];
    __shared__ int s_holes;
    const int tid = threadIdx.x;
    const bool vec = (reinterpret_cast<uintptr_t>(a.refs) & 15) == 0;
    constexpr int kPer = 16, kStep = kMetaThreads * kPer;
    int mine = 0, used = 0;
    for (int p0 = tid * kPer; p0 < a.pages; p0 += kStep) mine += __popc(page_mask<true, kPer>(a.refs, p0, a.pages, vec));
    block_inclusive_scan<kMetaWaves>(mine, scratch, used);
    if (tid == 0) {
        *a.used = used;
        s_holes = 0;
    }
    __syncthreads();
    int before = 0;  // used pages in earlier steps
    for (int base = 0; base < a.pages; base += kStep) {
        const int p0 = base + tid * kPer;
        const uint32_t m = p0 < a.pages ? page_mask<true, kPer>(a.refs, p0, a.pages, vec) : 0;
        int total;
        const int count = __popc(m);
        const int upto = before + block_inclusive_scan<kMetaWaves>(count, scratch, total) - count;
        const int end = min(p0 + kPer, a.pages);
        // page `used` is the border: the holes below it are all there are to fill
        if (p0 <= used && used < end) s_holes = used - (upto + __popc(m & ((1u << (used - p0)) - 1)));
        __syncthreads();
        int c = upto;  // used pages below p
        for (int p = p0; p < end; ++p) {
            const bool in_use = m >> (p - p0) & 1;
            if (!in_use && p < used) a.move_dst[p - c] = p;
            if (in_use && p >= used) a.move_src[c - (used - s_holes)] = p;
            if (!in_use && p >= used) a.new_name[p] = -1;
            c += in_use;
        }
        before += total;
    }
    __syncthreads();
    const int holes = s_holes;
    if (tid == 0) *a.moves = holes;
    for (int i = tid; i < holes; i += kMetaThreads) {
        const int s = a.move_src[i], d = a.move_dst[i];
        a.new_name[s] = d;
        a.refs[d] = a.refs[s];
        a.refs[s] = 0;
    }
}

// The first `table_blocks` workgroups rename the tables, the others move contents.
template <typename V>
__global__ __launch_bounds__(256) void compact_kernel(const CompactArgs a, const Pool pool, int table_blocks) {
    const int block = blockIdx.x;
    if (block >= table_blocks) {
        move_pages<V>(pool, a.move_src, a.move_dst, *a.moves, block - table_blocks, gridDim.x - table_blocks);
        return;
    }
    if (*a.moves == 0) return;
    const int used = *a.used;
    const int64_t entries = (int64_t)a.rows * a.width;
    for (int64_t e = (int64_t)block * 256 + threadIdx.x; e < entries; e += (int64_t)table_blocks * 256) {
        const int64_t row = e / a.width;
        int32_t* const at = a.tables + row * a.table_stride + (e - row * a.width);
        const int page = *at;
        // an entry that no count covers names a free page: it has no new name
        if (page >= used && page < a.pages && a.new_name[page] >= 0) *at = a.new_name[page];
    }
}

// ---- host ----------------------------------------------------------------------

bool small(int64_t v) { return v >= 0 && v <= INT_MAX; }

int check_launch() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

// The pool as the kernels take it, or an error.
int as_pool(const pw4_page_pool* p, Pool& out) {
    if (p == nullptr || p->planes < 0 || p->num_pages < 0 || p->page_bytes < 0) return PW4_ERR_ARG;
    if (!small(p->planes) || !small(p->num_pages)) return PW4_ERR_SHAPE;
    const int64_t pieces = ceil_div(p->page_bytes, kPieceBytes);
    if (!small(pieces * std::max<int64_t>(1, p->planes))) return PW4_ERR_SHAPE;
    if (p->base == nullptr && p->planes * p->num_pages * p->page_bytes != 0) return PW4_ERR_ARG;
    out = Pool{static_cast<uint8_t*>(p->base), p->plane_stride_bytes, p->page_stride_bytes, p->page_bytes,
               (int32_t)p->planes, (int32_t)p->num_pages, (int32_t)pieces};
    return PW4_OK;
}

// Bytes that every address and size of the pool is a multiple of: 16, 4 or 1.
int pool_unit(const Pool& p) {
    const uint64_t all = (uint64_t)(uintptr_t)p.base | (uint64_t)p.plane_stride | (uint64_t)p.page_stride |
                         (uint64_t)p.page_bytes;
    return (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : 1;
}

// Pages that compacting moves at most: there is a hole for each.
int64_t most_moves(int64_t pages) { return (pages + 1) / 2; }

// Workgroups that move `pairs` pages: a piece each, up to eight a CU.
int move_blocks(const Pool& p, int64_t pairs) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(pairs * p.planes * p.pieces, 8 * device_cus()));
}

template <typename F>
void with_unit(int unit, F&& f) {
    if (unit == 16) {
        f(u32x4{});
    } else if (unit == 4) {
        f(uint32_t{});
    } else {
        f(uint8_t{});
    }
}

int check_tables(const void* refs, const void* tables, int64_t pages, int64_t rows, int64_t width, int64_t stride) {
    if (rows < 0 || width < 0 || pages < 0) return PW4_ERR_ARG;
    if (!small(pages) || !small(rows) || !small(width) || stride < width) return PW4_ERR_SHAPE;
    if ((pages && refs == nullptr) || (rows && width && tables == nullptr)) return PW4_ERR_ARG;
    return PW4_OK;
}

}  // namespace

extern "C" {

int pw4_paged_cache_extend(int32_t* ref_counts, int64_t num_pages, int32_t* block_tables, int64_t table_width,
                           int64_t table_stride, int32_t* seq_lens, const int32_t* cu_q, int64_t rows,
                           int64_t num_tokens, int64_t page_size, int64_t* slots, int32_t* missing,
                           pw4_stream_t stream) {
    if (const int rc = check_tables(ref_counts, block_tables, num_pages, rows, table_width, table_stride)) return rc;
    if (num_tokens < 0 || missing == nullptr || (rows && (seq_lens == nullptr || cu_q == nullptr)) ||
        (num_tokens && slots == nullptr)) {
        return PW4_ERR_ARG;
    }
    if (page_size <= 0 || !small(page_size) || rows > kMaxRows || !small(num_tokens) ||
        !small(table_width * page_size)) {
        return PW4_ERR_SHAPE;
    }
    const ExtendArgs a{ref_counts, block_tables, seq_lens, cu_q, slots, missing, table_stride, num_tokens,
                       (int32_t)num_pages, (int32_t)table_width, (int32_t)rows, (int32_t)page_size};
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    // The one workgroup takes the slots of up to 2048 tokens, two a thread, with it.
    const bool inline_slots = num_tokens <= 2 * kMetaThreads;
    hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(kMetaThreads), (uint32_t)(2 * rows + 1) * 4, s, a,
                       inline_slots ? 1 : 0);
    if (!inline_slots) {
        hipLaunchKernelGGL(slots_kernel, dim3((unsigned)ceil_div(num_tokens, 256)), dim3(256), (uint32_t)(rows + 1) * 4,
                           s, a);
    }
    return check_launch();
}

int pw4_paged_cache_write(const void* k, const void* v, void* k_cache, void* v_cache, const int64_t* slots,
                          int64_t num_tokens, int64_t kv_heads, int64_t head_dim, int64_t k_token_stride,
                          int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int64_t num_pages,
                          int64_t page_size, int64_t page_stride, int64_t row_stride, int64_t kv_head_stride,
                          pw4_stream_t stream) {
    if (num_tokens < 0 || kv_heads < 0 || head_dim < 0 || num_pages < 0 || page_size <= 0) return PW4_ERR_ARG;
    if (!small(kv_heads * head_dim) || !small(page_size) || !small(num_tokens)) return PW4_ERR_SHAPE;
    if (num_tokens == 0 || kv_heads == 0 || head_dim == 0 || num_pages == 0) return PW4_OK;
    if (!k || !v || !k_cache || !v_cache || !slots) return PW4_ERR_ARG;
    const uint64_t addresses = (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v | (uint64_t)(uintptr_t)k_cache |
                               (uint64_t)(uintptr_t)v_cache;
    const uint64_t strides = (uint64_t)(head_dim | k_token_stride | k_head_stride | v_token_stride | v_head_stride |
                                        page_stride | row_stride | kv_head_stride);
    if (addresses & 1) return PW4_ERR_ARG;
    const int vec = (addresses & 15) == 0 && (strides & 7) == 0 ? 8 : 1;
    const int64_t token_units = kv_heads * (head_dim / vec), units = num_tokens * token_units;
    if (!small(units) || !small(num_pages) || !small(num_pages * page_size)) return PW4_ERR_SHAPE;
    const WriteArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), static_cast<uint16_t*>(k_cache),
                      static_cast<uint16_t*>(v_cache), slots, k_token_stride, k_head_stride, v_token_stride,
                      v_head_stride, page_stride, row_stride, kv_head_stride, num_pages * page_size, (uint32_t)units,
                      (uint32_t)page_size, (uint32_t)(head_dim / vec), (uint32_t)token_units};
    const dim3 grid((unsigned)ceil_div(units, 256));
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (vec == 8) {
        hipLaunchKernelGGL(write_kernel<8>, grid, dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL(write_kernel<1>, grid, dim3(256), 0, s, a);
    }
    return check_launch();
}

int pw4_paged_cache_copy(const pw4_page_pool* pool, const int32_t* src, const int32_t* dst, int64_t n,
                         pw4_stream_t stream) {
    Pool p;
    if (const int rc = as_pool(pool, p)) return rc;
    if (n < 0) return PW4_ERR_ARG;
    if (!small(n)) return PW4_ERR_SHAPE;
    if (n == 0 || p.planes == 0 || p.pages == 0 || p.page_bytes == 0) return PW4_OK;
    if (src == nullptr || dst == nullptr) return PW4_ERR_ARG;
    const int blocks = move_blocks(p, n);
    with_unit(pool_unit(p), [&](auto v) {
        hipLaunchKernelGGL(copy_kernel<decltype(v)>, dim3(blocks), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                           p, src, dst, (int)n);
    });
    return check_launch();
}

size_t pw4_paged_cache_fork_workspace_size(int64_t n) { return n > 0 ? (size_t)n * 8 : 0; }

int pw4_paged_cache_fork(const pw4_page_pool* pool, int32_t* ref_counts, int32_t* block_tables, int64_t rows,
                         int64_t table_width, int64_t table_stride, int32_t* seq_lens, const int32_t* src_rows,
                         const int32_t* dst_rows, int64_t n, int64_t page_size, int32_t* missing, void* workspace,
                         size_t workspace_bytes, pw4_stream_t stream) {
    Pool p;
    if (const int rc = as_pool(pool, p)) return rc;
    if (const int rc = check_tables(ref_counts, block_tables, p.pages, rows, table_width, table_stride)) return rc;
    if (n < 0 || missing == nullptr || (rows && seq_lens == nullptr) || (n && (!src_rows || !dst_rows))) {
        return PW4_ERR_ARG;
    }
    if (page_size <= 0 || !small(page_size) || n > kMaxRows || !small(table_width * page_size)) return PW4_ERR_SHAPE;
    if (workspace_bytes < pw4_paged_cache_fork_workspace_size(n) || (n && workspace == nullptr)) {
        return PW4_ERR_WORKSPACE;
    }
    int32_t* const pairs = static_cast<int32_t*>(workspace);
    const ForkArgs a{ref_counts, block_tables, seq_lens, src_rows, dst_rows, missing, pairs, pairs + n, table_stride,
                     p.pages, (int32_t)table_width, (int32_t)rows, (int32_t)page_size, (int32_t)n};
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(fork_pages_kernel, dim3(1), dim3(kMetaThreads), (uint32_t)n * 4, s, a);
    if (n > 0) {
        const int blocks = (int)n + move_blocks(p, n);
        with_unit(pool_unit(p), [&](auto v) {
            hipLaunchKernelGGL(fork_kernel<decltype(v)>, dim3(blocks), dim3(256), 0, s, a, p);
        });
    }
    return check_launch();
}

int pw4_paged_cache_free(int32_t* ref_counts, int64_t num_pages, int32_t* block_tables, int64_t rows,
                         int64_t table_width, int64_t table_stride, int32_t* seq_lens, const int32_t* which, int64_t n,
                         pw4_stream_t stream) {
    if (const int rc = check_tables(ref_counts, block_tables, num_pages, rows, table_width, table_stride)) return rc;
    if (n < 0 || (rows && seq_lens == nullptr) || (n && which == nullptr)) return PW4_ERR_ARG;
    if (!small(n) || table_width > 65535 * 256) return PW4_ERR_SHAPE;
    if (n == 0 || rows == 0) return PW4_OK;
    const unsigned cols = (unsigned)std::max<int64_t>(1, ceil_div(table_width, 256));
    hipLaunchKernelGGL(free_kernel, dim3((unsigned)n, cols), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       ref_counts, (int)num_pages, block_tables, (int)rows, (int)table_width, table_stride, seq_lens,
                       which);
    return check_launch();
}

size_t pw4_paged_cache_compact_workspace_size(int64_t num_pages) {
    return num_pages > 0 ? (size_t)(2 + 2 * most_moves(num_pages) + num_pages) * 4 : 8;
}

int pw4_paged_cache_compact(const pw4_page_pool* pool, int32_t* ref_counts, int32_t* block_tables, int64_t rows,
                            int64_t table_width, int64_t table_stride, int32_t* used, void* workspace,
                            size_t workspace_bytes, pw4_stream_t stream) {
    Pool p;
    if (const int rc = as_pool(pool, p)) return rc;
    if (const int rc = check_tables(ref_counts, block_tables, p.pages, rows, table_width, table_stride)) return rc;
    if (used == nullptr) return PW4_ERR_ARG;
    if (workspace == nullptr || workspace_bytes < pw4_paged_cache_compact_workspace_size(p.pages)) {
        return PW4_ERR_WORKSPACE;
    }
    int32_t* const ws = static_cast<int32_t*>(workspace);
    const int64_t most = most_moves(p.pages);
    const CompactArgs a{ref_counts, block_tables, used, ws, ws + 2, ws + 2 + most, ws + 2 + 2 * most, table_stride,
                        p.pages, (int32_t)rows, (int32_t)table_width};
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(compact_pages_kernel, dim3(1), dim3(kMetaThreads), 0, s, a);
    if (p.pages > 1) {
        const int table_blocks = (int)std::min<int64_t>(256, std::max<int64_t>(1, ceil_div(rows * table_width, 1024)));
        const int blocks = table_blocks + move_blocks(p, p.pages / 2);
        with_unit(pool_unit(p), [&](auto v) {
            hipLaunchKernelGGL(compact_kernel<decltype(v)>, dim3(blocks), dim3(256), 0, s, a, p, table_blocks);
        });
    }
    return check_launch();
}

}  // extern "C"

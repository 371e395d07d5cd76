// kv.cu -- the paged key/value cache: the batch's plan, append with rotation,
// read, and the C ABI of include/ttl_kv.h.  The attention kernels are in
// kv_tokens.cu (few columns), kv_prompt.cu (many) and kv_attend.cu (32 bits, and
// the choice among them).
//
// Reference: store_kv and apply_rope of tt-lab (src/model.cpp:230-253), there
// for one token of one sequence in a contiguous f32 cache.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>

#include "internal.h"
#include "kv.cuh"
#include "kv_internal.h"
#include "ttl_kv.h"

namespace {

using namespace ttl::kv;

// ---- plan ----

struct PlanArgs {
    Plan *plan;
    Tile *tiles[2][2];
    int32_t *prefix[2][2];
    Cut *cuts[2][2];
    int4 *row[2];
    uint32_t *counters;
    uint32_t *status;
    const int32_t *row_start, *length, *pages, *first, *prefix_len;
    uint32_t page_stride;
    int seqs, rows, max_new, group, kv_heads, window, page_tokens;
    int width[2], gran[2], cost[2], ctas[2];  // ctas 0: no sequence goes to this kind
    int few;                         // sequences of at most this many columns go to kind 0
    int tile_cap[2];
};

constexpr int kPlanThreads = 1024;
constexpr int kNearTiles = 1024;
constexpr int kFewShare = 4;  // granules of each CTA of the prompt kernel
constexpr int kMaxPosition = (1 << 29) - 128;  // a tile counts up to 2^23 - 1 granules

struct SeqState {
    int row0, n, len;
    bool good;
};

__device__ SeqState load_seq(const PlanArgs &a, int s) {
    SeqState r;
    r.row0 = a.row_start[s];
    const int end = a.row_start[s + 1];
    r.len = a.length[s];
    const bool order = r.row0 >= 0 && end >= r.row0 && end <= a.rows;
    r.n = order ? end - r.row0 : 0;
    const long long room = (long long)(a.page_stride) * a.page_tokens;
    r.good = order && r.len >= r.n && r.len <= room && r.len <= kMaxPosition && r.n <= a.max_new;
    if (!r.good) {
        r.n = 0;
        r.len = 0;
    }
    return r;
}

// Exclusive scan of one int per thread over the block; total in *sum.
__device__ int block_scan(int v, int *sum, int *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        x += lane >= o ? y : 0;
    }
    if (lane == 31) {
        warp_sums[warp] = x;
    }
    __syncthreads();
    if (warp == 0) {
        int y = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            y += lane >= o ? z : 0;
        }
        warp_sums[lane] = y;
    }
    __syncthreads();
    const int base = warp ? warp_sums[warp - 1] : 0;
    *sum = warp_sums[31];
    __syncthreads();
    return base + x - v;
}

// CTAs 0 .. 3 build the tile list of (kind, window); the others write the rows'
// visible ranges.  Everything is read from the caller's arrays, so no CTA
// waits for another.  Latency-bound, a few dependent loads and three scans: 6 us
// for up to 1024 tiles.
__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(PlanArgs a) {
    __shared__ int sums[32];
    __shared__ int starts[4096 + 1];  // first tile of a sequence
    __shared__ Cut shared_cuts[kMaxCtas + 1];
    __shared__ int near_prefix[kNearTiles + 1];  // the granules before a tile, where there are few tiles
    const int tid = threadIdx.x;
    wait_previous();
    if (blockIdx.x >= 4) {
        const int r = (blockIdx.x - 4) * kPlanThreads + tid;
        if (r >= a.rows) {
            return;
        }
        int lo = 0, hi = a.seqs;  // last sequence with row_start <= r
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.row_start[mid] <= r) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        SeqState s = load_seq(a, lo);
        if (!(s.good && r >= s.row0 && r < s.row0 + s.n) && r < a.row_start[a.seqs]) {
            // row_start is out of order: the first good sequence that claims the row
            for (lo = 0; lo < a.seqs - 1; ++lo) {
                s = load_seq(a, lo);
                if (s.good && r >= s.row0 && r < s.row0 + s.n) {
                    break;
                }
            }
            s = load_seq(a, lo);
        }
        int4 full = make_int4(0, 0, 0, -1), slide = full;
        if (s.good && r >= s.row0 && r < s.row0 + s.n) {
            const int p = s.len - s.n + r - s.row0;
            const int first = a.first ? a.first[r] : 0;
            const int end = a.prefix_len ? min(max(p + 1, a.prefix_len[lo]), s.len) : p + 1;
            full = make_int4(p, max(first, 0), end, lo);
            slide = make_int4(p, max(max(first, 0), p - a.window + 1), end, lo);
        }
        a.row[0][r] = full;
        a.row[1][r] = slide;
        return;
    }
    const int kind = blockIdx.x >> 1, sliding = blockIdx.x & 1;
    if (blockIdx.x == 0 && tid == 0) {
        a.plan->pages = a.pages;
        a.plan->page_stride = a.page_stride;
        a.plan->seqs = a.seqs;
        a.plan->rows = a.rows;
        if (a.row_start[0] != 0) {
            ttl::set_status(a.status, kKvBadBatch);
        }
    }
    if (!sliding) {  // the merge counters of the kind start at zero
        for (int i = tid; i < kMaxCtas; i += kPlanThreads) {
            a.counters[kind * kMaxCtas + i] = 0;
        }
    }
    if (sliding && a.window == 0) {
        if (tid == 0) {
            a.plan->list[kind][1] = List{0, 0, 0, 0, {0, 0, 0, 0}};
        }
        return;
    }
    const int width = a.width[kind], gran = a.gran[kind], cost = a.cost[kind];
    Tile *tiles = a.tiles[kind][sliding];
    Cut *cuts = a.cuts[kind][sliding];
    // Where little of the batch's work lies with sequences of few columns, the
    // prompt kernel takes them too: the other's launch, with nothing to do then,
    // costs about 3 us instead of the 30 that a pass over one long sequence takes.
    int few = a.few;
    if (a.ctas[0] && a.ctas[1]) {
        int work = 0;
        for (int base = 0; base < a.seqs; base += kPlanThreads) {
            int n = 0;
            if (base + tid < a.seqs) {
                const SeqState q = load_seq(a, base + tid);
                const int keys = sliding && !a.prefix_len ? min(q.len, a.window + q.n) : q.len;
                n = q.n > 0 && q.n * a.group <= a.few ? min(keys / a.gran[1], kMaxCtas) + a.cost[1] : 0;
            }
            int sum;
            block_scan(n, &sum, sums);
            work += sum;
        }
        few = (long long)(work) * a.kv_heads <= kFewShare * a.ctas[1] ? 0 : few;
    }
    // tiles of each sequence
    int total = 0;
    for (int base = 0; base < a.seqs; base += kPlanThreads) {
        const int s = base + tid;
        int count = 0;
        if (s < a.seqs) {
            const SeqState q = load_seq(a, s);
            if (!q.good && blockIdx.x == 0) {
                ttl::set_status(a.status, kKvBadBatch);
            }
            const int columns = q.n * a.group;
            const bool mine = (columns <= few) == (kind == 0);
            count = (mine && columns > 0) ? (columns + width - 1) / width : 0;
        }
        int sum;
        const int at = block_scan(count, &sum, sums);
        if (s < a.seqs) {
            starts[s] = total + at;
        }
        total += sum;
    }
    if (a.ctas[kind] == 0) {
        total = 0;  // no launch of this kind follows
    }
    if (total > a.tile_cap[kind]) {
        if (tid == 0) {
            ttl::set_status(a.status, kKvBadBatch);
        }
        total = 0;
    }
    if (tid == 0) {
        starts[a.seqs] = total;
    }
    __syncthreads();
    // their key ranges
    int32_t *prefix = total <= kNearTiles ? near_prefix : a.prefix[kind][sliding];
    int line = 0;
    long long whole_line = 0;
    for (int base = 0; base < total; base += kPlanThreads) {
        const int t = base + tid;
        int n = 0;
        if (t < total) {
            int lo = 0, hi = a.seqs;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (starts[mid] <= t) {
                    lo = mid;
                } else {
                    hi = mid;
                }
            }
            const SeqState q = load_seq(a, lo);
            const int col0 = (t - starts[lo]) * width;
            const int ncols = min(width, q.n * a.group - col0);
            const int r0 = col0 / a.group, r1 = (col0 + ncols - 1) / a.group;
            const int p0 = q.len - q.n + r0, p1 = q.len - q.n + r1;
            const int pre = a.prefix_len ? min(a.prefix_len[lo], q.len) : 0;
            int begin, end;
            if (a.first) {
                begin = q.len, end = 0;
                for (int r = r0; r <= r1; ++r) {  // rows that see something
                    const int p = q.len - q.n + r;
                    const int b = max(max(a.first[q.row0 + r], 0), sliding ? p - a.window + 1 : 0);
                    const int e = max(p + 1, pre);
                    if (b < e) {
                        begin = min(begin, b);
                        end = max(end, e);
                    }
                }
            } else {
                begin = sliding ? max(0, p0 - a.window + 1) : 0;
                end = max(p1 + 1, pre);
            }
            const int g0 = begin < end ? begin / gran : 0;
            // at least one granule: a tile whose rows see nothing is written too
            n = begin < end ? (end + gran - 1) / gran - g0 : 1;
            tiles[t] = Tile{lo, col0, g0, uint32_t(ncols) | uint32_t(n) << 9, q.row0 + r0, col0 - r0 * a.group, q.len,
                            begin < end ? begin : kNoPosition};
            n += cost;
        }
        int sum;
        const int at = block_scan(n, &sum, sums);
        if (t < total) {
            prefix[t] = line + at;
        }
        line += sum;
        if (total > 255) {
            // the line is counted in 32 bits, which 255 tiles cannot pass: the upper parts'
            // sum gives the whole to within 2^22, its lower bits the rest
            int upper;
            block_scan(n >> 12, &upper, sums);
            whole_line += ((long long)(upper) << 12) + (uint32_t(sum) - (uint32_t(upper) << 12));
        }
    }
    if (whole_line > 0x7fffffff) {  // more work than weeks: refused
        if (tid == 0) {
            ttl::set_status(a.status, kKvBadBatch);
        }
        total = line = 0;
        __syncthreads();
    }
    if (tid == 0) {
        prefix[total] = line;
        a.plan->list[kind][sliding] = List{total, a.ctas[kind], width, gran, {0, 0, 0, 0}};
    }
    __syncthreads();
    // the cuts: equal shares of the line of all heads; a tile of few granules
    // is not cut, and no tile is cut next to its ends
    const long long all = (long long)(line) * a.kv_heads;
    // at least one unit per share, so that cuts inside a tile differ
    const int shares = int(min((long long)(a.ctas[kind]), all));
    for (int c = tid; c <= a.ctas[kind]; c += kPlanThreads) {
        Cut cut{total == 0 ? 0 : a.kv_heads, 0, 0, 0u};
        if (c < shares) {
            const long long pos = all * c / shares;
            cut.head = int(pos / line);
            const int rest = int(pos - (long long)(cut.head) * line);
            int lo = 0, hi = total;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (prefix[mid] <= rest) {
                    lo = mid;
                } else {
                    hi = mid;
                }
            }
            const int g = rest - prefix[lo] - cost, n = prefix[lo + 1] - prefix[lo] - cost;
            cut.tile = lo;
            if (n <= kNoSplit ? 2 * g < n : g < 2) {
                cut.gran = 0;
            } else if (n <= kNoSplit || n - g < 2) {
                cut.gran = 0;
                if (++cut.tile == total) {
                    cut.tile = 0;
                    ++cut.head;
                }
            } else {
                cut.gran = g;
            }
        }
        shared_cuts[c] = cut;
    }
    __syncthreads();
    // a cut inside a tile knows the CTAs that share the tile: those of the
    // neighbouring cuts inside it
    for (int c = tid; c <= a.ctas[kind]; c += kPlanThreads) {
        Cut cut = shared_cuts[c];
        if (cut.gran > 0) {
            int first = c - 1, last = c;
            while (shared_cuts[first].head == cut.head && shared_cuts[first].tile == cut.tile && shared_cuts[first].gran > 0) {
                --first;
            }
            while (shared_cuts[last + 1].head == cut.head && shared_cuts[last + 1].tile == cut.tile) {
                ++last;
            }
            cut.span = uint32_t(first) | uint32_t(last) << 16;
        }
        cuts[c] = cut;
    }
}

// ---- append ----

struct AppendArgs {
    const Plan *plan;
    const int4 *row;
    const void *k, *v, *q;
    void *q_out;
    size_t k_stride, v_stride, q_stride, q_out_stride;
    uint8_t *pool;  // this layer
    const double *turns;
    const double2 *table;      // cosine and sine of -1, -1 + 1/64 .. 1 half turns
    double rope_scale;
    uint32_t *status;
    int rows, q_heads, kv_heads, page_shift, pages, half, interleaved;  // half: rotated pairs (0: none)
    uint32_t block_bytes;
    // Blocks [0, q_blocks) take Q, the others K and V: [0] and [1] below.
    int q_blocks;
    int deep;                  // rows of a thread, up to kAppendRows
    int subs[2];               // groups of threads that share a CTA, each with its own rows
    int units[2];              // of a row
    uint32_t unit_div[2], pair_div;  // ceil(2^32 / n) of units and of half
};

constexpr int kAppendThreads = 256;
// Rows of a thread at most (f32: half as many, as their values take twice the
// registers), groups of threads of a CTA at most.
constexpr int kAppendRows = 4, kAppendSubs = 4;
__host__ __device__ constexpr int append_rows(int rows_type) {
    return rows_type == kF32 ? kAppendRows / 2 : kAppendRows;
}
constexpr int kMaxPairs = 64;

// i / n by the reciprocal above: exact while i * n < 2^32.
__device__ __forceinline__ int quotient(int i, uint32_t div) {
    return int(__umulhi(uint32_t(i), div));
}

// A row of the plan on the device.  A captured call may have more rows than the
// batch that ran last: what the table holds behind that batch's rows is another's
// (or nobody's), and such a row is padding.
template <class Args> __device__ __forceinline__ int4 planned_row(const Args &a, int r) {
    int4 x = a.row[r];  // a.rows entries are there, whoever's; neither load waits for the other
    x.w = r < a.plan->rows ? x.w : -1;
    return x;
}
// Reports a plan of another number of rows (one thread of the grid).
template <class Args> __device__ __forceinline__ void check_rows_of_plan(const Args &a) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.plan->rows != a.rows) {
        ttl::set_status(a.status, kKvStalePlan);
    }
}

// The slot of a row: the block of (page, head 0) and the token in it, or
// nullptr for padding and for a page outside the pool.
template <class Args> __device__ __forceinline__ uint8_t *row_slot(const Args &a, const int4 &ri, int &token) {
    if (ri.w < 0) {
        return nullptr;
    }
    const int id = a.plan->pages[size_t(ri.w) * a.plan->page_stride + size_t(ri.x >> a.page_shift)];
    token = ri.x & ((1 << a.page_shift) - 1);
    if (uint32_t(id) >= uint32_t(a.pages)) {
        ttl::set_status(a.status, kKvBadPage);
        return nullptr;
    }
    return const_cast<uint8_t *>(a.pool) + size_t(id) * a.kv_heads * a.block_bytes;
}

// E2M1 codes of two values that are already divided by their scale.
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
    uint32_t out;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(out) : "f"(lo), "f"(hi));
    return out;
}

// hi + lo (hi their sum to nearest) as one f32 rounded to odd: the f32 below in
// size, its last bit set unless lo is 0.  It keeps the order against every f32
// with an even last bit, so that rounding it to E2M1, whose borders are such
// numbers, and taking its exponent equals doing so with hi + lo.
__device__ __forceinline__ float to_odd(float hi, float lo) {
    if (lo == 0.0f || !(fabsf(hi) < INFINITY)) {
        return hi;
    }
    uint32_t b = __float_as_uint(hi);
    b -= ((__float_as_uint(lo) ^ b) >> 31) && (b << 1) ? 1u : 0u;
    return __uint_as_float(b | 1u);
}

// x c - y s to about 48 bits: c and s as sums of two f32, the products' and the
// difference's rounding errors kept by fused multiply-adds and a two-sum.
__device__ __forceinline__ float turned_odd(float x, float y, float ch, float cl, float sh, float sl) {
    const float p = x * ch, q = -(y * sh);
    const float ep = fmaf(x, ch, -p), eq = -fmaf(y, sh, q);
    const float z = p + q;
    const float t = z - p;
    const float ez = (p - (z - t)) + (q - t);
    const float lo = ez + (ep + eq + (x * cl - y * sl));
    const float hi = z + lo;
    return to_odd(hi, lo - (hi - z));
}

// Eight values of a block of 32 that four neighbouring lanes hold: the block's
// scale and this lane's codes, stored where `write`.  An infinity or NaN in any
// of the four marks the block.
__device__ __forceinline__ void quantize8(const float (&x)[8], int lane, bool write, uint8_t *block, size_t code_at, size_t scale_at) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);  // sizes order like their bits, NaN above infinity
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const bool finite = top < 0x7f800000u;
    // floor(log2(top)) - 2; a subnormal top has a scale below the smallest
    const int exp = max(int(top >> 23) - 127 - 2, -127);
    uint32_t codes = 0;
    if (finite) {
        const float inv = __uint_as_float(uint32_t(127 - exp) << 23);  // exact: exp is -127 .. 125
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            codes |= e2m1x2(x[j] * inv, x[j + 1] * inv) << (4 * j);
        }
    }
    if (write) {
        *reinterpret_cast<uint32_t *>(block + code_at) = codes;
        if ((lane & 3) == 0) {
            block[scale_at] = finite ? uint8_t(exp + 127) : uint8_t(255);
        }
    }
}

// Cosine and sine of `turn` half turns, |turn| <= 1, to about 2^-52: a table of the
// angles of 1/64 half turn (kTurnSteps + 1 entries from -1 on), and the rest of at
// most 1/128 half turn (0.0246 rad) by Taylor's series, whose next terms are
// below 2^-60.
constexpr int kTurnSteps = 128;
__device__ __forceinline__ void cos_sin(double turn, const double2 *table, double &c, double &s) {
    const double k = rint(turn * 64.0);
    const double x = (turn - k * 0.015625) * 3.14159265358979323846;
    const double2 t = table[int(k) + 64];
    const double z = x * x;
    const double sx = x * fma(z, fma(z, fma(z, -1.0 / 5040.0, 1.0 / 120.0), -1.0 / 6.0), 1.0);
    const double cx = fma(z, fma(z, fma(z, fma(z, 1.0 / 40320.0, -1.0 / 720.0), 1.0 / 24.0), -0.5), 1.0);
    c = t.x * cx - t.y * sx;
    s = t.y * cx + t.x * sx;
}

// A CTA takes a few rows' Q, or their K and V: the cosines and sines of the rows'
// pairs once, for all heads, then every head in units of 16 values (two runs of
// 8 that are rotated with one another).  A thread keeps its unit and goes
// through the rows with it, their loads in flight together and before the
// cosines are computed, so that what depends on the unit is computed once.  The
// angle is a fraction of a revolution in 64 bits (in 32, position times
// frequency has lost 7 bits of its fraction at position 131072), cut to its
// fractional part there; its cosine and sine are then good to 32 bits.
// Over a 4-bit cache, K and V go in units of 8 values, four lanes to a block of
// 32; K's cosines and sines are pairs of f32 and its codes are rounded once,
// from about 48 bits, so that they are those of the exact rotation.
// Every row is read and written once.  16384 bf16 rows of 64 query and 8 KV heads
// of 64 values into 4 bits (311 MB): 75 us, 4.1 TB/s.  No unit is full (issue 55 % of
// clocks, integer pipe 49 %, a third of the warps): a CTA is one chain of loads,
// cosines, barrier, rotation and stores, and three of them on an SM do not cover it.
// 509-row chunks of 16 bits 12 us, one token 5 us, of which most is the chain from
// the page id to the store.
template <int kRows, int kCache, int D>
__global__ void __launch_bounds__(kAppendThreads, 3) kv_append_kernel(AppendArgs a) {
    constexpr bool kFour = kCache == kMxfp4;
    constexpr int kSize = kRows == kF32 ? 4 : 2, kVec = 8 * kSize / 16;  // 16-byte words of a run
    constexpr int kDeep = append_rows(kRows), kMost = kDeep * kAppendSubs;
    __shared__ float2 cs[kMost * kMaxPairs];
    __shared__ float2 low[kFour ? kMost * kMaxPairs : 1];  // what cos and sin lack in f32
    __shared__ uint8_t *slots[kMost];
    __shared__ int tokens[kMost], good[kMost];
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31;
    const bool is_q = int(blockIdx.x) < a.q_blocks;
    const int part = is_q ? 0 : 1, block = is_q ? blockIdx.x : blockIdx.x - a.q_blocks;
    wait_previous();
    const int units = a.units[part], subs = a.subs[part], per_cta = a.deep * subs;
    const int r0 = block * per_cta, count = min(per_cta, a.rows - r0);
    const int sub = subs > 1 ? quotient(tid, a.unit_div[part]) : 0;
    const int step = subs > 1 ? units : threads;  // to the next unit of a thread
    const int mine = sub < subs ? min(a.deep, count - sub * a.deep) : 0;  // this thread's rows
    const int rs = sub * a.deep;                  // the first of them, in the CTA
    int i = subs > 1 ? tid - sub * units : tid;

    // What a unit is: 16 values of Q, or of K or V in the rows' type, or 8 of K or V in 4 bits.
    struct Unit {
        bool is_v;
        int head, ax, ay, turn, pair;  // the runs; turn: 0 none, 1 pairs across the runs, 2 pairs inside; first pair
        const uint8_t *src;
        size_t stride;
    };
    auto decode = [&](int u) {
        Unit x;
        const bool four = kFour && !is_q;
        const int per_head = four ? D / 8 : D / 16, kv = a.kv_heads * per_head;
        x.is_v = !is_q && u >= kv;
        u -= x.is_v ? kv : 0;
        x.head = u / per_head;
        u -= x.head * per_head;
        const int half = x.is_v ? 0 : a.half;
        if (four) {
            const int d = 8 * u;
            x.turn = d < 2 * half ? 1 + a.interleaved : 0;
            x.ax = d;
            x.ay = d >= half ? d - half : d + half;  // the run it is rotated with
            x.pair = x.turn == 2 ? d / 2 : (d >= half ? d - half : d);
        } else {
            // the rotated values are a multiple of 16: a unit is rotated whole or not at all
            x.turn = 16 * u < 2 * half ? 1 + a.interleaved : 0;
            x.ax = x.turn == 1 ? 8 * u : 16 * u;
            x.ay = x.turn == 1 ? half + 8 * u : 16 * u + 8;
            x.pair = 8 * u;
        }
        x.stride = (is_q ? a.q_stride : (x.is_v ? a.v_stride : a.k_stride)) * kSize;
        x.src = static_cast<const uint8_t *>(is_q ? a.q : (x.is_v ? a.v : a.k)) + size_t(r0 + rs) * x.stride + size_t(x.head) * (D * kSize);
        return x;
    };
    uint4 x[kDeep][kVec], y[kDeep][kVec];
    auto load = [&](const Unit &u) {
        const bool both = !(kFour && !is_q) || u.turn == 1;
#pragma unroll
        for (int r = 0; r < kDeep; ++r) {
            if (r < mine) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    x[r][j] = reinterpret_cast<const uint4 *>(u.src + r * u.stride + u.ax * kSize)[j];
                    if (both) {
                        y[r][j] = reinterpret_cast<const uint4 *>(u.src + r * u.stride + u.ay * kSize)[j];
                    }
                }
            }
        }
    };
    Unit unit{};
    if (i < units) {
        unit = decode(i);
        load(unit);
    }
    check_rows_of_plan(a);
    for (int r = tid; r < count; r += threads) {
        const int4 ri = planned_row(a, r0 + r);
        int token = 0;
        slots[r] = is_q ? nullptr : row_slot(a, ri, token);
        tokens[r] = token;
        good[r] = ri.w >= 0;
    }
    for (int n = tid; n < count * a.half; n += threads) {
        const int r = quotient(n, a.pair_div), pair = n - r * a.half;
        const double turn = double(a.row[r0 + r].x) * a.turns[pair];
        const double part_turn = 2.0 * (turn - rint(turn));  // half turns in [-1, 1]
        if (kFour && !is_q) {
            double sn, c;
            cos_sin(part_turn, a.table, c, sn);
            sn *= a.rope_scale, c *= a.rope_scale;
            const float2 h = make_float2(float(c), float(sn));
            cs[n] = h;
            if constexpr (kFour) {
                low[n] = make_float2(float(c - double(h.x)), float(sn - double(h.y)));
            }
        } else {
            float sn, c;
            sincospif(float(part_turn), &sn, &c);
            cs[n] = make_float2(c * float(a.rope_scale), sn * float(a.rope_scale));
        }
    }
    __syncthreads();
    if (!(kFour && !is_q)) {
        while (i < units) {
            uint8_t *out = is_q ? static_cast<uint8_t *>(a.q_out) + (size_t(r0 + rs) * a.q_out_stride + size_t(unit.head) * D) * kSize : nullptr;
            const size_t in_slot = size_t(unit.head) * a.block_bytes + (unit.is_v ? a.block_bytes >> 1 : 0);
#pragma unroll
            for (int r = 0; r < kDeep; ++r) {
                if (r >= mine || !good[rs + r] || (!is_q && !slots[rs + r])) {
                    continue;
                }
                uint8_t *dst = is_q ? out + r * a.q_out_stride * kSize : slots[rs + r] + in_slot + size_t(tokens[rs + r]) * (D * kSize);
                if (unit.turn) {
                    const float2 *c = cs + (rs + r) * a.half + unit.pair;
                    float p[8], q[8];
                    load8<kRows>(x[r], 0, p);
                    load8<kRows>(y[r], 0, q);
                    if (unit.turn == 1) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 t = c[j];
                            const float v = p[j], w = q[j];
                            p[j] = v * t.x - w * t.y;
                            q[j] = v * t.y + w * t.x;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 t = c[j];
                            float *z = j < 4 ? p + 2 * j : q + 2 * (j - 4);
                            const float v = z[0], w = z[1];
                            z[0] = v * t.x - w * t.y;
                            z[1] = v * t.y + w * t.x;
                        }
                    }
                    store8<kRows>(dst, unit.ax, p);
                    store8<kRows>(dst, unit.ay, q);
                } else {
#pragma unroll
                    for (int j = 0; j < kVec; ++j) {
                        reinterpret_cast<uint4 *>(dst + unit.ax * kSize)[j] = x[r][j];
                        reinterpret_cast<uint4 *>(dst + unit.ay * kSize)[j] = y[r][j];
                    }
                }
            }
            i += step;
            if (subs > 1 || i >= units) {
                break;
            }
            unit = decode(i);
            load(unit);
        }
    }
    if constexpr (kFour) {
        // four lanes to a block of 32: units, threads and groups are multiples of four, so
        // a block's lanes are in the loop together; the shuffles name the lanes that are
        while (!is_q && __any_sync(0xffffffffu, i < units)) {
            const bool have = i < units;
#pragma unroll
            for (int r = 0; r < kDeep; ++r) {
                const bool row = have && r < mine;
                if (!__any_sync(0xffffffffu, row)) {
                    continue;
                }
                float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (row) {
                    load8<kRows>(x[r], 0, z);
                    const float2 *c = cs + (rs + r) * a.half + unit.pair, *e = low + (rs + r) * a.half + unit.pair;
                    if (unit.turn == 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 h = c[j], l = e[j];
                            const float p = z[2 * j], q = z[2 * j + 1];
                            z[2 * j] = turned_odd(p, q, h.x, l.x, h.y, l.y);
                            z[2 * j + 1] = turned_odd(q, -p, h.x, l.x, h.y, l.y);
                        }
                    } else if (unit.turn == 1) {
                        float w[8];
                        load8<kRows>(y[r], 0, w);
                        const float sign = unit.ax >= a.half ? -1.0f : 1.0f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 h = c[j], l = e[j];
                            z[j] = turned_odd(z[j], sign * w[j], h.x, l.x, h.y, l.y);
                        }
                    }
                }
                const bool write = row && slots[rs + r] != nullptr;
                const int token = write ? tokens[rs + r] : 0;
                quantize8(z, lane, write, write ? slots[rs + r] + size_t(unit.head) * a.block_bytes + (unit.is_v ? a.block_bytes >> 1 : 0) : nullptr,
                          size_t(token) * (D / 2) + unit.ax / 2,
                          (size_t(1) << a.page_shift) * (D / 2) + size_t(token) * (D / 32) + unit.ax / 32);
            }
            i += step;
            if (subs > 1) {
                break;
            }
            if (i < units) {
                unit = decode(i);
                load(unit);
            }
        }
    }
}

// ---- read ----

struct ReadArgs {
    const Plan *plan;
    const int4 *row;
    void *k, *v;
    size_t k_stride, v_stride;
    const uint8_t *pool;
    uint32_t *status;
    int rows, kv_heads, page_shift, pages;
    uint32_t block_bytes;
    int per_cta;
};

// A CTA takes a few rows; a thread keeps its 8 values of a head and goes through
// the rows with them, their loads in flight together.  16384 rows of 8 heads of 64
// values out of 4 bits to bf16 (43 MB) 16 us, 2.7 TB/s, two fifths of a copy's rate:
// a lane asks for 4 bytes of codes and one of scale at a time.
template <int kRows, int kCache, int D> __global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    __shared__ const uint8_t *slots[kAppendRows];
    __shared__ int tokens[kAppendRows];
    wait_previous();
    const int tid = threadIdx.x, r0 = blockIdx.x * a.per_cta;
    const int count = min(a.per_cta, a.rows - r0);
    check_rows_of_plan(a);
    if (tid < count) {
        int token = 0;
        slots[tid] = row_slot(a, planned_row(a, r0 + tid), token);
        tokens[tid] = token;
    }
    __syncthreads();
    constexpr int kUnits = D / 8;
    const int ku = a.kv_heads * kUnits;
    for (int i = tid; i < 2 * ku; i += int(blockDim.x)) {
        const bool is_v = i >= ku;
        const int u = is_v ? i - ku : i;
        const int head = u / kUnits, d = 8 * (u - head * kUnits);
        const size_t in_slot = size_t(head) * a.block_bytes + (is_v ? a.block_bytes >> 1 : 0);
        const size_t stride = is_v ? a.v_stride : a.k_stride, to = size_t(r0) * stride + size_t(head) * D + d;
        float x[kAppendRows][8];
#pragma unroll
        for (int r = 0; r < kAppendRows; ++r) {
            if (r < count && slots[r]) {
                const uint8_t *block = slots[r] + in_slot;
                if constexpr (kCache != kMxfp4) {
                    load8<kCache>(block, size_t(tokens[r]) * D + d, x[r]);
                } else {
                    const uint32_t codes = *reinterpret_cast<const uint32_t *>(block + size_t(tokens[r]) * (D / 2) + d / 2);
                    const float f = scale_of(block[(size_t(1) << a.page_shift) * (D / 2) + size_t(tokens[r]) * (D / 32) + d / 32]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v = __half22float2(ttl::e2m1x2_to_half2((codes >> (8 * j)) & 255u));
                        x[r][2 * j] = v.x * f, x[r][2 * j + 1] = v.y * f;
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kAppendRows; ++r) {
            if (r < count && slots[r]) {
                store8<kRows>(is_v ? a.v : a.k, to + r * stride, x[r]);
            }
        }
    }
}

// ---- host ----

int kv_fail(ttl_kv *h, int code, const std::string &msg) {
    if (h) {
        h->error = msg;
    }
    return ttl::fail(nullptr, code, msg);
}

#define TTL_KV_CUDA(h, expr)                                                                           \
    do {                                                                                               \
        const cudaError_t e_ = (expr);                                                                 \
        if (e_ != cudaSuccess) {                                                                       \
            cudaGetLastError();                                                                        \
            return kv_fail((h), TTL_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_));     \
        }                                                                                              \
    } while (0)

// Makes the handle's device current and the caller's again on return.
struct DeviceGuard {
    int before = -1;
    cudaError_t error;
    explicit DeviceGuard(int device) {
        error = cudaGetDevice(&before);
        if (error == cudaSuccess && before != device) {
            error = cudaSetDevice(device);
        } else {
            before = -1;
        }
    }
    ~DeviceGuard() {
        if (before >= 0) {
            cudaSetDevice(before);
        }
    }
};

template <class T> int kv_alloc(ttl_kv *h, T **p, size_t count) {
    void *q = nullptr;
    const cudaError_t e = cudaMalloc(&q, std::max<size_t>(count, 1) * sizeof(T));
    if (e != cudaSuccess) {
        cudaGetLastError();
        return kv_fail(h, TTL_ERR_CUDA, "device allocation of " + std::to_string(count * sizeof(T)) + " bytes failed");
    }
    h->allocations.push_back(q);
    *p = static_cast<T *>(q);
    return TTL_OK;
}

size_t type_size(int t) {
    return t == kF32 ? 4 : 2;
}

// A device array the kernels will read or write.
int check_pointer(ttl_kv *h, const void *p, const char *name, size_t align) {
    if (!p) {
        return kv_fail(h, TTL_ERR_ARGUMENT, std::string("null ") + name);
    }
    if (reinterpret_cast<uintptr_t>(p) % align) {
        return kv_fail(h, TTL_ERR_ARGUMENT, std::string(name) + " is not aligned to " + std::to_string(align) + " bytes");
    }
    unsigned kind = 0, managed = 0;
    int device = -1;
    CUpointer_attribute what[3] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, CU_POINTER_ATTRIBUTE_IS_MANAGED};
    void *into[3] = {&kind, &device, &managed};
    if (h->attributes(3, what, into, reinterpret_cast<CUdeviceptr>(p)) != CUDA_SUCCESS || kind == 0) {
        return kv_fail(h, TTL_ERR_ARGUMENT, std::string(name) + " is not a device pointer");
    }
    if (!managed && (kind != CU_MEMORYTYPE_DEVICE || device != h->device)) {
        return kv_fail(h, TTL_ERR_ARGUMENT, std::string(name) + " is not memory of the handle's GPU");
    }
    return TTL_OK;
}

// A row array: pointer, and a stride that holds a row and keeps its alignment.
int check_rows(ttl_kv *h, const void *p, size_t stride, int heads, const char *name) {
    if (h->rows == 0) {
        return TTL_OK;
    }
    const int rc = check_pointer(h, p, name, 16);
    if (rc) {
        return rc;
    }
    if (stride < size_t(heads) * h->dim || stride > (size_t(1) << 40) || stride * type_size(h->rows_type) % 16) {
        return kv_fail(h, TTL_ERR_ARGUMENT,
                       std::string(name) + ": a row stride is at least heads * head_dim and a multiple of 16 bytes");
    }
    return TTL_OK;
}

// Two row arrays of a call, one of which is written, that share memory: blocks write
// in no order what others still read.  Rows of one stride may lie side by side (views
// of one projection); of different strides they must not interleave.
int check_apart(ttl_kv *h, const void *out, size_t out_stride, int out_heads, const char *out_name, const void *in, size_t in_stride,
                int in_heads, const char *in_name) {
    if (h->rows == 0) {
        return TTL_OK;
    }
    const size_t size = type_size(h->rows_type), rows = size_t(h->rows), so = out_stride * size, si = in_stride * size;
    const size_t wo = size_t(out_heads) * h->dim * size, wi = size_t(in_heads) * h->dim * size;
    const uintptr_t o = reinterpret_cast<uintptr_t>(out), i = reinterpret_cast<uintptr_t>(in);
    if (o + (rows - 1) * so + wo <= i || i + (rows - 1) * si + wi <= o) {
        return TTL_OK;
    }
    if (rows > 1 && so == si) {
        const size_t from = i >= o ? (i - o) % so : (so - (o - i) % so) % so;  // of in's rows behind out's
        if (from >= wo && from + wi <= so) {
            return TTL_OK;
        }
    }
    return kv_fail(h, TTL_ERR_ARGUMENT, std::string(out_name) + " overlaps " + in_name);
}

int check_layer(ttl_kv *h, int layer) {
    if (layer < 0 || layer >= h->layers) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "layer " + std::to_string(layer) + " out of range");
    }
    if (!h->batched) {
        return kv_fail(h, TTL_ERR_STATE, "no batch: call ttl_kv_batch_async first");
    }
    return TTL_OK;
}

uint32_t reciprocal(int n) {
    return n > 1 ? uint32_t(((uint64_t(1) << 32) + n - 1) / n) : 0;
}

// Rows of a thread: one while there are too few to fill the GPU.
int rows_of_a_thread(const ttl_kv *h, int rows) {
    return rows <= 4 * h->sms ? 1 : append_rows(h->rows_type);
}

template <int kRows, int kCache, int D> cudaError_t launch_append(ttl_kv *h, const AppendArgs &args) {
    AppendArgs a = args;
    a.units[0] = a.q ? a.q_heads * (D / 16) : 0;
    a.units[1] = 2 * a.kv_heads * (kCache == kMxfp4 ? D / 8 : D / 16);
    // threads: the wider part's units in equal passes of at most 256; the
    // narrower part puts several rows side by side
    const int most = std::max(a.units[0], a.units[1]), passes = (most + kAppendThreads - 1) / kAppendThreads;
    const int threads = std::max(((most + passes - 1) / passes + 31) / 32 * 32, 64);
    a.deep = rows_of_a_thread(h, a.rows);
    int blocks[2] = {0, 0};
    for (int p = 0; p < 2; ++p) {
        if (a.units[p] == 0) {
            a.subs[p] = 1;
            continue;
        }
        // groups of a 4-bit part's lanes stay whole: its units are a multiple of 16
        a.subs[p] = a.deep > 1 ? std::min(std::max(threads / a.units[p], 1), kAppendSubs) : 1;
        a.unit_div[p] = reciprocal(a.units[p]);
        blocks[p] = (a.rows + a.deep * a.subs[p] - 1) / (a.deep * a.subs[p]);
    }
    a.q_blocks = blocks[0];
    a.pair_div = a.half > 1 ? reciprocal(a.half) : 0;
    return launch_chained(kv_append_kernel<kRows, kCache, D>, blocks[0] + blocks[1], threads, 0, h->stream, a);
}

template <int kRows, int kCache, int D> cudaError_t launch_read(ttl_kv *h, const ReadArgs &args) {
    ReadArgs a = args;
    a.per_cta = rows_of_a_thread(h, a.rows);
    const int threads = std::min(256, (2 * a.kv_heads * (D / 8) + 31) / 32 * 32);
    return launch_chained(kv_read_kernel<kRows, kCache, D>, (a.rows + a.per_cta - 1) / a.per_cta, threads, 0, h->stream, a);
}

// Tensor maps of a 16-bit pool, one per layer: rows of head_dim values (K and V
// of a head's page follow one another), boxes of 64 values x up to 64 rows, with
// the 128-byte swizzle that ldmatrix and the matrix instructions read.
int build_maps(ttl_kv *h) {
    if (h->rows_type == kF32 || h->cache_type == kMxfp4) {
        h->maps.resize(size_t(h->layers));
        return TTL_OK;
    }
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        return kv_fail(h, TTL_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    }
    h->maps.resize(size_t(h->layers));
    const cuuint64_t rows = cuuint64_t(h->pages) * h->kv_heads * 2 * h->page_tokens;
    if (rows > (cuuint64_t(1) << 31)) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "pages * kv_heads * page_tokens must be at most 2^30");  // coordinates are 32 bits
    }
    const cuuint64_t dims[2] = {cuuint64_t(h->dim), rows}, strides[1] = {cuuint64_t(h->dim) * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(std::min(h->page_tokens, 64))}, ones[2] = {1, 1};
    for (int i = 0; i < h->layers; ++i) {
        const CUresult r = reinterpret_cast<Encode>(fn)(
            &h->maps[size_t(i)], h->rows_type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
            h->pool + size_t(i) * h->layer_bytes, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) {
            return kv_fail(h, TTL_ERR_CUDA, "cuTensorMapEncodeTiled rejected the pool's map");
        }
    }
    return TTL_OK;
}

std::string config_error(const ttl_kv_config &c) {
    auto in = [](uint32_t v, uint32_t lo, uint32_t hi) { return v >= lo && v <= hi; };
    if (!in(c.layers, 1, 256)) return "layers must be 1..256";
    if (!in(c.pages, 1, 1u << 24)) return "pages must be 1..2^24";
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
        return "page_tokens must be 16, 32, 64 or 128";
    if (!in(c.q_heads, 1, 256) || !in(c.kv_heads, 1, 256) || c.q_heads % c.kv_heads)
        return "q_heads must be 1..256 and a multiple of kv_heads";
    if (c.head_dim != 64 && c.head_dim != 128) return "head_dim must be 64 or 128";
    if (c.rows_type > TTL_KV_BF16) return "rows_type must be TTL_KV_F32, TTL_KV_F16 or TTL_KV_BF16";
    if (c.cache_type != c.rows_type && c.cache_type != TTL_KV_MXFP4) return "cache_type must be rows_type or TTL_KV_MXFP4";
    if (!in(c.max_seqs, 1, 4096)) return "max_seqs must be 1..4096";
    if (!in(c.max_rows, 1, 1u << 20)) return "max_rows must be 1..2^20";
    if (c.window > (1u << 30)) return "window must be at most 2^30";
    if (c.rope_dims % 16 || c.rope_dims > c.head_dim) return "rope_dims must be a multiple of 16 up to head_dim";
    if (c.rope_interleaved > 1) return "rope_interleaved must be 0 or 1";
    if (c.rope_dims && !c.rope_freq) return "rope_dims without rope_freq";
    if (!std::isfinite(c.rope_scale)) return "rope_scale must be finite";
    for (uint32_t i = 0; i < c.rope_dims / 2; ++i) {
        if (!std::isfinite(c.rope_freq[i])) return "rope_freq must be finite";
    }
    return "";
}

int kv_create(const ttl_kv_config *c, ttl_kv **out) {
    if (!c || !out) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "null argument");
    }
    *out = nullptr;
    const std::string bad = config_error(*c);
    if (!bad.empty()) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, bad);
    }
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
        cudaGetLastError();
        return kv_fail(nullptr, TTL_ERR_UNSUPPORTED, "no CUDA device");
    }
    int device = c->device;
    if (device < 0 && cudaGetDevice(&device) != cudaSuccess) {
        return kv_fail(nullptr, TTL_ERR_CUDA, "cudaGetDevice failed");
    }
    if (device >= count) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "device ordinal out of range");
    }
    cudaDeviceProp prop{};
    if (cudaGetDeviceProperties(&prop, device) != cudaSuccess || prop.major != 10) {
        cudaGetLastError();
        return kv_fail(nullptr, TTL_ERR_UNSUPPORTED, "the kernels are built for sm_100a (B200)");
    }
    DeviceGuard guard(device);
    if (guard.error != cudaSuccess) {
        return kv_fail(nullptr, TTL_ERR_CUDA, "cudaSetDevice failed");
    }
    ttl_kv *h = new ttl_kv();
    auto bail = [&](int rc, const std::string &why) {
        ttl_kv_destroy(h);
        return kv_fail(nullptr, rc, why);
    };
    h->device = device;
    h->sms = prop.multiProcessorCount;
    h->layers = int(c->layers), h->pages = int(c->pages), h->page_tokens = int(c->page_tokens);
    h->page_shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
    h->q_heads = int(c->q_heads), h->kv_heads = int(c->kv_heads), h->dim = int(c->head_dim);
    h->rows_type = int(c->rows_type), h->cache_type = int(c->cache_type);
    h->max_seqs = int(c->max_seqs), h->max_rows = int(c->max_rows), h->window = int(c->window);
    h->rope_dims = int(c->rope_dims), h->interleaved = int(c->rope_interleaved);
    h->rope_scale = c->rope_scale == 0.0 ? 1.0 : c->rope_scale;
    h->block_bytes = 2 * uint32_t(h->page_tokens) * row_bytes(h->cache_type, h->dim);
    h->layer_bytes = size_t(h->pages) * h->kv_heads * h->block_bytes;
    if (c->stream) {
        h->stream = static_cast<cudaStream_t>(c->stream);
    } else {
        if (cudaStreamCreateWithFlags(&h->stream, cudaStreamNonBlocking) != cudaSuccess) {
            cudaGetLastError();
            return bail(TTL_ERR_CUDA, "cannot create a stream");
        }
        h->own_stream = true;
    }
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found{};
    if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &fn, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        return bail(TTL_ERR_CUDA, "cuPointerGetAttributes is not available");
    }
    h->attributes = reinterpret_cast<ttl_kv::Attributes>(fn);
    const int group = h->q_heads / h->kv_heads;
    // tiles of the narrowest width a list can have; see choose_shapes
    h->tile_cap[0] = int(std::min<long long>((long long)(h->max_rows) * group / kNarrow + h->max_seqs, 1 << 28));
    h->tile_cap[1] = int((long long)(h->max_rows) * group / kPromptWidth + h->max_seqs);
    const cudaError_t ec = kv_configure(*h);
    if (ec != cudaSuccess) {
        cudaGetLastError();
        return bail(TTL_ERR_CUDA, std::string("cannot configure the kernels: ") + cudaGetErrorString(ec));
    }
    const size_t part = kv_part_floats(*h);
    int rc = kv_alloc(h, &h->pool, h->layer_bytes * h->layers);
    rc = rc ? rc : kv_alloc(h, &h->turns, size_t(h->rope_dims / 2));
    rc = rc ? rc : kv_alloc(h, &h->table, kTurnSteps + 1);
    rc = rc ? rc : kv_alloc(h, &h->plan, 1);
    for (int k = 0; k < kKinds && !rc; ++k) {
        for (int w = 0; w < (h->window ? 2 : 1) && !rc; ++w) {
            rc = rc ? rc : kv_alloc(h, &h->tiles[k][w], size_t(h->tile_cap[k]));
            rc = rc ? rc : kv_alloc(h, &h->prefix[k][w], size_t(h->tile_cap[k]) + 1);
            rc = rc ? rc : kv_alloc(h, &h->cuts[k][w], kMaxCtas + 1);
        }
    }
    rc = rc ? rc : kv_alloc(h, &h->row[0], size_t(h->max_rows));
    rc = rc ? rc : kv_alloc(h, &h->row[1], size_t(h->max_rows));
    rc = rc ? rc : kv_alloc(h, &h->part, part);
    rc = rc ? rc : kv_alloc(h, &h->counters, size_t(kKinds) * kMaxCtas);
    rc = rc ? rc : kv_alloc(h, &h->status, 1);
    rc = rc ? rc : build_maps(h);
    if (rc) {
        return bail(rc, h->error);
    }
    double turns[kMaxPairs] = {};
    for (int i = 0; i < h->rope_dims / 2; ++i) {
        turns[i] = c->rope_freq[i] / 6.283185307179586476925286766559;
    }
    double2 table[kTurnSteps + 1];
    for (int i = 0; i <= kTurnSteps; ++i) {
        // from the first octant, so that equal angles have equal values
        const int k = std::abs(i - 64), m = std::min(k, 64 - k), n = std::min(m, 32 - m);
        const double x = n * (3.141592653589793238462643383279502884 / 64.0);
        const double c = m <= 16 ? std::cos(x) : std::sin(x), s = m <= 16 ? std::sin(x) : std::cos(x);
        table[i] = make_double2(k <= 32 ? c : -c, i < 64 ? -s : s);
    }
    cudaError_t e = cudaMemsetAsync(h->pool, 0, h->layer_bytes * h->layers, h->stream);
    e = e ? e : cudaMemsetAsync(h->plan, 0, sizeof(Plan), h->stream);
    e = e ? e : cudaMemsetAsync(h->counters, 0, sizeof(uint32_t) * kKinds * kMaxCtas, h->stream);
    e = e ? e : cudaMemsetAsync(h->status, 0, sizeof(uint32_t), h->stream);
    e = e ? e : cudaMemcpyAsync(h->turns, turns, sizeof(double) * size_t(h->rope_dims / 2), cudaMemcpyHostToDevice, h->stream);
    e = e ? e : cudaMemcpyAsync(h->table, table, sizeof(table), cudaMemcpyHostToDevice, h->stream);
    e = e ? e : cudaStreamSynchronize(h->stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return bail(TTL_ERR_CUDA, std::string("device initialisation: ") + cudaGetErrorString(e));
    }
    *out = h;
    return TTL_OK;
}

int kv_batch(ttl_kv *h, uint32_t seqs, uint32_t rows, uint32_t max_new, const int32_t *row_start, const int32_t *length,
             const int32_t *pages, uint32_t page_stride, const int32_t *first, const int32_t *prefix) {
    if (!h) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "null handle");
    }
    if (seqs == 0 || seqs > uint32_t(h->max_seqs)) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "seqs must be 1..max_seqs");
    }
    if (rows > uint32_t(h->max_rows)) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "rows exceed max_rows");
    }
    if (page_stride == 0 || page_stride > (1u << 26)) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "page_stride must be 1..2^26");
    }
    DeviceGuard guard(h->device);
    TTL_KV_CUDA(h, guard.error);
    int rc = check_pointer(h, row_start, "row_start", 4);
    rc = rc ? rc : check_pointer(h, length, "length", 4);
    rc = rc ? rc : check_pointer(h, pages, "pages", 4);
    rc = (rc || !first) ? rc : check_pointer(h, first, "first", 4);
    rc = (rc || !prefix) ? rc : check_pointer(h, prefix, "prefix", 4);
    if (rc) {
        return rc;
    }
    max_new = std::min(max_new, rows);
    PlanArgs a{};
    a.plan = h->plan;
    for (int k = 0; k < kKinds; ++k) {
        for (int w = 0; w < 2; ++w) {
            a.tiles[k][w] = h->tiles[k][w];
            a.prefix[k][w] = h->prefix[k][w];
            a.cuts[k][w] = h->cuts[k][w];
        }
    }
    a.row[0] = h->row[0], a.row[1] = h->row[1];
    a.counters = h->counters, a.status = h->status;
    a.row_start = row_start, a.length = length, a.pages = pages, a.first = first, a.prefix_len = prefix;
    a.page_stride = page_stride;
    a.seqs = int(seqs), a.rows = int(rows), a.max_new = int(max_new);
    a.group = h->q_heads / h->kv_heads, a.kv_heads = h->kv_heads, a.window = h->window, a.page_tokens = h->page_tokens;
    Shape shape[kKinds];
    a.few = choose_shapes(*h, int(seqs), int(max_new), shape);
    for (int k = 0; k < kKinds; ++k) {
        a.width[k] = h->width[k] = shape[k].width;
        a.gran[k] = shape[k].gran;
        a.cost[k] = shape[k].cost;
        a.ctas[k] = h->ctas[k] = shape[k].ctas;
        a.tile_cap[k] = h->tile_cap[k];
    }
    TTL_KV_CUDA(h, launch_chained(kv_plan_kernel, 4 + int((rows + kPlanThreads - 1) / kPlanThreads), kPlanThreads, 0, h->stream, a));
    h->batched = true;
    h->seqs = int(seqs), h->rows = int(rows);
    return TTL_OK;
}

int kv_append(ttl_kv *h, int layer, int rotate, const void *k, size_t k_stride, const void *v, size_t v_stride, const void *q,
              size_t q_stride, void *q_out, size_t q_out_stride) {
    if (!h) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "null handle");
    }
    int rc = check_layer(h, layer);
    if (rc) {
        return rc;
    }
    if ((q == nullptr) != (q_out == nullptr)) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "q and q_out go together");
    }
    if (q && q == q_out && q_stride != q_out_stride) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "q rotated in place has one stride");
    }
    DeviceGuard guard(h->device);
    TTL_KV_CUDA(h, guard.error);
    rc = check_rows(h, k, k_stride, h->kv_heads, "k");
    rc = rc ? rc : check_rows(h, v, v_stride, h->kv_heads, "v");
    rc = (rc || !q) ? rc : check_rows(h, q, q_stride, h->q_heads, "q");
    rc = (rc || !q) ? rc : check_rows(h, q_out, q_out_stride, h->q_heads, "q_out");
    rc = (rc || !q || q == q_out) ? rc : check_apart(h, q_out, q_out_stride, h->q_heads, "q_out", q, q_stride, h->q_heads, "q");
    rc = (rc || !q) ? rc : check_apart(h, q_out, q_out_stride, h->q_heads, "q_out", k, k_stride, h->kv_heads, "k");
    rc = (rc || !q) ? rc : check_apart(h, q_out, q_out_stride, h->q_heads, "q_out", v, v_stride, h->kv_heads, "v");
    if (rc || h->rows == 0) {
        return rc;
    }
    AppendArgs a{};
    a.plan = h->plan, a.row = h->row[0];
    a.k = k, a.v = v, a.q = q, a.q_out = q_out;
    a.k_stride = k_stride, a.v_stride = v_stride, a.q_stride = q_stride, a.q_out_stride = q_out_stride;
    a.pool = h->pool + size_t(layer) * h->layer_bytes;
    a.turns = h->turns, a.table = h->table, a.rope_scale = h->rope_scale, a.status = h->status;
    a.rows = h->rows, a.q_heads = h->q_heads, a.kv_heads = h->kv_heads, a.page_shift = h->page_shift, a.pages = h->pages;
    a.half = rotate ? h->rope_dims / 2 : 0, a.interleaved = h->interleaved, a.block_bytes = h->block_bytes;
    TTL_KV_CUDA(h, TTL_KV_DISPATCH(h, launch_append, h, a));
    return TTL_OK;
}

int kv_read(ttl_kv *h, int layer, void *k, size_t k_stride, void *v, size_t v_stride) {
    if (!h) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "null handle");
    }
    int rc = check_layer(h, layer);
    if (rc) {
        return rc;
    }
    DeviceGuard guard(h->device);
    TTL_KV_CUDA(h, guard.error);
    rc = check_rows(h, k, k_stride, h->kv_heads, "k");
    rc = rc ? rc : check_rows(h, v, v_stride, h->kv_heads, "v");
    rc = rc ? rc : check_apart(h, v, v_stride, h->kv_heads, "v", k, k_stride, h->kv_heads, "k");
    if (rc || h->rows == 0) {
        return rc;
    }
    ReadArgs a{h->plan, h->row[0], k, v, k_stride, v_stride, h->pool + size_t(layer) * h->layer_bytes, h->status,
               h->rows, h->kv_heads, h->page_shift, h->pages, h->block_bytes, 0};
    TTL_KV_CUDA(h, TTL_KV_DISPATCH(h, launch_read, h, a));
    return TTL_OK;
}

int kv_attend(ttl_kv *h, int layer, uint32_t flags, const void *q, size_t q_stride, void *out, size_t out_stride, float scale,
              float cap, const float *sinks, const float *slopes) {
    if (!h) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "null handle");
    }
    int rc = check_layer(h, layer);
    if (rc) {
        return rc;
    }
    if (flags & ~TTL_KV_SLIDING) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "unknown flags");
    }
    if ((flags & TTL_KV_SLIDING) && h->window == 0) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "a sliding call on a handle without a window");
    }
    if (!std::isfinite(scale) || !std::isfinite(cap) || cap < 0.0f) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "scale must be finite, cap finite and not negative");
    }
    if (q == out && h->rows > 0) {
        return kv_fail(h, TTL_ERR_ARGUMENT, "out must not be q");
    }
    DeviceGuard guard(h->device);
    TTL_KV_CUDA(h, guard.error);
    rc = check_rows(h, q, q_stride, h->q_heads, "q");
    rc = rc ? rc : check_rows(h, out, out_stride, h->q_heads, "out");
    rc = rc ? rc : check_apart(h, out, out_stride, h->q_heads, "out", q, q_stride, h->q_heads, "q");
    rc = (rc || !sinks) ? rc : check_pointer(h, sinks, "sinks", 4);
    rc = (rc || !slopes) ? rc : check_pointer(h, slopes, "slopes", 4);
    if (rc || h->rows == 0) {
        return rc;
    }
    const int w = (flags & TTL_KV_SLIDING) ? 1 : 0;
    for (int kind = 0; kind < kKinds; ++kind) {
        if (h->ctas[kind] == 0) {
            continue;
        }
        AttendArgs a{};
        a.walk = Walk{h->plan, &h->plan->list[kind][w], h->tiles[kind][w], h->cuts[kind][w], h->row[w]};
        a.pool = h->pool + size_t(layer) * h->layer_bytes;
        a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
        a.sinks = sinks, a.slopes = slopes;
        a.part = h->part, a.counters = h->counters + kind * kMaxCtas, a.status = h->status;
        a.scale = scale == 0.0f ? 1.0f / std::sqrt(float(h->dim)) : scale;
        a.cap = cap;
        a.rows = h->rows, a.group = h->q_heads / h->kv_heads, a.page_shift = h->page_shift, a.pages = h->pages;
        a.kv_heads = h->kv_heads, a.block_bytes = h->block_bytes;
        a.other_ctas = h->ctas[1 - kind];
        a.group_div = uint32_t(((1 << 20) + a.group - 1) / a.group);
        TTL_KV_CUDA(h, launch_attend(*h, a, kind, layer));
    }
    return TTL_OK;
}

int kv_sync(ttl_kv *h) {
    if (!h) {
        return kv_fail(nullptr, TTL_ERR_ARGUMENT, "null handle");
    }
    DeviceGuard guard(h->device);
    TTL_KV_CUDA(h, guard.error);
    uint32_t st = 0;
    TTL_KV_CUDA(h, cudaMemcpyAsync(&st, h->status, sizeof(st), cudaMemcpyDeviceToHost, h->stream));
    TTL_KV_CUDA(h, cudaStreamSynchronize(h->stream));
    if (!st) {
        return TTL_OK;
    }
    // a kernel that gave up leaves counters behind: both start again at zero
    TTL_KV_CUDA(h, cudaMemsetAsync(h->status, 0, sizeof(uint32_t), h->stream));
    TTL_KV_CUDA(h, cudaMemsetAsync(h->counters, 0, sizeof(uint32_t) * kKinds * kMaxCtas, h->stream));
    TTL_KV_CUDA(h, cudaStreamSynchronize(h->stream));
    std::string why = "device status:";
    why += (st & kKvBadBatch) ? " row_start or length out of order or range;" : "";
    why += (st & kKvBadPage) ? " a page id outside the pool;" : "";
    why += (st & kKvWait) ? " bounded-wait-timeout;" : "";
    why += (st & kKvStalePlan) ? " the plan on the device has another shape than the call;" : "";
    return kv_fail(h, TTL_ERR_DEVICE, why);
}

// No exception (an allocation of a message) leaves a C entry.
template <class F> int guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return TTL_ERR_STATE;
    } catch (...) {
        return TTL_ERR_STATE;
    }
}

}  // namespace

extern "C" {

int ttl_kv_create(const ttl_kv_config *config, ttl_kv **handle_out) {
    return guarded([&] { return kv_create(config, handle_out); });
}

void ttl_kv_destroy(ttl_kv *h) {
    if (!h) {
        return;
    }
    DeviceGuard guard(h->device);
    if (h->stream || !h->own_stream) {
        cudaStreamSynchronize(h->stream);
    }
    for (void *p : h->allocations) {
        cudaFree(p);
    }
    if (h->own_stream && h->stream) {
        cudaStreamDestroy(h->stream);
    }
    delete h;
}

const char *ttl_kv_last_error(const ttl_kv *h) {
    return h ? h->error.c_str() : ttl::thread_error().c_str();
}

size_t ttl_kv_page_bytes(const ttl_kv *h) {
    return h ? size_t(h->kv_heads) * h->block_bytes : 0;
}

int ttl_kv_batch_async(ttl_kv *h, uint32_t seqs, uint32_t rows, uint32_t max_new, const int32_t *row_start,
                       const int32_t *length, const int32_t *pages, uint32_t page_stride, const int32_t *first,
                       const int32_t *prefix) {
    return guarded([&] { return kv_batch(h, seqs, rows, max_new, row_start, length, pages, page_stride, first, prefix); });
}

int ttl_kv_append_async(ttl_kv *h, int layer, int rotate, const void *k, size_t k_stride, const void *v, size_t v_stride,
                        const void *q, size_t q_stride, void *q_out, size_t q_out_stride) {
    return guarded([&] { return kv_append(h, layer, rotate, k, k_stride, v, v_stride, q, q_stride, q_out, q_out_stride); });
}

int ttl_kv_read_async(ttl_kv *h, int layer, void *k, size_t k_stride, void *v, size_t v_stride) {
    return guarded([&] { return kv_read(h, layer, k, k_stride, v, v_stride); });
}

int ttl_kv_attend_async(ttl_kv *h, int layer, uint32_t flags, const void *q, size_t q_stride, void *out, size_t out_stride,
                        float scale, float cap, const float *sinks, const float *slopes) {
    return guarded([&] { return kv_attend(h, layer, flags, q, q_stride, out, out_stride, scale, cap, sinks, slopes); });
}

int ttl_kv_sync(ttl_kv *h) {
    return guarded([&] { return kv_sync(h); });
}

void *ttl_kv_stream(ttl_kv *h) {
    return h ? static_cast<void *>(h->stream) : nullptr;
}

}  // extern "C"

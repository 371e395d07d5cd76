// kv.cuh -- what the kernels of the paged cache share: the plan that a batch
// call leaves on the device, the walk over it, the pool's layout, and the end
// of a tile (merge of partial results, sink, rounding, rows with infinities).
//
// Columns.  The query rows of one sequence and one KV head are n x group
// vectors over the same keys; they are numbered c = i * group + g (row i,
// query head kv * group + g).  A tile is up to `width` columns of a sequence.
//
// Plan.  A tile's visible key range is counted in granules (of 64 or 128
// keys); tiles are laid end to end, once per KV head, each as long as its
// granules and the few that its start and end cost, and the line is cut into
// one piece of equal length per CTA.  So every CTA gets the same work
// whatever the batch's shape, in one wave; a tile cut by a CTA border leaves
// partial sums in the workspace, and the CTA that arrives last merges them, in
// the order of the keys, so results do not depend on timing.  (A second kernel
// for the merges, in place of the last CTA, cost 7 to 10 us more per call.)  The
// plan takes 6 us on the device, once for all layers of a batch; times in these
// files that say so hold it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "tc.cuh"

namespace ttl {
namespace kv {

enum : int { kF32 = 0, kF16 = 1, kBf16 = 2, kMxfp4 = 3 };

// Status bits (device word of a ttl_kv handle).
enum : uint32_t {
    kKvBadBatch = 1u << 0,   // row_start / length out of order or range
    kKvBadPage = 1u << 1,    // a page id outside the pool
    kKvWait = 1u << 2,       // a bounded wait gave up
    kKvStalePlan = 1u << 3,  // the plan on the device is not of this launch's shape
};

constexpr int kKinds = 2;          // tiles of few columns, tiles of a prompt
constexpr int kMaxCtas = 1024;     // CTAs of a list (cuts)
constexpr int kNoPosition = 1 << 30;  // above all
constexpr int kNoSplit = 4;        // a tile of at most this many granules is not cut

struct __align__(32) Tile {
    int32_t seq, col0, gran0;
    uint32_t size;                 // columns (9 bits), granules
    int32_t row0, rem, len, low;   // row and head (in its group) of the first column; the sequence's length; the
                                   // lowest position a column sees (kNoPosition: none)
};
struct __align__(16) Cut {
    int32_t head, tile, gran;      // gran: granules into the tile
    uint32_t span;                 // gran > 0: first and last CTA (<< 16) that hold a part of the tile
};
struct __align__(16) List {
    int32_t tiles, ctas, width, gran;
    int32_t pad[4];
};
struct Plan {
    const int32_t *pages;
    uint32_t page_stride;
    int32_t seqs, rows;            // rows: entries of Walk::row that are this batch's
    List list[kKinds][2];          // [kind][0 full, 1 sliding]
};

// What one list's walk reads.
struct Walk {
    const Plan *plan;
    const List *list;
    const Tile *tiles;
    const Cut *cuts;               // [ctas + 1]
    const int4 *row;               // [rows] {position, lo, hi, seq} of this window; seq -1: padding
};

struct Piece {
    int head, tile, seq, ncols, row0, rem, len, low;
    int k0, k1;        // keys of the piece (k1 <= the tile's last granule; clip to the sequence's length)
    int first, last;   // first and last CTA that hold a part of the tile (equal: the whole tile is here)
};

struct AttendArgs {
    Walk walk;
    const uint8_t *pool;           // this layer
    const void *q;
    void *out;
    size_t q_stride, out_stride;   // elements
    const float *sinks, *slopes;
    float *part;                   // [2 * ctas][width][part_pitch(D)]
    uint32_t *counters;            // [ctas]
    uint32_t *status;
    float scale, cap;              // natural units; cap 0: none
    int rows, group, page_shift, pages, kv_heads;
    int other_ctas;                // of the call's launch of the other kind (0: none)
    uint32_t block_bytes;          // one KV head of a page
    uint32_t group_div;            // ceil(2^20 / group)

    // Row and query head of column c of a tile.  (rem + c < 512, so the product
    // is below 2^29 and the quotient exact for any group up to 256.)
    __device__ __forceinline__ void column(const Piece &p, int c, int &row, int &qhead) const {
        const int t = p.rem + c, r = int(uint32_t(t) * group_div >> 20);
        row = p.row0 + r;
        qhead = p.head * group + t - r * group;
    }
};

__host__ __device__ constexpr uint32_t row_bytes(int cache, int d) {
    return cache == kMxfp4 ? uint32_t(d / 2 + d / 32) : uint32_t(cache == kF32 ? 4 * d : 2 * d);
}

// 2^(e - 127) of an E8M0 byte: 0 is the smallest (a subnormal float), 255 NaN.
__device__ __forceinline__ float scale_of(uint32_t e) {
    return e == 255u ? __uint_as_float(0x7fffffffu) : (e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23));
}

// ---- the pool: [page][KV head][K rows, V rows] ----
// f32, f16, bf16: [page_tokens][D].  MXFP4: codes [page_tokens][D / 2] (value k
// in byte k / 2, low nibble for even k), then scales [page_tokens][D / 32].

template <int kCache, int D> __device__ __forceinline__ float pool_value(const uint8_t *rows, int tokens, int t, int d) {
    if constexpr (kCache == kF32) {
        return reinterpret_cast<const float *>(rows)[size_t(t) * D + d];
    } else if constexpr (kCache == kF16) {
        return __half2float(reinterpret_cast<const __half *>(rows)[size_t(t) * D + d]);
    } else if constexpr (kCache == kBf16) {
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(rows)[size_t(t) * D + d]);
    } else {
        const uint32_t byte = rows[t * (D / 2) + d / 2];
        const uint32_t code = (d & 1) ? byte >> 4 : byte & 15u;
        const uint32_t e = rows[tokens * (D / 2) + t * (D / 32) + d / 32];
        const float2 v = __half22float2(e2m1x2_to_half2(code));
        return v.x * scale_of(e);
    }
}

template <int kRows> __device__ __forceinline__ float row_value(const void *base, size_t i) {
    if constexpr (kRows == kF32) {
        return static_cast<const float *>(base)[i];
    } else if constexpr (kRows == kF16) {
        return __half2float(static_cast<const __half *>(base)[i]);
    } else {
        return __bfloat162float(static_cast<const __nv_bfloat16 *>(base)[i]);
    }
}
template <int kRows> __device__ __forceinline__ void store_value(void *base, size_t i, float v) {
    if constexpr (kRows == kF32) {
        static_cast<float *>(base)[i] = v;
    } else if constexpr (kRows == kF16) {
        static_cast<__half *>(base)[i] = __float2half_rn(v);
    } else {
        static_cast<__nv_bfloat16 *>(base)[i] = __float2bfloat16_rn(v);
    }
}
// Eight values as 16-bit or 32-bit rows (16-byte aligned).
template <int kRows> __device__ __forceinline__ void store8(void *base, size_t i, const float (&v)[8]) {
    if constexpr (kRows == kF32) {
        float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(base) + i);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kRows == kF16) {
                const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// Four values (on their size).
template <int kRows> __device__ __forceinline__ void store4(void *base, size_t i, const float (&v)[4]) {
    if constexpr (kRows == kF32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(base) + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if constexpr (kRows == kF16) {
                const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + i) = make_uint2(w[0], w[1]);
    }
}
template <int kRows> __device__ __forceinline__ void load8(const void *base, size_t i, float (&v)[8]) {
    if constexpr (kRows == kF32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + i);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 f;
            if constexpr (kRows == kF16) {
                f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
            } else {
                f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u[j]));
            }
            v[2 * j] = f.x, v[2 * j + 1] = f.y;
        }
    }
}

// Eight values of a pool row, from a multiple of 8 on.
template <int kCache, int D> __device__ __forceinline__ void pool8(const uint8_t *rows, int tokens, int t, int d, float (&x)[8]) {
    if constexpr (kCache != kMxfp4) {
        load8<kCache>(rows, size_t(t) * D + d, x);
    } else {
        const uint32_t codes = *reinterpret_cast<const uint32_t *>(rows + t * (D / 2) + d / 2);
        const float f = scale_of(rows[tokens * (D / 2) + t * (D / 32) + d / 32]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = __half22float2(e2m1x2_to_half2((codes >> (8 * j)) & 255u));
            x[2 * j] = v.x * f, x[2 * j + 1] = v.y * f;
        }
    }
}

// Page id of position `pos` of a sequence; an id outside the pool is read as page 0,
// and reported unless the whole page lies below position `low`.  The caller keeps
// pos below the sequence's length.
__device__ __forceinline__ int page_of(const Plan &plan, int seq, int pos, int low, int page_shift, int pages, uint32_t *status) {
    const int id = plan.pages[size_t(seq) * plan.page_stride + size_t(pos >> page_shift)];
    if (uint32_t(id) >= uint32_t(pages)) {
        if (pos >> page_shift >= low >> page_shift) {
            set_status(status, kKvBadPage);
        }
        return 0;
    }
    return id;
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// cap * tanh(x / cap) in log2 units, from the raw product: `in` is the scale
// times 2 log2(e) / cap, `out` cap * log2(e).  tanh y = 1 - 2 / (e^2y + 1), whose
// absolute error is about 2^-22 (the hardware's tanh.approx has 2^-11; e^2y =
// infinity gives 1); up to y = 1/4, where that would be much of a small score
// under a large cap, y P(y^2), P fitted to tanh(y) / y for the least relative
// error (4e-7).
__device__ __forceinline__ float capped(float dot, float in, float out) {
    const float e = dot * in, y = e * 0.34657359f, t = y * y;  // ln 2 / 2
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ex2(e) + 1.0f));
    const float small = out * y * fmaf(t, fmaf(t, 0.12841587f, -0.33321908f), 0.99999958f);
    return t <= 0.0625f ? small : fmaf(-2.0f * out, r, out);
}

// The same for |x / cap| up to kSmallScore: tanh y = y P(y^2) without the
// special-function unit, P fitted to tanh(y) / y over y <= 0.5 for the least
// relative error (1.4e-8).  Two at a time (one instruction works on a pair of f32):
// x, y raw products, to log2 units; scale and ratio bring them there and to x / cap.
constexpr float kSmallScore = 0.5f;
__device__ __forceinline__ void capped_small(float &x, float &y, float scale, float ratio) {
    asm("{\n\t.reg .b64 x, r, t, p, c;\n\t"
        "mov.b64 x, {%0, %1};\n\t"
        "mov.b64 c, {%3, %3};\n\tmul.rn.f32x2 r, x, c;\n\tmul.rn.f32x2 t, r, r;\n\t"
        "mov.b64 c, {%2, %2};\n\tmul.rn.f32x2 x, x, c;\n\t"
        "mov.b64 p, {%4, %4};\n\t"
        "mov.b64 c, {%5, %5};\n\tfma.rn.f32x2 p, p, t, c;\n\t"
        "mov.b64 c, {%6, %6};\n\tfma.rn.f32x2 p, p, t, c;\n\t"
        "mov.b64 c, {%7, %7};\n\tfma.rn.f32x2 p, p, t, c;\n\t"
        "mov.b64 c, 0x3f8000003f800000;\n\tfma.rn.f32x2 p, p, t, c;\n\t"
        "mul.rn.f32x2 x, x, p;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(scale), "f"(ratio), "f"(0.017134985f), "f"(-0.052986064f), "f"(0.13324779f), "f"(-0.33333069f));
}
// x = x * f + (b + c), with b a pair.
__device__ __forceinline__ void bias_pair(float &x, float &y, float f, float b0, float b1, float c) {
    asm("{\n\t.reg .b64 x, b, c;\n\t"
        "mov.b64 x, {%0, %1};\n\tmov.b64 b, {%3, %4};\n\tmov.b64 c, {%5, %5};\n\tadd.rn.f32x2 b, b, c;\n\t"
        "mov.b64 c, {%2, %2};\n\tfma.rn.f32x2 x, x, c, b;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(f), "f"(b0), "f"(b1), "f"(c));
}

// Pairs of f32 in one instruction: x * f + c, and a + b.
__device__ __forceinline__ void fma_pair(float &x0, float &x1, float f, float c) {
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 d, {%3, %3};\n\t"
        "fma.rn.f32x2 a, a, b, d;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(x0), "+f"(x1)
        : "f"(f), "f"(c));
}
__device__ __forceinline__ void add_pair(float &a0, float &a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1));
}
// 2^x and 2^y on the multiply-add units, for x, y <= 127; 0 from -127 on.  x = n +
// f with n the nearest integer (it comes out of the sum with 1.5 * 2^23), 2^f by a
// polynomial fitted over [-1/2, 1/2] with P(0) = 1 for the least relative error
// (9e-8), n added to its exponent: at -127 that leaves the zero word.  NaN gives 0:
// the caller looks for it in the maximum.
__device__ __forceinline__ void pow2_pair(float x, float y, float &px, float &py) {
    uint32_t bx, by;
    asm("{\n\t.reg .b64 x, t, r, p, c;\n\t.reg .b32 tx, ty, qx, qy;\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mov.b64 c, 0x4b4000004b400000;\n\tadd.rn.f32x2 t, x, c;\n\t"
        "mov.b64 c, 0xcb400000cb400000;\n\tadd.rn.f32x2 r, t, c;\n\t"
        "mov.b64 c, 0xbf800000bf800000;\n\tfma.rn.f32x2 x, r, c, x;\n\t"
        "mov.b64 p, {%4, %4};\n\t"
        "mov.b64 c, {%5, %5};\n\tfma.rn.f32x2 p, p, x, c;\n\t"
        "mov.b64 c, {%6, %6};\n\tfma.rn.f32x2 p, p, x, c;\n\t"
        "mov.b64 c, {%7, %7};\n\tfma.rn.f32x2 p, p, x, c;\n\t"
        "mov.b64 c, {%8, %8};\n\tfma.rn.f32x2 p, p, x, c;\n\t"
        "mov.b64 c, 0x3f8000003f800000;\n\tfma.rn.f32x2 p, p, x, c;\n\t"
        "mov.b64 {tx, ty}, t;\n\tmov.b64 {qx, qy}, p;\n\t"
        "mad.lo.u32 %0, tx, 8388608, qx;\n\tmad.lo.u32 %1, ty, 8388608, qy;\n\t}"
        : "=r"(bx), "=r"(by)
        : "f"(fmaxf(x, -127.0f)), "f"(fmaxf(y, -127.0f)), "f"(0.001326472731307149f), "f"(0.009671512991189957f),
          "f"(0.05550733581185341f), "f"(0.24022242426872253f), "f"(0.6931470036506653f));
    px = __uint_as_float(bx), py = __uint_as_float(by);
}
// Largest and smallest of three; NaN if any is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Whether the plan on the device is of this call's shape; where it is not, says so.
// A captured call may meet the plan of another batch.  That plan's work may lie
// with the other kind as well, which the call did not launch, so both kinds are
// compared; rows that the call's arrays lack are left out and reported.
__device__ __forceinline__ bool plan_fits(const AttendArgs &a, int width, int gran) {
    const List *lists = &a.walk.plan->list[0][0];  // [kind][window]
    const int4 mine = *reinterpret_cast<const int4 *>(a.walk.list);
    const int other = lists[(a.walk.list - lists) ^ 2].ctas, rows = a.walk.plan->rows;  // three loads at once
    const bool fits = (mine.y == int(gridDim.x)) & (mine.z == width) & (mine.w == gran) & (other == a.other_ctas);
    if (threadIdx.x == 0 && (!fits || (blockIdx.x == 0 && rows != a.rows))) {
        set_status(a.status, kKvStalePlan);
    }
    return fits;
}

// ---- the walk ----

// The descriptor of the tile after the one handed out is loaded ahead.
struct Walker {
    const Tile *list;
    int head, tile, gran;  // next piece
    Cut end;
    uint32_t start_span;   // of the tile that the CTA's range begins in, where it begins inside
    int cta, count, gsize;
    int4 t4;               // tile `tile`
    int4 t2;

    __device__ __forceinline__ Walker(const Walk &w, int cta_, int gsize_) : list(w.tiles), cta(cta_), gsize(gsize_) {
        const Cut a = w.cuts[cta];
        end = w.cuts[cta + 1];
        count = w.list->tiles;
        head = a.head, tile = a.tile, gran = a.gran;
        start_span = a.span;
        load();
    }
    __device__ __forceinline__ void load() {
        if (before(head, tile, gran, end)) {
            t4 = *reinterpret_cast<const int4 *>(list + tile);
            t2 = *reinterpret_cast<const int4 *>(&list[tile].row0);
        }
    }
    __device__ __forceinline__ static bool before(int h, int t, int g, const Cut &c) {
        return h != c.head ? h < c.head : (t != c.tile ? t < c.tile : g < c.gran);
    }
    __device__ __forceinline__ bool next(Piece &p) {
        if (!before(head, tile, gran, end)) {
            return false;
        }
        const int n = int(uint32_t(t4.w) >> 9);
        int stop = n;
        if (end.head == head && end.tile == tile) {
            stop = end.gran;  // > gran
        }
        p.head = head, p.tile = tile, p.seq = t4.x, p.row0 = t2.x, p.rem = t2.y, p.len = t2.z, p.low = t2.w;
        p.ncols = int(uint32_t(t4.w) & 511u);
        p.k0 = (t4.z + gran) * gsize;
        p.k1 = (t4.z + stop) * gsize;
        p.first = p.last = cta;
        const uint32_t span = gran > 0 ? start_span : end.span;
        if (gran > 0 || stop < n) {
            p.first = int(span & 0xffffu);
            p.last = int(span >> 16);
        }
        if (stop == n) {
            gran = 0;
            if (++tile == count) {
                tile = 0;
                ++head;
            }
        } else {
            gran = stop;
        }
        load();
        return true;
    }
};

// Slots behind a sequence's end hold what was left there, and 0 * NaN is NaN in every
// column, so V's values there become 0 before the product: by a warp, `rows` rows of
// 64 values (128 bytes each) from `addr` on in shared memory that copies fill.
__device__ __forceinline__ void clear_rows(uint32_t addr, int rows) {
#pragma unroll 1
    for (int i = (threadIdx.x & 31) * 16; i < rows * 128; i += 512) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr + i), "r"(0) : "memory");
    }
}

// Whether a phase of a barrier is complete, without waiting for it.
__device__ __forceinline__ bool phase_done(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(tc::smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// Waits for a phase of a barrier unless the CTA has given up; a wait of about two
// seconds gives the CTA up (every later wait returns at once, so that all warps
// still meet at their barriers and leave).  kSleep lets the hardware put the
// warp to sleep for up to a millisecond a try.  It pays where other warps of the
// scheduler compute meanwhile.
//
// Two things take as long as their keys are many, and their time does not count.
// While warps compute columns again (`Halt::busy`) nobody gives up.  And the prompt
// kernel's next tile waits for the last scores of the one in hand, over all the keys
// of its piece: such a wait (kLong) begins again where the beat that goes with the
// keys has changed.  The keys are finite, and so are these waits.
constexpr long long kWaitClocks = 4000000000ll;

struct Halt {
    int state;  // bit 0: the CTA has given up; above: warps that compute columns again
    int beat;   // changes while the CTA gets on
    __device__ __forceinline__ bool aborted() const {
        return *const_cast<const volatile int *>(&state) & 1;
    }
    __device__ __forceinline__ void busy(bool on) {
        atomicAdd(&state, on ? 2 : -2);
    }
    __device__ __forceinline__ void alive() {
        *const_cast<volatile int *>(&beat) = int(clock());
    }
};

template <bool kSleep, bool kLong = false> __device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, Halt *halt, uint32_t *status) {
    const uint32_t addr = tc::smem_u32(bar);
    long long start = 0;
    int beat = 0;
    while (true) {
        uint32_t ok;
        if constexpr (kSleep) {
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(addr), "r"(parity), "r"(1000000u)
                : "memory");
        } else {
            ok = tc::mbar_try_wait(bar, parity);
        }
        if (ok) {
            return true;
        }
        const int state = *const_cast<volatile int *>(&halt->state);
        if (state & 1) {
            return false;
        }
        const long long now = clock64();
        if (start == 0 || state) {
            start = now;
        } else if (now - start > kWaitClocks) {
            const int last = kLong ? *const_cast<volatile int *>(&halt->beat) : 0;
            if (last == beat) {
                set_status(status, kKvWait);
                atomicOr(&halt->state, 1);
                return false;
            }
            start = now;
            beat = last;
        }
    }
}

// Programmatic dependent launch: lets the next kernel on the stream start, and
// waits for what ran before this one.  Every kernel of the cache waits before it
// touches global memory, so whatever follows a kernel also follows its
// predecessors.
__device__ __forceinline__ void wait_previous() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Slot of the partial result that CTA c keeps for a tile whose parts begin in
// CTA `first`: its own first tile (slot 2c) or the one it begins (2c + 1).
__device__ __forceinline__ int part_slot(int c, int first) {
    return 2 * c + (c == first ? 1 : 0);
}

// ---- the end of a tile ----

// The sink's part of a column: adds it to the sum l of weights relative to m, and
// returns the factor that brings the column's sums to the same measure.  An
// infinite sink takes everything.
__device__ __forceinline__ float add_sink(float m, float &l, float sink) {
    sink *= kLog2e;
    const float mn = fmaxf(m, sink), safe = mn == -INFINITY ? 0.0f : mn;
    const float f = exp2f(m - safe);
    l = l * f + (sink == INFINITY ? 1.0f : exp2f(sink - safe));
    return f;
}

// Partial results: [slot][width][part_pitch(D)] floats, a column's D sums, then
// its maximum and sum; rows of a multiple of 16 bytes.  (Prompts lay the same
// space out by columns.)
__host__ __device__ constexpr int part_pitch(int d) {
    return d + 4;
}
constexpr int kPromptColumns = 256;  // of a prompt tile

// ---- columns with infinities or NaN ----
// The matrix products multiply every value of a tile, so an infinity or NaN in a
// place that a column does not see reaches its sums as 0 * x.  A column whose sums
// over a piece of a tile are not finite is computed again over that piece, by a
// warp, and unseen keys are not touched.  Being cut as the tiles are, this takes the
// whole GPU for a long sequence too.  Lanes are keys for the scores (each reads its
// own K row, Q comes by shuffles) and values of the head for the sums, eight V rows
// in flight; a hundred clocks a key, most of them waiting.
//
// The column's sums go over those in the partial result `part` of the piece, laid out
// as in the kernel for few columns or (kPrompt) in that for prompts; without `part` the
// piece is a whole tile, and the column is finished and stored.
template <int kRows, int kCache, int D, bool kPrompt>
__device__ __forceinline__ void redo_column(const AttendArgs &a, const Piece &p, int c, float *part) {
    constexpr int kPer = D / 32, kDeep = 8;
    const int lane = threadIdx.x & 31;
    const Plan &plan = *a.walk.plan;
    int row, qhead;
    a.column(p, c, row, qhead);
    const int4 ri = a.walk.row[row];
    const int lo = max(max(ri.y, 0), p.k0), hi = min(min(ri.z, p.len), p.k1);
    const float scale_log2 = a.scale * kLog2e;
    const float slope = a.slopes ? a.slopes[qhead] * kLog2e : 0.0f;
    const int tokens = 1 << a.page_shift;
    auto block = [&](int page) { return a.pool + (size_t(page) * a.kv_heads + p.head) * a.block_bytes; };
    float q[kPer], o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        q[i] = row_value<kRows>(a.q, size_t(row) * a.q_stride + size_t(qhead) * D + lane * kPer + i);
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int base = lo; base < hi; base += 32) {
        const int j = base + lane, n = min(32, hi - base);
        const bool seen = lane < n;
        const int page = seen ? page_of(plan, p.seq, j, 0, a.page_shift, a.pages, a.status) : 0;
        const uint8_t *kb = block(page);
        float s = 0.0f;
#pragma unroll
        for (int d = 0; d < D; d += 8) {
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (seen) {
                pool8<kCache, D>(kb, tokens, j & (tokens - 1), d, x);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s = fmaf(__shfl_sync(0xffffffffu, q[i % kPer], (d + i) / kPer), x[i], s);
            }
        }
        const float x = a.cap != 0.0f ? a.cap * tanhf(s * a.scale / a.cap) * kLog2e : s * scale_log2;
        const float z = seen ? x - slope * float(abs(ri.x - j)) : -INFINITY;
        float top = z;  // NaN drops out here and is met in the weight
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        }
        const float mn = fmaxf(m, top), safe = mn == -INFINITY ? 0.0f : mn;
        const float up = exp2f(m - safe), w = seen ? exp2f(z - safe) : 0.0f;
        m = mn;
        l = l * up + warp_sum(w);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            o[i] *= up;
        }
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += kDeep) {
            float v[kDeep][kPer];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const uint8_t *vb = block(__shfl_sync(0xffffffffu, page, k0 + k)) + (a.block_bytes >> 1);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    v[k][i] = k0 + k < n ? pool_value<kCache, D>(vb, tokens, (base + k0 + k) & (tokens - 1), lane * kPer + i) : 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const float wk = __shfl_sync(0xffffffffu, w, k0 + k);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    o[i] = fmaf(wk, v[k][i], o[i]);
                }
            }
        }
    }
    if (part) {
        float *dst = kPrompt ? part + 4 * c : part + size_t(c) * part_pitch(D);
        constexpr int kQuad = kPrompt ? 4 * kPromptColumns : 4;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane * kPer + i;
            dst[(d >> 2) * kQuad + (d & 3)] = o[i];
        }
        if (lane == 0) {
            *reinterpret_cast<float2 *>(kPrompt ? part + kPromptColumns * D + 2 * c : dst + D) = make_float2(m, l);
        }
        return;
    }
    const float f = a.sinks ? add_sink(m, l, a.sinks[qhead]) : 1.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        store_value<kRows>(a.out, size_t(row) * a.out_stride + size_t(qhead) * D + lane * kPer + i, lo < hi ? o[i] * f / l : 0.0f);
    }
}

// Adds the sink, divides, rounds and stores columns [c0, ncols) step `step` of
// a tile, by warps: D / 8 lanes per column, eight values a lane.  value(c, d,
// v) gives the eight unnormalised sums, stats(c) {max, sum} in log2 units,
// info(c, row, head) what the column may see.  Returns whether the thread stored
// something that is not finite.
struct ColumnInfo {
    int lo, hi, seq;
    float sink;
};
// From the plan's rows, for kernels that do not keep them.
__device__ __forceinline__ ColumnInfo column_info(const AttendArgs &a, int row, int qhead) {
    const int4 ri = a.walk.row[row];
    return ColumnInfo{ri.y, ri.z, ri.w, a.sinks ? a.sinks[qhead] : 0.0f};
}

template <int kRows, int D, class Value, class Stats, class Info>
__device__ __forceinline__ bool store_columns(const AttendArgs &a, const Piece &p, int warp, int warps, Value value, Stats stats,
                                              Info info) {
    constexpr int kLanes = D / 8, kCols = 32 / kLanes;
    const int lane = threadIdx.x & 31;
    bool bad = false;
    for (int base = warp * kCols; base < p.ncols; base += warps * kCols) {
        const int c = base + lane / kLanes;
        if (c < p.ncols) {
            int row, qhead;
            a.column(p, c, row, qhead);
            const ColumnInfo ci = info(c, row, qhead);
            const bool sees = max(ci.lo, 0) < min(ci.hi, p.len);
            const float2 ml = stats(c);
            float l = ml.y;
            const float f = (a.sinks ? add_sink(ml.x, l, ci.sink) : 1.0f) / l;
            float v[8];
            value(c, (lane % kLanes) * 8, v);
            const bool write = row < a.rows && ci.seq == p.seq;  // a row that two sequences claim belongs to the first
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = sees ? v[j] * f : 0.0f;
                bad = bad || (write && !(fabsf(v[j]) < INFINITY));
            }
            if (write) {
                store8<kRows>(a.out, size_t(row) * a.out_stride + size_t(qhead) * D + (lane % kLanes) * 8, v);
            }
        }
    }
    return bad;
}

// Merges the partial results of a tile over the CTAs [first, last] that hold
// them, in that order, and stores its columns: D / 4 lanes per column.  The
// parts come from other SMs through L2, about a microsecond each way, so what
// counts is how many are asked for at once: kBatch parts' sums and statistics
// per lane.
template <int kRows, int D, int kBatch>
__device__ __forceinline__ void merge_tile(const AttendArgs &a, const Piece &p, int warp, int warps, int width) {
    constexpr int kLanes = D / 4, kCols = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane / kLanes, d = 4 * (lane % kLanes);
    const int parts = p.last - p.first + 1;
    for (int base = warp * kCols; base < p.ncols; base += warps * kCols) {
        const int c = min(base + sub, p.ncols - 1);
        const bool have = base + sub < p.ncols;
        int row, qhead;
        a.column(p, c, row, qhead);
        const ColumnInfo ci = column_info(a, row, qhead);
        const float *col = a.part + size_t(c) * part_pitch(D);
        auto slot = [&](int k) { return col + size_t(part_slot(p.first + k, p.first)) * width * part_pitch(D); };
        float m = -INFINITY;
        if (parts > kBatch) {
            for (int k = lane % kLanes; k < parts; k += kLanes) {
                m = fmaxf(m, __ldcg(slot(k) + D));
            }
#pragma unroll
            for (int off = kLanes / 2; off; off >>= 1) {
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            }
        }
        float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < parts; k0 += kBatch) {
            float2 ml[kBatch];
            float4 x[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (k0 + k < parts) {
                    ml[k] = __ldcg(reinterpret_cast<const float2 *>(slot(k0 + k) + D));
                    x[k] = __ldcg(reinterpret_cast<const float4 *>(slot(k0 + k) + d));
                }
            }
            if (parts <= kBatch) {
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    m = k < parts ? fmaxf(m, ml[k].x) : m;
                }
            }
            const float safe = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (k0 + k < parts) {
                    const float w = exp2f(ml[k].x - safe);
                    l = fmaf(ml[k].y, w, l);
                    o[0] = fmaf(x[k].x, w, o[0]), o[1] = fmaf(x[k].y, w, o[1]);
                    o[2] = fmaf(x[k].z, w, o[2]), o[3] = fmaf(x[k].w, w, o[3]);
                }
            }
        }
        const float f = (a.sinks ? add_sink(m, l, ci.sink) : 1.0f) / l;
        const bool sees = max(ci.lo, 0) < min(ci.hi, p.len);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = sees ? o[j] * f : 0.0f;
        }
        if (have && row < a.rows && ci.seq == p.seq) {
            store4<kRows>(a.out, size_t(row) * a.out_stride + size_t(qhead) * D + d, o);
        }
    }
}

// After a CTA wrote its partial result of a tile: counts it, and returns true
// in the CTA that arrived last (all threads that `sync` joins, thread 0 among
// them), with the others' results visible.  A part that is held back is not counted;
// it arrives later.  That CTA leaves the tile's counter at zero for the next launch.
struct NeverHeld {
    __device__ __forceinline__ bool operator()() const {
        return false;
    }
};
template <class Sync, class Held = NeverHeld>
__device__ __forceinline__ bool arrive_last(const AttendArgs &a, const Piece &p, int *flag, Sync sync, Held held = Held()) {
    __threadfence();
    sync();
    if (threadIdx.x == 0) {
        const uint32_t parts = uint32_t(p.last - p.first + 1);
        const bool is_last = !held() && atomicAdd(&a.counters[p.first], 1u) + 1u == parts;
        if (is_last) {
            a.counters[p.first] = 0;
        }
        *flag = is_last;
        __threadfence();
    }
    sync();
    return *flag != 0;
}

}  // namespace kv
}  // namespace ttl

// kv_prompt.cu -- attention of many columns per KV head (prompts and chunks of
// prompts) over the paged cache on tcgen05, for f16 and bf16 rows.
//
//   S [128 cols x 128 keys] = Q K^T      A = Q, B = K from shared memory (K-major)
//   O [128 cols x D]       += P V        A = P from tensor memory, B = V (D-major)
//
// What bounds it is neither of these: per score the tensor pipe does 4 D
// operations (at D = 64, 256 of its 8192 a clock) and the special-function unit
// one exponential (16 a clock), so 128 x 128 scores take 512 clocks of the one
// and 1024 of the other.  So the exponentials must never wait:
//   - a tile is 2 x 128 columns, each with a warpgroup of its own: while one
//     turns its scores into weights, the tensor pipe works for the other;
//   - a thread owns a column: its 128 scores of a granule come from tensor
//     memory into registers once, the maximum and the sum need no shuffles, and
//     the weights go back over the scores as P;
//   - the maximum moves only when a weight would pass 2^8 (f16: 2^4), and only
//     then are the sums in tensor memory read, rescaled and written.
// One warp loads K and V (TMA, 128-byte swizzle, a ring of granules), one thread
// issues the matrix instructions.  The scores of granule j + 1 are issued right
// behind the product of granule j, over the weights it has just read.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv.cuh"
#include "kv_internal.h"
#include "tc.cuh"

namespace ttl {
namespace kv {

namespace {

constexpr int kGran = 128;
constexpr int kHalf = 128;                 // columns of a warpgroup
constexpr int kLoader = 8, kIssuer = 9;    // warps
constexpr int kExpander = 12;              // first of the four warps that expand a 4-bit cache
constexpr uint32_t kTmemCols = 512;

// Threads, and registers of the softmax warpgroups, of the loader's and of the
// expanders': a warpgroup may only take what the launch holds (168 or 128 a
// thread), 256 * 208 + 128 * 80 <= 384 * 168 and 256 * 168 + 128 * 64 + 128 * 104
// <= 512 * 128.
template <int kCache> struct PromptShape {
    static constexpr bool kFour = kCache == kMxfp4;
    static constexpr int kThreads = kFour ? 512 : 384;
    static constexpr int kSoftmaxRegs = kFour ? 168 : 208, kOtherRegs = kFour ? 64 : 80, kExpandRegs = 104;
    static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs + (kFour ? 128 * kExpandRegs : 0) <= kThreads * (kFour ? 128 : 168), "registers");
};

template <int kCache, int D> struct PromptSmem {
    static constexpr int kStages = D == 64 ? 3 : 2;
    static constexpr uint32_t kRawBytes = kCache == kMxfp4 ? 2 * kGran * row_bytes(kMxfp4, D) : 16;  // a granule as the cache holds it
    alignas(1024) uint8_t q[2][kHalf * D * 2];
    alignas(1024) uint8_t k[kStages][kGran * D * 2];
    alignas(1024) uint8_t v[kStages][kGran * D * 2];
    alignas(16) uint8_t raw[2][kRawBytes];
    uint64_t raw_full[2], raw_empty[2];
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int last, abort;
};

__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort, uint32_t *status) {
    if (tc::mbar_try_wait(bar, parity)) {
        return true;
    }
    if (*abort) {
        return false;
    }
    if (!tc::mbar_wait(bar, parity)) {
        set_status(status, kKvWait);
        *abort = 1;
        return false;
    }
    return true;
}

__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void softmax_sync() {
    asm volatile("bar.sync 1, 256;" ::: "memory");
}

// kind::f16: D f32, A and B f16 or bf16, M = 128; b_mn: B is N-major.
template <int kType> __device__ __forceinline__ constexpr uint32_t f16_desc(uint32_t n, bool b_mn) {
    const uint32_t t = kType == kBf16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// N-major, 128-byte swizzle: rows of 64 N-values (128 bytes), 8-row groups 1024
// bytes apart along K (SBO), 64-value blocks `lbo` bytes apart along N.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t lbo) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | uint64_t((lbo >> 4) & 0x3FFFu) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 |
           uint64_t(2) << 61;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

#define KV_R8(a, i) "=f"(a[i]), "=f"(a[i + 1]), "=f"(a[i + 2]), "=f"(a[i + 3]), "=f"(a[i + 4]), "=f"(a[i + 5]), "=f"(a[i + 6]), "=f"(a[i + 7])
// This warp's 32 lanes, 32 consecutive f32 columns into v[0 .. 31].
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : KV_R8(v, 0), KV_R8(v, 8), KV_R8(v, 16), KV_R8(v, 24)
        : "r"(taddr)
        : "memory");
}
#undef KV_R8
#define KV_F8(a, i) "f"(a[i]), "f"(a[i + 1]), "f"(a[i + 2]), "f"(a[i + 3]), "f"(a[i + 4]), "f"(a[i + 5]), "f"(a[i + 6]), "f"(a[i + 7])
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        KV_F8(v, 0), KV_F8(v, 8), KV_F8(v, 16), KV_F8(v, 24)
        : "memory");
}
#undef KV_F8

template <int kType> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kType == kF16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

template <int kCache, int D>
__device__ __forceinline__ void load_granules(const AttendArgs &a, const Plan &plan, const CUtensorMap *map, PromptSmem<kCache, D> &sm) {
    const int lane = threadIdx.x & 31;
    // 16 bits: boxes of 64 values x up to 64 keys; 4 bits: a head's whole part of a page
    constexpr int kParts = kCache == kMxfp4 ? 1 : D / 64;
    const int seg = min(1 << a.page_shift, kCache == kMxfp4 ? kGran : 64), segs = kGran / seg, copies = segs * kParts;
    const int s = lane / kParts, x = lane % kParts;
    int stage = 0;
    uint32_t phase = 0;
    Walker walk(a.walk, int(blockIdx.x), kGran);
    Piece p;
    while (walk.next(p)) {
        const int len = p.len;
        const int32_t *table = plan.pages + size_t(p.seq) * plan.page_stride;
        const int last = max(len - 1, 0) >> a.page_shift;
        int base = -64, id = 0;
        for (int k0 = p.k0; k0 < p.k1; k0 += kGran) {
            const int first = k0 >> a.page_shift;
            if (((k0 + kGran - 1) >> a.page_shift) >= base + 32) {
                base = first;
                id = len > 0 ? table[min(base + lane, last)] : 0;
                if (uint32_t(id) >= uint32_t(a.pages)) {
                    if (base + lane <= min(last, (p.k1 - 1) >> a.page_shift)) {
                        set_status(a.status, kKvBadPage);
                    }
                    id = 0;
                }
            }
            const int key = k0 + (lane < copies ? s : 0) * seg;
            const int page = __shfl_sync(0xffffffffu, id, (key >> a.page_shift) - base);
            if constexpr (kCache == kMxfp4) {
                const bool ok = wait_or_abort(&sm.raw_empty[stage], phase ^ 1, &sm.abort, a.status);
                if (__all_sync(0xffffffffu, ok)) {
                    if (lane == 0) {
                        tc::mbar_expect_tx(&sm.raw_full[stage], PromptSmem<kCache, D>::kRawBytes);
                    }
                    __syncwarp();
                    if (lane < copies) {
                        const uint8_t *src = a.pool + (size_t(page) * a.kv_heads + p.head) * a.block_bytes;
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                         tc::smem_u32(sm.raw[stage] + lane * a.block_bytes)),
                                     "l"(src), "r"(a.block_bytes), "r"(tc::smem_u32(&sm.raw_full[stage]))
                                     : "memory");
                    }
                }
                if (++stage == 2) {
                    stage = 0;
                    phase ^= 1;
                }
                continue;
            }
            const int y = ((page * a.kv_heads + p.head) * 2) * (1 << a.page_shift) + (key & ((1 << a.page_shift) - 1));
            const uint32_t to = uint32_t(x * kGran + s * seg) * 128;
            bool ok = wait_or_abort(&sm.k_empty[stage], phase ^ 1, &sm.abort, a.status);
            if (__all_sync(0xffffffffu, ok)) {
                if (lane == 0) {
                    tc::mbar_expect_tx(&sm.k_full[stage], kGran * D * 2);
                }
                __syncwarp();
                if (lane < copies) {
                    tc::tma_load_2d(sm.k[stage] + to, map, 64 * x, y, &sm.k_full[stage]);
                }
            }
            ok = wait_or_abort(&sm.v_empty[stage], phase ^ 1, &sm.abort, a.status);
            if (__all_sync(0xffffffffu, ok)) {
                if (lane == 0) {
                    tc::mbar_expect_tx(&sm.v_full[stage], kGran * D * 2);
                }
                __syncwarp();
                if (lane < copies) {
                    tc::tma_load_2d(sm.v[stage] + to, map, 64 * x, y + (1 << a.page_shift), &sm.v_full[stage]);
                }
            }
            if (++stage == PromptSmem<kCache, D>::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
    }
}

// A granule of a 4-bit cache to bf16, which holds every code times its scale
// exactly: a thread per key, K then V, into the places that TMA fills for a
// 16-bit cache.
template <int kCache, int D> __device__ __forceinline__ void expand(const AttendArgs &a, PromptSmem<kCache, D> &sm) {
    const int key = threadIdx.x - 32 * kExpander;
    int stage = 0, raw = 0;
    uint32_t phase = 0, raw_phase = 0;
    const int tokens = 1 << a.page_shift;
    const uint32_t at = uint32_t(key >> a.page_shift) * a.block_bytes;
    const int t = key & (tokens - 1);
    auto half = [&](const uint8_t *src, uint8_t *dst) {
        const uint8_t *scales = src + tokens * (D / 2) + t * (D / 32);
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const float f = scale_of(scales[b]);
            const uint4 w = *reinterpret_cast<const uint4 *>(src + t * (D / 2) + 16 * b);
            const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 v = __half22float2(e2m1x2_to_half2((c[i] >> (8 * j)) & 255u));
                    o[j] = pack2<kBf16>(v.x * f, v.y * f);
                }
                const int chunk = 4 * (b & 1) + i;
                *reinterpret_cast<uint4 *>(dst + (b / 2) * (kGran * 128) + key * 128 + ((chunk ^ (key & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    Walker walk(a.walk, int(blockIdx.x), kGran);
    Piece p;
    while (walk.next(p)) {
        for (int k0 = p.k0; k0 < p.k1; k0 += kGran) {
            wait_or_abort(&sm.raw_full[raw], raw_phase, &sm.abort, a.status);
            wait_or_abort(&sm.k_empty[stage], phase ^ 1, &sm.abort, a.status);
            half(sm.raw[raw] + at, sm.k[stage]);
            arrive(&sm.k_full[stage]);
            wait_or_abort(&sm.v_empty[stage], phase ^ 1, &sm.abort, a.status);
            half(sm.raw[raw] + at + (a.block_bytes >> 1), sm.v[stage]);
            arrive(&sm.v_full[stage]);
            arrive(&sm.raw_empty[raw]);
            raw_phase ^= uint32_t(raw);
            raw ^= 1;
            if (++stage == PromptSmem<kCache, D>::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
    }
}

// The matrix instructions, from one thread.
template <int kRows, int kCache, int D> __device__ __forceinline__ void issue(const AttendArgs &a, PromptSmem<kCache, D> &sm, uint32_t tmem) {
    constexpr int kStages = PromptSmem<kCache, D>::kStages;
    constexpr uint32_t kSDesc = f16_desc<kRows>(kGran, false), kODesc = f16_desc<kRows>(D, true);
    const uint32_t s_at[2] = {tmem, tmem + 128}, o_at[2] = {tmem + 256, tmem + 256 + D};
    int ks = 0, vs = 0;
    uint32_t k_phase = 0, v_phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
    auto scores = [&](int w) {
        const uint32_t q = tc::smem_u32(sm.q[w]), k = tc::smem_u32(sm.k[ks]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const uint32_t off = uint32_t(i / 4) * 128 * 128 + uint32_t(i % 4) * 32;
            mma_ss(s_at[w], tc::smem_desc_sw128(q + off), tc::smem_desc_sw128(k + off), kSDesc, i > 0);
        }
        tc::mma_commit(&sm.s_full[w]);
    };
    Walker walk(a.walk, int(blockIdx.x), kGran);
    Piece p, ahead;
    bool any = walk.next(p), more;
    for (; any; any = more, p = ahead) {
        more = walk.next(ahead);
        const int n = (p.k1 - p.k0) / kGran, halves = p.ncols > kHalf ? 2 : 1;
        wait_or_abort(&sm.k_full[ks], k_phase, &sm.abort, a.status);
        for (int w = 0; w < halves; ++w) {
            wait_or_abort(&sm.q_full[w], q_phase[w], &sm.abort, a.status);
            q_phase[w] ^= 1;
            tc::fence_after_sync();
            if (!*const_cast<volatile int *>(&sm.abort)) {
                scores(w);
            }
        }
        tc::mma_commit(&sm.k_empty[ks]);
        if (++ks == kStages) {
            ks = 0;
            k_phase ^= 1;
        }
        for (int j = 0; j < n; ++j) {
            wait_or_abort(&sm.v_full[vs], v_phase, &sm.abort, a.status);
            const uint32_t v = tc::smem_u32(sm.v[vs]);
            for (int w = 0; w < halves; ++w) {
                wait_or_abort(&sm.p_full[w], p_phase[w], &sm.abort, a.status);
                p_phase[w] ^= 1;
                tc::fence_after_sync();
                if (j + 1 < n && w == 0) {
                    wait_or_abort(&sm.k_full[ks], k_phase, &sm.abort, a.status);
                }
                if (*const_cast<volatile int *>(&sm.abort)) {
                    continue;
                }
#pragma unroll
                for (int i = 0; i < kGran / 16; ++i) {
                    mma_ts(o_at[w], s_at[w] + 8 * i, desc_mn(v + uint32_t(i) * 2048, kGran * 128), kODesc, j > 0 || i > 0);
                }
                if (j + 1 < n) {
                    scores(w);
                } else {
                    tc::mma_commit(&sm.o_full[w]);
                }
            }
            tc::mma_commit(&sm.v_empty[vs]);
            if (++vs == kStages) {
                vs = 0;
                v_phase ^= 1;
            }
            if (j + 1 < n) {
                tc::mma_commit(&sm.k_empty[ks]);
                if (++ks == kStages) {
                    ks = 0;
                    k_phase ^= 1;
                }
            }
        }
    }
}

// A warpgroup: the columns [128 w, 128 w + 128) of each tile, one per thread.
template <int kRows, int kCache, int D>
__device__ __forceinline__ void soften(const AttendArgs &a, const Plan &plan, PromptSmem<kCache, D> &sm, uint32_t tmem) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, w = warp >> 2;
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // (32 * quadrant) << 16
    const uint32_t s_at = tmem + 128 * w + lanes, o_at = tmem + 256 + D * w + lanes;
    constexpr float kSlack = kRows == kF16 ? 4.0f : 8.0f;
    constexpr float kLift = kRows == kF16 ? 11.0f : 0.0f;
    const float scale = a.scale * kLog2e, cap_log2 = a.cap * kLog2e;
    const float cap_in = a.cap != 0.0f ? scale * 2.0f / a.cap : 0.0f;
    const float sign = scale < 0.0f ? -1.0f : 1.0f;  // the largest score is the smallest product where the scale is negative
    const bool special = a.cap != 0.0f || a.slopes;
    uint32_t s_phase = 0, o_phase = 0;
    Walker walk(a.walk, int(blockIdx.x), kGran);
    // The tile after the one in hand is looked up while that one runs, and its Q
    // rows are copied as soon as the last scores of this one are there, so that
    // its first scores are under way before this one has ended.
    struct Column {
        Piece p;
        bool any, active, have;
        int row, qhead;
        int4 ri;
        float slope;
    };
    auto look_up = [&](Column &c) {
        c.any = walk.next(c.p);
        c.active = c.any && (w == 0 || c.p.ncols > kHalf);
        c.have = c.any && tid < c.p.ncols;
        c.row = 0, c.qhead = 0, c.slope = 0.0f;
        c.ri = make_int4(0, 0, 1 << 30, -1);
        if (c.have) {
            const int cc = c.p.col0 + tid, r = cc / a.group;
            c.qhead = c.p.head * a.group + cc - r * a.group;
            c.row = c.p.row0 + r;
            c.ri = a.walk.row[c.row];
            c.ri.y = max(c.ri.y, 0), c.ri.z = min(c.ri.z, c.p.len);
            c.slope = a.slopes ? a.slopes[c.qhead] * kLog2e : 0.0f;
        }
    };
    // Q, 16 bytes at a time, swizzled as the matrix instruction reads it
    auto copy_q = [&](const Column &c) {
        const bool read = c.have && c.row < a.rows;
        const uint16_t *src = static_cast<const uint16_t *>(a.q) + (read ? size_t(c.row) * a.q_stride + size_t(c.qhead) * D : 0);
        const int r = tid & (kHalf - 1);
        const uint32_t to = tc::smem_u32(sm.q[w]) + r * 128;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + uint32_t(i / 8) * (kHalf * 128) + (((i & 7) ^ (r & 7)) << 4)),
                         "l"(src + (read ? 8 * i : 0)), "r"(read ? 16 : 0)
                         : "memory");
        }
    };
    auto publish_q = [&] {
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc::fence_before_sync();
        arrive(&sm.q_full[w]);
    };
    Column cur, next;
    look_up(cur);
    if (cur.active) {
        copy_q(cur);
        publish_q();
    }
    for (; cur.any; cur = next) {
        look_up(next);
        const Piece &p = cur.p;
        const int c = tid;  // column of the tile
        const bool active = cur.active, have = cur.have;
        const int row = cur.row, qhead = cur.qhead;
        const int4 ri = cur.ri;
        const float slope = cur.slope;
        const bool sees = ri.y < ri.z;
        float m = -INFINITY, l = 0.0f;
        if (!active && next.active) {
            copy_q(next);
            publish_q();
        }
        if (active) {
            for (int k0 = p.k0; k0 < p.k1; k0 += kGran) {
                const bool ok = wait_or_abort(&sm.s_full[w], s_phase, &sm.abort, a.status);
                s_phase ^= 1;
                if (!__all_sync(0xffffffffu, ok)) {
                    continue;
                }
                tc::fence_after_sync();
                if (k0 + kGran >= p.k1 && next.active) {
                    copy_q(next);  // the last scores of this tile: its Q has been read
                }
                // ---- the maximum; scores that are capped, biased or masked go back as they then are ----
                float f = scale, top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                const bool mask = __any_sync(0xffffffffu, k0 < ri.y || k0 + kGran > ri.z);
                if (mask || special) {
                    f = 1.0f;
                    const int from = ri.y - k0, to = ri.z - k0;
#pragma unroll 1
                    for (int i = 0; i < kGran; i += 32) {
                        float s[32];
                        tmem_ld32(s_at + i, s);
                        tc::wait_ld();
                        if (a.cap != 0.0f) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                s[j] = capped(s[j], cap_in, cap_log2);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                s[j] *= scale;
                            }
                        }
                        if (a.slopes) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                s[j] = fmaf(-slope, fabsf(float(ri.x - k0 - i - j)), s[j]);
                            }
                        }
                        if (mask) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                s[j] = i + j >= from && i + j < to ? s[j] : -INFINITY;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            top[j & 3] = fmaxf(top[j & 3], s[j]);
                        }
                        tmem_st32(s_at + i, s);
                    }
                    tc::wait_st();
                } else {
                    float s[2][32];
                    tmem_ld32(s_at, s[0]);
                    tc::wait_ld();
#pragma unroll
                    for (int i = 0; i < kGran / 32; ++i) {
                        if (i + 1 < kGran / 32) {
                            tmem_ld32(s_at + 32 * (i + 1), s[(i + 1) & 1]);
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            top[j & 3] = fmaxf(top[j & 3], s[i & 1][j] * sign);
                        }
                        tc::wait_ld();
                    }
                }
                const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * (f == 1.0f ? 1.0f : f * sign);
                float s[2][32];
                tmem_ld32(s_at, s[0]);
                if (__any_sync(0xffffffffu, most > m + (kSlack + kLift))) {
                    const float mn = fmaxf(m, most - kLift);
                    const float up = ex2(m - (mn == -INFINITY ? 0.0f : mn));
                    m = mn;
                    l *= up;
                    if (k0 != p.k0) {
                        // the product before has ended: its scores came behind it
#pragma unroll 1
                        for (int i = 0; i < D; i += 32) {
                            float o[32];
                            tmem_ld32(o_at + i, o);
                            tc::wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                o[j] *= up;
                            }
                            tmem_st32(o_at + i, o);
                        }
                    }
                }
                // ---- the weights, over the scores ----
                const float base = m == -INFINITY ? 0.0f : m;
                float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
                tc::wait_ld();
#pragma unroll
                for (int i = 0; i < kGran / 32; ++i) {
                    if (i + 1 < kGran / 32) {
                        tmem_ld32(s_at + 32 * (i + 1), s[(i + 1) & 1]);
                    }
                    uint32_t w2[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float *x = s[i & 1] + j;
                        const float p0 = ex2(fmaf(x[0], f, -base)), p1 = ex2(fmaf(x[1], f, -base));
                        const float p2 = ex2(fmaf(x[2], f, -base)), p3 = ex2(fmaf(x[3], f, -base));
                        l0 += p0, l1 += p1, l2 += p2, l3 += p3;
                        w2[j / 2] = pack2<kRows>(p0, p1);
                        w2[j / 2 + 1] = pack2<kRows>(p2, p3);
                    }
                    tc::wait_ld();
                    tc::tmem_st16(s_at + 16 * i, w2);
                }
                l += (l0 + l1) + (l2 + l3);
                tc::wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    arrive(&sm.p_full[w]);
                }
            }
            if (next.active) {
                publish_q();
            }
        }
        // ---- the end of the tile ----
        const bool whole = p.first == p.last;
        bool bad = false;
        if (active) {
            const bool ok = wait_or_abort(&sm.o_full[w], o_phase, &sm.abort, a.status);
            o_phase ^= 1;
            tc::fence_after_sync();
            float g = 1.0f;
            float *part = a.part + (size_t(part_slot(int(blockIdx.x), p.first)) * kPromptWidth + c) * (D + 2);
            if (whole) {
                float mm = m, ll = l;
                if (a.sinks && have) {
                    const float sink = a.sinks[qhead] * kLog2e;
                    mm = fmaxf(m, sink);
                    const float safe = mm == -INFINITY ? 0.0f : mm;
                    g = exp2f(m - safe);
                    ll = l * g + exp2f(sink - safe);
                }
                g = g / ll;
            } else if (have) {
                part[D] = m, part[D + 1] = l;
            }
            const bool write = have && row < a.rows && ri.w == p.seq;
            if (__all_sync(0xffffffffu, ok)) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    float o[32];
                    tmem_ld32(o_at + 32 * i, o);
                    tc::wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        float v[8];
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            v[t] = whole ? (sees ? o[j + t] * g : 0.0f) : o[j + t];
                            bad = bad || !(fabsf(v[t]) < INFINITY);
                        }
                        if (whole && write) {
                            store8<kRows>(a.out, size_t(row) * a.out_stride + size_t(qhead) * D + 32 * i + j, v);
                        } else if (!whole && have) {
#pragma unroll
                            for (int t = 0; t < 8; t += 2) {
                                *reinterpret_cast<float2 *>(part + 32 * i + j + t) = make_float2(v[t], v[t + 1]);
                            }
                        }
                    }
                }
            }
            tc::fence_before_sync();
            uint32_t redo = __ballot_sync(0xffffffffu, bad && whole && write);
            while (redo) {
                const int src = __ffs(redo) - 1;
                redo &= redo - 1;
                attend_column<kRows, kCache, D>(a, plan, p.head, p.seq, p.len, __shfl_sync(0xffffffffu, row, src),
                                               __shfl_sync(0xffffffffu, qhead, src));
            }
        }
        if (!whole) {
            if (arrive_last(a, p, &sm.last, softmax_sync)) {
                merge_tile<kRows, kCache, D>(a, plan, p, warp, 8, kPromptWidth);
            }
            softmax_sync();
        }
    }
}

template <int kRows, int kCache, int D>
__global__ void __launch_bounds__(PromptShape<kCache>::kThreads, 1)
    kv_attend_prompt_kernel(AttendArgs a, const __grid_constant__ CUtensorMap map) {
    using Shape = PromptShape<kCache>;
    using Smem = PromptSmem<kCache, D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5;
    const Plan &plan = *a.walk.plan;
    wait_previous();
    if (a.walk.list->ctas != int(gridDim.x) || a.walk.list->width != kPromptWidth || a.walk.list->gran != kGran) {
        if (tid == 0) {
            set_status(a.status, kKvStalePlan);
        }
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < Smem::kStages; ++i) {
            tc::mbar_init(&sm.k_full[i], Shape::kFour ? 128 : 1);
            tc::mbar_init(&sm.k_empty[i], 1);
            tc::mbar_init(&sm.v_full[i], Shape::kFour ? 128 : 1);
            tc::mbar_init(&sm.v_empty[i], 1);
        }
        for (int w = 0; w < 2; ++w) {
            tc::mbar_init(&sm.raw_full[w], 1);
            tc::mbar_init(&sm.raw_empty[w], 128);
            tc::mbar_init(&sm.q_full[w], kHalf);
            tc::mbar_init(&sm.s_full[w], 1);
            tc::mbar_init(&sm.p_full[w], 4);
            tc::mbar_init(&sm.o_full[w], 1);
        }
        sm.abort = 0;
        tc::fence_mbar_init();
    }
    if (warp == kIssuer) {
        tc::tmem_alloc(&sm.tmem, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sm.tmem;
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::kSoftmaxRegs));
        soften<kRows, kCache, D>(a, plan, sm, tmem);
    } else if (warp < kExpander) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kOtherRegs));
        if (warp == kLoader) {
            load_granules<kCache, D>(a, plan, &map, sm);
        } else if (threadIdx.x == 32 * kIssuer) {
            issue<kRows, kCache, D>(a, sm, tmem);
        }
    } else if constexpr (Shape::kFour) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kExpandRegs));
        expand<kCache, D>(a, sm);
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kIssuer) {
        if (*const_cast<volatile int *>(&sm.abort)) {
            // copies and products that are still in flight end before their memory goes
            for (uint32_t ph = 0; ph < 2; ++ph) {
                for (int i = 0; i < Smem::kStages; ++i) {
                    tc::mbar_wait(&sm.k_full[i], ph, 1000000ull);
                    tc::mbar_wait(&sm.v_full[i], ph, 1000000ull);
                    tc::mbar_wait(&sm.k_empty[i], ph, 1000000ull);
                    tc::mbar_wait(&sm.v_empty[i], ph, 1000000ull);
                }
                for (int i = 0; i < 2; ++i) {
                    tc::mbar_wait(&sm.raw_full[i], ph, 1000000ull);
                }
            }
        }
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

// f16 rows over a 4-bit cache stay with the kernel for few columns: bf16, which
// a 4-bit value times its scale needs for its exponent, would cut their Q.
template <int kRows, int kCache> constexpr bool built() {
    return kRows != kF32 && (kCache != kMxfp4 || kRows == kBf16);
}

template <int kRows, int kCache, int D> cudaError_t launch(const ttl_kv &h, const AttendArgs &a, int layer) {
    if constexpr (!built<kRows, kCache>()) {
        return cudaErrorInvalidValue;
    } else {
        return launch_chained(kv_attend_prompt_kernel<kRows, kCache, D>, h.ctas[1], PromptShape<kCache>::kThreads,
                              sizeof(PromptSmem<kCache, D>), h.stream, a, h.maps[size_t(layer)]);
    }
}

template <int kRows, int kCache, int D> cudaError_t configure(ttl_kv &h) {
    if constexpr (!built<kRows, kCache>()) {
        return cudaSuccess;
    } else {
        h.prompt_ctas = std::min(h.sms, kMaxCtas);
        return cudaFuncSetAttribute(kv_attend_prompt_kernel<kRows, kCache, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(sizeof(PromptSmem<kCache, D>)));
    }
}

}  // namespace

cudaError_t prompt_configure(ttl_kv &h) {
    return TTL_KV_DISPATCH(&h, configure, h);
}

cudaError_t launch_prompt(const ttl_kv &h, const AttendArgs &a, int layer) {
    return TTL_KV_DISPATCH(&h, launch, h, a, layer);
}

}  // namespace kv
}  // namespace ttl

// kv_prompt.cu -- attention of many columns per KV head (prompts and chunks of
// prompts) over the paged cache on tcgen05, for f16 and bf16 rows.
//
//   S [128 cols x 64 keys] = Q K^T      A = Q, B = K from shared memory (K-major)
//   O [128 cols x D]      += P V        A = P from tensor memory, B = V (D-major)
//
// What bounds it is neither of these: per score the tensor pipe does 4 D
// operations (at D = 64, 256 of its 8192 a clock) and the special-function unit
// one exponential (16 a clock), so 128 x 128 scores take 512 clocks of the one
// and 1024 of the other.  So the exponentials must never wait:
//   - a tile is 2 x 128 columns, each with a warpgroup of its own: while one
//     turns its scores into weights, the tensor pipe works for the other;
//   - a granule of 128 keys is taken in two halves with scores of their own, so
//     that a warpgroup has the next half's scores while the products of this one
//     are under way;
//   - a thread owns a column: its 64 scores of a half come from tensor memory
//     into registers once, the maximum and the sum need no shuffles, and the
//     weights go back over the scores as P;
//   - the maximum moves only when a weight would pass 2^8 (f16: 2^4 times the
//     lift), and only then are the sums in tensor memory read, rescaled and
//     written;
//   - a quarter of the exponentials is computed on the multiply-add units.
// One warp loads K and V (TMA, 128-byte swizzle, a ring of granules), one issues
// the matrix instructions, two look tiles up and copy their Q rows, and over a
// 4-bit cache four turn codes into bf16.  The scores of the half after next are
// issued right behind the product of this one, over the weights it has just read.
//
// Measured, with the plan's 6 us: a 4096-token prompt of 64 query and 8 KV heads, D
// = 64, bf16: 252 us, 545 TFLOP/s of the 1675 that a plain product reaches; the
// special-function unit alone needs 88 us (40 % busy), the tensor pipe (27 %) 82.  A
// half takes a warp about 1900 clocks: 400 for loads and the maximum, 900 for the
// weights, the rest for hand-overs, with one other warp on its scheduler to fill the
// gaps; the third that would need 576 columns of tensor memory.  Ends of tiles are
// 7 %.  f16 chunks of up to 509 rows, D = 128, a cap: 124 us, 323 TFLOP/s.  A
// 1500-token prompt over 4 bits with a distance bias: 120 us, of which the four
// expanding warps cost about 15.  In these two a CTA has 20 to 25 granules in two or
// three pieces: starts, ends and merges weigh more, and the plan's equal shares come
// out unequal, the last CTA 15 % behind the mean.
//
// Registers: 64-wide heads over 16 bits keep everything in them; 128-wide ones spill
// 32 bytes, over 4 bits 56 (64-wide) and 224.
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
constexpr int kKeys = 64;                  // keys of a step: half a granule
constexpr int kLoader = 8, kIssuer = 9;    // warps
constexpr int kScout = 10;                 // two warps
constexpr int kExpander = 12;              // first of the four warps that expand a 4-bit cache
constexpr uint32_t kTmemCols = 512;

// Threads, and registers of the softmax warpgroups, of the loader's and of the
// expanders': a warpgroup may only take what the launch holds (168 or 128 a
// thread), 256 * 208 + 128 * 80 <= 384 * 168 and 256 * 176 + 128 * 64 + 128 * 96
// <= 512 * 128.
template <int kCache> struct PromptShape {
    static constexpr bool kFour = kCache == kMxfp4;
    static constexpr int kThreads = kFour ? 512 : 384;
    static constexpr int kSoftmaxRegs = kFour ? 176 : 208, kOtherRegs = kFour ? 64 : 80, kExpandRegs = 96;
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
    uint64_t v_tail[kStages];                               // V of a granule that passes the sequence's end, as it was read
    Piece piece[2];                                         // the tile in hand and the next; ncols 0: no more
    uint64_t piece_full[2], piece_empty[2], q_full, q_empty;
    uint64_t s_full[2][2], p_full[2][2], o_done[2][2];  // [warpgroup][half of a granule]
    uint32_t tmem;
    int last;
    Halt halt;
};

__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
// True in all softmax warps when it is in any.
__device__ __forceinline__ bool softmax_any(bool x) {
    uint32_t y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(y)
        : "r"(x ? 1u : 0u)
        : "memory");
    return y != 0;
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
// Issued by the lane with `lead` set, the operands alike in all lanes of the warp:
// so the compiler can keep them in uniform registers, which the instruction
// takes.  (Code of one thread that has left its warp costs about 120 clocks per
// instruction, twice what the tensor pipe needs for it.)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc::smem_u32(bar)),
        "r"(lead)
        : "memory");
}
__device__ __forceinline__ uint32_t elected() {
    uint32_t lead;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(lead));
    return lead;
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
                    // (a granule may begin on pages below all that the tile sees: not reported)
                    if (base + lane >= p.low >> a.page_shift && base + lane <= min(last, (p.k1 - 1) >> a.page_shift)) {
                        set_status(a.status, kKvBadPage);
                    }
                    id = 0;
                }
            }
            const int key = k0 + (lane < copies ? s : 0) * seg;
            const int page = __shfl_sync(0xffffffffu, id, (key >> a.page_shift) - base);
            if constexpr (kCache == kMxfp4) {
                const bool ok = wait_or_abort<true>(&sm.raw_empty[stage], phase ^ 1, &sm.halt, a.status);
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
            bool ok = wait_or_abort<true>(&sm.k_empty[stage], phase ^ 1, &sm.halt, a.status);
            if (__all_sync(0xffffffffu, ok)) {
                if (lane == 0) {
                    tc::mbar_expect_tx(&sm.k_full[stage], kGran * D * 2);
                }
                __syncwarp();
                if (lane < copies) {
                    tc::tma_load_2d(sm.k[stage] + to, map, 64 * x, y, &sm.k_full[stage]);
                }
            }
            ok = wait_or_abort<true>(&sm.v_empty[stage], phase ^ 1, &sm.halt, a.status);
            if (__all_sync(0xffffffffu, ok)) {
                uint64_t *bar = k0 + kGran > len ? &sm.v_tail[stage] : &sm.v_full[stage];  // the scouts hand a tail on
                if (lane == 0) {
                    tc::mbar_expect_tx(bar, kGran * D * 2);
                }
                __syncwarp();
                if (lane < copies) {
                    tc::tma_load_2d(sm.v[stage] + to, map, 64 * x, y + (1 << a.page_shift), bar);
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
// exactly (below 2^-126 as a subnormal): a thread per key, K then V, into the
// places that TMA fills for a 16-bit cache.
template <int kCache, int D> __device__ __forceinline__ void expand(const AttendArgs &a, PromptSmem<kCache, D> &sm) {
    const int key = threadIdx.x - 32 * kExpander;
    int stage = 0, raw = 0;
    uint32_t phase = 0, raw_phase = 0;
    const int tokens = 1 << a.page_shift;
    const uint32_t at = uint32_t(key >> a.page_shift) * a.block_bytes;
    const int t = key & (tokens - 1);
    const __nv_bfloat162 unit = __bfloat162bfloat162(__ushort_as_bfloat16(0x7e80));  // 2^126
    // dead: V behind the sequence's end, whatever was left there, becomes 0
    auto half = [&](const uint8_t *src, uint8_t *dst, bool dead) {
        const uint8_t *scales = src + tokens * (D / 2) + t * (D / 32);
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const __nv_bfloat162 f = __bfloat162bfloat162(__float2bfloat16_rn(dead ? 1.0f : scale_of(scales[b])));  // a power of two
            const uint4 w = dead ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4 *>(src + t * (D / 2) + 16 * b);
            const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // byte j's codes to the top of the halves: sign at bit 15, the three bits of
                    // exponent and mantissa to bits 6 to 8, a bf16 of 2^-126 times the value
                    // (0.5 and 0 are subnormal in either format); both products are exact but
                    // for results below bf16's normal range
                    const uint32_t x = __byte_perm(c[i] << 4, c[i], j << 4 | (4 + j) << 12);
                    const uint32_t bits = (x & 0x80008000u) | ((x >> 6) & 0x01c001c0u);
                    __nv_bfloat162 v;
                    memcpy(&v, &bits, 4);
                    v = __hmul2(__hmul2(v, unit), f);
                    memcpy(&o[j], &v, 4);
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
            wait_or_abort<true>(&sm.raw_full[raw], raw_phase, &sm.halt, a.status);
            wait_or_abort<true>(&sm.k_empty[stage], phase ^ 1, &sm.halt, a.status);
            half(sm.raw[raw] + at, sm.k[stage], false);
            arrive(&sm.k_full[stage]);
            wait_or_abort<true>(&sm.v_empty[stage], phase ^ 1, &sm.halt, a.status);
            half(sm.raw[raw] + at + (a.block_bytes >> 1), sm.v[stage], k0 + key >= p.len);
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

// The matrix instructions: a warp, one lane of which issues them.
template <int kRows, int kCache, int D> __device__ __forceinline__ void issue(const AttendArgs &a, PromptSmem<kCache, D> &sm, uint32_t tmem) {
    constexpr int kStages = PromptSmem<kCache, D>::kStages;
    constexpr uint32_t kSDesc = f16_desc<kRows>(kKeys, false), kODesc = f16_desc<kRows>(D, true);
    constexpr uint32_t kTileBytes = kGran * D * 2;
    const uint32_t lead = elected();
    // descriptors of the first Q, K and V; offsets go to their low bits in units of 16 bytes
    const uint64_t q_desc = tc::smem_desc_sw128(tc::smem_u32(sm.q[0])), k_desc = tc::smem_desc_sw128(tc::smem_u32(sm.k[0])),
                   v_desc = desc_mn(tc::smem_u32(sm.v[0]), kGran * 128);
    int ks = 0, vs = 0;
    uint32_t k_phase = 0, v_phase = 0, q_phase = 0, p_phase = 0;  // p: bit 2 h + w
    auto scores = [&](int w, int h) {
        const uint64_t q = q_desc + uint64_t(uint32_t(w) * (kHalf * D * 2) >> 4), k = k_desc + uint64_t((uint32_t(ks) * kTileBytes + h * kKeys * 128) >> 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const uint64_t off = (uint32_t(i / 4) * 128 * 128 + uint32_t(i % 4) * 32) >> 4;
            mma_ss(tmem + 128 * w + h * kKeys, q + off, k + off, kSDesc, i > 0, lead);
        }
        commit(&sm.s_full[w][h], lead);
    };
    auto next_k = [&] {
        commit(&sm.k_empty[ks], lead);
        if (++ks == kStages) {
            ks = 0;
            k_phase ^= 1;
        }
    };
    Walker walk(a.walk, int(blockIdx.x), kGran);
    Piece p, ahead;
    bool any = walk.next(p), more, ok = true;
    for (; any; any = more, p = ahead) {
        more = walk.next(ahead);
        const int n = (p.k1 - p.k0) / kGran, halves = p.ncols > kHalf ? 2 : 1;
        ok = wait_or_abort<true>(&sm.k_full[ks], k_phase, &sm.halt, a.status) && ok;
        ok = wait_or_abort<true>(&sm.q_full, q_phase, &sm.halt, a.status) && ok;
        q_phase ^= 1;
        tc::fence_after_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w < halves && __all_sync(0xffffffffu, ok)) {
                    scores(w, h);
                }
            }
        }
        next_k();
        if (n == 1) {
            commit(&sm.q_empty, lead);
        }
        for (int j = 0; j < n; ++j) {
            if ((j & 255) == 255 && lead && ok) {
                sm.halt.alive();  // about twice a millisecond
            }
            ok = wait_or_abort<true>(&sm.v_full[vs], v_phase, &sm.halt, a.status) && ok;
            if (j + 1 < n) {
                ok = wait_or_abort<true>(&sm.k_full[ks], k_phase, &sm.halt, a.status) && ok;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint64_t v = v_desc + uint64_t((uint32_t(vs) * kTileBytes + h * kKeys * 128) >> 4);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (w < halves) {
                        ok = wait_or_abort<true>(&sm.p_full[w][h], (p_phase >> (2 * h + w)) & 1u, &sm.halt, a.status) && ok;
                        p_phase ^= 1u << (2 * h + w);
                        tc::fence_after_sync();
                        if (!__all_sync(0xffffffffu, ok)) {
                            continue;
                        }
#pragma unroll
                        for (int i = 0; i < kKeys / 16; ++i) {
                            mma_ts(tmem + 256 + D * w, tmem + 128 * w + h * kKeys + 8 * i, v + uint64_t(i * 2048 >> 4), kODesc,
                                   j > 0 || h > 0 || i > 0, lead);
                        }
                        commit(&sm.o_done[w][h], lead);
                        if (j + 1 < n) {
                            scores(w, h);
                        }
                    }
                }
            }
            commit(&sm.v_empty[vs], lead);
            if (++vs == kStages) {
                vs = 0;
                v_phase ^= 1;
            }
            if (j + 1 < n) {
                next_k();
            }
            if (j + 2 == n) {
                commit(&sm.q_empty, lead);  // the tile's last scores are under way
            }
        }
    }
}

// Two warps that look the tiles up: each tile's description for the softmax
// warps, and its Q rows, 16 bytes at a time, swizzled as the matrix instruction
// reads them, as soon as the last scores of the tile before are computed.  Over a
// 16-bit cache the first of them hands V of a granule that passes the sequence's
// end on, with the slots behind the end set to 0 (over 4 bits the expanders write
// 0 there): long before its product, and before the next tile's Q can go anywhere.
template <int kCache, int D> __device__ __forceinline__ void scout(const AttendArgs &a, PromptSmem<kCache, D> &sm) {
    const int lane = threadIdx.x - 32 * kScout;  // 0 .. 63
    Walker walk(a.walk, int(blockIdx.x), kGran);
    Piece p;
    uint32_t side_phase = 0, q_phase = 0, tail_phase = 0;  // tail: a bit per stage
    int granules = 0;                                      // before this tile, modulo the stages
    for (int side = 0;; side ^= 1) {
        const bool more = walk.next(p);
        p.ncols = more ? p.ncols : 0;
        wait_or_abort<true, true>(&sm.piece_empty[side], side_phase ^ 1, &sm.halt, a.status);
        side_phase ^= uint32_t(side);
        if (lane == 0) {
            sm.piece[side] = p;
        }
        arrive(&sm.piece_full[side]);
        if (!more) {
            break;
        }
        wait_or_abort<true, true>(&sm.q_empty, q_phase ^ 1, &sm.halt, a.status);
        q_phase ^= 1;
        const int columns = p.ncols > kHalf ? 2 * kHalf : kHalf;
        for (int i = lane; i < columns * (D / 8); i += 64) {
            const int c = i / (D / 8), chunk = i % (D / 8), r = c & (kHalf - 1);
            int row, qhead;
            a.column(p, c, row, qhead);
            const bool have = c < p.ncols && row < a.rows;
            const uint16_t *src = static_cast<const uint16_t *>(a.q) + (have ? size_t(row) * a.q_stride + size_t(qhead) * D + 8 * chunk : 0);
            const uint32_t to = tc::smem_u32(sm.q[c / kHalf]) + uint32_t(chunk / 8) * (kHalf * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(have ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        arrive(&sm.q_full);
        if constexpr (kCache != kMxfp4) {
            constexpr int kStages = PromptSmem<kCache, D>::kStages;
            const int stage = (granules + (p.k1 - p.k0) / kGran - 1) % kStages;  // of the last granule
            granules = (stage + 1) % kStages;
            if (lane < 32 && p.k1 > p.len) {
                const bool ok = wait_or_abort<true, true>(&sm.v_tail[stage], (tail_phase >> stage) & 1u, &sm.halt, a.status);
                tail_phase ^= 1u << stage;
                if (__all_sync(0xffffffffu, ok)) {
                    const int first = max(p.len - (p.k1 - kGran), 0);
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        clear_rows(tc::smem_u32(sm.v[stage]) + (x * kGran + first) * 128, kGran - first);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        arrive(&sm.v_full[stage]);
                    }
                }
            }
        }
    }
}

// A CTA's partial result of a tile: D / 4 rows of a float4 per column, then a
// row of {maximum, sum}: a warp, whose threads hold a column each, writes and
// reads 512 bytes at a time.
template <int D> __device__ __forceinline__ float *part_of(const AttendArgs &a, int cta, int first) {
    static_assert(kPromptWidth * (D + 2) <= kPromptWidth * part_pitch(D), "the space of a slot");
    return a.part + size_t(part_slot(cta, first)) * kPromptWidth * part_pitch(D);
}

// Merges the parts of a thread's column in the order of the keys, and stores it.
// What counts is the time of a load through L2: eight are under way per thread
// (two warps' worth of columns at a time, two loads each, took 30 us for 256
// columns of 128 values in three parts).
template <int kRows, int D>
__device__ __forceinline__ void merge_column(const AttendArgs &a, const Piece &p, int c, int row, int qhead, bool write, bool sees) {
    float m = -INFINITY, l = 0.0f;
    for (int k = p.first; k <= p.last; ++k) {
        const float2 y = __ldcg(reinterpret_cast<const float2 *>(part_of<D>(a, k, p.first) + kPromptWidth * D) + c);
        const float mn = fmaxf(m, y.x), safe = mn == -INFINITY ? 0.0f : mn;
        l = l * exp2f(m - safe) + y.y * exp2f(y.x - safe);
        m = mn;
    }
    const float safe = m == -INFINITY ? 0.0f : m;
    const float g = (a.sinks && write ? add_sink(m, l, a.sinks[qhead]) : 1.0f) / l;
#pragma unroll 1
    for (int i = 0; i < D / 4; i += 8) {
        float o[32] = {};
#pragma unroll 1
        for (int k = p.first; k <= p.last; ++k) {
            const float *part = part_of<D>(a, k, p.first);
            const float4 *src = reinterpret_cast<const float4 *>(part) + i * kPromptWidth + c;
            float4 x[8];
            const float y = __ldcg(part + kPromptWidth * D + 2 * c);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __ldcg(src + j * kPromptWidth);
            }
            const float w = exp2f(y - safe);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[4 * j] = fmaf(x[j].x, w, o[4 * j]), o[4 * j + 1] = fmaf(x[j].y, w, o[4 * j + 1]);
                o[4 * j + 2] = fmaf(x[j].z, w, o[4 * j + 2]), o[4 * j + 3] = fmaf(x[j].w, w, o[4 * j + 3]);
            }
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
            float v[8];
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                v[t] = sees ? o[j + t] * g : 0.0f;
            }
            if (write) {
                store8<kRows>(a.out, size_t(row) * a.out_stride + size_t(qhead) * D + 4 * i + j, v);
            }
        }
    }
}

// The columns base + i of the bits i of `bad`, the same in all lanes.
template <int kRows, int kCache, int D>
__device__ __noinline__ void redo_columns(const AttendArgs &a, const Piece &p, uint32_t bad, int base, Halt *halt, float *part) {
    const bool lead = (threadIdx.x & 31) == 0;
    if (lead) {
        halt->busy(true);
    }
    __syncwarp();  // what is written again was written before by another lane
    for (; bad; bad &= bad - 1) {
        redo_column<kRows, kCache, D, true>(a, p, base + __ffs(bad) - 1, part);
    }
    __syncwarp();
    if (lead) {
        halt->busy(false);
    }
}

// A warpgroup: the columns [128 w, 128 w + 128) of each tile, one per thread.
template <int kRows, int kCache, int D>
__device__ __forceinline__ void soften(const AttendArgs &a, PromptSmem<kCache, D> &sm, uint32_t tmem) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, w = warp >> 2;
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // (32 * quadrant) << 16
    const uint32_t s_at = tmem + 128 * w + lanes, o_at = tmem + 256 + D * w + lanes;
    constexpr float kSlack = kRows == kF16 ? 4.0f : 8.0f;
    constexpr float kLift = kRows == kF16 ? 11.0f : 0.0f;
    const float scale = a.scale * kLog2e, cap_log2 = a.cap * kLog2e;
    const float cap_in = a.cap != 0.0f ? scale * 2.0f / a.cap : 0.0f;
    const float ratio = a.cap != 0.0f ? a.scale / a.cap : 0.0f;
    const bool special = a.cap != 0.0f || a.slopes;
    uint32_t phase = 0;       // of the granule, for the barriers of both halves
    uint32_t side_phase = 0;
    for (int side = 0;; side ^= 1) {
        bool ok = wait_or_abort<true>(&sm.piece_full[side], side_phase, &sm.halt, a.status);
        side_phase ^= uint32_t(side);
        const Piece &p = sm.piece[side];
        // all softmax warps go on with the tile, or none
        if (softmax_any(!ok || p.ncols == 0)) {
            break;
        }
        const int c = tid;    // column of the tile
        const bool active = w == 0 || p.ncols > kHalf, have = c < p.ncols;
        int4 ri = make_int4(0, 0, 1 << 30, -1);
        float slope = 0.0f;
        if (have) {
            int row, qhead;
            a.column(p, c, row, qhead);
            ri = a.walk.row[row];
            ri.y = max(ri.y, 0), ri.z = min(ri.z, p.len);
            slope = a.slopes ? a.slopes[qhead] * kLog2e : 0.0f;
        }
        float m = -INFINITY, l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
        if (active) {
            const int begin = p.k0, end = p.k1;
            int h = 0;
            bool ready = false;  // the scores of this half are there
            for (int k0 = begin; k0 < end; k0 += kKeys, h ^= 1) {
                const uint32_t now = phase;
                phase ^= uint32_t(h);
                ok = ready || wait_or_abort<true>(&sm.s_full[w][h], now, &sm.halt, a.status);
                if (!__all_sync(0xffffffffu, ok)) {
                    continue;
                }
                tc::fence_after_sync();
                const uint32_t at = s_at + kKeys * h;
                float s[kKeys];
                tmem_ld32(at, s);
                tmem_ld32(at + 32, s + 32);
                tc::wait_ld();
                float f = scale;
                if (special) {
                    f = 1.0f;
                    if (a.cap != 0.0f) {
                        float big[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int j = 0; j < kKeys; j += 4) {
                            big[0] = max3(big[0], fabsf(s[j]), fabsf(s[j + 1]));
                            big[1] = max3(big[1], fabsf(s[j + 2]), fabsf(s[j + 3]));
                        }
                        if (__any_sync(0xffffffffu, !(fmaxf(big[0], big[1]) * fabsf(ratio) <= kSmallScore))) {
#pragma unroll
                            for (int j = 0; j < kKeys; ++j) {
                                s[j] = capped(s[j], cap_in, cap_log2);
                            }
                        } else {
                            // most scores are far below their cap: one special function per score, not three
#pragma unroll
                            for (int j = 0; j < kKeys; j += 2) {
                                capped_small(s[j], s[j + 1], scale, ratio);
                            }
                        }
                    }
                    if (a.slopes) {
                        const float by = a.cap != 0.0f ? 1.0f : scale;
                        const float away = float(ri.x - k0);
                        if (__all_sync(0xffffffffu, away <= 0.0f || away >= float(kKeys - 1))) {
                            // no row lies between the keys: the bias is a line, +-slope (j - away);
                            // eight keys share its start
                            const float turn = away <= 0.0f ? -slope : slope;
                            float step[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                step[j] = turn * float(j);
                            }
#pragma unroll
                            for (int j = 0; j < kKeys; j += 8) {
                                const float start = turn * (float(j) - away);
#pragma unroll
                                for (int t = 0; t < 8; t += 2) {
                                    bias_pair(s[j + t], s[j + t + 1], by, step[t], step[t + 1], start);
                                }
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < kKeys; ++j) {
                                s[j] = fmaf(-slope, fabsf(away - float(j)), s[j] * by);
                            }
                        }
                    }
                }
                if (__any_sync(0xffffffffu, k0 < ri.y || k0 + kKeys > ri.z)) {
                    const int from = ri.y - k0, to = ri.z - k0;
#pragma unroll
                    for (int j = 0; j < kKeys; ++j) {
                        s[j] = j >= from && j < to ? s[j] : (f < 0.0f ? INFINITY : -INFINITY);  // f turns it
                    }
                }
                // ---- the maximum ----
                float top[2] = {s[0], s[1]};
                if (f >= 0.0f) {
#pragma unroll
                    for (int j = 2; j + 3 < kKeys; j += 4) {
                        top[0] = max3(top[0], s[j], s[j + 1]);
                        top[1] = max3(top[1], s[j + 2], s[j + 3]);
                    }
                    top[0] = max3(max3(top[0], s[kKeys - 2], s[kKeys - 1]), top[1], top[1]);
                } else {
#pragma unroll
                    for (int j = 2; j + 3 < kKeys; j += 4) {
                        top[0] = min3(top[0], s[j], s[j + 1]);
                        top[1] = min3(top[1], s[j + 2], s[j + 3]);
                    }
                    top[0] = min3(min3(top[0], s[kKeys - 2], s[kKeys - 1]), top[1], top[1]);
                }
                // NaN where a score is, or the scale a zero in log2 units
                const float most = top[0] * f;
                if (__any_sync(0xffffffffu, !(most <= m + (kSlack + kLift)))) {
                    l0 = most < INFINITY ? l0 : NAN;  // the column is computed again
                    const float mn = fmaxf(m, most - kLift);
                    const float up = ex2(m - (mn == -INFINITY ? 0.0f : mn));
                    m = mn;
                    l0 *= up, l1 *= up, l2 *= up, l3 *= up;
                    if (k0 != begin) {
                        // The product of the half before ends, and with it those before it:
                        // rescale their sums.  (A barrier per half: the scores in hand came
                        // behind this half's last product, so no barrier is ever more than
                        // the one phase behind that its parity can tell.)
                        wait_or_abort<true>(&sm.o_done[w][h ^ 1], now ^ uint32_t(h ^ 1), &sm.halt, a.status);
                        __syncwarp();
                        tc::fence_after_sync();
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
                float pairs[kKeys / 2];  // of 16-bit weights
                // A quarter of the exponentials goes to the multiply-add units: the special
                // functions alone take 16 a clock and SM.  (4096-token prompt 248 us; with an
                // eighth 256, three eighths 252, half 267.  With a cap, which keeps those units
                // busy already, 112, with an eighth 111.)
#pragma unroll
                for (int j = 0; j < kKeys; j += 4) {
                    // Are the next half's scores there?  Asked here, the answer's way through the
                    // queue that the special functions fill costs nothing.  (4096-token prompt
                    // 264 us without, 249 so.  Over 4 bits the expanding warps take the gaps: 112
                    // us without, 116.)
                    if (kCache != kMxfp4 && j == kKeys / 2) {
                        ready = k0 + kKeys < end && phase_done(&sm.s_full[w][h ^ 1], phase);
                    }
                    fma_pair(s[j], s[j + 1], f, -base);
                    fma_pair(s[j + 2], s[j + 3], f, -base);
                    const float p0 = ex2(s[j]), p1 = ex2(s[j + 1]);
                    float p2, p3;
                    if (j % 8 == 0) {
                        pow2_pair(s[j + 2], s[j + 3], p2, p3);
                    } else {
                        p2 = ex2(s[j + 2]), p3 = ex2(s[j + 3]);
                    }
                    add_pair(l0, l1, p0, p1);
                    add_pair(l2, l3, p2, p3);
                    pairs[j / 2] = __uint_as_float(pack2<kRows>(p0, p1));
                    pairs[j / 2 + 1] = __uint_as_float(pack2<kRows>(p2, p3));
                }
                tmem_st32(at, pairs);
                tc::wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    arrive(&sm.p_full[w][h]);
                }
            }
        }
        // ---- the end of the tile ----
        const bool whole = p.first == p.last, sees = ri.y < ri.z;
        int row = 0, qhead = 0;
        if (have) {
            a.column(p, c, row, qhead);
        }
        bool bad = false;
        if (active) {
            ok = wait_or_abort<true>(&sm.o_done[w][0], phase ^ 1, &sm.halt, a.status) && ok;
            ok = wait_or_abort<true>(&sm.o_done[w][1], phase ^ 1, &sm.halt, a.status) && ok;
            tc::fence_after_sync();
            float l = (l0 + l1) + (l2 + l3);
            float g = 1.0f;
            float *part = part_of<D>(a, int(blockIdx.x), p.first);
            float2 *const stats = reinterpret_cast<float2 *>(part + kPromptWidth * D);
            if (whole) {
                g = (a.sinks && have ? add_sink(m, l, a.sinks[qhead]) : 1.0f) / l;
            } else if (have) {
                stats[c] = make_float2(m, l);
                bad = !(l < INFINITY);
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
                            float4 *dst = reinterpret_cast<float4 *>(part) + (8 * i + j / 4) * kPromptWidth + c;
                            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                            dst[kPromptWidth] = make_float4(v[4], v[5], v[6], v[7]);
                        }
                    }
                }
            }
            tc::fence_before_sync();
            const uint32_t again = __ballot_sync(0xffffffffu, bad && write);
            if (again) {
                redo_columns<kRows, kCache, D>(a, p, again, c & ~31, &sm.halt, whole ? nullptr : part);
            }
        }
        if (!whole) {
            if (arrive_last(a, p, &sm.last, softmax_sync)) {
                merge_column<kRows, D>(a, p, c, row, qhead, have && row < a.rows && ri.w == p.seq, sees);
            }
            softmax_sync();
        }
        __syncwarp();
        if (lane == 0) {
            arrive(&sm.piece_empty[side]);
        }
    }
}

template <int kRows, int kCache, int D>
__global__ void __launch_bounds__(PromptShape<kCache>::kThreads, 1)
    kv_attend_prompt_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap map) {
    using Shape = PromptShape<kCache>;
    using Smem = PromptSmem<kCache, D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5;
    const Plan &plan = *a.walk.plan;
    wait_previous();
    if (!plan_fits(a, kPromptWidth, kGran)) {
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < Smem::kStages; ++i) {
            tc::mbar_init(&sm.k_full[i], Shape::kFour ? 128 : 1);
            tc::mbar_init(&sm.k_empty[i], 1);
            tc::mbar_init(&sm.v_full[i], Shape::kFour ? 128 : 1);
            tc::mbar_init(&sm.v_empty[i], 1);
            tc::mbar_init(&sm.v_tail[i], 1);
        }
        for (int w = 0; w < 2; ++w) {
            tc::mbar_init(&sm.raw_full[w], 1);
            tc::mbar_init(&sm.raw_empty[w], 128);
            tc::mbar_init(&sm.piece_full[w], 64);
            tc::mbar_init(&sm.piece_empty[w], 8);
            for (int h = 0; h < 2; ++h) {
                tc::mbar_init(&sm.s_full[w][h], 1);
                tc::mbar_init(&sm.p_full[w][h], 4);
                tc::mbar_init(&sm.o_done[w][h], 1);
            }
        }
        tc::mbar_init(&sm.q_full, 64);
        tc::mbar_init(&sm.q_empty, 1);
        sm.halt = Halt{0, 0};
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
        soften<kRows, kCache, D>(a, sm, tmem);
    } else if (warp < kExpander) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kOtherRegs));
        if (warp == kLoader) {
            load_granules<kCache, D>(a, plan, &map, sm);
        } else if (warp == kIssuer) {
            issue<kRows, kCache, D>(a, sm, tmem);
        } else {
            scout<kCache, D>(a, sm);
        }
    } else if constexpr (Shape::kFour) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kExpandRegs));
        expand<kCache, D>(a, sm);
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kIssuer) {
        if (sm.halt.aborted()) {
            // copies and products that are still in flight end before their memory goes
            for (uint32_t ph = 0; ph < 2; ++ph) {
                for (int i = 0; i < Smem::kStages; ++i) {
                    tc::mbar_wait(&sm.k_full[i], ph, 1000000ull);
                    tc::mbar_wait(&sm.v_full[i], ph, 1000000ull);
                    tc::mbar_wait(&sm.v_tail[i], ph, 1000000ull);
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

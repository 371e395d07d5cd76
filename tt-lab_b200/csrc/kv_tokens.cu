// kv_tokens.cu -- attention of a few columns per KV head (single tokens, a few
// rows) over the paged cache, for f16 and bf16 rows: the decode side of
// ttl_kv_attend_async.
//
// What it must do is read K and V once: 2 x D x 2 bytes per key and KV head
// (17/64 of that in 4 bits) against 4 x group x D operations, so HBM bounds it
// and the work per byte has to stay small.
//
// Both products are taken with the keys as the rows of the matrix instruction
// (mma.sync m16n8k16) and the columns as its N, 8 to a step: the 8 query heads
// of a KV head fill it, where they would fill half of an M = 16.
//   S^T [16 keys x 8 cols] = K [16 x D] Q^T       A = K rows as they lie in memory
//   O^T [D x 8 cols]      += V^T [D x 16 keys] P^T  A = V^T by ldmatrix.trans
// The weights go from S^T's accumulator layout to the B operand by one 8 x 8
// transpose in registers (movmatrix).  tcgen05 has nothing to give here: its M
// is 128 rows for 8 columns, and the tensor pipe is not what bounds.
//
// A CTA is four warps that compute and one that loads.  The loader walks the
// CTA's piece of the plan and keeps kStages granules of 64 keys in flight (TMA
// boxes with the 128-byte swizzle, or bulk copies of 4-bit pages), across
// tiles.  Each computing warp takes 16 keys of a granule with its own running
// maximum, sum and accumulators; the four are merged when the tile ends.  The
// maximum moves only when a weight would pass 2^8 (bf16) or 2^4 (f16) times 1,
// so that most granules need one vote instead of shuffles and a rescaling;
// weights that large are as exact as weights up to 1.  f16 weights are lifted
// by a power of two, so that the smallest step of f16 (2^-24) is 2^-35 (4 bits:
// 2^-33) of the largest weight.
//
// 4 bits.  K's codes become f16 exactly (cvt e2m1x2 -> f16x2); a block's scale
// multiplies the 32-term partial score of the block, in f32.  V's codes are
// gathered to key pairs (ldmatrix.trans moves 4 codes of a key as one b16) and
// the scale of (key, block) is multiplied into the weight, taken relative to the
// largest scale a column has seen in the block, so that it stays in f16's
// range whatever the values' size.
//
// Measured, with the plan's 6 us: 128 single tokens over 1 to 8192 keys, 64 query
// and 8 KV heads, D = 64, bf16 (985 MB): 151 to 156 us, 6.3 to 6.5 TB/s, a plain
// copy's rate.  One token over 131072 keys (268 MB): 58 us, 41 of them at that rate;
// the rest is two launches, the first loads and the merge of 55 parts a head.  256
// tokens with a window of 128 (70 MB): 29.5 us: the two or three granules of a
// sequence leave nothing to fetch ahead, and each waits for the page ids that name
// it.  64 tokens over 4 bits, up to 16384 keys (287 MB): 95 us, 3 TB/s: the
// schedulers issue in 58 % of all clocks, with the integer pipe busy in 53 %, for
// taking codes apart, so the bytes, 44 us of them, do not bound it.
//
// Registers: tiles of 8 columns, which single tokens have, keep everything in them.
// Wider ones spill: 16 columns of 128-wide heads 64 to 100 bytes, 32 columns 124 to
// 228, in loops that are bound elsewhere or had no narrower form that was faster.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv.cuh"
#include "kv_internal.h"
#include "tc.cuh"

namespace ttl {
namespace kv {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * (kWarps + 1);

template <int kRows, int kCache, int D, int NT> struct TokenShape {
    static constexpr int kCols = 8 * NT;
    static constexpr bool kFour = kCache == kMxfp4;
    static constexpr int kSub = token_sub(kCache, 8 * NT);  // steps of 16 keys a warp takes at once
    static constexpr int kGran = 16 * kWarps * kSub;
    static constexpr uint32_t kStageBytes = kFour ? 2 * kGran * row_bytes(kMxfp4, D) : 2 * kGran * D * 2;
    // Granules in flight: about 96 KB per SM in its two CTAs.  More reads slower
    // (128 tokens of 64 values: three granules 151 us, five 158, six 162), less too
    // (two: 161); with three CTAs on an SM 160.
    static constexpr int kStages = D == 64 || kFour ? 3 : 2;
    // Parts that a lane merges at once.  More of them take registers from the loop over
    // the keys: 64 sequences of two rows, D = 128, 189 us, with eight 226 (four rows, D
    // = 64: 127 and 171; over 4 bits one row, D = 128, 92, with two 96, with three 100).
    // Fewer wait longer where parts are many: one token over 131072 keys 2 us more with
    // two, 4 us with one; over 4 bits, where the loop is what counts, 6 us less.
    static constexpr int kMergeBatch = kFour ? 1 : 4;
    // A column's sums in shared memory: over a 16-bit cache rows of D values whose
    // groups of 8 are swapped by the column, over 4 bits rows with 4 values of
    // padding; either way the accumulators' stores do not collide.
    static constexpr int kOPitch = kFour ? D + 4 : D;
    __device__ static __forceinline__ int o_at(int c, int d) {
        return kFour ? d : d ^ (((c >> 1) & 3) << 3);
    }
    // Q rows: 16-byte chunks swapped by the column.
    __device__ static __forceinline__ int q_at(int c, int d) {
        return d ^ ((c & 7) << 3);
    }
};

template <int kRows, int kCache, int D, int NT> struct TokenSmem {
    using T = TokenShape<kRows, kCache, D, NT>;
    alignas(1024) uint8_t stage[T::kStages][(T::kStageBytes + 1023) / 1024 * 1024];
    float o[kWarps][T::kCols][T::kOPitch];
    float m[kWarps][T::kCols], l[kWarps][T::kCols];
    // the tile in hand and the next: what it is, its Q rows, the plan's rows, slopes and sinks
    Piece piece[2];                // ncols 0: no more
    alignas(16) uint16_t q[2][T::kCols][D];
    int4 row[2][T::kCols];
    float slope[2][T::kCols], sink[2][T::kCols];
    uint64_t tile_full[2], tile_empty[2];
    uint64_t full[T::kStages], empty[T::kStages];
    int last;
    Halt halt;
    int again;                     // some column has a sum that is not finite
    int held[2];                   // so it has in the part of a tile that began in an earlier CTA, or begins here
};

__device__ __forceinline__ void consumer_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
}

// True in all computing warps when it is in any.
__device__ __forceinline__ bool consumers_any(bool x) {
    uint32_t y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(y)
        : "r"(x ? 1u : 0u), "n"(32 * kWarps)
        : "memory");
    return y != 0;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix2_trans(uint32_t &r0, uint32_t &r1, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// C += A B, 16 x 8 x 16, f16 or bf16 operands, f32 sums.
template <int kType> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kType == kF16) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
template <int kType> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kType == kF16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
// Eight E2M1 codes to four f16 pairs.
__device__ __forceinline__ void halves8(uint32_t codes, uint32_t &h0, uint32_t &h1, uint32_t &h2, uint32_t &h3) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h0), "=r"(h1), "=r"(h2), "=r"(h3)
        : "r"(codes));
}
// 2^d for |d| beyond f32's exponents too (0 or infinity there).
__device__ __forceinline__ float pow2i(int d) {
    return ex2(float(max(d, -1000)));
}

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     tc::smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
                 : "memory");
}

// Where this CTA leaves its partial result of a tile.
template <int D, int kCols> __device__ __forceinline__ float *own_part(const AttendArgs &a, const Piece &p) {
    return a.part + size_t(part_slot(int(blockIdx.x), p.first)) * kCols * part_pitch(D);
}

// The loader: one warp, a granule a step.
template <class Smem, int kCache, int D, int kCols, int kGran, int kStages, uint32_t kStageBytes>
__device__ __forceinline__ void load_granules(const AttendArgs &a, const Plan &plan, const CUtensorMap *map, Smem &sm) {
    const int lane = threadIdx.x & 31;
    const int seg = min(1 << a.page_shift, kGran);       // keys of one copy (a TMA box has up to 64 rows)
    static_assert(kCache == kMxfp4 || kGran == 64, "box rows");
    const int segs = kGran / seg;
    int stage = 0;
    uint32_t phase = 0;
    Walker walk(a.walk, int(blockIdx.x), kGran);
    // Page ids, 32 at a time; past the sequence's end its last page stands in.  The
    // first of the next tile are loaded while this one is.
    auto ids = [&](const Piece &p, int base) {
        const int last = max(p.len - 1, 0) >> a.page_shift;
        return p.len > 0 ? plan.pages[size_t(p.seq) * plan.page_stride + min(base + lane, last)] : 0;
    };
    auto checked = [&](const Piece &p, int base, int id) {
        if (uint32_t(id) >= uint32_t(a.pages)) {
            // (a granule may begin on pages below all that the tile sees: not reported)
            if (base + lane >= p.low >> a.page_shift && base + lane <= min(max(p.len - 1, 0), p.k1 - 1) >> a.page_shift) {
                set_status(a.status, kKvBadPage);
            }
            return 0;
        }
        return id;
    };
    // Hands a tile to the computing warps: its description now, its columns
    // asynchronously.  A lane arrives once for what it stored and once, by itself,
    // when its copies are there.
    int side = 0;
    uint32_t side_phase = 0;
    auto hand_over = [&](const Piece &p) {
        wait_or_abort<false>(&sm.tile_empty[side], side_phase ^ 1, &sm.halt, a.status);
        __syncwarp();
        if (lane == 0) {
            sm.piece[side] = p;
        }
        if (p.ncols > 0) {
            for (int i = lane; i < kCols * (D / 8); i += 32) {
                const int c = i / (D / 8), d = 8 * (i - c * (D / 8));
                int row, qhead;
                a.column(p, c, row, qhead);
                const bool have = c < p.ncols && row < a.rows;
                const uint16_t *src = static_cast<const uint16_t *>(a.q) + (have ? size_t(row) * a.q_stride + size_t(qhead) * D + d : 0);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(&sm.q[side][c][d ^ ((c & 7) << 3)])), "l"(src), "r"(have ? 16 : 0)
                             : "memory");
            }
            if (lane < p.ncols) {
                int row, qhead;
                a.column(p, lane, row, qhead);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc::smem_u32(&sm.row[side][lane])), "l"(a.walk.row + row) : "memory");
                if (a.slopes) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(&sm.slope[side][lane])), "l"(a.slopes + qhead) : "memory");
                }
                if (a.sinks) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(&sm.sink[side][lane])), "l"(a.sinks + qhead) : "memory");
                }
            } else if (lane < kCols) {
                sm.row[side][lane] = make_int4(0, 0, 1 << 30, -1);  // past the tile: all keys, so that it asks for no mask
                sm.slope[side][lane] = sm.sink[side][lane] = 0.0f;
            }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(tc::smem_u32(&sm.tile_full[side])) : "memory");
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(&sm.tile_full[side])) : "memory");
        side_phase ^= uint32_t(side);
        side ^= 1;
    };
    Piece p, ahead;
    bool any = walk.next(p), more = false;
    int first_ids = any ? ids(p, p.k0 >> a.page_shift) : 0;
    if (any) {
        hand_over(p);
    }
    for (; any; any = more, p = ahead) {
        int base = p.k0 >> a.page_shift, id = checked(p, base, first_ids);
        more = walk.next(ahead);
        first_ids = more ? ids(ahead, ahead.k0 >> a.page_shift) : 0;
        for (int k0 = p.k0; k0 < p.k1; k0 += kGran) {
            if (((k0 + kGran - 1) >> a.page_shift) >= base + 32) {
                base = k0 >> a.page_shift;
                id = checked(p, base, ids(p, base));
            }
            const bool free = wait_or_abort<false>(&sm.empty[stage], phase ^ 1, &sm.halt, a.status);
            if (__all_sync(0xffffffffu, free)) {
                if (lane == 0) {
                    tc::mbar_expect_tx(&sm.full[stage], kStageBytes);
                }
                __syncwarp();
                if constexpr (kCache != kMxfp4) {
                    // copy c: (segment, K or V, 64 values of the head)
                    const int copies = segs * 2 * (D / 64);
                    const int c = lane;
                    const int s = c / (2 * (D / 64)), is_v = c / (D / 64) & 1, x = c & (D / 64 - 1);
                    const int key = k0 + (c < copies ? s : 0) * seg;
                    const int page = __shfl_sync(0xffffffffu, id, (key >> a.page_shift) - base);
                    if (c < copies) {
                        const int y = ((page * a.kv_heads + p.head) * 2 + is_v) * (1 << a.page_shift) + (key & ((1 << a.page_shift) - 1));
                        tc::tma_load_2d(sm.stage[stage] + ((is_v * (D / 64) + x) * kGran + s * seg) * 128, map, 64 * x, y, &sm.full[stage]);
                    }
                } else {
                    // pages up to a granule: one copy of a head's block; larger: its four parts
                    const bool whole = (1 << a.page_shift) <= kGran;
                    const int copies = whole ? segs : 4;
                    const int c = lane;
                    const int key = k0 + (whole && c < copies ? c * seg : 0);
                    const int page = __shfl_sync(0xffffffffu, id, (key >> a.page_shift) - base);
                    if (c < copies) {
                        const uint8_t *src = a.pool + (size_t(page) * a.kv_heads + p.head) * a.block_bytes;
                        if (whole) {
                            bulk_load(sm.stage[stage] + c * a.block_bytes, src, a.block_bytes, &sm.full[stage]);
                        } else {
                            const uint32_t codes = kGran * (D / 2), scales = kGran * (D / 32);
                            const uint32_t t0 = uint32_t(key & ((1 << a.page_shift) - 1));
                            const uint32_t from = (c >> 1) * (a.block_bytes >> 1) + ((c & 1) ? 128u * (D / 2) + t0 * (D / 32) : t0 * (D / 2));
                            const uint32_t to = (c >> 1) * (codes + scales) + (c & 1) * codes;
                            bulk_load(sm.stage[stage] + to, src + from, (c & 1) ? scales : codes, &sm.full[stage]);
                        }
                    }
                }
            }
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
        if (more) {
            hand_over(ahead);  // while the last granules of this tile are worked on
        }
    }
    p.ncols = 0;
    hand_over(p);
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (sm.halt.aborted()) {
        // what is still in flight lands before the shared memory goes away
        for (int i = 0; i < kStages; ++i) {
            tc::mbar_wait(&sm.full[i], 0, 1000000ull);
            tc::mbar_wait(&sm.full[i], 1, 1000000ull);
        }
    }
}

// Columns whose sums are not finite, after the CTA's last tile: found by what was
// left of them, computed again, and the parts held back are counted.  (In the loop
// over the tiles this would hold registers that the loop over the keys needs: 64
// tokens over 4 bits 4 us more.)
template <int kRows, int kCache, int D, int NT>
__device__ __forceinline__ void redo_pieces(const AttendArgs &a, TokenSmem<kRows, kCache, D, NT> &sm) {
    using T = TokenShape<kRows, kCache, D, NT>;
    constexpr int kPer = D / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Walker walk(a.walk, int(blockIdx.x), T::kGran);
    Piece p;
    while (walk.next(p)) {
        const bool whole = p.first == p.last;
        if (!whole && !sm.held[p.first == int(blockIdx.x)]) {
            continue;
        }
        float *part = whole ? nullptr : own_part<D, T::kCols>(a, p);
        for (int c = warp; c < p.ncols; c += kWarps) {
            int row, qhead;
            a.column(p, c, row, qhead);
            if (row >= a.rows || a.walk.row[row].w != p.seq) {
                continue;  // nobody stores it
            }
            bool bad = false;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int d = lane + 32 * i;
                const float x = whole ? row_value<kRows>(a.out, size_t(row) * a.out_stride + size_t(qhead) * D + d)
                                      : part[size_t(c) * part_pitch(D) + d];
                bad = bad || !(fabsf(x) < INFINITY);
            }
            bad = bad || (!whole && !(part[size_t(c) * part_pitch(D) + D + 1] < INFINITY));
            if (__any_sync(0xffffffffu, bad)) {
                redo_column<kRows, kCache, D, false>(a, p, c, part);
            }
        }
        if (!whole && arrive_last(a, p, &sm.last, consumer_sync)) {
            merge_tile<kRows, D, T::kMergeBatch>(a, p, warp, kWarps, T::kCols);
        }
    }
}

template <int kRows, int kCache, int D, int NT>
__global__ void __launch_bounds__(kThreads, kCache == kMxfp4 && NT == 1 && D == 64 ? 3 : 2)
    kv_attend_tokens_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap map) {
    using T = TokenShape<kRows, kCache, D, NT>;
    using Smem = TokenSmem<kRows, kCache, D, NT>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    constexpr int kCols = T::kCols;
    constexpr int kBlocks = D / 32, kSub = T::kSub;
    constexpr int kMma = kCache == kMxfp4 ? kF16 : kRows;
    constexpr int kMTiles = D / 16;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Plan &plan = *a.walk.plan;
    if (tid == 0) {
        for (int i = 0; i < T::kStages; ++i) {
            tc::mbar_init(&sm.full[i], 1);
            tc::mbar_init(&sm.empty[i], kWarps);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&sm.tile_full[i], 64);
            tc::mbar_init(&sm.tile_empty[i], kWarps);
        }
        sm.halt = Halt{0, 0};
        sm.again = sm.held[0] = sm.held[1] = 0;
        tc::fence_mbar_init();
    }
    __syncthreads();
    wait_previous();
    if (!plan_fits(a, kCols, T::kGran)) {
        return;
    }
    if (warp == kWarps) {
        load_granules<Smem, kCache, D, kCols, T::kGran, T::kStages, T::kStageBytes>(a, plan, &map, sm);
        return;
    }
    const int g = lane >> 2, t = lane & 3;
    const float cap_log2 = a.cap * kLog2e;
    const float two_over_cap = a.cap != 0.0f ? 2.0f / a.cap : 0.0f;
    // 4 bits: keys and bytes of a copied part
    const int seg_shift = min(a.page_shift, T::kGran == 64 ? 6 : 7), seg = 1 << seg_shift;
    const uint32_t block = 2u * uint32_t(seg) * row_bytes(kMxfp4, D);
    // largest weight 2^(kSlack + kLift), times 2^kScaleSlack over a 4-bit cache: 2^15 in f16
    constexpr float kSlack = kMma == kF16 ? 4.0f : 8.0f;
    constexpr int kScaleSlack = 2;
    constexpr float kLift = kMma != kF16 ? 0.0f : (kCache == kMxfp4 ? 9.0f : 11.0f);
    int stage = 0;
    uint32_t phase = 0;
    uint32_t side_phase = 0;
    for (int side = 0;; side ^= 1) {
        const bool ok = wait_or_abort<false>(&sm.tile_full[side], side_phase, &sm.halt, a.status);
        side_phase ^= uint32_t(side);
        // all warps go on with the tile, or none
        if (consumers_any(!ok || sm.piece[side].ncols == 0)) {
            break;
        }
        const Piece &p = sm.piece[side];
        uint32_t q[NT][D / 16][2];
        float scale[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int c = 8 * n + g;
            const uint16_t *src = sm.q[side][c];
            if constexpr (kCache != kMxfp4) {
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    q[n][s][0] = *reinterpret_cast<const uint32_t *>(src + T::q_at(c, 16 * s) + 2 * t);
                    q[n][s][1] = *reinterpret_cast<const uint32_t *>(src + T::q_at(c, 16 * s + 8) + 2 * t);
                }
            } else {
                // values 8t .. 8t + 7 of each block of 32, as the codes' words lie
                uint4 w[kBlocks];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    w[b] = *reinterpret_cast<const uint4 *>(src + T::q_at(c, 32 * b + 8 * t));
                }
                float unscale = 1.0f;
                if constexpr (kRows == kBf16) {
                    // bf16 -> f16 by a power of two per column: exact down to 2^-39 of its largest value
                    uint32_t top = 0;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        const uint32_t u[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            top = max(top, max(u[j] & 0x7fffu, (u[j] >> 16) & 0x7fffu));
                        }
                    }
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = int(top >> 7);  // biased exponent of the largest value
                    // to [2^14, 2^15); infinities and NaN as they are
                    const int up = e == 255 ? 0 : min(14 - (e - 127), 120);
                    const float f = __uint_as_float(uint32_t(127 + max(up, -120)) << 23);
                    unscale = __uint_as_float(uint32_t(127 - max(up, -120)) << 23);
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        uint32_t u[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            u[j] = pack2<kF16>(__uint_as_float(u[j] << 16) * f, __uint_as_float(u[j] & 0xffff0000u) * f);
                        }
                        w[b] = make_uint4(u[0], u[1], u[2], u[3]);
                    }
                }
                // the column's factor, from the lane that holds it to those that hold its scores
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    scale[n][j] = __shfl_sync(0xffffffffu, a.scale * kLog2e * unscale, 4 * (2 * t + j));
                }
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    q[n][2 * b][0] = w[b].x, q[n][2 * b][1] = w[b].y;
                    q[n][2 * b + 1][0] = w[b].z, q[n][2 * b + 1][1] = w[b].w;
                }
            }
        }
        // lowest and highest borders over the columns
        int lo_min, lo_max, hi_min, hi_max;
        {
            const int4 ri = sm.row[side][min(lane, kCols - 1)];
            const int l = max(ri.y, 0), h = min(ri.z, p.len);
            const bool real = lane < p.ncols;
            lo_max = __reduce_max_sync(0xffffffffu, real ? l : 0);
            hi_min = __reduce_min_sync(0xffffffffu, real ? h : 1 << 30);
            lo_min = __reduce_min_sync(0xffffffffu, real && l < h ? l : 1 << 30);
            hi_max = __reduce_max_sync(0xffffffffu, real && l < h ? h : 0);
        }
        float m[NT][2], l[NT][2];
        float o[NT][kMTiles][4];
        // 4 bits: 1 / the scale that o is in units of; 0 until the column sees a key, so
        // that the scales of unseen keys make 0 with it, however large
        float unit[kCache == kMxfp4 ? NT : 1][2][kBlocks];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                scale[n][c] = kCache == kMxfp4 ? scale[n][c] : a.scale * kLog2e;
                m[n][c] = -INFINITY, l[n][c] = 0.0f;
                if constexpr (kCache == kMxfp4) {
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        unit[n][c][b] = 0.0f;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kMTiles; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[n][i][j] = 0.0f;
                }
            }
        }
        const int end = p.k1;
        for (int k0 = p.k0; k0 < end; k0 += T::kGran) {
            wait_or_abort<false>(&sm.full[stage], phase, &sm.halt, a.status);
            const int key0 = k0 + 16 * kSub * warp;
            if (key0 < hi_max && key0 + 16 * kSub > lo_min) {
                const uint32_t buf = tc::smem_u32(sm.stage[stage]);
                if constexpr (kCache != kMxfp4) {
                    if (key0 + 16 > hi_max) {  // the warp's own rows behind all that the tile sees
                        const int first = hi_max - key0;
#pragma unroll 1
                        for (int x = 0; x < D / 64; ++x) {
                            clear_rows(buf + ((D / 64 + x) * T::kGran + 16 * warp + first) * 128, 16 - first);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                }
                float s[kSub][NT][4];
                float sv[kSub][2][kBlocks];  // 4 bits: V's scales of keys g, g + 8
                uint32_t vcodes[kSub];
                float sv_max[kBlocks];
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    const int at = 16 * (kSub * warp + u);  // first key in the granule
                    if constexpr (kCache != kMxfp4) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                s[u][n][j] = 0.0f;
                            }
                        }
                        const int row = at + (lane & 15);
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            uint32_t ka[4];
                            const int chunk = (2 * ks + (lane >> 4)) & 7, x = ks >> 2;
                            ldmatrix4(ka, buf + (x * T::kGran + row) * 128 + ((chunk ^ (row & 7)) << 4));
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma<kMma>(s[u][n], ka, q[n][ks][0], q[n][ks][1]);
                            }
                        }
                    } else {
                        const int in_seg = at & (seg - 1);
                        const uint32_t kc = buf + uint32_t(at >> seg_shift) * block;
                        const uint32_t ksc = kc + uint32_t(seg) * (D / 2);
                        const uint32_t vc = kc + (block >> 1), vsc = vc + uint32_t(seg) * (D / 2);
                        vcodes[u] = vc + uint32_t(in_seg) * (D / 2);
                        float sk[2][kBlocks];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t from = uint32_t(in_seg + g + 8 * h) * kBlocks;
                            uint32_t bk, bv;
                            if constexpr (kBlocks == 2) {
                                asm volatile("ld.shared.u16 %0, [%1];" : "=r"(bk) : "r"(ksc + from));
                                asm volatile("ld.shared.u16 %0, [%1];" : "=r"(bv) : "r"(vsc + from));
                            } else {
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(bk) : "r"(ksc + from));
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(bv) : "r"(vsc + from));
                            }
                            // 2^(e - 127): the byte is the float's exponent (0: below f32's
                            // normal range, taken as 0; 255: infinity here, NaN below)
                            float nan = 0.0f;
#pragma unroll
                            for (int b = 0; b < kBlocks; ++b) {
                                sk[h][b] = __uint_as_float(((bk >> (8 * b)) & 255u) << 23);
                                sv[u][h][b] = __uint_as_float(((bv >> (8 * b)) & 255u) << 23);
                                nan += sk[h][b] - sk[h][b];
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                s[u][n][2 * h] = s[u][n][2 * h + 1] = nan;
                            }
                        }
#pragma unroll
                        for (int b = 0; b < kBlocks; ++b) {
                            const float top = fmaxf(sv[u][0][b], sv[u][1][b]);
                            sv_max[b] = u == 0 ? top : fmaxf(sv_max[b], top);
                            uint32_t w0, w1, a0[4], a1[4];
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0) : "r"(kc + uint32_t(in_seg + g) * (D / 2) + 16 * b + 4 * t));
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1) : "r"(kc + uint32_t(in_seg + g + 8) * (D / 2) + 16 * b + 4 * t));
                            halves8(w0, a0[0], a0[2], a1[0], a1[2]);
                            halves8(w1, a0[1], a0[3], a1[1], a1[3]);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma<kMma>(c, a0, q[n][2 * b][0], q[n][2 * b][1]);
                                mma<kMma>(c, a1, q[n][2 * b + 1][0], q[n][2 * b + 1][1]);
                                s[u][n][0] = fmaf(c[0], sk[0][b], s[u][n][0]);
                                s[u][n][1] = fmaf(c[1], sk[0][b], s[u][n][1]);
                                s[u][n][2] = fmaf(c[2], sk[1][b], s[u][n][2]);
                                s[u][n][3] = fmaf(c[3], sk[1][b], s[u][n][3]);
                            }
                        }
                    }
                }
                // ---- scores in log2 units ----
                const bool masked = key0 < lo_max || key0 + 16 * kSub > hi_min;
                if (cap_log2 == 0.0f && !a.slopes) {
#pragma unroll
                    for (int u = 0; u < kSub; ++u) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                s[u][n][j] *= scale[n][j & 1];
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < kSub; ++u) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int c = 8 * n + 2 * t + (j & 1), key = key0 + 16 * u + g + (j >> 1) * 8;
                                const float f = scale[n][j & 1];
                                const float x = cap_log2 != 0.0f ? capped(s[u][n][j], f * two_over_cap, cap_log2) : s[u][n][j] * f;
                                s[u][n][j] = a.slopes ? fmaf(-kLog2e * sm.slope[side][c], float(abs(sm.row[side][c].x - key)), x) : x;
                            }
                        }
                    }
                }
                if (masked) {
#pragma unroll
                    for (int u = 0; u < kSub; ++u) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int c = 8 * n + 2 * t + (j & 1), key = key0 + 16 * u + g + (j >> 1) * 8;
                                const int4 ri = sm.row[side][c];
                                s[u][n][j] = key >= ri.y && key < ri.z ? s[u][n][j] : -INFINITY;
                            }
                        }
                        if constexpr (kCache == kMxfp4) {  // behind all that the tile sees: any scale, NaN too
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
#pragma unroll
                                for (int b = 0; b < kBlocks; ++b) {
                                    sv[u][h][b] = key0 + 16 * u + g + 8 * h < hi_max ? sv[u][h][b] : 0.0f;
                                }
                            }
                        }
                    }
                }
                // ---- the running maximum ----
                bool move = false;
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        top[n][c] = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
                        for (int u = 1; u < kSub; ++u) {
                            top[n][c] = fmaxf(top[n][c], fmaxf(s[u][n][c], s[u][n][c + 2]));
                        }
                        move = move || top[n][c] > m[n][c] + (kSlack + kLift);
                        if constexpr (kCache == kMxfp4) {
#pragma unroll
                            for (int b = 0; b < kBlocks; ++b) {
                                // unseen keys may ask for nothing; the scale moves by seen ones below
                                move = move || sv_max[b] * unit[n][c][b] > float(1 << kScaleSlack);
                            }
                        }
                    }
                }
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float up[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float most = top[n][c];
#pragma unroll
                            for (int off = 4; off < 32; off <<= 1) {
                                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                            }
                            // m is what weights are relative to: the maximum less the lift
                            const float mn = fmaxf(m[n][c], most - kLift);
                            up[c] = ex2(m[n][c] - (mn == -INFINITY ? 0.0f : mn));
                            m[n][c] = mn;
                            l[n][c] *= up[c];
                        }
                        if constexpr (kCache == kMxfp4) {
#pragma unroll
                            for (int b = 0; b < kBlocks; ++b) {
                                float f[2];
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    // the largest finite scale of a seen key
                                    float e = 0.0f;
#pragma unroll
                                    for (int u = 0; u < kSub; ++u) {
#pragma unroll
                                        for (int h = 0; h < 2; ++h) {
                                            e = s[u][n][c + 2 * h] != -INFINITY && sv[u][h][b] < INFINITY ? fmaxf(e, sv[u][h][b]) : e;
                                        }
                                    }
#pragma unroll
                                    for (int off = 4; off < 32; off <<= 1) {
                                        e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, off));
                                    }
                                    // the unit's reciprocal: 2^(254 - byte) as a float's exponent; a byte
                                    // that a finite value has is at most 252
                                    const float r = __uint_as_float(0x7f000000u - max(__float_as_uint(e), 0x00800000u));
                                    const bool begun = unit[n][c][b] != 0.0f;
                                    const float less = begun ? fminf(unit[n][c][b], r) : r;
                                    f[c] = up[c] * (!begun || less == unit[n][c][b] ? 1.0f : pow2i(int(__float_as_uint(less) >> 23) - int(__float_as_uint(unit[n][c][b]) >> 23)));
                                    unit[n][c][b] = m[n][c] == -INFINITY ? 0.0f : less;
                                }
#pragma unroll
                                for (int i = 2 * b; i < 2 * b + 2; ++i) {
                                    o[n][i][0] *= f[0], o[n][i][1] *= f[1], o[n][i][2] *= f[0], o[n][i][3] *= f[1];
                                }
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < kMTiles; ++i) {
                                o[n][i][0] *= up[0], o[n][i][1] *= up[1], o[n][i][2] *= up[0], o[n][i][3] *= up[1];
                            }
                        }
                    }
                }
                // ---- weights, and their products with V ----
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float mm = m[n][c] == -INFINITY ? 0.0f : m[n][c];
#pragma unroll
                        for (int u = 0; u < kSub; ++u) {
                            s[u][n][c] = ex2(s[u][n][c] - mm);
                            s[u][n][c + 2] = ex2(s[u][n][c + 2] - mm);
                            l[n][c] += s[u][n][c] + s[u][n][c + 2];
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    if constexpr (kCache != kMxfp4) {
                        uint32_t w[NT][2];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            w[n][0] = transpose8(pack2<kMma>(s[u][n][0], s[u][n][1]));
                            w[n][1] = transpose8(pack2<kMma>(s[u][n][2], s[u][n][3]));
                        }
                        const uint32_t vbuf = buf + (D / 64) * T::kGran * 128;
                        const int row = 16 * (kSub * warp + u) + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                        for (int i = 0; i < kMTiles; ++i) {
                            uint32_t va[4];
                            const int chunk = (2 * i + ((lane >> 3) & 1)) & 7, x = i >> 2;
                            ldmatrix4_trans(va, vbuf + (x * T::kGran + row) * 128 + ((chunk ^ (row & 7)) << 4));
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma<kMma>(o[n][i], va, w[n][0], w[n][1]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < kBlocks; ++b) {
                            // 8 x 8 b16 of 4 codes each: keys 0-7 and 8-15, the block's 32 values
                            uint32_t r0, r1, va0[4], va1[4];
                            ldmatrix2_trans(r0, r1, vcodes[u] + uint32_t(lane & 15) * (D / 2) + 16 * b);
                            // r: codes 4g .. 4g + 3 of key 2t (low half) and of key 2t + 1, to
                            // bytes of a value's two keys: rows 0-7 of a tile are values 4g + 2i,
                            // rows 8-15 values 4g + 2i + 1
                            const uint32_t x0 = (r0 & 0x0F0Fu) | ((r0 >> 12) & 0xF0F0u), y0 = ((r0 >> 4) & 0x0F0Fu) | ((r0 >> 16) & 0xF0F0u);
                            const uint32_t x1 = (r1 & 0x0F0Fu) | ((r1 >> 12) & 0xF0F0u), y1 = ((r1 >> 4) & 0x0F0Fu) | ((r1 >> 16) & 0xF0F0u);
                            halves8(x0 | y0 << 16, va0[0], va1[0], va0[1], va1[1]);
                            halves8(x1 | y1 << 16, va0[2], va1[2], va0[3], va1[3]);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                // the scale over the unit: at most 2^kScaleSlack where the key is seen
                                // (a NaN scale makes infinity or NaN here, and the column is computed again)
                                const float f0 = sv[u][0][b] * unit[n][0][b], f1 = sv[u][0][b] * unit[n][1][b];
                                const float f2 = sv[u][1][b] * unit[n][0][b], f3 = sv[u][1][b] * unit[n][1][b];
                                const uint32_t w0 = transpose8(pack2<kF16>(s[u][n][0] * f0, s[u][n][1] * f1));
                                const uint32_t w1 = transpose8(pack2<kF16>(s[u][n][2] * f2, s[u][n][3] * f3));
                                mma<kF16>(o[n][2 * b], va0, w0, w1);
                                mma<kF16>(o[n][2 * b + 1], va1, w0, w1);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) {
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(&sm.empty[stage])) : "memory");
            }
            if (++stage == T::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
        // ---- the four warps' results ----
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
                }
                if (g == 0) {
                    sm.m[warp][8 * n + 2 * t + c] = m[n][c];
                    sm.l[warp][8 * n + 2 * t + c] = l[n][c];
                }
            }
#pragma unroll
            for (int i = 0; i < kMTiles; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 8 * n + 2 * t + (j & 1);
                    if constexpr (kCache == kMxfp4) {
                        const int d = 32 * (i >> 1) + 4 * g + 2 * (i & 1) + (j >> 1);
                        sm.o[warp][c][d] = o[n][i][j] * __uint_as_float(0x7f000000u - __float_as_uint(unit[n][j & 1][i >> 1]));
                    } else {
                        sm.o[warp][c][T::o_at(c, 16 * i + g + 8 * (j >> 1))] = o[n][i][j];
                    }
                }
            }
        }
        consumer_sync();
        auto top = [&](int c) {
            return fmaxf(fmaxf(sm.m[0][c], sm.m[1][c]), fmaxf(sm.m[2][c], sm.m[3][c]));
        };
        auto stats = [&](int c) {
            const float mm = top(c), safe = mm == -INFINITY ? 0.0f : mm;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                sum = fmaf(sm.l[w][c], ex2(sm.m[w][c] - safe), sum);
            }
            return make_float2(mm, sum);
        };
        auto value = [&](int c, int d, float(&v)[8]) {
            const float mm = top(c), safe = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = 0.0f;
            }
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(sm.m[w][c] - safe);
                const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][c][T::o_at(c, d)]);
                const float4 y = *reinterpret_cast<const float4 *>(&sm.o[w][c][T::o_at(c, d + 4)]);
                v[0] = fmaf(x.x, f, v[0]), v[1] = fmaf(x.y, f, v[1]), v[2] = fmaf(x.z, f, v[2]), v[3] = fmaf(x.w, f, v[3]);
                v[4] = fmaf(y.x, f, v[4]), v[5] = fmaf(y.y, f, v[5]), v[6] = fmaf(y.z, f, v[6]), v[7] = fmaf(y.w, f, v[7]);
            }
        };
        if (p.first == p.last) {
            const bool bad = store_columns<kRows, D>(a, p, warp, kWarps, value, stats, [&](int c, int, int) {
                const int4 ri = sm.row[side][c];
                return ColumnInfo{ri.y, ri.z, ri.w, sm.sink[side][c]};
            });
            if (bad) {
                sm.again = 1;
            }
        } else {
            float *part = own_part<D, kCols>(a, p);
            bool bad = false;
            for (int i = tid; i < p.ncols * (D / 8); i += 32 * kWarps) {
                const int c = i / (D / 8), d = 8 * (i % (D / 8));
                float v[8];
                value(c, d, v);
                float4 *dst = reinterpret_cast<float4 *>(part + size_t(c) * part_pitch(D) + d);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    bad = bad || !(fabsf(v[j]) < INFINITY);
                }
                if (d == 0) {
                    const float2 ml = stats(c);
                    *reinterpret_cast<float2 *>(part + size_t(c) * part_pitch(D) + D) = ml;
                    bad = bad || !(ml.y < INFINITY);
                }
            }
            int &held = sm.held[p.first == int(blockIdx.x)];
            if (bad) {
                sm.again = held = 1;
            }
            if (arrive_last(a, p, &sm.last, consumer_sync, [&] { return held != 0; })) {
                merge_tile<kRows, D, T::kMergeBatch>(a, p, warp, kWarps, kCols);
            }
        }
        __syncwarp();
        if (lane == 0) {
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(&sm.tile_empty[side])) : "memory");
        }
    }
    consumer_sync();
    if (sm.again && !sm.halt.aborted()) {
        redo_pieces<kRows, kCache, D, NT>(a, sm);
    }
}

template <int kRows, int kCache, int D, int NT> cudaError_t launch_nt(const ttl_kv &h, const AttendArgs &a, int layer) {
    return launch_chained(kv_attend_tokens_kernel<kRows, kCache, D, NT>, h.ctas[0], kThreads,
                          sizeof(TokenSmem<kRows, kCache, D, NT>), h.stream, a, h.maps[size_t(layer)]);
}

template <int kRows, int kCache, int D> cudaError_t launch(const ttl_kv &h, const AttendArgs &a, int layer) {
    if constexpr (kRows == kF32) {
        return cudaErrorInvalidValue;
    } else {
        if (h.width[0] == 8) {
            return launch_nt<kRows, kCache, D, 1>(h, a, layer);
        }
        if (h.width[0] == 16) {
            return launch_nt<kRows, kCache, D, 2>(h, a, layer);
        }
        if constexpr (D == 64) {
            return launch_nt<kRows, kCache, D, 4>(h, a, layer);
        }
        return cudaErrorInvalidValue;
    }
}

template <int kRows, int kCache, int D, int NT> cudaError_t configure_nt(ttl_kv &h, int i) {
    const int bytes = int(sizeof(TokenSmem<kRows, kCache, D, NT>));
    cudaError_t e = cudaFuncSetAttribute(kv_attend_tokens_kernel<kRows, kCache, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    int n = 0;
    e = e ? e : cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv_attend_tokens_kernel<kRows, kCache, D, NT>, kThreads, size_t(bytes));
    h.token_ctas[i] = std::min(std::max(n, 1) * h.sms, kMaxCtas);
    return e;
}

template <int kRows, int kCache, int D> cudaError_t configure(ttl_kv &h) {
    if constexpr (kRows == kF32) {
        return cudaSuccess;
    } else {
        cudaError_t e = configure_nt<kRows, kCache, D, 1>(h, 0);
        e = e ? e : configure_nt<kRows, kCache, D, 2>(h, 1);
        if constexpr (D == 64) {
            e = e ? e : configure_nt<kRows, kCache, D, 4>(h, 2);
        }
        return e;
    }
}

}  // namespace

cudaError_t tokens_configure(ttl_kv &h) {
    return TTL_KV_DISPATCH(&h, configure, h);
}

cudaError_t launch_tokens(const ttl_kv &h, const AttendArgs &a, int layer) {
    return TTL_KV_DISPATCH(&h, launch, h, a, layer);
}

}  // namespace kv
}  // namespace ttl

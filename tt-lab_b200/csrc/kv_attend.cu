// kv_attend.cu -- attention over the paged cache (ttl_kv_attend_async): the
// choice of kernels, and the kernel that computes in 32-bit arithmetic.
//
// Reference: attention_from_cache of tt-lab (src/model.cpp:255-290), there for
// one token over a contiguous f32 cache.
#include <cuda_runtime.h>

#include <algorithm>

#include "kv.cuh"
#include "kv_internal.h"

namespace ttl {
namespace kv {

namespace {

// ---- 32-bit arithmetic ----
// o = sum_j p_j v_j / sum_j p_j with p_j = exp(score_j), one pass over the
// keys with a running maximum and sum per column.  A CTA holds a tile of CT
// columns; per granule of 64 keys it stages K and V as f32 in shared memory,
// computes the CT x 64 scores (a thread: one key, CT / 4 columns), turns them
// into weights (a warp: a column at a time) and adds the weighted values (a
// thread: four values of CT * D / 1024 columns).  For f32 rows alone, whose
// products the tensor cores would round.  A single token bounds it by latency:
// 64 query and 8 KV heads over 1040 keys (4.3 MB) 19.8 us with the plan; prompts by
// the 32-bit multiply-adds, fed from shared memory, with five barriers per granule:
// 1024 rows 578 us, 15 TFLOP/s.  64 tokens over 4096 keys in 4 bits 729 us, where
// bf16 rows take 57: a byte is loaded for every code and another for its scale.
constexpr int kSimpleThreads = 256;
constexpr int kSimpleGran = 64;

template <int CT, int D> struct SimpleSmem {
    static constexpr int kKPitch = D + 4;  // rows 16 bytes apart modulo 128: a warp's 16-byte loads of 32 rows do not collide
    static constexpr int kSPitch = kSimpleGran + 4;
    float k[kSimpleGran * kKPitch];
    float v[kSimpleGran * D];
    float q[CT * D];
    float s[CT * kSPitch];
    float m[CT], l[CT], up[CT];
    int lo[CT], hi[CT], pos[CT];
    float slope[CT];
    int pages[kSimpleGran / 16];
    int last;
};

template <int kRows, int kCache, int D, int CT>
__global__ void __launch_bounds__(kSimpleThreads) kv_attend_simple_kernel(AttendArgs a) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    using Smem = SimpleSmem<CT, D>;
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Plan &plan = *a.walk.plan;
    wait_previous();
    if (!plan_fits(a, CT, kSimpleGran)) {
        return;
    }
    constexpr int kD4 = D / 4;
    constexpr int kGroups = kSimpleThreads / kD4;                // groups of threads that each cover D
    constexpr int kKeySplit = kGroups > CT ? kGroups / CT : 1;   // groups that share a column's keys
    constexpr int kCols = CT > kGroups ? CT / kGroups : 1;       // columns of a thread
    const int d4 = tid % kD4, grp = tid / kD4;
    const int col0 = (grp / kKeySplit) * kCols, half = grp % kKeySplit;
    const int tokens = 1 << a.page_shift;
    const float scale_log2 = a.scale * kLog2e;
    Walker walk(a.walk, int(blockIdx.x), kSimpleGran);
    Piece p;
    while (walk.next(p)) {
        for (int i = tid; i < CT * (D / 8); i += kSimpleThreads) {
            const int c = i / (D / 8), d = 8 * (i % (D / 8));
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (c < p.ncols) {
                int row, qhead;
                a.column(p, c, row, qhead);
                if (row < a.rows) {
                    load8<kRows>(a.q, size_t(row) * a.q_stride + size_t(qhead) * D + d, x);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sm.q[c * D + d + j] = x[j];
            }
        }
        for (int c = tid; c < CT; c += kSimpleThreads) {
            int4 ri = make_int4(0, 0, 0, -1);
            float slope = 0.0f;
            if (c < p.ncols) {
                int row, qhead;
                a.column(p, c, row, qhead);
                ri = a.walk.row[row];
                slope = a.slopes ? a.slopes[qhead] * kLog2e : 0.0f;
            }
            sm.pos[c] = ri.x, sm.lo[c] = max(ri.y, 0), sm.hi[c] = min(ri.z, p.len);
            sm.slope[c] = slope;
            sm.m[c] = -INFINITY, sm.l[c] = 0.0f;
        }
        float o[kCols][4] = {};
        for (int k0 = p.k0; k0 < p.k1; k0 += kSimpleGran) {
            const int keys = min(kSimpleGran, p.len - k0);  // <= 0: a tile that sees nothing
            __syncthreads();
            if (tid < kSimpleGran / 16) {
                const int j = k0 + 16 * tid;
                sm.pages[tid] = j < p.len ? page_of(plan, p.seq, j, p.low, a.page_shift, a.pages, a.status) : 0;
            }
            __syncthreads();
            if constexpr (kCache != kMxfp4) {
                for (int i = tid; i < 2 * kSimpleGran * (D / 8); i += kSimpleThreads) {
                    const int t = (i / (D / 8)) % kSimpleGran, d = 8 * (i % (D / 8));
                    const bool is_v = i >= kSimpleGran * (D / 8);
                    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (t < keys) {
                        const uint8_t *b = a.pool + (size_t(sm.pages[t / 16]) * a.kv_heads + p.head) * a.block_bytes +
                                           (is_v ? a.block_bytes >> 1 : 0);
                        load8<kCache>(b, size_t((k0 + t) & (tokens - 1)) * D + d, x);
                    }
                    float *dst = is_v ? &sm.v[t * D + d] : &sm.k[t * Smem::kKPitch + d];
                    *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                    *reinterpret_cast<float4 *>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
                }
            } else {
                for (int i = tid; i < 2 * kSimpleGran * (D / 8); i += kSimpleThreads) {
                    const int t = (i / (D / 8)) % kSimpleGran, d = 8 * (i % (D / 8));
                    const bool is_v = i >= kSimpleGran * (D / 8);
                    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (t < keys) {
                        const uint8_t *b = a.pool + (size_t(sm.pages[t / 16]) * a.kv_heads + p.head) * a.block_bytes +
                                           (is_v ? a.block_bytes >> 1 : 0);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            x[j] = pool_value<kCache, D>(b, tokens, (k0 + t) & (tokens - 1), d + j);
                        }
                    }
                    float *dst = is_v ? &sm.v[t * D + d] : &sm.k[t * Smem::kKPitch + d];
                    *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                    *reinterpret_cast<float4 *>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
                }
            }
            __syncthreads();
            {
                const int key = tid & (kSimpleGran - 1), cg = tid / kSimpleGran;
                constexpr int kPer = CT / 4;
                float acc[kPer] = {};
                for (int d = 0; d < D; d += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(&sm.k[key * Smem::kKPitch + d]);
#pragma unroll
                    for (int c = 0; c < kPer; ++c) {
                        const float4 y = *reinterpret_cast<const float4 *>(&sm.q[(cg * kPer + c) * D + d]);
                        acc[c] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, acc[c]))));
                    }
                }
#pragma unroll
                for (int c = 0; c < kPer; ++c) {
                    const int col = cg * kPer + c, j = k0 + key;
                    const bool sees = j >= sm.lo[col] && j < sm.hi[col];
                    const float t = a.cap != 0.0f ? a.cap * tanhf(acc[c] * a.scale / a.cap) * kLog2e : acc[c] * scale_log2;
                    // -1 in the sign of a weight marks an unseen key below
                    sm.s[col * Smem::kSPitch + key] = sees ? t - sm.slope[col] * float(abs(sm.pos[col] - j)) : __uint_as_float(0xffc00001u);
                }
            }
            __syncthreads();
            for (int c = warp; c < CT; c += kSimpleThreads / 32) {
                float *s = &sm.s[c * Smem::kSPitch];
                const float x0 = s[lane], x1 = s[lane + 32];
                const bool see0 = __float_as_uint(x0) != 0xffc00001u, see1 = __float_as_uint(x1) != 0xffc00001u;
                float top = fmaxf(see0 ? x0 : -INFINITY, see1 ? x1 : -INFINITY);
#pragma unroll
                for (int off = 16; off; off >>= 1) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                }
                const float m = sm.m[c], mn = fmaxf(m, top);
                const float safe = mn == -INFINITY ? 0.0f : mn;
                const float p0 = see0 ? exp2f(x0 - safe) : -1.0f, p1 = see1 ? exp2f(x1 - safe) : -1.0f;
                const float sum = warp_sum((see0 ? p0 : 0.0f) + (see1 ? p1 : 0.0f));
                const float up = exp2f(m - safe);
                __syncwarp();
                s[lane] = p0, s[lane + 32] = p1;
                if (lane == 0) {
                    sm.m[c] = mn, sm.l[c] = sm.l[c] * up + sum, sm.up[c] = up;
                }
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                const float up = sm.up[col0 + c];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[c][j] *= up;
                }
            }
            for (int t = half; t < keys; t += kKeySplit) {
                const float4 x = *reinterpret_cast<const float4 *>(&sm.v[t * D + 4 * d4]);
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const float w = sm.s[(col0 + c) * Smem::kSPitch + t];
                    if (!(w < 0.0f)) {  // an unseen value is not touched, whatever it is
                        o[c][0] = fmaf(w, x.x, o[c][0]);
                        o[c][1] = fmaf(w, x.y, o[c][1]);
                        o[c][2] = fmaf(w, x.z, o[c][2]);
                        o[c][3] = fmaf(w, x.w, o[c][3]);
                    }
                }
            }
        }
        __syncthreads();
        // the sums of the tile's columns, in the place of K
        float *sum = sm.k;
#pragma unroll
        for (int h = 0; h < kKeySplit; ++h) {
            if (half == h) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    float4 *dst = reinterpret_cast<float4 *>(&sum[(col0 + c) * D + 4 * d4]);
                    float4 x = make_float4(o[c][0], o[c][1], o[c][2], o[c][3]);
                    if (h) {
                        const float4 y = *dst;
                        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
                    }
                    *dst = x;
                }
            }
            __syncthreads();
        }
        if (p.first == p.last) {
            store_columns<kRows, D>(
                a, p, warp, kSimpleThreads / 32,
                [&](int c, int d, float(&v)[8]) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[j] = sum[c * D + d + j];
                    }
                },
                [&](int c) { return make_float2(sm.m[c], sm.l[c]); },
                [&](int, int row, int qhead) { return column_info(a, row, qhead); });  // unseen values were not touched
        } else {
            float *part = a.part + size_t(part_slot(int(blockIdx.x), p.first)) * CT * part_pitch(D);
            for (int i = tid; i < p.ncols * part_pitch(D); i += kSimpleThreads) {
                const int c = i / part_pitch(D), d = i - c * part_pitch(D);
                part[i] = d < D ? sum[c * D + d] : (d == D ? sm.m[c] : sm.l[c]);
            }
            if (arrive_last(a, p, &sm.last, [] { __syncthreads(); })) {
                merge_tile<kRows, D, 8>(a, p, warp, kSimpleThreads / 32, CT);
            }
        }
        __syncthreads();
    }
}

template <int kRows, int kCache, int D, int CT> cudaError_t launch_simple_ct(const ttl_kv &h, const AttendArgs &a, int ctas) {
    return launch_chained(kv_attend_simple_kernel<kRows, kCache, D, CT>, ctas, kSimpleThreads, sizeof(SimpleSmem<CT, D>), h.stream, a);
}

template <int kRows, int kCache, int D> cudaError_t launch_simple(const ttl_kv &h, const AttendArgs &a) {
    if constexpr (kRows != kF32) {
        return cudaErrorInvalidValue;
    } else {
        return h.width[0] == 8 ? launch_simple_ct<kRows, kCache, D, 8>(h, a, h.ctas[0])
                           : launch_simple_ct<kRows, kCache, D, 32>(h, a, h.ctas[0]);
    }
}

template <int kRows, int kCache, int D> cudaError_t configure_simple(const ttl_kv &) {
    if constexpr (kRows != kF32) {
        return cudaErrorInvalidValue;
    } else {
    cudaError_t e = cudaFuncSetAttribute(kv_attend_simple_kernel<kRows, kCache, D, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         int(sizeof(SimpleSmem<8, D>)));
    return e ? e
             : cudaFuncSetAttribute(kv_attend_simple_kernel<kRows, kCache, D, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(sizeof(SimpleSmem<32, D>)));
    }
}

}  // namespace

namespace {

// Sequences of more columns than the widest tile of the kernel for few columns
// go to the prompt kernel: from there on that one would read the cache more
// than once.  64 sequences of 4096 keys, bf16, 8 KV heads: D = 64, 32 columns
// 129 us against the prompt kernel's 171, 64 columns 230 against 173; over 4
// bits 172 and 243, 316 and 238; D = 128, 16 columns 189 and 210, 32 columns 342
// and 212.
constexpr int few_columns(int dim) {
    return dim == 128 ? 16 : 32;
}

int token_index(int columns, int dim) {
    return columns <= 8 ? 0 : (columns <= 16 || dim == 128 ? 1 : 2);
}

}  // namespace

int choose_shapes(const ttl_kv &h, int seqs, int max_new, Shape shape[kKinds]) {
    const int group = h.q_heads / h.kv_heads, columns = max_new * group;
    shape[0] = shape[1] = Shape{kPromptWidth, 128, 2, 0};
    if (h.rows_type == kF32) {
        shape[0] = Shape{columns <= 8 ? 8 : 32, kSimpleGran, 1, 2 * h.sms};
        return 1 << 30;
    }
    const bool prompt = h.prompt_ctas > 0 && columns > few_columns(h.dim);
    if (prompt) {
        shape[1].ctas = h.prompt_ctas;
    }
    if (prompt && seqs == 1) {
        return 0;  // one launch: whatever the sequence's rows turn out to be
    }
    // Beside a prompt most sequences bring one token: a tile is as wide as that
    // (64 tokens over 8192 keys and a prompt of 512, bf16: 201 us, with tiles of
    // 32 columns 270; over 4 bits 131 and 348).
    const int i = token_index(prompt ? std::min(columns, group) : columns, h.dim);
    shape[0] = Shape{8 << i, 64 * token_sub(h.cache_type, 8 << i), 1, h.token_ctas[i]};
    return prompt ? few_columns(h.dim) : 1 << 30;
}

size_t kv_part_floats(const ttl_kv &h) {
    size_t most = h.rows_type == kF32 ? size_t(2 * h.sms) * 32 : size_t(h.prompt_ctas) * kPromptWidth;
    for (int i = 0; i < 3; ++i) {
        most = std::max(most, size_t(h.token_ctas[i]) * (8 << i));
    }
    return 2 * most * part_pitch(h.dim);
}

cudaError_t kv_configure(ttl_kv &h) {
    if (h.rows_type == kF32) {
        return TTL_KV_DISPATCH(&h, configure_simple, h);
    }
    const cudaError_t e = tokens_configure(h);
    return e ? e : prompt_configure(h);
}

cudaError_t launch_attend(const ttl_kv &h, const AttendArgs &a, int kind, int layer) {
    if (h.rows_type == kF32) {
        return TTL_KV_DISPATCH(&h, launch_simple, h, a);
    }
    return kind == 0 ? launch_tokens(h, a, layer) : launch_prompt(h, a, layer);
}

}  // namespace kv
}  // namespace ttl

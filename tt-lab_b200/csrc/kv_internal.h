// kv_internal.h -- the handle of ttl_kv and the launchers of its kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <string>
#include <utility>
#include <vector>

#include "kv.cuh"

struct ttl_kv {
    int device = 0, sms = 148;
    int layers = 0, pages = 0, page_tokens = 0, page_shift = 0, q_heads = 0, kv_heads = 0, dim = 0;
    int rows_type = 0, cache_type = 0, max_seqs = 0, max_rows = 0, window = 0, rope_dims = 0, interleaved = 0;
    double rope_scale = 1.0;
    uint32_t block_bytes = 0;      // one KV head of a page
    size_t layer_bytes = 0;
    typedef CUresult (*Attributes)(unsigned, CUpointer_attribute *, void **, CUdeviceptr);
    Attributes attributes = nullptr;  // cuPointerGetAttributes
    cudaStream_t stream = nullptr;
    bool own_stream = false;
    std::vector<void *> allocations;
    uint8_t *pool = nullptr;
    double *turns = nullptr;       // [rope_dims / 2] revolutions per position
    double2 *table = nullptr;      // cosines and sines of 129 angles (append over 4 bits)
    ttl::kv::Plan *plan = nullptr;
    ttl::kv::Tile *tiles[2][2] = {};
    int32_t *prefix[2][2] = {};
    ttl::kv::Cut *cuts[2][2] = {};
    int4 *row[2] = {};
    int tile_cap[2] = {};
    float *part = nullptr;
    uint32_t *counters = nullptr;  // [2 kinds][kMaxCtas]
    uint32_t *status = nullptr;
    std::vector<CUtensorMap> maps; // per layer: the 16-bit pool as rows of head_dim values
    int token_ctas[3] = {};        // CTAs that are resident at once, tiles of 8, 16, 32 columns
    int prompt_ctas = 0;           // 0: no prompt kernel for the handle's types
    // the last batch call
    bool batched = false;
    int seqs = 0, rows = 0;
    int width[2] = {}, ctas[2] = {};  // ctas 0: the kind is not launched
    std::string error;
};

// Calls F<rows type, cache type, head size> for the handle's types.
#define TTL_KV_DISPATCH_D(h, F, R, C, ...) ((h)->dim == 64 ? F<R, C, 64>(__VA_ARGS__) : F<R, C, 128>(__VA_ARGS__))
#define TTL_KV_DISPATCH_C(h, F, R, ...)                                          \
    ((h)->cache_type == ttl::kv::kMxfp4 ? TTL_KV_DISPATCH_D(h, F, R, ttl::kv::kMxfp4, __VA_ARGS__) \
                                        : TTL_KV_DISPATCH_D(h, F, R, R, __VA_ARGS__))
#define TTL_KV_DISPATCH(h, F, ...)                                               \
    ((h)->rows_type == ttl::kv::kF32   ? TTL_KV_DISPATCH_C(h, F, ttl::kv::kF32, __VA_ARGS__) \
     : (h)->rows_type == ttl::kv::kF16 ? TTL_KV_DISPATCH_C(h, F, ttl::kv::kF16, __VA_ARGS__) \
                                       : TTL_KV_DISPATCH_C(h, F, ttl::kv::kBf16, __VA_ARGS__))

namespace ttl {
namespace kv {

// Launches `kernel` so that it may start while its predecessor on the stream
// ends (programmatic dependent launch; see wait_previous).
template <class... Params, class... Args>
cudaError_t launch_chained(void (*kernel)(Params...), int blocks, int threads, size_t smem, cudaStream_t stream, Args &&...args) {
    cudaLaunchAttribute chained[1];
    chained[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    chained[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(blocks));
    c.blockDim = dim3(unsigned(threads));
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    c.attrs = chained;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, std::forward<Args>(args)...);
}

constexpr int kNarrow = 8;         // columns of the narrowest tile
constexpr int kPromptWidth = kPromptColumns;

// The kernel for few columns: steps of 16 keys that each of its four warps takes
// at once.  Two over a 4-bit cache (less bookkeeping per byte) where the
// registers allow it.
constexpr int token_sub(int cache, int width) {
    return cache == kMxfp4 && width == 8 ? 2 : 1;
}

// Shape of one kind's launch.
struct Shape {
    int width, gran, cost, ctas;   // columns per tile, keys per granule, granules a tile's ends cost, CTAs (0: no launch)
};

// Chooses the kernels of a batch; returns the most columns of a sequence that
// goes to kind 0.
int choose_shapes(const ttl_kv &h, int seqs, int max_new, Shape shape[kKinds]);
// Floats of the workspace that holds partial results.
size_t kv_part_floats(const ttl_kv &h);
// Sets the kernels' attributes once per handle.
cudaError_t kv_configure(ttl_kv &h);
cudaError_t tokens_configure(ttl_kv &h);
cudaError_t launch_tokens(const ttl_kv &h, const AttendArgs &a, int layer);
cudaError_t prompt_configure(ttl_kv &h);
cudaError_t launch_prompt(const ttl_kv &h, const AttendArgs &a, int layer);
cudaError_t launch_attend(const ttl_kv &h, const AttendArgs &a, int kind, int layer);

}  // namespace kv
}  // namespace ttl

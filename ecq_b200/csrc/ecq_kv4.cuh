// ecq_kv4.cuh -- the layout of the 4-bit KV cache's pool (ecq_kv4.h) and the
// checks that its entry points share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ecq_kernels.cuh"
#include "ecq_kv4.h"

namespace ecq_kv4 {

constexpr int kBlockTokens = 16;

__host__ __device__ constexpr int block_bytes(int dim, int groups) { return 16 * dim + 128 * groups; }
__host__ __device__ constexpr int v_codes_at(int dim) { return 8 * dim; }
__host__ __device__ constexpr int k_params_at(int dim) { return 16 * dim; }
__host__ __device__ constexpr int v_params_at(int dim, int groups) { return 16 * dim + 64 * groups; }

inline bool sizes_ok(int head_dim, int page_size, int group_size) {
    if (head_dim != 64 && head_dim != 128) return false;
    if (group_size != 32 && group_size != 64 && group_size != 128) return false;
    if (group_size > head_dim) return false;
    return page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0;
}
inline int log2i(int v) {
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}
inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) == 0; }

// f(Layout<element, head_dim, groups per row>) for a call that sizes_ok and
// the dtype check let through
template <typename T_, int D_, int G_>
struct Layout {
    using T = T_;
    static constexpr int D = D_, G = G_;
};
template <typename F>
int32_t by_layout(int dtype, int dim, int groups, F&& f) {
    const bool h = dtype == ECQ_KV4_F16;
    using B = __nv_bfloat16;
    if (dim == 64) {
        if (groups == 1) return h ? f(Layout<__half, 64, 1>{}) : f(Layout<B, 64, 1>{});
        return h ? f(Layout<__half, 64, 2>{}) : f(Layout<B, 64, 2>{});
    }
    if (groups == 1) return h ? f(Layout<__half, 128, 1>{}) : f(Layout<B, 128, 1>{});
    if (groups == 2) return h ? f(Layout<__half, 128, 2>{}) : f(Layout<B, 128, 2>{});
    return h ? f(Layout<__half, 128, 4>{}) : f(Layout<B, 128, 4>{});
}

inline bool pool_ok(const void* pages, int64_t n_pages, int kv_heads, int page_size) {
    return pages && aligned(pages, 16) && n_pages >= 1 && kv_heads >= 1 && kv_heads <= 65535 && n_pages <= ((1ll << 31) - 1) / page_size;
}
inline int32_t result(cudaError_t rc) { return rc == cudaSuccess ? ECQ_OK : (cudaGetLastError(), ECQ_ERR_CUDA); }

__device__ __forceinline__ void raise_status(int32_t* status, uint32_t bits) {
    if (status) atomicOr(reinterpret_cast<unsigned int*>(status), bits);
}

}  // namespace ecq_kv4

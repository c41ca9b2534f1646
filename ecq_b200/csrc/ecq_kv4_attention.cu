// ecq_kv4_attention.cu -- attention over the 4-bit KV cache. One CTA per query
// token and head; its warps take every 4th key, each with a running maximum
// and sum, and are joined in shared memory.
#include <cuda_runtime.h>

#include "ecq_kv4.cuh"

namespace {

using namespace ecq_kv4;
using ecq_dev::launch_pdl;
using ecq_dev::pdl_launch_dependents;
using ecq_dev::pdl_wait;

constexpr int kWarps = 4;

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <typename T, int D, int G>
__global__ void __launch_bounds__(kWarps * 32) attention_kernel(
    const T* __restrict__ q, int64_t q_token, int64_t q_head, T* __restrict__ out, int64_t o_token, int64_t o_head,
    const uint8_t* __restrict__ pages, int64_t n_pages, int kv_heads, int share, int page_shift,
    const int32_t* __restrict__ table, int64_t table_stride, int max_pages, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ starts, int batch, float scale, int32_t* status) {
    constexpr int E = D / 32;
    __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][D];
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int b = t, i = 0, n = 1;
    if (starts) {
        if (t >= starts[batch]) return;
        int lo = 0, hi = batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= t) lo = mid;
            else hi = mid;
        }
        b = lo;
        i = t - starts[b];
        n = starts[b + 1] - starts[b];
    }
    int len = lens[b];
    const long long room = static_cast<long long>(max_pages) << page_shift;
    if (len > room) {
        if (threadIdx.x == 0) raise_status(status, ECQ_STATUS_BADARG);
        len = static_cast<int>(room);
    }
    const int keys = min(len, len - n + i + 1);
    const int page_size = 1 << page_shift;
    float qv[E], m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = to_float(q[t * q_token + h * q_head + lane + 32 * e]) * scale;
        o[e] = 0.f;
    }
    for (int j = warp; j < keys; j += kWarps) {
        const int page = table[b * table_stride + (j >> page_shift)];
        if (page < 0 || page >= n_pages) {
            if (lane == 0) raise_status(status, ECQ_STATUS_BADARG);
            continue;
        }
        const int at = j & (page_size - 1), tok = at % kBlockTokens;
        const uint8_t* blk = pages + ((static_cast<int64_t>(page) * kv_heads + h / share) * (page_size / kBlockTokens) +
                                      at / kBlockTokens) * block_bytes(D, G);
        float dot = 0.f, vv[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = lane + 32 * e;
            const int nk = ((d % 32) / 8) * (D / 4) + (d / 32) * 8 + d % 8, nv = (d % 8) * (D / 8) + d / 8;
            const int ck = blk[tok * (D / 2) + nk / 2] >> (4 * (nk % 2)) & 15;
            const int cv = blk[v_codes_at(D) + tok * (D / 2) + nv / 2] >> (4 * (nv % 2)) & 15;
            const int g = d / (D / G);
            const float2 pk = __half22float2(*reinterpret_cast<const __half2*>(blk + k_params_at(D) + (tok * G + g) * 4));
            const float2 pv = __half22float2(*reinterpret_cast<const __half2*>(blk + v_params_at(D, G) + (tok * G + g) * 4));
            dot = fmaf(qv[e], fmaf(static_cast<float>(ck), pk.x, pk.y), dot);
            vv[e] = fmaf(static_cast<float>(cv), pv.x, pv.y);
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
        const float mx = fmaxf(m, dot), keep = expf(m - mx), p = expf(dot - mx);
        l = fmaf(l, keep, p);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], keep, p * vv[e]);
        m = mx;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
    __syncthreads();
    if (threadIdx.x >= D) return;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
    for (int w = 0; w < kWarps; ++w) {
        const float a = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - M);
        L = fmaf(a, s_l[w], L);
        O = fmaf(a, s_o[w][threadIdx.x], O);
    }
    store(out + t * o_token + h * o_head + threadIdx.x, L == 0.f ? 0.f : O / L);
}

}  // namespace

extern "C" {

int64_t ecq_kv4_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_q, int32_t max_pages, int32_t page_size) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || max_q < 1 || max_pages < 1)
        return ECQ_ERR_ARG;
    if (!sizes_ok(head_dim, page_size, 32) || heads / kv_heads > 64) return ECQ_ERR_UNSUPPORTED;
    return 0;
}

int32_t ecq_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* out,
                          int64_t out_token_stride, int64_t out_head_stride, int32_t dtype, const void* pages,
                          int64_t n_pages, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t page_size,
                          int32_t group_size, const void* block_table, int64_t table_stride, int32_t max_pages,
                          const void* seq_lens, const void* q_starts, int32_t batch, int32_t total_q, int32_t max_q,
                          float scale, void* workspace, int64_t workspace_bytes, void* status, void* stream) {
    if (!sizes_ok(head_dim, page_size, group_size) || (dtype != ECQ_KV4_F16 && dtype != ECQ_KV4_BF16))
        return ECQ_ERR_UNSUPPORTED;
    const int64_t need =
        ecq_kv4_attention_workspace_bytes(batch, heads, kv_heads, head_dim, max_q, max_pages, page_size);
    if (need < 0) return static_cast<int32_t>(need);
    if (total_q < 0 || !pool_ok(pages, n_pages, kv_heads, page_size)) return ECQ_ERR_ARG;
    if (!block_table || !seq_lens || table_stride < max_pages) return ECQ_ERR_ARG;
    if (static_cast<int64_t>(max_pages) * page_size >= (1ll << 31) - 256) return ECQ_ERR_ARG;
    if (!q_starts && (total_q != batch || max_q != 1)) return ECQ_ERR_ARG;
    if (total_q == 0) return ECQ_OK;
    if (!q || !out || !aligned(q, 16) || !aligned(out, 8)) return ECQ_ERR_ARG;
    if (((q_token_stride | q_head_stride) & 7) || ((out_token_stride | out_head_stride) & 3)) return ECQ_ERR_ARG;
    if (workspace_bytes < need || (need > 0 && !workspace)) return ECQ_ERR_WORKSPACE;
    return by_layout(dtype, head_dim, head_dim / group_size, [&](auto layout) {
        using L = decltype(layout);
        using T = typename L::T;
        return result(launch_pdl(attention_kernel<T, L::D, L::G>, dim3(total_q, heads), dim3(kWarps * 32), 0,
                                 static_cast<cudaStream_t>(stream), static_cast<const T*>(q), q_token_stride,
                                 q_head_stride, static_cast<T*>(out), out_token_stride, out_head_stride,
                                 static_cast<const uint8_t*>(pages), n_pages, kv_heads, heads / kv_heads,
                                 log2i(page_size), static_cast<const int32_t*>(block_table), table_stride, max_pages,
                                 static_cast<const int32_t*>(seq_lens), static_cast<const int32_t*>(q_starts), batch,
                                 scale, static_cast<int32_t*>(status)));
    });
}

}  // extern "C"

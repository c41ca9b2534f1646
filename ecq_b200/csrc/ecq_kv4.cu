// ecq_kv4.cu -- the 4-bit KV cache's bookkeeping and storage:
//   ecq_kv4_extend   lengths, block tables, slots and positions of a step
//   ecq_kv4_release  pages of finished requests back on the free stack
//   ecq_kv4_append   K and V rows quantised into their slots
//   ecq_kv4_gather   rows read back
#include <cuda_runtime.h>

#include "ecq_kv4.cuh"

namespace {

using namespace ecq_kv4;
using ecq_dev::launch_pdl;
using ecq_dev::launch_pdl_cluster;
using ecq_dev::pdl_launch_dependents;
using ecq_dev::pdl_wait;

// ---------------------------------------------------------------------------
// Block tables and slot maps. One launch: every CTA of one cluster scans all
// requests (a few KB from L2) into its own shared memory -- tokens and pages
// before each request -- and then writes its share of the outputs. The cluster
// barrier between the two parts is what lets lengths and count be updated in
// place: nothing is written before every CTA has read. Work per token and per
// page is found by a binary search in the scanned starts, so one request with
// all the tokens is spread like many with few. Bound by launch and barrier
// latency.
// ---------------------------------------------------------------------------
constexpr int kTableThreads = 512;
constexpr int kRun = 4;  // outputs that a thread takes in a row

struct Totals {
    long long tokens;  // sums of 2^13 lengths below 2^31
    int pages;
};

// Exclusive sums over the CTA of (tokens, pages); returns the totals.
__device__ __forceinline__ Totals block_exclusive(long long& tokens, int& pages, long long* s_tok, int* s_pg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long t = tokens;
    int p = pages;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long tt = __shfl_up_sync(0xffffffffu, t, o);
        const int pp = __shfl_up_sync(0xffffffffu, p, o);
        if (lane >= o) {
            t += tt;
            p += pp;
        }
    }
    __syncthreads();  // the last round's readers are done
    if (lane == 31) {
        s_tok[warp] = t;
        s_pg[warp] = p;
    }
    __syncthreads();
    Totals all = {0, 0};
    long long bt = 0;
    int bp = 0;
#pragma unroll
    for (int w = 0; w < kTableThreads / 32; ++w) {
        if (w == warp) {
            bt = all.tokens;
            bp = all.pages;
        }
        all.tokens += s_tok[w];
        all.pages += s_pg[w];
    }
    tokens = bt + t - tokens;
    pages = bp + p - pages;
    return all;
}

// The last b in [0, n) with start[b] <= i (start ascending, start[0] = 0): of
// equal starts the last, which is the one that owns i.
__device__ __forceinline__ int owner(const int* start, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kTableThreads) extend_kernel(
    const int32_t* lens_in, const int32_t* __restrict__ new_lens, int32_t* lens_out, int32_t* table,
    int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_shift, const int32_t* __restrict__ free_pages,
    int32_t free_capacity, const int32_t* count_in, int32_t* count_out, int32_t* __restrict__ q_starts,
    int32_t* __restrict__ slots, int32_t* __restrict__ positions, int32_t max_tokens, int32_t* status) {
    extern __shared__ int32_t sm[];
    int32_t* s_len = sm;
    int32_t* s_tok = sm + batch;      // tokens before request b
    int32_t* s_page = s_tok + batch;  // new pages before request b
    __shared__ long long w_tok[kTableThreads / 32];
    __shared__ int w_pg[kTableThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int32_t count = *count_in;
    const long long room = static_cast<long long>(max_pages) << page_shift;
    const int page_size = 1 << page_shift;
    Totals sum = {0, 0};
    long long pages_sum = 0;
    bool bad = count < 0 || count > free_capacity;
    for (int base = 0; base < batch; base += kTableThreads) {
        const int b = base + threadIdx.x;
        long long tok = 0;
        int pg = 0, len = 0;
        if (b < batch) {
            len = lens_in[b];
            const int add = new_lens[b];
            if (len < 0 || add < 0 || static_cast<long long>(len) + add > room) {
                bad = true;
            } else {
                tok = add;
                // room < 2^31 (checked on the host), so the sums fit
                pg = ((len + add + page_size - 1) >> page_shift) - ((len + page_size - 1) >> page_shift);
            }
        }
        const Totals all = block_exclusive(tok, pg, w_tok, w_pg);
        if (b < batch) {
            s_len[b] = len;
            // beyond 2^31 the call is refused below and nothing uses these
            s_tok[b] = static_cast<int>(min(sum.tokens + tok, 0x7fffffffll));
            s_page[b] = static_cast<int>(min(pages_sum + pg, 0x7fffffffll));
        }
        sum.tokens += all.tokens;
        pages_sum += all.pages;
    }
    bad = __syncthreads_or(bad || sum.tokens > max_tokens);
    const bool dry = !bad && pages_sum > count;
    ecq_dev::cluster_sync();
    const int rank = static_cast<int>(ecq_dev::cluster_rank()), ranks = static_cast<int>(ecq_dev::cluster_size());
    const int tid = rank * kTableThreads + threadIdx.x, threads = ranks * kTableThreads;
    if (bad || dry) {
        if (tid == 0) {
            raise_status(status, bad ? ECQ_STATUS_BADARG : ECQ_STATUS_NO_PAGES);
            *count_out = count;
        }
        for (int b = tid; b <= batch; b += threads) {
            q_starts[b] = 0;
            if (b < batch) lens_out[b] = s_len[b];
        }
        for (int i = tid; i < max_tokens; i += threads) {
            slots[i] = -1;
            positions[i] = -1;
        }
        return;
    }
    const int total = static_cast<int>(sum.tokens), pages = static_cast<int>(pages_sum);
    if (tid == 0) *count_out = count - pages;
    for (int b = tid; b <= batch; b += threads) {
        const int start = b < batch ? s_tok[b] : total;
        q_starts[b] = start;
        if (b < batch) lens_out[b] = s_len[b] + ((b + 1 < batch ? s_tok[b + 1] : total) - start);
    }
    for (int j = tid; j < pages; j += threads) {
        const int b = owner(s_page, batch, j);
        const int held = (s_len[b] + page_size - 1) >> page_shift;
        table[b * table_stride + held + (j - s_page[b])] = free_pages[count - 1 - j];
    }
    // a thread takes kRun tokens in a row: one search, and mostly one page, for all of them
    for (int i0 = tid * kRun; i0 < max_tokens; i0 += threads * kRun) {
        int b = 0, held = 0, next = -1, page = -1, have = -1;
        if (i0 < total) b = owner(s_tok, batch, i0);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const int i = i0 + k;
            int slot = -1, pos = -1;
            if (i < total) {
                if (i >= next) {  // the first token, or the next request that has any
                    if (next >= 0) do ++b;
                        while ((b + 1 < batch ? s_tok[b + 1] : total) <= i);
                    next = b + 1 < batch ? s_tok[b + 1] : total;
                    held = (s_len[b] + page_size - 1) >> page_shift;
                    have = -1;
                }
                pos = s_len[b] + (i - s_tok[b]);
                const int col = pos >> page_shift;
                if (col != have) {
                    have = col;
                    // a page of this step comes off the stack again: the table entry is another thread's write
                    page = col < held ? table[b * table_stride + col] : free_pages[count - 1 - (s_page[b] + col - held)];
                }
                const long long at = (static_cast<long long>(page) << page_shift) + (pos & (page_size - 1));
                slot = page < 0 || at > 0x7fffffffll ? -1 : static_cast<int>(at);
            }
            if (i < max_tokens) {
                slots[i] = slot;
                positions[i] = pos;
            }
        }
    }
}

__global__ void __launch_bounds__(kTableThreads) release_kernel(
    const uint8_t* __restrict__ done, const int32_t* lens_in, int32_t* lens_out, const int32_t* __restrict__ table,
    int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_shift, int32_t* __restrict__ free_pages,
    int32_t free_capacity, const int32_t* count_in, int32_t* count_out, int32_t* status) {
    extern __shared__ int32_t sm[];
    int32_t* s_len = sm;              // length after the call
    int32_t* s_page = sm + batch;     // pages given back before request b
    __shared__ long long w_tok[kTableThreads / 32];
    __shared__ int w_pg[kTableThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int32_t count = *count_in;
    const int page_size = 1 << page_shift;
    long long pages_sum = 0;
    bool bad = count < 0 || count > free_capacity;
    for (int base = 0; base < batch; base += kTableThreads) {
        const int b = base + threadIdx.x;
        long long none = 0;
        int pg = 0, len = 0;
        bool give = false;
        if (b < batch) {
            len = lens_in[b];
            give = done[b] != 0;
            const long long held = (static_cast<long long>(len) + page_size - 1) >> page_shift;
            if (len < 0 || held > max_pages) bad = true;
            else if (give) pg = static_cast<int>(held);
        }
        const Totals all = block_exclusive(none, pg, w_tok, w_pg);
        if (b < batch) {
            s_len[b] = give ? 0 : len;
            s_page[b] = static_cast<int>(min(pages_sum + pg, 0x7fffffffll));
        }
        pages_sum += all.pages;
    }
    bad = __syncthreads_or(bad);
    const bool full = !bad && pages_sum + count > free_capacity;
    ecq_dev::cluster_sync();
    const int rank = static_cast<int>(ecq_dev::cluster_rank()), ranks = static_cast<int>(ecq_dev::cluster_size());
    const int tid = rank * kTableThreads + threadIdx.x, threads = ranks * kTableThreads;
    if (bad || full) {
        if (tid == 0) {
            raise_status(status, bad ? ECQ_STATUS_BADARG : ECQ_STATUS_NO_PAGES);
            *count_out = count;
        }
        // done requests' lengths were read by this thread's own CTA: take them from the input again
        if (lens_out != lens_in)
            for (int b = tid; b < batch; b += threads) lens_out[b] = lens_in[b];
        return;
    }
    const int pages = static_cast<int>(pages_sum);
    if (tid == 0) *count_out = count + pages;
    for (int b = tid; b < batch; b += threads) lens_out[b] = s_len[b];
    for (int j0 = tid * kRun; j0 < pages; j0 += threads * kRun) {
        int b = owner(s_page, batch, j0);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const int j = j0 + k;
            if (j < pages) {
                while (b + 1 < batch && s_page[b + 1] <= j) ++b;  // the last request that starts at or before j: the one with it
                free_pages[count + j] = table[b * table_stride + (j - s_page[b])];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Storage. D / 8 lanes take a K row of one token and head, 8 channels (16
// bytes) each, and as many the V row: a warp holds one token and head at D =
// 128, two at 64. Minimum and maximum of a group go over its g / 8 lanes by
// shuffles. A K lane's 8 channels are one 32-bit word of codes; V words want
// every 8th channel, which an 8 x 8 transposition of nibbles over 8 lanes
// gives (3 shuffles). Bound by latency for steps and by instructions for
// prompts. Codes are those of the IEEE quotient, so that a value on the border
// between two codes goes the same way everywhere.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t u);
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t from_float2(float a, float b);
template <>
__device__ __forceinline__ uint32_t from_float2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t from_float2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Nibble j of lane i of 8 neighbouring lanes <-> nibble i of lane j.
__device__ __forceinline__ uint32_t transpose8(uint32_t x, int lane) {
    constexpr uint32_t kLow[3] = {0x0000ffffu, 0x00ff00ffu, 0x0f0f0f0fu};
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        const int j = 4 >> s;
        const uint32_t m = kLow[s], y = __shfl_xor_sync(0xffffffffu, x, j);
        x = (lane & j) ? ((x & ~m) | ((y & ~m) >> (4 * j))) : ((x & m) | ((y & m) << (4 * j)));
    }
    return x;
}

// This thread's row: token (of head blockIdx.y), whether V, and which 8 channels.
template <int D>
struct RowLane {
    static constexpr int kUnit = D / 4;  // lanes per token and head
    static constexpr int kTokens = kRowThreads / kUnit;
    int token, c;  // channels 8c .. 8c + 7
    bool is_v;
    __device__ __forceinline__ RowLane() {
        const int l = threadIdx.x % kUnit;
        token = static_cast<int>(blockIdx.x) * kTokens + threadIdx.x / kUnit;
        is_v = l >= D / 8;
        c = l % (D / 8);
    }
};

// Where the lane's word of codes and its group's pair lie in the token's block.
template <int D, int G>
__device__ __forceinline__ int code_at(bool is_v, int tok, int c) {
    const int word = is_v ? (c % 8) * (D / 16) + (c / 8) * 4 : (c % 4) * (D / 8) + (c / 4) * 4;
    return (is_v ? v_codes_at(D) : 0) + tok * (D / 2) + word;
}
template <int D, int G>
__device__ __forceinline__ int params_at(bool is_v, int tok, int c) {
    return (is_v ? v_params_at(D, G) : k_params_at(D)) + tok * 4 * G + (c * 8 / (D / G)) * 4;
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kRowThreads) append_kernel(const T* __restrict__ k, int64_t k_token, int64_t k_head,
                                                            const T* __restrict__ v, int64_t v_token, int64_t v_head,
                                                            uint8_t* __restrict__ pages, int64_t n_slots, int heads,
                                                            int page_shift, const int32_t* __restrict__ slots,
                                                            int tokens, int32_t* status) {
    constexpr int kGroupLanes = D / G / 8;
    pdl_launch_dependents();
    const RowLane<D> me;
    pdl_wait();
    const int token = me.token, head = blockIdx.y;
    const bool in = token < tokens;
    const int32_t slot = in ? slots[token] : -1;
    const bool keep = slot >= 0 && slot < n_slots;
    if (in && slot >= n_slots && head == 0 && me.c == 0) raise_status(status, ECQ_STATUS_BADARG);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (keep) {
        const T* row = me.is_v ? v + token * v_token + head * v_head : k + token * k_token + head * k_head;
        const uint4 u = *reinterpret_cast<const uint4*>(row + 8 * me.c);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = to_float2<T>(w[i]);
            x[2 * i] = min_nan(max_nan(f.x, -65504.f), 65504.f);
            x[2 * i + 1] = min_nan(max_nan(f.y, -65504.f), 65504.f);
        }
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = min_nan(lo, x[i]);
        hi = max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < kGroupLanes; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const __half zero = __float2half_rn(lo), scale = __float2half_rn(__fdiv_rn(hi - lo, 15.f));
    const float z = __half2float(zero), s = __half2float(scale);
    // (x - zero) / scale by the reciprocal; where that comes so near to the border between two codes that the rounded
    // quotient might fall on the other side, the division itself decides. 1.5 2^23 + q holds q rounded to even in its
    // low bits. A NaN's code is 0 (fmaxf takes the other operand).
    const float inv = s == 0.f ? 0.f : __frcp_rn(s);
    constexpr float kInt = 12582912.f;
    uint32_t word = 0;
    bool near = false;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float q = fminf(fmaxf((x[i] - z) * inv, 0.f), 15.f), y = q + kInt;
        near |= fabsf(q - (y - kInt)) > 0.49999f;
        word = word * 16u + (__float_as_uint(y) - 0x4b400000u);
    }
    if (near) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = s == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x[i] - z, s)), 0.f), 15.f);
            word |= static_cast<uint32_t>(t) << (4 * i);
        }
    }
    const uint32_t turned = transpose8(word, threadIdx.x & 31);
    if (!keep) return;
    const int page_size = 1 << page_shift, at = slot & (page_size - 1);
    uint8_t* blk = pages + ((static_cast<int64_t>(slot >> page_shift) * heads + head) * (page_size / kBlockTokens) +
                            at / kBlockTokens) * block_bytes(D, G);
    const int tok = at % kBlockTokens;
    *reinterpret_cast<uint32_t*>(blk + code_at<D, G>(me.is_v, tok, me.c)) = me.is_v ? turned : word;
    if (me.c % kGroupLanes == 0)
        *reinterpret_cast<__half2*>(blk + params_at<D, G>(me.is_v, tok, me.c)) = __halves2half2(scale, zero);
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(T* __restrict__ k, T* __restrict__ v,
                                                            const uint8_t* __restrict__ pages, int64_t n_slots,
                                                            int heads, int page_shift,
                                                            const int32_t* __restrict__ slots, int tokens,
                                                            int32_t* status) {
    pdl_launch_dependents();
    const RowLane<D> me;
    pdl_wait();
    const int token = me.token, head = blockIdx.y;
    const bool in = token < tokens;
    const int32_t slot = in ? slots[token] : -1;
    const bool have = slot >= 0 && slot < n_slots;
    if (in && slot >= n_slots && head == 0 && me.c == 0) raise_status(status, ECQ_STATUS_BADARG);
    uint32_t word = 0;
    float2 par = make_float2(0.f, 0.f);
    if (have) {
        const int page_size = 1 << page_shift, at = slot & (page_size - 1);
        const uint8_t* blk = pages + ((static_cast<int64_t>(slot >> page_shift) * heads + head) *
                                      (page_size / kBlockTokens) + at / kBlockTokens) * block_bytes(D, G);
        const int tok = at % kBlockTokens;
        word = *reinterpret_cast<const uint32_t*>(blk + code_at<D, G>(me.is_v, tok, me.c));
        par = __half22float2(*reinterpret_cast<const __half2*>(blk + params_at<D, G>(me.is_v, tok, me.c)));
    }
    const uint32_t turned = transpose8(word, threadIdx.x & 31);
    if (!in) return;
    if (me.is_v) word = turned;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = from_float2<T>(fmaf(static_cast<float>((word >> (8 * i)) & 15u), par.x, par.y),
                              fmaf(static_cast<float>((word >> (8 * i + 4)) & 15u), par.x, par.y));
    T* row = (me.is_v ? v : k) + (static_cast<int64_t>(token) * heads + head) * D + 8 * me.c;
    *reinterpret_cast<uint4*>(row) = make_uint4(o[0], o[1], o[2], o[3]);
}

bool table_args_ok(int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_size, int32_t free_capacity) {
    if (batch < 1 || max_pages < 1 || free_capacity < 0 || table_stride < max_pages) return false;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return false;
    return static_cast<int64_t>(max_pages) * page_size < (1ll << 31) - 256;
}

cudaError_t allow(const void* fn, size_t smem) {
    if (smem <= 48 * 1024) return cudaSuccess;
    return ecq_dev::ensure_smem_limit(fn, 112 * 1024) ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace

extern "C" {

int64_t ecq_kv4_page_bytes(int32_t head_dim, int32_t page_size, int32_t group_size) {
    if (!sizes_ok(head_dim, page_size, group_size)) return ECQ_ERR_UNSUPPORTED;
    return static_cast<int64_t>(page_size / kBlockTokens) * block_bytes(head_dim, head_dim / group_size);
}

int32_t ecq_kv4_extend(const void* seq_lens, const void* new_lens, void* seq_lens_out, void* block_table,
                       int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_size,
                       const void* free_pages, int32_t free_capacity, const void* free_count, void* free_count_out,
                       void* q_starts, void* slots, void* positions, int32_t max_tokens, void* status, void* stream) {
    if (!seq_lens || !new_lens || !seq_lens_out || !block_table || !free_count || !free_count_out || !q_starts)
        return ECQ_ERR_ARG;
    if ((free_capacity > 0 && !free_pages) || max_tokens < 0 || (max_tokens > 0 && (!slots || !positions)))
        return ECQ_ERR_ARG;
    if (!table_args_ok(table_stride, max_pages, batch, page_size, free_capacity)) return ECQ_ERR_ARG;
    if (batch > ECQ_KV4_MAX_BATCH) return ECQ_ERR_UNSUPPORTED;
    const size_t smem = static_cast<size_t>(batch) * 12;
    if (cudaError_t rc = allow(reinterpret_cast<const void*>(extend_kernel), smem); rc != cudaSuccess) return result(rc);
    // one CTA while its threads cover the outputs in a few rounds, a cluster of 8 above
    const unsigned ctas = (max_tokens > 4 * kTableThreads || batch > 2 * kTableThreads) ? 8 : 1;
    return result(launch_pdl_cluster(extend_kernel, dim3(ctas), dim3(kTableThreads), smem,
                                     static_cast<cudaStream_t>(stream), ctas, static_cast<const int32_t*>(seq_lens),
                                     static_cast<const int32_t*>(new_lens), static_cast<int32_t*>(seq_lens_out),
                                     static_cast<int32_t*>(block_table), table_stride, max_pages, batch,
                                     log2i(page_size), static_cast<const int32_t*>(free_pages), free_capacity,
                                     static_cast<const int32_t*>(free_count), static_cast<int32_t*>(free_count_out),
                                     static_cast<int32_t*>(q_starts), static_cast<int32_t*>(slots),
                                     static_cast<int32_t*>(positions), max_tokens, static_cast<int32_t*>(status)));
}

int32_t ecq_kv4_release(const void* done, const void* seq_lens, void* seq_lens_out, const void* block_table,
                        int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_size, void* free_pages,
                        int32_t free_capacity, const void* free_count, void* free_count_out, void* status,
                        void* stream) {
    if (!done || !seq_lens || !seq_lens_out || !block_table || !free_pages || !free_count || !free_count_out)
        return ECQ_ERR_ARG;
    if (!table_args_ok(table_stride, max_pages, batch, page_size, free_capacity)) return ECQ_ERR_ARG;
    if (batch > ECQ_KV4_MAX_BATCH) return ECQ_ERR_UNSUPPORTED;
    const size_t smem = static_cast<size_t>(batch) * 8;
    if (cudaError_t rc = allow(reinterpret_cast<const void*>(release_kernel), smem); rc != cudaSuccess) return result(rc);
    const unsigned ctas = static_cast<int64_t>(batch) * max_pages > 8 * kTableThreads ? 8 : 1;
    return result(launch_pdl_cluster(release_kernel, dim3(ctas), dim3(kTableThreads), smem,
                                     static_cast<cudaStream_t>(stream), ctas, static_cast<const uint8_t*>(done),
                                     static_cast<const int32_t*>(seq_lens), static_cast<int32_t*>(seq_lens_out),
                                     static_cast<const int32_t*>(block_table), table_stride, max_pages, batch,
                                     log2i(page_size), static_cast<int32_t*>(free_pages), free_capacity,
                                     static_cast<const int32_t*>(free_count), static_cast<int32_t*>(free_count_out),
                                     static_cast<int32_t*>(status)));
}

int32_t ecq_kv4_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                       int64_t v_token_stride, int64_t v_head_stride, int32_t dtype, void* pages, int64_t n_pages,
                       int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t group_size, const void* slots,
                       int32_t tokens, void* status, void* stream) {
    if (!sizes_ok(head_dim, page_size, group_size) || (dtype != ECQ_KV4_F16 && dtype != ECQ_KV4_BF16))
        return ECQ_ERR_UNSUPPORTED;
    if (tokens < 0 || !pool_ok(pages, n_pages, kv_heads, page_size)) return ECQ_ERR_ARG;
    if (tokens == 0) return ECQ_OK;
    if (!k || !v || !slots || !aligned(k, 16) || !aligned(v, 16)) return ECQ_ERR_ARG;
    if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return ECQ_ERR_ARG;
    const int per_block = kRowThreads / (head_dim / 4);
    const dim3 grid((tokens + per_block - 1) / per_block, kv_heads);
    return by_layout(dtype, head_dim, head_dim / group_size, [&](auto layout) {
        using L = decltype(layout);
        using T = typename L::T;
        return result(launch_pdl(append_kernel<T, L::D, L::G>, grid, dim3(kRowThreads), 0,
                                 static_cast<cudaStream_t>(stream), static_cast<const T*>(k), k_token_stride,
                                 k_head_stride, static_cast<const T*>(v), v_token_stride, v_head_stride,
                                 static_cast<uint8_t*>(pages), n_pages * page_size, kv_heads, log2i(page_size),
                                 static_cast<const int32_t*>(slots), tokens, static_cast<int32_t*>(status)));
    });
}

int32_t ecq_kv4_gather(void* k, void* v, int32_t dtype, const void* pages, int64_t n_pages, int32_t kv_heads,
                       int32_t head_dim, int32_t page_size, int32_t group_size, const void* slots, int32_t tokens,
                       void* status, void* stream) {
    if (!sizes_ok(head_dim, page_size, group_size) || (dtype != ECQ_KV4_F16 && dtype != ECQ_KV4_BF16))
        return ECQ_ERR_UNSUPPORTED;
    if (tokens < 0 || !pool_ok(pages, n_pages, kv_heads, page_size)) return ECQ_ERR_ARG;
    if (tokens == 0) return ECQ_OK;
    if (!k || !v || !slots || !aligned(k, 16) || !aligned(v, 16)) return ECQ_ERR_ARG;
    const int per_block = kRowThreads / (head_dim / 4);
    const dim3 grid((tokens + per_block - 1) / per_block, kv_heads);
    return by_layout(dtype, head_dim, head_dim / group_size, [&](auto layout) {
        using L = decltype(layout);
        using T = typename L::T;
        return result(launch_pdl(gather_kernel<T, L::D, L::G>, grid, dim3(kRowThreads), 0,
                                 static_cast<cudaStream_t>(stream), static_cast<T*>(k), static_cast<T*>(v),
                                 static_cast<const uint8_t*>(pages), n_pages * page_size, kv_heads, log2i(page_size),
                                 static_cast<const int32_t*>(slots), tokens, static_cast<int32_t*>(status)));
    });
}

}  // extern "C"

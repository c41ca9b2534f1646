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
// Block tables and slot maps. One launch: every CTA scans all requests (a few
// KB from L2) into its own shared memory -- tokens and pages before each
// request -- and then writes its share of the outputs. Where lengths or count
// are updated in place the CTAs are one cluster, whose barrier between the two
// parts keeps anything from being written before every CTA has read; otherwise
// there are more of them. Work per token and per
// page is found by a binary search in the scanned starts, so one request with
// all the tokens is spread like many with few. Release is one CTA or one cluster
// in any case: whether all of its pages were good decides what it says. Bound by
// launch and barrier latency: one token of 17 requests 4.5 us, 512 prompts of up
// to 255 tokens 6.0 us, 17 requests released 2.6 us, 256 of 512 with up to 512
// pages 5.9 us.
// ---------------------------------------------------------------------------
constexpr int kTableThreads = 512;
constexpr int kRun = 4;  // outputs that a thread takes in a row

struct Totals {
    long long first;  // tokens, or pages that are given back: of 2^13 requests below 2^31 each
    int second;       // new pages, or parts of those
};

// Exclusive sums over the CTA of two counts; returns the totals.
__device__ __forceinline__ Totals block_exclusive(long long& first, int& second, long long* s_tok, int* s_pg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long t = first;
    int p = second;
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
            bt = all.first;
            bp = all.second;
        }
        all.first += s_tok[w];
        all.second += s_pg[w];
    }
    first = bt + t - first;
    second = bp + p - second;
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

// A page number whose slots are no int32.
__device__ __forceinline__ bool bad_page(int32_t page, int page_shift) {
    return static_cast<uint32_t>(page) > static_cast<uint32_t>(INT32_MAX >> page_shift);
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
    int32_t* s_part = s_page + batch;  // its last page, where new tokens go on in that
    __shared__ long long w_tok[kTableThreads / 32];
    __shared__ int w_pg[kTableThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int32_t count = *count_in;
    const long long room = static_cast<long long>(max_pages) << page_shift;
    const int page_size = 1 << page_shift;
    long long tokens_sum = 0, pages_sum = 0;
    const bool stack = count >= 0 && count <= free_capacity;
    bool bad = !stack;
    // the first pages to be popped, on their way while the lengths are scanned
    int32_t first_page[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        const int j = k * kTableThreads + threadIdx.x;
        first_page[k] = stack && j < count ? free_pages[count - 1 - j] : 0;
    }
    for (int base = 0; base < batch; base += kTableThreads) {
        const int b = base + threadIdx.x;
        long long tok = 0;
        int pg = 0, len = 0, part = 0;
        if (b < batch) {
            len = lens_in[b];
            const int add = new_lens[b];
            if (len < 0 || add < 0 || static_cast<long long>(len) + add > room) {
                bad = true;
            } else {
                tok = add;
                // room < 2^31 (checked on the host), so the sums fit
                pg = ((len + add + page_size - 1) >> page_shift) - ((len + page_size - 1) >> page_shift);
                if (add && (len & (page_size - 1))) part = table[b * table_stride + (len >> page_shift)];
            }
        }
        const Totals all = block_exclusive(tok, pg, w_tok, w_pg);
        bad |= bad_page(part, page_shift);
        if (b < batch) {
            s_len[b] = len;
            s_part[b] = part;
            // beyond 2^31 the call is refused below and nothing uses these
            s_tok[b] = static_cast<int>(min(tokens_sum + tok, 0x7fffffffll));
            s_page[b] = static_cast<int>(min(pages_sum + pg, 0x7fffffffll));
        }
        tokens_sum += all.first;
        pages_sum += all.second;
    }
    if (stack && tokens_sum <= max_tokens && pages_sum <= count) {  // (the pages of more tokens may not fit an int)
#pragma unroll
        for (int k = 0; k < kRun; ++k) bad |= k * kTableThreads + static_cast<int>(threadIdx.x) < pages_sum && bad_page(first_page[k], page_shift);
        for (unsigned j = threadIdx.x + kRun * kTableThreads; j < static_cast<unsigned>(pages_sum); j += kTableThreads)
            bad |= bad_page(free_pages[count - 1 - static_cast<int>(j)], page_shift);
    }
    bad = __syncthreads_or(bad || tokens_sum > max_tokens);
    const bool dry = !bad && pages_sum > count;
    ecq_dev::cluster_sync();
    // unsigned: the counts are below 2^31, so an index that has gone past its end by a stride is below 2^32
    const unsigned tid = blockIdx.x * kTableThreads + threadIdx.x, threads = gridDim.x * kTableThreads;
    const unsigned n = batch, most = max_tokens;
    if (bad || dry) {
        if (tid == 0) {
            raise_status(status, bad ? ECQ_STATUS_BADARG : ECQ_STATUS_NO_PAGES);
            *count_out = count;
        }
        for (unsigned b = tid; b <= n; b += threads) {
            q_starts[b] = 0;
            if (b < n) lens_out[b] = s_len[b];
        }
        for (unsigned i = tid; i < most; i += threads) {
            slots[i] = -1;
            positions[i] = -1;
        }
        return;
    }
    const int total = static_cast<int>(tokens_sum), pages = static_cast<int>(pages_sum);
    if (tid == 0) *count_out = count - pages;
    for (unsigned b = tid; b <= n; b += threads) {
        const int start = b < n ? s_tok[b] : total;
        q_starts[b] = start;
        if (b < n) lens_out[b] = s_len[b] + ((b + 1 < n ? s_tok[b + 1] : total) - start);
    }
    for (unsigned j0 = tid; j0 < static_cast<unsigned>(pages); j0 += threads) {
        const int j = static_cast<int>(j0), b = owner(s_page, batch, j);
        const int held = (s_len[b] + page_size - 1) >> page_shift;
        table[b * table_stride + held + (j - s_page[b])] = free_pages[count - 1 - j];
    }
    // a thread takes kRun tokens in a row: one search, and mostly one page, for all of them
    for (unsigned i0 = tid * kRun; i0 < most; i0 += threads * kRun) {
        int b = 0, held = 0, next = -1, page = -1, have = -1;
        if (i0 < static_cast<unsigned>(total)) b = owner(s_tok, batch, static_cast<int>(i0));
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const unsigned at_token = i0 + k;
            const int i = static_cast<int>(at_token);
            int slot = -1, pos = -1;
            if (at_token < static_cast<unsigned>(total)) {
                if (i >= next) {  // the first token, or the next request that has any
                    while ((b + 1 < batch ? s_tok[b + 1] : total) <= i) ++b;
                    next = b + 1 < batch ? s_tok[b + 1] : total;
                    held = (s_len[b] + page_size - 1) >> page_shift;
                    have = -1;
                }
                pos = s_len[b] + (i - s_tok[b]);
                const int col = pos >> page_shift;
                if (col != have) {
                    have = col;
                    // a page of this step comes off the stack again: the table entry is another thread's write
                    page = col < held ? s_part[b] : free_pages[count - 1 - (s_page[b] + col - held)];
                }
                slot = (page << page_shift) + (pos & (page_size - 1));
            }
            if (at_token < most) {
                slots[at_token] = slot;
                positions[at_token] = pos;
            }
        }
    }
}

// One CTA or one cluster. The pages are written behind the stack's end first, where nothing is yet, and looked at on the
// way; lengths and count say so only if all of them were good.
constexpr int kPart = 256;  // pages that a warp takes at a time
__global__ void __launch_bounds__(kTableThreads) release_kernel(
    const uint8_t* __restrict__ done, const int32_t* lens_in, int32_t* lens_out, const int32_t* __restrict__ table,
    int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_shift, int32_t* __restrict__ free_pages,
    int32_t free_capacity, const int32_t* count_in, int32_t* count_out, int32_t* status) {
    extern __shared__ int32_t sm[];
    int32_t* s_len = sm;              // length after the call
    int32_t* s_page = sm + batch;     // pages given back before request b
    int32_t* s_part = s_page + batch;  // parts of up to kPart pages before it
    __shared__ long long w_tok[kTableThreads / 32];
    __shared__ int w_pg[kTableThreads / 32];
    __shared__ float s_bad;           // this CTA found something wrong
    pdl_launch_dependents();
    pdl_wait();
    const int32_t count = *count_in;
    const int page_size = 1 << page_shift;
    long long pages_sum = 0, parts_sum = 0;
    bool bad = count < 0 || count > free_capacity;
    for (int base = 0; base < batch; base += kTableThreads) {
        const int b = base + threadIdx.x;
        long long pg = 0;
        int parts = 0, len = 0;
        bool give = false;
        if (b < batch) {
            len = lens_in[b];
            give = done[b] != 0;
            const long long held = (static_cast<long long>(len) + page_size - 1) >> page_shift;
            if (len < 0 || held > max_pages) bad = true;
            else if (give) pg = held;
        }
        parts = static_cast<int>((pg + kPart - 1) / kPart);
        const Totals all = block_exclusive(pg, parts, w_tok, w_pg);
        if (b < batch) {
            s_len[b] = give ? 0 : len;
            s_page[b] = static_cast<int>(min(pages_sum + pg, 0x7fffffffll));
            s_part[b] = static_cast<int>(parts_sum + parts);
        }
        pages_sum += all.first;
        parts_sum += all.second;
    }
    bad = __syncthreads_or(bad);
    const bool full = pages_sum + count > free_capacity;
    // unsigned, as above
    const unsigned tid = blockIdx.x * kTableThreads + threadIdx.x, threads = gridDim.x * kTableThreads, n = batch;
    const int pages = bad || full ? 0 : static_cast<int>(pages_sum), parts = bad || full ? 0 : static_cast<int>(parts_sum);
    const int lane = threadIdx.x & 31;
    for (int i = tid >> 5; i < parts; i += threads >> 5) {  // a warp takes a part of a request's pages
        const int b = owner(s_part, batch, i), first = (i - s_part[b]) * kPart + lane;
        const int held = (b + 1 < batch ? s_page[b + 1] : pages) - s_page[b];
        const int32_t* from = table + b * table_stride;
        int32_t* to = free_pages + count + s_page[b];
        int32_t page[kPart / 32];
#pragma unroll
        for (int k = 0; k < kPart / 32; ++k) page[k] = first + 32 * k < held ? from[first + 32 * k] : 0;
#pragma unroll
        for (int k = 0; k < kPart / 32; ++k) {
            bad |= bad_page(page[k], page_shift);
            if (first + 32 * k < held) to[first + 32 * k] = page[k];
        }
    }
    bad = __syncthreads_or(bad);
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) s_bad = bad ? 1.f : 0.f;
        ecq_dev::cluster_sync();  // every CTA has read the lengths and the count, too
        for (unsigned r = 0; r < gridDim.x; ++r) bad |= ecq_dev::ld_cluster_f32(&s_bad, r) != 0.f;
        ecq_dev::cluster_arrive();
    }
    if (tid == 0) {
        if (bad || full) raise_status(status, bad ? ECQ_STATUS_BADARG : ECQ_STATUS_NO_PAGES);
        *count_out = count + (bad ? 0 : pages);
    }
    for (unsigned b = tid; b < n; b += threads) {
        if (!bad && !full) lens_out[b] = s_len[b];
        else if (lens_out != lens_in) lens_out[b] = lens_in[b];
    }
    if (gridDim.x > 1) ecq_dev::cluster_wait();  // no CTA leaves while another reads its flag
}

// ---------------------------------------------------------------------------
// Storage. D / 8 lanes take a K row of one token and head, 8 channels (16
// bytes) each, and as many the V row: a warp holds one token and head at D =
// 128, two at 64. Minimum and maximum of a group go over its g / 8 lanes by
// shuffles. A K lane's 8 channels are one 32-bit word of codes; V words want
// every 8th channel, which an 8 x 8 transposition of nibbles over 8 lanes
// gives (3 shuffles). Bound by latency for steps and by instructions for
// prompts. Codes are those of the IEEE quotient, so that a value on the border
// between two codes goes the same way everywhere. Measured: 16 tokens of 8 heads
// stored and read 3.7 us, 8191 tokens 32.5 us (2.7 TB/s).
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// Packed minimum that passes NaN on.
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t min2<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <>
__device__ __forceinline__ uint32_t min2<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// x / 15, correctly rounded: the product with the rounded reciprocal is within
// a unit of the quotient, and one step with the exact remainder rounds it
// (Markstein's theorem).
__device__ __forceinline__ float fifteenth(float x) {
    constexpr float r = 1.f / 15.f;
    const float q = x * r;
    return fmaf(fmaf(-q, 15.f, x), r, q);
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

// This thread's rows: tokens token, token + kTokens, ... (of head blockIdx.y),
// whether V, and which 8 channels. kPer rows a thread: their loads overlap.
template <int D, int kPer>
struct RowLane {
    static constexpr int kUnit = D / 4;  // lanes per token and head
    static constexpr int kTokens = kRowThreads / kUnit;
    int token, c;  // channels 8c .. 8c + 7
    int left;      // tokens from there on (an index behind 2^31 - 1 of them is no int)
    bool is_v;
    __device__ __forceinline__ RowLane(int tokens) {
        const int l = threadIdx.x % kUnit;
        const unsigned first = blockIdx.x * (kTokens * kPer) + threadIdx.x / kUnit;
        token = static_cast<int>(first);
        left = first < static_cast<unsigned>(tokens) ? tokens - token : 0;
        is_v = l >= D / 8;
        c = l % (D / 8);
    }
};
// The slots of the thread's rows; -1: none. One beyond the pool is reported.
template <int D, int kPer>
__device__ __forceinline__ void row_slots(int (&slot)[kPer], const RowLane<D, kPer>& me, const int32_t* slots,
                                          int64_t n_slots, int32_t* status) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) slot[i] = i * me.kTokens < me.left ? slots[me.token + i * me.kTokens] : -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (slot[i] >= n_slots) {
            if (blockIdx.y == 0 && me.c == 0) raise_status(status, ECQ_STATUS_BADARG);
            slot[i] = -1;
        }
}
__device__ __forceinline__ int64_t block_of(int slot, int heads, int page_shift) {
    return (static_cast<int64_t>(slot >> page_shift) * heads + blockIdx.y) * (1 << page_shift) / kBlockTokens +
           (slot & ((1 << page_shift) - 1)) / kBlockTokens;
}

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

template <typename T, int D, int G, int kPer>
__global__ void __launch_bounds__(kRowThreads) append_kernel(const T* __restrict__ k, int64_t k_token, int64_t k_head,
                                                            const T* __restrict__ v, int64_t v_token, int64_t v_head,
                                                            uint8_t* __restrict__ pages, int64_t n_slots, int heads,
                                                            int page_shift, const int32_t* __restrict__ slots,
                                                            int tokens, int32_t* status) {
    constexpr int kGroupLanes = D / G / 8;
    pdl_launch_dependents();
    const RowLane<D, kPer> me(tokens);
    const int64_t step = me.is_v ? v_token : k_token;
    const T* src = (me.is_v ? v + blockIdx.y * v_head : k + blockIdx.y * k_head) + me.token * step + 8 * me.c;
    pdl_wait();
    int slot[kPer];
    row_slots(slot, me, slots, n_slots, status);
    uint4 raw[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        raw[i] = make_uint4(0, 0, 0, 0);
        if (slot[i] >= 0) raw[i] = *reinterpret_cast<const uint4*>(src + i * me.kTokens * step);
    }
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
        const uint32_t w[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
        // (minimum, minus maximum) of the group as one packed minimum
        const uint32_t lo2 = min2<T>(min2<T>(w[0], w[1]), min2<T>(w[2], w[3]));
        const uint32_t hi2 = min2<T>(min2<T>(w[0] ^ 0x80008000u, w[1] ^ 0x80008000u), min2<T>(w[2] ^ 0x80008000u, w[3] ^ 0x80008000u));
        uint32_t ends = min2<T>(__byte_perm(lo2, hi2, 0x5410), __byte_perm(lo2, hi2, 0x7632));
#pragma unroll
        for (int o = 1; o < kGroupLanes; o <<= 1) ends = min2<T>(ends, __shfl_xor_sync(0xffffffffu, ends, o));
        const float2 e = to_float2<T>(ends);
        const bool wide = e.x < -65504.f || e.y < -65504.f;
        // a NaN is neither wide nor changed by what follows
        const float lo = wide ? fmaxf(e.x, -65504.f) : e.x, hi = wide ? fminf(-e.y, 65504.f) : -e.y;
        const __half zero = __float2half_rn(lo), scale = __float2half_rn(fifteenth(hi - lo));
        const float z = __half2float(zero), s = __half2float(scale);
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = to_float2<T>(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
        if (wide) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
        }
        // (x - zero) / (15 scale), held to 0..1, by the reciprocal (its roundings: under 2^-20 of it); where 15 of that come
        // so near to the border between two codes that the rounded quotient might fall on the other side, the division
        // itself decides. 1.5 2^23 + q holds q rounded to even in its low bits. A NaN's code is 0 (.sat).
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s * 15.f));
        if (s == 0.f) inv = 0.f;
        constexpr float kInt = 12582912.f;
        uint32_t word = 0;
        float far = 0.f;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const float t = __saturatef((x[i] - z) * inv), y = fmaf(t, 15.f, kInt);
            far = fmaxf(far, fabsf(fmaf(t, 15.f, kInt - y)));
            word = word * 16u + __float_as_uint(y);
        }
        word -= 0x4b400000u * 0x11111111u;  // the bits of 1.5 2^23, eight times
        if (far > 0.49997f) {
            word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = s == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x[i] - z, s)), 0.f), 15.f);
                word |= static_cast<uint32_t>(t) << (4 * i);
            }
        }
        const uint32_t turned = transpose8(word, threadIdx.x & 31);
        if (slot[n] >= 0) {
            const int tok = slot[n] % kBlockTokens;
            uint8_t* blk = pages + block_of(slot[n], heads, page_shift) * block_bytes(D, G);
            *reinterpret_cast<uint32_t*>(blk + code_at<D, G>(me.is_v, tok, me.c)) = me.is_v ? turned : word;
            if (me.c % kGroupLanes == 0)
                *reinterpret_cast<__half2*>(blk + params_at<D, G>(me.is_v, tok, me.c)) = __halves2half2(scale, zero);
        }
    }
}

template <typename T, int D, int G, int kPer>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(T* __restrict__ k, T* __restrict__ v,
                                                            const uint8_t* __restrict__ pages, int64_t n_slots,
                                                            int heads, int page_shift,
                                                            const int32_t* __restrict__ slots, int tokens,
                                                            int32_t* status) {
    pdl_launch_dependents();
    const RowLane<D, kPer> me(tokens);
    const int64_t step = static_cast<int64_t>(heads) * D;
    T* dst = (me.is_v ? v : k) + me.token * step + blockIdx.y * D + 8 * me.c;
    pdl_wait();
    int slot[kPer];
    row_slots(slot, me, slots, n_slots, status);
    uint32_t word[kPer], par[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        word[i] = par[i] = 0u;
        if (slot[i] >= 0) {
            const int tok = slot[i] % kBlockTokens;
            const uint8_t* blk = pages + block_of(slot[i], heads, page_shift) * block_bytes(D, G);
            word[i] = *reinterpret_cast<const uint32_t*>(blk + code_at<D, G>(me.is_v, tok, me.c));
            par[i] = *reinterpret_cast<const uint32_t*>(blk + params_at<D, G>(me.is_v, tok, me.c));
        }
    }
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
        const uint32_t turned = transpose8(word[n], threadIdx.x & 31), x = me.is_v ? turned : word[n];
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&par[n]));
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // a code in the low bits of 2^23, less that, is exact
            const uint32_t c = (x >> (4 * i)) & 15u;
            f[i] = fmaf(__uint_as_float(c | 0x4b000000u) - 8388608.f, p.x, p.y);
        }
        if (n * me.kTokens < me.left)
            *reinterpret_cast<uint4*>(dst + n * me.kTokens * step) =
                make_uint4(from_float2<T>(f[0], f[1]), from_float2<T>(f[2], f[3]), from_float2<T>(f[4], f[5]),
                           from_float2<T>(f[6], f[7]));
    }
}

// Rows a thread takes: one while one round of CTAs covers them (a step: the
// shortest way), four above (a prompt: loads overlap, addresses are shared).
int rows_per_thread(int tokens, int kv_heads, int head_dim) {
    const int64_t threads = static_cast<int64_t>(tokens) * kv_heads * (head_dim / 4);
    return threads <= 2048ll * ecq_dev::sm_count_cached() ? 1 : 4;
}
dim3 row_grid(int tokens, int kv_heads, int head_dim, int per) {
    const int block = kRowThreads / (head_dim / 4) * per;
    return dim3((static_cast<unsigned>(tokens) + block - 1) / block, kv_heads);
}

bool table_args_ok(int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_size, int32_t free_capacity) {
    if (batch < 1 || max_pages < 1 || free_capacity < 0 || table_stride < max_pages) return false;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return false;
    return static_cast<int64_t>(max_pages) * page_size < (1ll << 31) - 256;
}

// Whether n bytes at a and m at b share any.
bool shares(const void* a, int64_t n, const void* b, int64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x < static_cast<uintptr_t>(n) : x - y < static_cast<uintptr_t>(m);
}
// Lengths and count that are written must be apart from all that is read and written, but for the inputs that they may be.
struct Span {
    const void* at;
    int64_t bytes;
};
template <size_t N>
bool outputs_apart(const void* lens, const void* lens_out, const void* count, const void* count_out, int32_t batch,
                   const Span (&others)[N]) {
    const int64_t n = 4ll * batch;
    if (shares(lens_out, n, count_out, 4) || shares(lens_out, n, count, 4) || shares(count_out, 4, lens, n)) return false;
    if ((lens_out != lens && shares(lens_out, n, lens, n)) || (count_out != count && shares(count_out, 4, count, 4))) return false;
    for (const Span& s : others)
        if (s.bytes && (shares(lens_out, n, s.at, s.bytes) || shares(count_out, 4, s.at, s.bytes))) return false;
    return true;
}
int64_t table_bytes(int64_t table_stride, int32_t max_pages, int32_t batch) {
    return 4 * ((batch - 1) * table_stride + max_pages);
}

// CTAs for so many outputs, kRun to a thread: one, a cluster, or (not in
// place) several clusters.
unsigned table_ctas(int64_t outputs, bool in_place) {
    const int64_t want = (outputs + kTableThreads * kRun - 1) / (kTableThreads * kRun);
    if (want <= 1) return 1;
    if (in_place || want <= 8) return 8;
    return want < 64 ? static_cast<unsigned>((want + 7) / 8 * 8) : 64;
}

cudaError_t allow(const void* fn, size_t smem) {
    if (smem <= 48 * 1024) return cudaSuccess;
    return ecq_dev::ensure_smem_limit(fn, 16 * ECQ_KV4_MAX_BATCH) ? cudaSuccess : cudaErrorInvalidValue;
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
    const Span others[] = {{new_lens, 4ll * batch}, {block_table, table_bytes(table_stride, max_pages, batch)},
                           {free_pages, 4ll * free_capacity}, {q_starts, 4ll * batch + 4}, {slots, 4ll * max_tokens},
                           {positions, 4ll * max_tokens}};
    if (!outputs_apart(seq_lens, seq_lens_out, free_count, free_count_out, batch, others)) return ECQ_ERR_ARG;
    const size_t smem = static_cast<size_t>(batch) * 16;
    if (cudaError_t rc = allow(reinterpret_cast<const void*>(extend_kernel), smem); rc != cudaSuccess) return result(rc);
    const unsigned ctas = table_ctas(static_cast<int64_t>(max_tokens) + batch,
                                     seq_lens == seq_lens_out || free_count == free_count_out);
    return result(launch_pdl_cluster(extend_kernel, dim3(ctas), dim3(kTableThreads), smem,
                                     static_cast<cudaStream_t>(stream), ctas < 8 ? ctas : 8, static_cast<const int32_t*>(seq_lens),
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
    const Span others[] = {{done, batch}, {block_table, table_bytes(table_stride, max_pages, batch)}, {free_pages, 4ll * free_capacity}};
    if (!outputs_apart(seq_lens, seq_lens_out, free_count, free_count_out, batch, others)) return ECQ_ERR_ARG;
    const size_t smem = static_cast<size_t>(batch) * 12;
    if (cudaError_t rc = allow(reinterpret_cast<const void*>(release_kernel), smem); rc != cudaSuccess) return result(rc);
    // a cluster where the warps of one CTA would take more than a part each, should half of the pages come back
    const unsigned ctas = static_cast<int64_t>(batch) * max_pages / 2 > kTableThreads / 32 * kPart ? 8 : 1;
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
    const int per = rows_per_thread(tokens, kv_heads, head_dim);
    const dim3 grid = row_grid(tokens, kv_heads, head_dim, per);
    return by_layout(dtype, head_dim, head_dim / group_size, [&](auto layout) {
        using L = decltype(layout);
        using T = typename L::T;
        const auto kernel = per == 1 ? append_kernel<T, L::D, L::G, 1> : append_kernel<T, L::D, L::G, 4>;
        return result(launch_pdl(kernel, grid, dim3(kRowThreads), 0, static_cast<cudaStream_t>(stream), static_cast<const T*>(k), k_token_stride,
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
    const int per = rows_per_thread(tokens, kv_heads, head_dim);
    const dim3 grid = row_grid(tokens, kv_heads, head_dim, per);
    return by_layout(dtype, head_dim, head_dim / group_size, [&](auto layout) {
        using L = decltype(layout);
        using T = typename L::T;
        const auto kernel = per == 1 ? gather_kernel<T, L::D, L::G, 1> : gather_kernel<T, L::D, L::G, 4>;
        return result(launch_pdl(kernel, grid, dim3(kRowThreads), 0, static_cast<cudaStream_t>(stream), static_cast<T*>(k), static_cast<T*>(v),
                                 static_cast<const uint8_t*>(pages), n_pages * page_size, kv_heads, log2i(page_size),
                                 static_cast<const int32_t*>(slots), tokens, static_cast<int32_t*>(status)));
    });
}

}  // extern "C"

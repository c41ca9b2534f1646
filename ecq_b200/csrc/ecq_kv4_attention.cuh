// ecq_kv4_attention.cuh -- what the attention kernels over the 4-bit KV cache
// share: their arguments, a request's part of the work, conversions and the
// launch of the one for prompts.
#pragma once

#include <float.h>

#include "ecq_kv4.cuh"

namespace ecq_kv4 {

struct Args {
    const void* q;
    void* out;
    const uint8_t* pages;
    const int32_t *table, *lens, *starts;
    float* parts;     // per CTA two parts: one that starts inside a pair, one that starts a pair and does not end it
    int4* cuts;       // per CTA: request, pair, CTAs that follow; x < 0: none
    int32_t* status;
    int64_t q_token, q_head, o_token, o_head, n_pages, table_stride;
    int kv_heads, share, page_shift, max_pages, batch, total_q;
    int most_rows;    // requests with more rows (queries times share) are the prompt kernel's
    float scale;
};

// A request's queries and keys, as far as they are sound.
struct Range {
    int first_q, queries, rows, len;
};
__device__ __forceinline__ Range range_of(const Args& a, int b) {
    int lo = b, hi = b + 1;
    if (a.starts) {
        lo = a.starts[b];
        hi = a.starts[b + 1];
        if (lo < 0 || hi < lo || hi > a.total_q) {
            raise_status(a.status, ECQ_STATUS_BADARG);
            lo = hi = 0;
        }
    }
    int len = a.lens[b];
    const long long room = static_cast<long long>(a.max_pages) << a.page_shift;
    if (len < 0 || len > room) {
        raise_status(a.status, ECQ_STATUS_BADARG);
        len = len < 0 ? 0 : static_cast<int>(room);
    }
    return {lo, hi - lo, (hi - lo) * a.share, len};
}

// A table's entry; a negative one is as bad as one behind the pool, and -1 is free to mean that there is none.
__device__ __forceinline__ int page_at(const int32_t* p) {
    return static_cast<int>(min(static_cast<uint32_t>(__ldg(p)), static_cast<uint32_t>(INT32_MAX)));
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A row's weights are exp2(score * factor - m), where the reference m is `lift` below the row's largest product. The
// products are exact and m is a float: from 2^27 on m's rounding would carry weights out of fp16, or all of them to 0. So
// rows with such products have a factor that is less by a power of two than their own, and a lift of kFarLift,
// with which m is exact: what fp32 tells apart is then still 4 and more apart, and that is less than its error.
constexpr float kFarLift = 8.f;
__device__ __forceinline__ float power2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ int power_of(float x) { return (__float_as_int(x) >> 23 & 255) - 127; }

constexpr float kNoMax = -FLT_MAX;       // m of a row without scores: below them all
constexpr float kNear = 33554432.f;      // 2^25: m of rows with less is what the plain form makes it

// Raising m for a new largest score, top: m = max(top factor - lift, held), and exp2(held - m) is what earlier weights are
// to be multiplied by. This puts that right for a row that is raised where the new m is beyond kNear, or the factor has gone
// down already.
__device__ __forceinline__ void raise_far(float& m, float& held, float& factor, float top, float own, float lift) {
    const float held_lift = factor == own ? lift : kFarLift;
    const int over = max(power_of(top * own) - 26, 0);
    const float f = own * power2(-over);
    held = (held + held_lift) * power2(power_of(f) - power_of(factor)) - held_lift;
    m = fmaf(top, f, over ? -kFarLift : -lift);
    factor = f;
}
// m as it compares with those of other parts of the row, whose factors may differ.
__device__ __forceinline__ float reference(float m, float factor, float own) {
    return factor == own ? m : (m + kFarLift) * power2(power_of(own) - power_of(factor));
}
__device__ __forceinline__ uint32_t h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 f2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

__device__ __forceinline__ float2 cvt2(uint32_t u, __half) { return f2(u); }
__device__ __forceinline__ float2 cvt2(uint32_t u, __nv_bfloat16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { return h2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Row `row` of a (request, head) in the output.
template <typename T>
__device__ __forceinline__ T* out_row(const Args& a, int first_q, int head, int row) {
    const int i = row / a.share;
    return static_cast<T*>(a.out) + static_cast<int64_t>(first_q + i) * a.o_token +
           static_cast<int64_t>(head * a.share + row - i * a.share) * a.o_head;
}

int32_t launch_prompt(const Args& a, int dtype, int head_dim, int groups, int max_q, cudaStream_t stream);

}  // namespace ecq_kv4

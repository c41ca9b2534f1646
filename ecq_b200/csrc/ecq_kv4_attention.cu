// ecq_kv4_attention.cu -- attention of a few query rows over the 4-bit KV
// cache (ecq_kv4.h has the layout).
//
// Mathematics. With codes c, scales s and zeros z per group G of channels,
//   q . k_j = sum_G s_jG (sum_{d in G} q_d c_jd) + z_jG (sum_{d in G} q_d)
//   o_d     = sum_j (p_j s_jG) c_jd + sum_j p_j z_jG
// so the codes go to the tensor cores as they are: a nibble in the low bits of
// an fp16 is the subnormal c 2^-24, exact, and one in the next four bits is
// c 2^-20; an AND (and a shift by 8 for half of them) makes two operands, where
// scaling every channel would cost a conversion and an fma each. Scales and
// zeros come in per token and group, in fp32. The products are
//   S^T[16 tokens x 8 rows] = K codes x q^T   and   o^T[16 d x 8 rows] = V codes^T x (p s)
// with query rows (tokens x heads that share a cache head) as the narrow side:
// mma.sync m16n8k16 holds 8 rows of keys' work at full use, where a tcgen05
// tile would be 64 or 128 rows, of which a decode step has 1 to 8.
// For fp16 outputs p and p s are fp16 twice (value and remainder: 22 bits), so
// V's side keeps fp32 accuracy. With up to 4 rows the remainders take the
// columns that would be idle: rows n and n + 4 of the narrow side are one row
// (7 % on a decode step of 32 requests). For bf16 they
// are fp16 once: 2^-12 of each weight beside the output's 2^-9, for 30
// instructions fewer of 330. q is scaled to its row's largest power of two and
// exact in fp16.
//
// What bounds it: the latency of instructions that wait for one another, with
// two warps per scheduler (8 per SM, 255 registers each) to hide it. Of ~267
// instructions per 16 tokens and head a scheduler issues one in 39 % of the
// cycles, the ALU is busy in 47 % and the tensor cores in 27 %. For short contexts
// it is launches and joins. Measured: 32 requests of 4-8k tokens, 8 cache heads
// shared by 4: 58 us, 3.9 TB/s of the 6.55 that a copy reaches; one request of
// 131071 tokens, shared by 8: 40 us, 3.8 TB/s; 32 heads of 2049 tokens: 8.9 us,
// 1.0 TB/s; 16 requests of 3-6 tokens and 1.5-4k keys, 8 shared by 4: 48 us.
//
// Layout of the work. The (request, cache head, row tile, unit of 32 or 64 tokens) space
// is flattened and cut into one even range per CTA (one wave of CTAs), from the
// lengths on the device, so ragged batches balance and no host knows them.
// Within a range unit f belongs to warp f % kWarps. Each warp streams its
// units through a ring of its own with cp.async.bulk and
// keeps its own running maximum and sum; at the end of a (request, head, tile)
// the CTA joins its warps in shared memory. Where a range's end cuts one, its
// parts go to the workspace and a second kernel joins them in order, so results
// do not depend on timing.
#include <cuda_runtime.h>

#include <type_traits>

#include "ecq_kv4_attention.cuh"

namespace {

using namespace ecq_kv4;
using ecq_dev::launch_pdl;
using ecq_dev::pdl_launch_dependents;
using ecq_dev::pdl_wait;
using ecq_dev::smem_addr;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// Two CTAs of 4 warps: 8 warps with 255 registers each hide their latencies
// better inside a step than 12 with 168 or 16 with 128 do among themselves (32
// requests of 4-8k tokens: 58, 65 and 71 us).
constexpr int kCtasPerSm = 2;
// Blocks of 16 tokens that a warp takes at a time: what it costs to fetch and
// to wait for them, and the look at the running maximum, are paid once, and
// their products are independent (1, 2 and 4 at a time: 71, 65 and 58 us). With
// four groups four blocks do not fit the registers (16
// requests of 3-6 tokens and four groups: 55 us, with two blocks 48).
__host__ __device__ constexpr int unit_blocks(int groups) { return groups <= 2 ? 4 : 2; }
// A warp takes one tile of 8 rows. Two at once were one pass over the keys for
// 16 rows, but left registers for two blocks a step only, and took as long (128
// pairs of 4096 tokens, 16 rows: 49.6 against 47.4 us).
constexpr int kTileRows = 8;
// Weights are exp2(score - reference + kLift). The reference is raised when a
// score passes it by more than kSlack, so few blocks raise it and the others
// need no reduction over their tokens. The lift keeps the weights of keys far
// below the largest (most of a long context) out of fp16's subnormals, whose
// step of 2^-24 would be felt in sums of thousands of them. weight * scale
// then overflows fp16 from a scale of 16: that is seen, and the unit's weights go
// in times 2^-15 (at most 2^-1 then, for a weight is up to 2^14 where the
// reference's own step is 8: any finite scale's product is finite; what fp16
// loses of them there is 2^-25) and its part of o comes out times 2^15. The
// reference stays as it is: raised by less than a step of its own, it would not
// be what the earlier sums are then multiplied for.
constexpr float kSlack = 2.f, kLift = 10.f;
constexpr int kMostRanks = 8;  // CTAs that share a pair

// How the weights are held: once, twice, or twice in the columns of a row.
enum Weights { kOnce, kTwice, kFolded };
template <int W>
__host__ __device__ constexpr int tile_rows() { return W == kFolded ? 4 : kTileRows; }

__host__ __device__ constexpr int ring_slots(int dim, int groups, int unit, int besides) {
    const int room = 110 * 1024 - kWarps * 8 * (dim + 4) * 4 - besides;
    const int n = room / (kWarps * unit * block_bytes(dim, groups));
    return n < 4 ? n : 4;
}

// One request's part of the work.
struct Request {
    int first_q, queries, rows, len, units, tiles, pairs;
};

template <int TR, int kUnit>  // rows per tile, blocks per unit
__device__ __forceinline__ Request request(const Args& a, int b) {
    const Range x = range_of(a, b);
    Request r = {x.first_q, x.queries, x.rows > a.most_rows ? 0 : x.rows, x.len, 0, 0, 0};
    r.tiles = (r.rows + TR - 1) / TR;
    r.pairs = r.tiles * a.kv_heads;
    // a request without keys has one (empty) unit, so that its rows are written
    constexpr int kUnitTokens = kUnit * kBlockTokens;
    r.units = r.rows ? max((r.len + kUnitTokens - 1) / kUnitTokens, 1) : 0;
    return r;
}

__device__ __forceinline__ long long block_sum(long long v, long long* s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += s[w];
    return v;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// o += t up
__device__ __forceinline__ void add4(float (&o)[4], const float (&t)[4], uint64_t up) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint64_t x = ecq_dev::fma2(ecq_dev::pack2(__float_as_uint(t[i]), __float_as_uint(t[i + 1])), up,
                                         ecq_dev::pack2(__float_as_uint(o[i]), __float_as_uint(o[i + 1])));
        ecq_dev::unpack2(x, o[i], o[i + 1]);
    }
}
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// N words at shared address addr + kAt
template <int N, int kAt>
__device__ __forceinline__ void lds(uint32_t (&w)[N], uint32_t addr) {
    if constexpr (N == 4) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(addr), "n"(kAt));
    } else if constexpr (N == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr), "n"(kAt));
    } else {
        asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(w[0]) : "r"(addr), "n"(kAt));
    }
}

template <typename T>
__device__ __forceinline__ T one(float x);
template <>
__device__ __forceinline__ __half one<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 one<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// V neighbouring channels
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&x)[V]) {
    if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()));
    else *reinterpret_cast<uint32_t*>(p) = pack2(x[0], x[1], T());
}
template <int V>
__device__ __forceinline__ void load(float (&x)[V], const float* p) {
    if constexpr (V == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[0] = v.x, x[1] = v.y;
    }
}
// The query rows of one tile as B operands, and what their scores need.
template <int D, int G>
struct Rows {
    uint32_t b[D / 16][2];
    uint32_t sums[2];  // B operand that takes (scale, zero) pairs: (0, sum of the group's q), high and low part
    float factor[2];   // scale log2(e) 2^24 / the row's power of two, less where scores are huge (raise_far)
    uint32_t own;      // where that is in shared memory as it was
    int limit[2];      // keys that the column's row sees
    int least;         // the smallest limit of rows that exist
};

// A lane's share of the tile's rows as they lie in memory: the loads are issued
// early and set_rows makes the operands of them.
template <typename T, int D, int W>
__device__ __forceinline__ void load_rows(uint4 (&raw)[D / 32], const Args& a, const Request& rq, int head, int tile) {
    const int lane = threadIdx.x & 31, t = lane & 3, n = lane >> 2;
    const int row = W == kFolded ? tile * 4 + (n & 3) : tile * 8 + n, i = row / a.share;
    const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(rq.first_q + i) * a.q_token +
                   static_cast<int64_t>(head * a.share + row - i * a.share) * a.q_head + 8 * t;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
        raw[w] = make_uint4(0, 0, 0, 0);
        if (row < rq.rows) raw[w] = __ldg(reinterpret_cast<const uint4*>(src + 32 * w));
    }
}

template <typename T, int D, int G, int W>
__device__ __forceinline__ void set_rows(Rows<D, G>& R, const uint4 (&raw)[D / 32], const Args& a,
                                         const Request& rq, int tile, float (*own)[2]) {
    const int lane = threadIdx.x & 31, t = lane & 3, n = lane >> 2;
    R.least = rq.len;
    const int row = W == kFolded ? tile * 4 + (n & 3) : tile * 8 + n;
    const bool in = row < rq.rows;
    float x[D / 32][8];
    float top = 0.f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
        const uint32_t us[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = cvt2(us[e], T());
            x[w][2 * e] = f.x;
            x[w][2 * e + 1] = f.y;
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // rows are brought to [2^14, 2^15): elements down to 2^-28 of the largest, and a sixteenth of them, keep
    // their bits in fp16. A negative scale turns the row's sign; with none every score is 0.
    const int ex = top == 0.f ? 0 : max((__float_as_int(top) >> 23) - 127, -100);
    float up = __int_as_float((14 - ex + 127) << 23);
    // the products reach 2^14 (128 channels of 65504 times 2^15, times 2^-24): a factor of up to 2^112 keeps scores
    // finite. What a larger one would tell apart (nonzero differences of products are 2^-72 and more) this one does.
    constexpr float kMostFactor = 5.192296858534828e33f;
    float factor = fabsf(a.scale) * 1.4426950408889634f * (__int_as_float((ex - 14 + 127) << 23) * 16777216.f);
    if (factor > kMostFactor) factor = kMostFactor;
    if (a.scale < 0.f) up = -up;
    if (factor == 0.f) {
        up = 0.f;
        factor = 1.f;
    }
    float sums[G];
#pragma unroll
    for (int g = 0; g < G; ++g) sums[g] = 0.f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[w][e] = __half2float(__float2half_rn(x[w][e] * up));
            sums[w * 32 * G / D] += x[w][e];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            R.b[2 * w + h][0] = h2(x[w][2 * h], x[w][4 + 2 * h]);
            R.b[2 * w + h][1] = h2(x[w][1 + 2 * h] * 0.0625f, x[w][5 + 2 * h] * 0.0625f);
        }
    }
    // query i sees keys up to len - queries + i
    const int limit = in ? rq.len - rq.queries + row / a.share + 1 : rq.len;
    int least = max(limit, 0);
#pragma unroll
    for (int o = 16; o; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
    R.least = min(R.least, least);
    float mine = 0.f;  // lane t has group t's sum (at most 2^22), times 2^-24
#pragma unroll
    for (int g = 0; g < G; ++g) {
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
        if (t == g) mine = sums[g] * 5.9604644775390625e-8f;
    }
    const float high = __half2float(__float2half_rn(mine));
    R.sums[0] = h2(0.f, high);
    R.sums[1] = h2(0.f, mine - high);
#pragma unroll
    for (int c = 0; c < 2; ++c) {  // column 2t + c is row 2t + c of the tile: lane 4 (2t + c) has it
        const int from = 4 * (2 * t + c);
        R.factor[c] = __shfl_sync(0xffffffffu, factor, from);
        R.limit[c] = __shfl_sync(0xffffffffu, limit, from);
    }
    if (n == 0) own[t][0] = R.factor[0], own[t][1] = R.factor[1];
    R.own = smem_addr(own) + 8 * t;
    __syncwarp();
}

// Running softmax of one warp over its blocks.
template <int D, int G>
struct State {
    float o[D / 16][4];
    float sums[2];  // columns 2t, 2t + 1; lanes of row r < G: sum p zero of group r; of row G: sum p
    float m[2];
    bool far;  // some row's factor has gone down
    __device__ __forceinline__ void reset() {
        far = false;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
        sums[0] = sums[1] = 0.f;
        m[0] = m[1] = kNoMax;
    }
};

// The block's token that row i (< 8) of the products stands for. Rows 2t and
// 2t + 1 are tokens t and t + 4, so that what a lane reads for the second lies
// at a constant from the first.
__device__ __forceinline__ int token_of(int i) { return (i >> 1) + 4 * (i & 1); }

// Where a lane's words lie in a block, from the block's start.
template <int D, int G>
struct Lane {
    uint32_t k, k_params, k_pair, v, v_params, v_pair;
    __device__ __forceinline__ Lane() {
        const int lane = threadIdx.x & 31, t = lane & 3, r = lane >> 2;
        k = token_of(r) * (D / 2) + t * (D / 8);
        k_params = k_params_at(D) + token_of(r) * 4 * G;
        k_pair = k_params + 4 * min(t, G - 1);
        v = v_codes_at(D) + t * (D / 2) + r * (D / 16);
        v_params = v_params_at(D, G) + t * 4 * G;
        v_pair = v_params + 4 * min(r, G - 1);
    }
};

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2_rn(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t fma2h(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t abs2(uint32_t a) {
    const __half2 r = __habs2(*reinterpret_cast<const __half2*>(&a));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t neg2(uint32_t a) {
    const __half2 r = __hneg2(*reinterpret_cast<const __half2*>(&a));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// A unit's blocks at shared address at; first[u]: the request's token that
// block u starts with (used with kMask; beyond all limits: leave it out).
template <int D, int G, int U, bool kMask, int kWeights>
__device__ __forceinline__ void blocks(State<D, G>& S, Rows<D, G>& R, const Lane<D, G>& me, uint32_t at,
                                       const int (&first)[U]) {
    constexpr int W = D / 32, BB = block_bytes(D, G);
    const int r = (threadIdx.x & 31) >> 2, tok = token_of(r);
    float s[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        uint32_t k0[W], k1[W], kp[2][G], pair[2][1];
        lds<W, 0>(k0, at + u * BB + me.k);
        lds<W, 8 * (D / 2)>(k1, at + u * BB + me.k);
        lds<G, 0>(kp[0], at + u * BB + me.k_params);
        lds<G, 32 * G>(kp[1], at + u * BB + me.k_params);
        lds<1, 0>(pair[0], at + u * BB + me.k_pair);
        lds<1, 32 * G>(pair[1], at + u * BB + me.k_pair);
        // sum over the groups of zero * (sum of q): the pairs (scale, zero) as they lie are an A operand (lanes past the
        // last group meet zeros in B). Then, per group, the codes.
        constexpr int A = G > 2 ? G : 2;  // accumulators: neighbouring steps go to different ones
        float acc[A][4];
        mma_first(s[u], pair[0][0], pair[1][0], pair[0][0], pair[1][0], R.sums[0], R.sums[1]);
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
            const int n = i % A, step = n * (2 * W / A) + i / A, w = step / 2, h = step % 2;
            const uint32_t x0 = h ? k0[w] >> 8 : k0[w], x1 = h ? k1[w] >> 8 : k1[w];
            const uint32_t a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu, a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
            if (i < A) mma_first(acc[n], a0, a1, a2, a3, R.b[step][0], R.b[step][1]);
            else mma(acc[n], a0, a1, a2, a3, R.b[step][0], R.b[step][1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < A; ++n) {
                const float scale = f2(kp[i][n * G / A]).x;
#pragma unroll
                for (int c = 0; c < 2; ++c) s[u][2 * i + c] = fmaf(scale, acc[n][2 * i + c], s[u][2 * i + c]);
            }
        if (kMask) {
            // a token out of sight, or behind the last, may hold anything: it is chosen away, not computed away
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (first[u] + tok + 8 * (c >> 1) >= R.limit[c & 1]) s[u][c] = -INFINITY;
        }
    }
    float top[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        top[c] = fmaxf(s[0][c], s[0][c + 2]);
#pragma unroll
        for (int u = 1; u < U; ++u) top[c] = fmaxf(top[c], fmaxf(s[u][c], s[u][c + 2]));
    }
    if (__any_sync(0xffffffffu, fmaf(top[0], R.factor[0], -S.m[0]) > kSlack + kLift ||
                                    fmaf(top[1], R.factor[1], -S.m[1]) > kSlack + kLift)) {
        float held[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
            held[c] = S.m[c];
            S.m[c] = fmaxf(fmaf(top[c], R.factor[c], -kLift), held[c]);
        }
        if (S.far || __any_sync(0xffffffffu, fmaxf(fabsf(S.m[0]), fabsf(S.m[1])) > kNear)) {
            uint32_t own[2];
            lds<2, 0>(own, R.own);
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (S.m[c] > held[c]) raise_far(S.m[c], held[c], R.factor[c], top[c], __uint_as_float(own[c]), kLift);
            S.far = S.far || __any_sync(0xffffffffu, R.factor[0] != __uint_as_float(own[0]) || R.factor[1] != __uint_as_float(own[1]));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float keep = exp2_fast(held[c] - S.m[c]);
            S.sums[c] *= keep;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                S.o[i][c] *= keep;
                S.o[i][c + 2] *= keep;
            }
        }
    }
    uint32_t ph[U][2], pl[U][2], hi[U][G][2], lo[U][G][2];
    // the weights and their products with V's scales, those of kDown times 2^-15; the largest of them
    auto weights = [&](auto down) {
        constexpr bool kDown = decltype(down)::value;
        uint32_t most = 0u;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float p[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) p[c] = exp2_fast(fmaf(s[u][2 * i + c], R.factor[c], -S.m[c]));
                const uint32_t x = h2(p[0], p[1]);
                const float2 back = f2(x);
                ph[u][i] = transpose(x);
                if (kWeights != kOnce) pl[u][i] = transpose(h2(p[0] - back.x, p[1] - back.y));
            }
            uint32_t sa[2][G], sb[2][G];
            lds<G, 0>(sa[0], at + u * BB + me.v_params);
            lds<G, 16 * G>(sb[0], at + u * BB + me.v_params);
            lds<G, 32 * G>(sa[1], at + u * BB + me.v_params);
            lds<G, 48 * G>(sb[1], at + u * BB + me.v_params);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t sc = __byte_perm(sa[i][g], sb[i][g], 0x5410);
                    // (weight * scale) in two parts: the product, and what its rounding lost (exact) with the weight's rest
                    constexpr uint32_t kScale = 0x02000200u;  // 2^-15
                    const uint32_t w = kDown ? mul2(ph[u][i], kScale) : ph[u][i];
                    uint32_t h = mul2(w, sc), l = 0u;
                    if (kWeights != kOnce) l = fma2h(kDown ? mul2(pl[u][i], kScale) : pl[u][i], sc, fma2h(w, sc, neg2(h)));
                    if (kMask) {  // weight 0: 0, whatever the scale is
                        const uint32_t keep = (w & 0xffffu ? 0xffffu : 0u) | (w & 0xffff0000u ? 0xffff0000u : 0u);
                        h &= keep;
                        l &= keep;
                    }
                    hi[u][g][i] = kWeights == kFolded && r >= 4 ? l : h;
                    lo[u][g][i] = l;
                    most = max2(most, abs2(h));  // a NaN passes by
                }
        }
        return most;
    };
    const uint32_t most = weights(std::false_type());
    uint64_t up = 0x3f8000003f800000ull;
    if (__any_sync(0xffffffffu, (most & 0xffffu) == 0x7c00u || most >> 16 == 0x7c00u)) {
        weights(std::true_type());
        up = 0x4700000047000000ull;  // 2^15
    }
    // rows of A: the groups' zeros, then ones (the sum of the weights)
    float sums[4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        uint32_t za[2][1], zb[2][1], z[2];
        lds<1, 0>(za[0], at + u * BB + me.v_pair);
        lds<1, 16 * G>(zb[0], at + u * BB + me.v_pair);
        lds<1, 32 * G>(za[1], at + u * BB + me.v_pair);
        lds<1, 48 * G>(zb[1], at + u * BB + me.v_pair);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            z[i] = __byte_perm(za[i][0], zb[i][0], 0x7632);
            if (kMask) {  // where a zero is not finite its scale is not either, and that reaches the rows that see the token
                if ((z[i] & 0x7c00u) == 0x7c00u) z[i] &= 0xffff0000u;
                if ((z[i] & 0x7c000000u) == 0x7c000000u) z[i] &= 0xffffu;
            }
            z[i] = r == G ? 0x3c003c00u : z[i];
        }
        const bool rest = kWeights == kFolded && r >= 4;
        const uint32_t p0 = rest ? pl[u][0] : ph[u][0], p1 = rest ? pl[u][1] : ph[u][1];
        if (u == 0) mma_first(sums, z[0], 0u, z[1], 0u, p0, p1);
        else mma(sums, z[0], 0u, z[1], 0u, p0, p1);
        if (kWeights == kTwice) mma(sums, z[0], 0u, z[1], 0u, pl[u][0], pl[u][1]);
    }
    S.sums[0] += sums[0];
    S.sums[1] += sums[1];
    // The unit's part of o starts from 0 and is added with a rounded fp32 sum: codes are 0..15 and the zeros take about 7.5
    // of that away again, so what a running sum loses to the tensor core's truncation would be many times as much in o.
    constexpr int VW = D / 64;  // words of a lane's chunk of a V row
    uint32_t v[U][4][VW];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        lds<VW, 0>(v[u][0], at + u * BB + me.v);
        lds<VW, 4 * (D / 2)>(v[u][1], at + u * BB + me.v);
        lds<VW, 8 * (D / 2)>(v[u][2], at + u * BB + me.v);
        lds<VW, 12 * (D / 2)>(v[u][3], at + u * BB + me.v);
    }
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t pick = half ? 0x7632u : 0x5410u;
            float t[2][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t x = __byte_perm(v[u][0][w], v[u][1][w], pick), y = __byte_perm(v[u][2][w], v[u][3][w], pick);
#pragma unroll
                for (int part = 0; part < (kWeights == kTwice ? 2 : 1); ++part)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int g = (4 * w + 2 * half + j) * 16 * G / D;
                        const uint32_t xs = j ? x >> 8 : x, ys = j ? y >> 8 : y;
                        const uint32_t a0 = xs & 0x000f000fu, a1 = xs & 0x00f000f0u, a2 = ys & 0x000f000fu, a3 = ys & 0x00f000f0u;
                        const uint32_t(&p)[2] = part ? lo[u][g] : hi[u][g];
                        if (u == 0 && part == 0) mma_first(t[j], a0, a1, a2, a3, p[0], p[1]);
                        else mma(t[j], a0, a1, a2, a3, p[0], p[1]);
                    }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
                add4(S.o[4 * w + 2 * half + j], t[j], up);
        }
}

template <int D, int TR>
__host__ __device__ constexpr int part_floats() { return TR * (D + 2); }

template <typename T, int D, int G, bool kPairs, int kWeights>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_kernel(const Args a, const int tiles) {
    constexpr int kUnit = unit_blocks(G), kUnitTokens = kUnit * kBlockTokens;
    constexpr int TR = tile_rows<kWeights>(), NS = ring_slots(D, G, kUnit, kPairs ? TR * (D + 4) * 4 : 0), BB = block_bytes(D, G),
                  UB = kUnit * BB, OS = D + 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_sum[kWarps];
    __shared__ long long s_before;
    __shared__ int s_request;
    __shared__ Request s_own;
    __shared__ uint64_t s_bar[kWarps][NS];
    __shared__ float s_m[kWarps][8], s_l[kWarps][8];
    __shared__ __align__(8) float s_factor[kWarps][4][2];  // the rows' factors
    float* s_o = reinterpret_cast<float*>(smem + kWarps * NS * UB);
    float* s_part = s_o + kWarps * 8 * OS;  // kPairs: this CTA's part of the pair
    const int lane = threadIdx.x & 31, cta = blockIdx.x;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // the compiler sees that it is one for the warp
    if (lane < NS) ecq_dev::mbar_init(smem_addr(&s_bar[warp][lane]), 1);
    ecq_dev::fence_proxy_async();
    pdl_launch_dependents();
    pdl_wait();

    // which units of which pair come first: number unit0 + mine of (request b, head, tile), then every step-th, `range` in all
    int b, head, tile, unit0 = 0, mine = warp, step = kWarps;
    long long range, each = 0, longer = 0;
    Request rq;
    if constexpr (kPairs) {
        const int ranks = static_cast<int>(ecq_dev::cluster_size()), pair = cta / ranks;
        b = pair / (a.kv_heads * tiles);
        head = pair / tiles - b * a.kv_heads;
        tile = pair % tiles;
        rq = request<TR, kUnit>(a, b);
        // more queries than the call said: their rows are not computed
        if (tile == tiles - 1 && rq.tiles > tiles && threadIdx.x == 0) raise_status(a.status, ECQ_STATUS_BADARG);
        if (tile >= rq.tiles) return;  // the whole cluster
        mine += static_cast<int>(ecq_dev::cluster_rank()) * kWarps;
        step *= ranks;
        range = rq.units;
    } else {
        // this CTA's range of the flattened units, and the request that it starts in
        long long total = 0, weight = 0;
        Request own = {};
        for (int r = threadIdx.x; r < a.batch; r += kThreads) {
            own = request<TR, kUnit>(a, r);
            weight = static_cast<long long>(own.units) * own.pairs;
            total += weight;
        }
        total = block_sum(total, s_sum);
        const long long ctas = min(static_cast<long long>(gridDim.x), (total + kWarps - 1) / kWarps);
        if (threadIdx.x == 0) a.cuts[cta] = make_int4(-1, 0, 0, 0);
        if (cta >= ctas) return;
        // the first `longer` ranges have one unit more
        each = total / ctas;
        longer = total - each * ctas;
        const long long f0 = each * cta + min(static_cast<long long>(cta), longer);
        range = each + (cta < longer);
        long long before = 0;
        for (int first = 0; first < a.batch; first += kThreads) {
            const int r = first + threadIdx.x;
            if (a.batch > kThreads) {  // more than one round: not the last one's any more
                weight = 0;
                if (r < a.batch) {
                    own = request<TR, kUnit>(a, r);
                    weight = static_cast<long long>(own.units) * own.pairs;
                }
            }
            long long incl = weight;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            __syncthreads();
            if (lane == 31) s_sum[warp] = incl;
            if (threadIdx.x == 0) s_request = -1;
            __syncthreads();
            long long start = before + incl - weight;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) start += s_sum[w];
                before += s_sum[w];
            }
            if (weight && start <= f0 && f0 < start + weight) {
                s_request = r;
                s_before = start;
                s_own = own;
            }
            __syncthreads();
            if (s_request >= 0) break;
        }
        if (s_request < 0) return;  // lengths that change meanwhile: no range, but no endless search either
        b = s_request;
        rq = s_own;
        const long long at = f0 - s_before;
        const int pair = static_cast<int>(at / rq.units);
        unit0 = static_cast<int>(at - static_cast<long long>(pair) * rq.units);
        head = pair / rq.tiles;
        tile = pair - head * rq.tiles;
    }

    // where this warp fetches next; the same in all its lanes
    const int shift = a.page_shift - 4;  // blocks per page
    const int page_bytes = BB << shift;
    const int64_t pool_row = static_cast<int64_t>(page_bytes) * a.kv_heads;
    const Request rq0 = rq;
    const int head0 = head, tile0 = tile;
    uint4 raw[D / 32];
    load_rows<T, D, kWeights>(raw, a, rq, head, tile);  // before the ring's copies fill the memory's queues
    int fb = b, f_head = head, f_tile = tile, f_unit = unit0 + mine, f_page[kUnit];
    int f_left = range > mine ? static_cast<int>((range - mine + step - 1) / step) : 0;
    Request fr = rq;
    const int32_t* f_row = a.table + fb * a.table_stride;
    const uint8_t* f_src = a.pages + static_cast<int64_t>(f_head) * page_bytes;
    constexpr uint32_t kAll = (1u << kUnit) - 1u;
    uint32_t f_bad = 0;  // a bit per ring slot and block: its page number is out of range
    int f_slot = 0;
    auto look = [&]() {  // the pages of the next unit, one fetch ahead of their use
        if (f_left <= 0) return;
        while (f_unit >= fr.units) {
            f_unit -= fr.units;
            if (++f_tile == fr.tiles) {
                f_tile = 0;
                if (++f_head == a.kv_heads) {
                    f_head = 0;
                    do {
                        if (++fb >= a.batch) {
                            f_left = 0;
                            return;
                        }
                        fr = request<TR, kUnit>(a, fb);
                    } while (fr.units == 0);
                    f_row = a.table + fb * a.table_stride;
                }
                f_src = a.pages + static_cast<int64_t>(f_head) * page_bytes;
            }
        }
        if (kBlockTokens << shift >= kUnitTokens) {  // a page has the whole unit
            f_page[0] = -1;  // nothing there: the one unit of a request without keys
            if (fr.len) f_page[0] = page_at(f_row + (f_unit * kUnit >> shift));
        } else {
#pragma unroll
            for (int u = 0; u < kUnit; ++u) {
                f_page[u] = -1;
                if ((f_unit * kUnit + u) * kBlockTokens < fr.len)
                    f_page[u] = page_at(f_row + ((f_unit * kUnit + u) >> shift));
            }
        }
    };
    const uint32_t ring = smem_addr(smem) + warp * NS * UB, bars = smem_addr(&s_bar[warp][0]);
    auto fetch = [&]() {
        if (f_left <= 0) return;
        const uint32_t bar = bars + 8 * f_slot, dst = ring + f_slot * UB;
        f_bad &= ~(kAll << kUnit * f_slot);
        const bool one_page = kBlockTokens << shift >= kUnitTokens;
        if (one_page && static_cast<uint32_t>(f_page[0]) < a.n_pages) {
            if (lane == 0) {
                ecq_dev::mbar_expect_tx(bar, UB);
                ecq_dev::bulk_copy_g2s(dst, f_src + f_page[0] * pool_row + ((f_unit * kUnit) & ((1 << shift) - 1)) * BB, UB, bar);
            }
        } else {
            uint32_t there = 0;
#pragma unroll
            for (int u = 0; u < kUnit; ++u) {
                const int page = one_page ? f_page[0] : f_page[u];
                if (page >= 0 && page < a.n_pages) there |= 1u << u;
                else if (page >= 0) f_bad |= 1u << (kUnit * f_slot + u);
            }
            if (lane == 0) {
                ecq_dev::mbar_expect_tx(bar, __popc(there) * BB);
#pragma unroll
                for (int u = 0; u < kUnit; ++u)
                    if (there >> u & 1u)
                        ecq_dev::bulk_copy_g2s(dst + u * BB, f_src + f_page[u] * pool_row + ((f_unit * kUnit + u) & ((1 << shift) - 1)) * BB,
                                               BB, bar);
                if (f_bad) raise_status(a.status, ECQ_STATUS_BADARG);
            }
        }
        f_slot = f_slot + 1 == NS ? 0 : f_slot + 1;
        --f_left;
        f_unit += step;
        look();
    };
    __syncwarp();
    look();
#pragma unroll 1
    for (int i = 0; i < NS; ++i) fetch();

    // segment by segment: what the range has of one (request, head, tile)
    int slot = 0;
    uint32_t phase = 0;
    bool late = false;  // a copy did not come: nothing more is fetched or read
    Rows<D, G> rows;
    State<D, G> st;
    const Lane<D, G> me;
#pragma unroll 1
    for (long long f = 0; f < range;) {
        const int n = static_cast<int>(min(static_cast<long long>(rq.units - unit0), range - f));
        set_rows<T, D, G, kWeights>(rows, raw, a, rq, tile, s_factor[warp]);
        st.reset();
        // this warp's first unit in [f, f + n)
        int i = kPairs ? mine : (warp - static_cast<int>(f % kWarps) + kWarps) % kWarps;
        auto wait = [&]() {
            if (late || __any_sync(0xffffffffu, !ecq_dev::mbar_wait(bars + 8 * slot, phase))) {
                if (!late && lane == 0) raise_status(a.status, ECQ_STATUS_TIMEOUT);
                late = true;
                f_left = 0;
                i = n;
            }
            return !late;
        };
        auto done = [&]() {
            __syncwarp();
            if (++slot == NS) {
                slot = 0;
                phase ^= 1;
            }
            i += step;
            fetch();
        };
        // units that every row sees, then (or between, where a page number is bad) those with a mask
        const int seen = rows.least / kUnitTokens - unit0;
#pragma unroll 1
        while (i < n) {
            int first[kUnit] = {};
#pragma unroll 1
            while (i < min(n, seen) && !(f_bad >> kUnit * slot & kAll)) {
                if (!wait()) break;
                blocks<D, G, kUnit, false, kWeights>(st, rows, me, ring + slot * UB, first);
                done();
            }
            if (i >= n || !wait()) break;
#pragma unroll
            for (int u = 0; u < kUnit; ++u)
                first[u] = f_bad >> (kUnit * slot + u) & 1u ? INT32_MAX - kUnitTokens : (unit0 + i) * kUnitTokens + u * kBlockTokens;
            blocks<D, G, kUnit, true, kWeights>(st, rows, me, ring + slot * UB, first);
            done();
        }
        // the next segment's rows are on their way while the warps join
        const Request now = rq;
        const int b_now = b, head_now = head, tile_now = tile;
        const bool starts = unit0 == 0, ends = unit0 + n == rq.units;
        const long long rest = rq.units - unit0 - n;
        f += n;
        unit0 = 0;
        if (++tile == rq.tiles) {
            tile = 0;
            if (++head == a.kv_heads) head = 0;
        }
        if (!kPairs && f < range) {
            if (head == 0 && tile == 0) {
                do {
                    if (++b >= a.batch) break;
                    rq = request<TR, kUnit>(a, b);
                } while (rq.units == 0);
                if (b >= a.batch) late = true;
            }
            if (!late) load_rows<T, D, kWeights>(raw, a, rq, head, tile);
        }
        float* part = kPairs ? s_part : a.parts + (2 * static_cast<size_t>(cta) + starts) * part_floats<D, TR>();
        if (!kPairs && starts && !ends && threadIdx.x == 0) {
            // how many of the ranges that follow it takes to the pair's end
            const long long k = max(longer - cta - 1, 0ll);
            const long long more = rest <= k * (each + 1) ? (rest + each) / (each + 1) : k + (rest - k * (each + 1) + each - 1) / each;
            a.cuts[cta] = make_int4(b_now, head_now * now.tiles + tile_now, static_cast<int>(more), 0);
        }
        constexpr int V = D / 32;
        const int t = lane & 3, r = lane >> 2;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float z[G];
#pragma unroll
            for (int g = 0; g < G; ++g) z[g] = __shfl_sync(0xffffffffu, st.sums[c], 4 * g + t);
            if (r == 0) s_m[warp][2 * t + c] = st.far ? reference(st.m[c], rows.factor[c], s_factor[warp][t][c]) : st.m[c];
            if (r == G) s_l[warp][2 * t + c] = st.sums[c];
            float* dst = s_o + (warp * 8 + 2 * t + c) * OS + r;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                dst[16 * i] = fmaf(st.o[i][c], 16777216.f, z[i * 16 * G / D]);
                dst[16 * i + 8] = fmaf(st.o[i][c + 2], 1048576.f, z[i * 16 * G / D]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int tr = warp; tr < TR; tr += kWarps) {
            float M = kNoMax, L = 0.f, o[V];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][tr]);
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float k = exp2_fast(s_m[w][tr] - M);
                float x[V], l = s_l[w][tr];
                load<V>(x, s_o + (w * 8 + tr) * OS + V * lane);
                if (kWeights == kFolded) {
                    float y[V];
                    load<V>(y, s_o + (w * 8 + tr + 4) * OS + V * lane);
                    l += s_l[w][tr + 4];
#pragma unroll
                    for (int v = 0; v < V; ++v) x[v] += y[v];
                }
                L = fmaf(k, l, L);
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] = fmaf(k, x[v], o[v]);
            }
            const int qr = tile_now * TR + tr;
            if (qr >= now.rows) continue;
            if (!kPairs && starts && ends) {
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] = L == 0.f ? 0.f : o[v] / L;
                store<T, V>(out_row<T>(a, now.first_q, head_now, qr) + V * lane, o);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) part[TR * 2 + tr * D + V * lane + v] = o[v];
                if (lane == 0) {
                    part[2 * tr] = M;
                    part[2 * tr + 1] = L;
                }
            }
        }
        // a warp that gave up takes the others with it: they would wait for it at the next segment's barriers
        if (__syncthreads_or(late)) late = true, f = range;
    }
    if constexpr (kPairs) {
        // the cluster's parts: rank r joins rows r, r + ranks, ...
        constexpr int V = D / 32;
        const int ranks = static_cast<int>(ecq_dev::cluster_size()), rank = static_cast<int>(ecq_dev::cluster_rank());
        ecq_dev::cluster_sync();
#pragma unroll 1
        for (int tr = rank + warp * ranks; tr < TR; tr += ranks * kWarps) {
            const int qr = tile0 * TR + tr;
            if (qr >= rq0.rows) break;
            float M[kMostRanks], L[kMostRanks], x[kMostRanks][V];
#pragma unroll
            for (int k = 0; k < kMostRanks; ++k) {
                M[k] = kNoMax;
                L[k] = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v) x[k][v] = 0.f;
                if (k < ranks) {
                    M[k] = ecq_dev::ld_cluster_f32(s_part + 2 * tr, k);
                    L[k] = ecq_dev::ld_cluster_f32(s_part + 2 * tr + 1, k);
#pragma unroll
                    for (int v = 0; v < V; ++v) x[k][v] = ecq_dev::ld_cluster_f32(s_part + 2 * TR + tr * D + 32 * v + lane, k);
                }
            }
            float top = kNoMax, sum = 0.f, val[V];
#pragma unroll
            for (int k = 0; k < kMostRanks; ++k) top = fmaxf(top, M[k]);
#pragma unroll
            for (int v = 0; v < V; ++v) val[v] = 0.f;
#pragma unroll
            for (int k = 0; k < kMostRanks; ++k) {
                const float w = exp2_fast(M[k] - top);
                sum = fmaf(w, L[k], sum);
#pragma unroll
                for (int v = 0; v < V; ++v) val[v] = fmaf(w, x[k][v], val[v]);
            }
            T* dst = out_row<T>(a, rq0.first_q, head0, qr) + lane;
#pragma unroll
            for (int v = 0; v < V; ++v) dst[32 * v] = one<T>(sum == 0.f ? 0.f : val[v] / sum);
        }
        ecq_dev::cluster_sync();  // no CTA leaves while another reads its part
    }
    if (late) {
        // let the copies in flight land before the shared memory is given back (a slot without one waits in vain)
        for (int i = 0; i < NS; ++i) ecq_dev::mbar_wait(bars + 8 * i, i < slot ? phase ^ 1u : phase);
    }
}

// CTA i joins the parts of the pair that range i starts and does not end. A
// row's parts are dealt to kJoinWarps / rows warps, whose sums meet in shared
// memory: few rows with many parts (one long request) are the slow case, and
// loads of the same thread would queue up behind one another.
constexpr int kJoinWarps = 32;

template <typename T, int D, int TR>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const Args a) {
    constexpr int kDeal = kJoinWarps / TR, V = D / 32, PF = part_floats<D, TR>();
    __shared__ __align__(16) float s_o[kDeal][TR][D];
    __shared__ float s_l[kDeal][TR], s_m[kDeal][TR];
    pdl_launch_dependents();
    pdl_wait();
    const int4 cut = a.cuts[blockIdx.x];
    if (cut.x < 0) return;
    const int lane = threadIdx.x & 31, row = (threadIdx.x >> 5) % TR, deal = (threadIdx.x >> 5) / TR;
    // the first part is the range's second one, the others the first ones of the ranges that follow: part c is at c * 2 PF
    // from there, but for the first
    const float* parts = a.parts + 2 * static_cast<size_t>(blockIdx.x) * PF;
    const int n = cut.z + 1;
    float M = kNoMax, L = 0.f, o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = 0.f;
    for (int c0 = deal; c0 < n; c0 += 4 * kDeal) {  // four parts at a time
        float m[4], l[4], x[4][V];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + j * kDeal;
            m[j] = kNoMax;
            l[j] = 0.f;
            if (c < n) {
                const float* p = parts + (c ? 2 * static_cast<size_t>(c) * PF : PF);
                m[j] = p[2 * row];
                l[j] = p[2 * row + 1];
                load<V>(x[j], p + 2 * TR + row * D + V * lane);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) x[j][v] = 0.f;
            }
        }
        float top = M;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, m[j]);
        const float keep = exp2_fast(M - top);
        M = top;
        L *= keep;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] *= keep;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float k = exp2_fast(m[j] - top);
            L = fmaf(k, l[j], L);
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] = fmaf(k, x[j][v], o[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) s_o[deal][row][V * lane + v] = o[v];
    if (lane == 0) {
        s_m[deal][row] = M;
        s_l[deal][row] = L;
    }
    __syncthreads();
    const Request rq = request<TR, 1>(a, cut.x);
    if (rq.rows == 0) return;
    const int head = cut.y / rq.tiles, tile = cut.y - head * rq.tiles;
    const int tr = threadIdx.x >> 5, qr = tile * TR + tr;
    if (tr >= TR || qr >= rq.rows) return;
    float top = kNoMax, sum = 0.f, val[V];
#pragma unroll
    for (int k = 0; k < kDeal; ++k) top = fmaxf(top, s_m[k][tr]);
#pragma unroll
    for (int v = 0; v < V; ++v) val[v] = 0.f;
#pragma unroll
    for (int k = 0; k < kDeal; ++k) {
        const float w = exp2_fast(s_m[k][tr] - top);
        float x[V];
        load<V>(x, s_o[k][tr] + V * lane);
        sum = fmaf(w, s_l[k][tr], sum);
#pragma unroll
        for (int v = 0; v < V; ++v) val[v] = fmaf(w, x[v], val[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) val[v] = sum == 0.f ? 0.f : val[v] / sum;
    store<T, V>(out_row<T>(a, rq.first_q, head, qr) + V * lane, val);
}

int grid_ctas() { return kCtasPerSm * ecq_dev::sm_count_cached(); }

// Requests with up to so many rows (queries times heads that share a cache
// head) are streamed by attention_kernel, those with more are the prompt
// kernel's; a call that may have such launches both. A row costs the stream
// kernel the same wherever it is, the prompt kernel works by 256 rows of a pair
// on one SM: many pairs fill the GPU with those, few do not. Measured (us,
// stream / prompt kernel, shared by 4): 128 pairs of 4096 tokens 32 rows
// 79 / 85; 32 pairs of 8192 96 rows 106 / 146; 8 pairs of 65536 256 rows
// 481 / 1139: they meet at about 4500 rows of all pairs.
int stream_rows(int batch, int kv_heads) {
    const int64_t rows = 4500 / (static_cast<int64_t>(batch) * kv_heads);
    return rows > 32 ? static_cast<int>(rows) : 32;
}

// CTAs of a cluster for each (request, head, tile); 0: ranges instead. Ranges
// balance lengths that differ and spread a few long requests over the GPU, at
// the price of a look at all lengths, and of a second kernel that joins what
// was cut. Clusters have neither, and are taken where that counts: all of them
// fit on the GPU at once, and the longest request that the tables have room for
// is a few steps of its cluster's warps (7b step, 32 pairs of up to 2112 tokens:
// 13.8 us with ranges, 8.9 with clusters).
constexpr int kMostTokens = 192;  // per warp
struct Plan {
    int most_rows;  // of a request that is streamed
    bool prompts;   // some may have more
    int rows;       // of a tile
    int tiles;      // of a streamed request at most
    int ranks;      // CTAs of a cluster; 0: ranges
};
Plan plan(int batch, int kv_heads, int share, int max_q, int max_pages, int page_size, int dtype) {
    Plan p;
    const int64_t rows = static_cast<int64_t>(share) * max_q;
    p.most_rows = stream_rows(batch, kv_heads);
    p.prompts = rows > p.most_rows;
    if (!p.prompts) p.most_rows = INT32_MAX;
    p.rows = rows <= 4 && dtype == ECQ_KV4_F16 ? 4 : 8;
    p.tiles = static_cast<int>(((rows < p.most_rows ? rows : p.most_rows) + p.rows - 1) / p.rows);
    const int64_t pairs = static_cast<int64_t>(batch) * kv_heads * p.tiles;
    p.ranks = kMostRanks;
    while (p.ranks && pairs * p.ranks > grid_ctas()) p.ranks /= 2;
    if (static_cast<int64_t>(max_pages) * page_size > kMostTokens * p.ranks * kWarps) p.ranks = 0;
    return p;
}

template <typename L, int W>
int32_t launch(const Args& a, const Plan& plan, cudaStream_t stream) {
    using T = typename L::T;
    constexpr int kUnit = unit_blocks(L::G), UB = kUnit * block_bytes(L::D, L::G), join = kWarps * 8 * (L::D + 4) * 4, part = tile_rows<W>() * (L::D + 4) * 4;
    if (plan.ranks) {
        constexpr int smem = kWarps * ring_slots(L::D, L::G, kUnit, part) * UB + join + part;
        const auto kernel = attention_kernel<T, L::D, L::G, true, W>;
        if (!ecq_dev::ensure_smem_limit(reinterpret_cast<const void*>(kernel), smem)) return ECQ_ERR_CUDA;
        const unsigned ctas = static_cast<unsigned>(a.batch * a.kv_heads * plan.tiles * plan.ranks);
        return result(
            ecq_dev::launch_pdl_cluster(kernel, dim3(ctas), dim3(kThreads), smem, stream, plan.ranks, a, plan.tiles));
    }
    constexpr int smem = kWarps * ring_slots(L::D, L::G, kUnit, 0) * UB + join;
    const auto kernel = attention_kernel<T, L::D, L::G, false, W>;
    if (!ecq_dev::ensure_smem_limit(reinterpret_cast<const void*>(kernel), smem)) return ECQ_ERR_CUDA;
    const dim3 grid(grid_ctas());
    cudaError_t rc = launch_pdl(kernel, grid, dim3(kThreads), smem, stream, a, 0);
    if (rc == cudaSuccess) rc = launch_pdl(join_kernel<T, L::D, tile_rows<W>()>, grid, dim3(kJoinWarps * 32), 0, stream, a);
    return result(rc);
}

}  // namespace

extern "C" {

int64_t ecq_kv4_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_q, int32_t max_pages, int32_t page_size) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || max_q < 1 || max_pages < 1)
        return ECQ_ERR_ARG;
    if (!sizes_ok(head_dim, page_size, 32) || heads / kv_heads > 64) return ECQ_ERR_UNSUPPORTED;
    // the same clusters or ranges for both types: tiles of 4 rows are taken where there is one tile of 8
    const Plan p = plan(batch, kv_heads, heads / kv_heads, max_q, max_pages, page_size, ECQ_KV4_BF16);
    return p.ranks ? 0 : grid_ctas() * (16 + 2 * 4 * 8ll * (head_dim + 2));
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
    if (static_cast<int64_t>(total_q) * (heads / kv_heads) >= (1ll << 31)) return ECQ_ERR_UNSUPPORTED;
    if (!q || !out || !aligned(q, 16) || !aligned(out, 8)) return ECQ_ERR_ARG;
    if (((q_token_stride | q_head_stride) & 7) || ((out_token_stride | out_head_stride) & 3)) return ECQ_ERR_ARG;
    if (need && (workspace_bytes < need || !workspace || !aligned(workspace, 16))) return ECQ_ERR_WORKSPACE;
    const Plan p = plan(batch, kv_heads, heads / kv_heads, max_q, max_pages, page_size, dtype);
    Args a;
    a.q = q;
    a.out = out;
    a.pages = static_cast<const uint8_t*>(pages);
    a.table = static_cast<const int32_t*>(block_table);
    a.lens = static_cast<const int32_t*>(seq_lens);
    a.starts = static_cast<const int32_t*>(q_starts);
    a.cuts = static_cast<int4*>(workspace);
    a.parts = reinterpret_cast<float*>(a.cuts + grid_ctas());
    a.status = static_cast<int32_t*>(status);
    a.q_token = q_token_stride;
    a.q_head = q_head_stride;
    a.o_token = out_token_stride;
    a.o_head = out_head_stride;
    a.n_pages = n_pages;
    a.table_stride = table_stride;
    a.kv_heads = kv_heads;
    a.share = heads / kv_heads;
    a.page_shift = log2i(page_size);
    a.max_pages = max_pages;
    a.batch = batch;
    a.total_q = total_q;
    a.scale = scale;
    a.most_rows = p.most_rows;
    if (p.prompts) {
        const int32_t rc = launch_prompt(a, dtype, head_dim, head_dim / group_size, max_q, static_cast<cudaStream_t>(stream));
        if (rc != ECQ_OK) return rc;
    }
    return by_layout(dtype, head_dim, head_dim / group_size, [&](auto layout) {
        using L = decltype(layout);
        const auto st = static_cast<cudaStream_t>(stream);
        if constexpr (std::is_same<typename L::T, __half>::value) {
            return p.rows == 4 ? launch<L, kFolded>(a, p, st) : launch<L, kTwice>(a, p, st);
        } else {
            return launch<L, kOnce>(a, p, st);
        }
    });
}

}  // extern "C"

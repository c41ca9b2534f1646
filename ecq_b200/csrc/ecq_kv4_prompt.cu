// ecq_kv4_prompt.cu -- attention of many query rows (prompt chunks) over the
// 4-bit KV cache, on the tcgen05 tensor cores.
//
// A CTA takes 256 rows (queries x heads that share a cache head) of one
// (request, cache head) as two tiles of 128 and walks the keys 64 at a time:
//   loader   one warp copies the packed blocks of 16 tokens into a ring
//            (cp.async.bulk, a lane per block, its page number read one step
//            ahead);
//   decoders four warps turn codes into fp16 K [64 x D] and four into V^T [D x
//            64], in the tensor core's K-major, no-swizzle layout: code * scale +
//            zero, rounded once to fp16, shared by all 256 rows;
//   MMA      one warp issues S = Q K^T and O += P V for both tiles;
//   softmax  eight warps per tile, two threads per row with 32 keys each: S from
//            tensor memory (its place is free for the next step's scores at
//            once), running maximum (the two threads exchange theirs; it is
//            raised only when a score passes it by 2^8, and the row's O is
//            rescaled then), exp2, P as fp16 to tensor memory, sums in fp32. With
//            one thread per row the warps' own latencies took twice the time of
//            the exponentials.
// So the next scores and the last step's O += P V are made while the
// exponentials of a step are computed. Tensor memory is full (512 columns): Q
// of the first tile, S, P and O of both; the second tile's Q lies in shared
// memory (its scores then read both operands there: 384 cycles a step instead
// of 256).
//
// fp16 for K, V and P costs a relative 2^-12 on average of each, next to the
// output's own rounding; q is brought to its row's power of two and keeps its
// bits. A group whose scale was rounded up holds values past fp16's end, up to
// 65584 where ecq_kv4_append wrote it: they count as 65504 (2^-9 less at most),
// which a look at code 15's value of each group finds.
//
// What bounds it: instructions and the exponentials (16 a cycle and SM: 1024
// cycles a step at D = 128, the products 1152, measured 2250). Measured: 37
// heads, 1024 rows and 32768 keys 606 us, 1050 TFLOP/s of 1718; four prompt
// chunks of 500-632 tokens with 2.5-4k keys, 32 heads 158 us, 922 TFLOP/s: two
// waves of CTAs, each of which starts and ends alone on its SM.
//
// Masks. Keys beyond a row's own are chosen away in S. A V row whose scale or
// zero is not finite would reach rows that do not see it (0 * NaN), so it
// enters as 0 and the first such token per group of channels is remembered:
// rows that see it get NaN there at the end. Keys of a page whose
// number is bad are left out.
//
// Every wait is bounded and looks at a flag that a wait sets which gave up; all
// roles then leave, and tensor memory is given back after the products in
// flight.
#include <cuda_runtime.h>
#include <stddef.h>

#include "ecq_kv4_attention.cuh"

namespace {

using namespace ecq_kv4;
using ecq_dev::bulk_copy_g2s;
using ecq_dev::fence_proxy_async;
using ecq_dev::mbar_expect_tx;
using ecq_dev::mbar_init;
using ecq_dev::smem_addr;

constexpr int kKeys = 64;                       // keys a step
constexpr int kTileBlocks = kKeys / kBlockTokens;
constexpr int kRows = 128, kCtaRows = 2 * kRows;
constexpr int kSoftmaxWarps = 16, kDecodeWarps = 8;  // decoders: four for K, four for V
constexpr int kThreads = (kSoftmaxWarps + kDecodeWarps + 2) * 32;
constexpr int kHalf = kKeys / 2;                // keys of a step that a softmax thread takes
constexpr int kMmaWarp = kSoftmaxWarps + kDecodeWarps;  // the loader is the one behind it
constexpr int kRing = 4;
constexpr uint32_t kTmemColumns = 512;
// P is exp2(score - reference + kLift), at most 2^15; the lift keeps the weights of keys far below the largest out of
// fp16's subnormals
constexpr float kSlack = 8.f, kLift = 7.f;

template <int D, int G>
struct Smem {
    static constexpr int kPacked = kTileBlocks * block_bytes(D, G);
    // K: core columns of 8 channels, 64 keys of 16 bytes each; 32 more bytes put a warp's stores in different banks
    static constexpr uint32_t kLboK = kKeys * 16 + 32, kBytesK = D / 8 * kLboK;
    static constexpr uint32_t kLboV = D * 16, kBytesV = kKeys / 8 * kLboV;
    // Q of both tiles: the first one's on its way to tensor memory; a tile's output at the end. 16 more bytes a core column:
    // a warp writes rows
    static constexpr uint32_t kLboQ = kRows * 16 + 16, kBytesQ = D / 8 * kLboQ;
    static constexpr int kRingAt = 0, kAtK = kRing * kPacked, kAtV = kAtK + 2 * kBytesK, kAtQ = kAtV + 2 * kBytesV,
                         kBytes = kAtQ + 2 * kBytesQ;
};

// Tensor memory columns (of tile x)
struct Tmem {
    static constexpr uint32_t kQ = 0;
    static __device__ constexpr uint32_t s(int x) { return 64 + x * 64; }
    static __device__ constexpr uint32_t p(int x) { return 192 + x * 32; }
    static __device__ constexpr uint32_t o(int x) { return 256 + x * 128; }
};

struct Control {
    uint64_t packed_full[kRing], packed_empty[kRing];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_full[2], s_full[2], s_read[2], p_full[2], p_read[2], drained;
    uint64_t rows[2];        // a tile's q is in shared memory
    uint64_t pair[8];        // of the two warps that share 32 rows
    float top[2][2][2 * kRows], sum[2][2 * kRows];  // by step parity and half: a row's maximum; by half: its sum
    float factor[2 * kRows];
    uint32_t tmem, gave_up;
    uint32_t hidden[8];  // by step: a bit per block where nothing is, or a bad page (the loader is at most 6 steps ahead of a softmax)
    int poison[4];           // per group: the first token whose V is not finite
};

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
// The whole warp comes here and one lane issues: what the instruction takes from
// uniform registers stays in them (issued under a branch on the lane, a product
// took 90 cycles to issue, which is three times what it takes to run).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ uint64_t kmajor(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | (static_cast<uint64_t>((lbo >> 4) & 0x3fffu) << 16) |
           (static_cast<uint64_t>((sbo >> 4) & 0x3fffu) << 32) | (1ull << 46);
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* v) {  // 32 columns of this thread's lane
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t lds1(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint4 lds4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}

// Waits for a phase of bar; false (and everybody told) after the limit, or
// where another wait gave up. (A time hint at the wait makes it a loop of
// sleeps, which cost a third of the speed.)
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up, int32_t* status) {
    const uint64_t t0 = ecq_dev::global_timer_ns();
    for (;;) {
        if (ecq_dev::mbar_try_wait(bar, parity)) return true;
        if (*gave_up) return false;
        if (ecq_dev::global_timer_ns() - t0 > ecq_dev::kWaitLimitNs) {
            *gave_up = 1u;
            raise_status(status, ECQ_STATUS_TIMEOUT);
            return false;
        }
    }
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up, int32_t* status) {
    return ecq_dev::mbar_try_wait(bar, parity) || wait_longer(bar, parity, gave_up, status);
}

__device__ __forceinline__ uint32_t hfma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t hadd(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Held to +-65504; a NaN stays one.
__device__ __forceinline__ uint32_t hold(uint32_t x) {
    asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7bff7bffu));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xfbfffbffu));
    return x;
}
// 0 where both halves of x are finite (their products with 0, summed up), else NaN in one of them
__device__ __forceinline__ uint32_t not_finite(uint32_t x, uint32_t before) { return hfma(x, 0u, before); }
__device__ __forceinline__ bool any_nan(uint32_t probe) { return (probe & 0x7fff7fffu) != 0u; }
constexpr uint32_t kTop = 0x4b804b80u;  // 15, twice: a group's values are finite where its first and its last are
// code * scale + zero of the nibbles at bits 0..3 (low) or 4..7 of both halves
// of x: a nibble in the mantissa of 1024 is 1024 + code (or 1024 + 16 code),
// what takes that off is exact, and the fma rounds once.
__device__ __forceinline__ uint32_t value_low(uint32_t x, uint32_t scale, uint32_t zero) {
    return hfma(hadd((x & 0x000f000fu) | 0x64006400u, 0xe400e400u), scale, zero);
}
__device__ __forceinline__ uint32_t value_high(uint32_t x, uint32_t scale, uint32_t zero) {
    return hfma(hfma((x & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd400d400u), scale, zero);
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const Args a) {
    using S = Smem<D, G>;
    using M = Tmem;
    constexpr int BB = block_bytes(D, G);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Control ctl;
    const uint32_t bars = smem_addr(&ctl);  // once: each look at a shared variable's address costs three instructions
    const int lane = threadIdx.x & 31;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    volatile uint32_t* gave_up = &ctl.gave_up;

    ecq_dev::pdl_wait();
    // this CTA's request and tile: every request has as many tiles as its rows fill, and the grid is as large as all rows
    // together may need. Last tiles, which see the most keys, come first.
    const int head = blockIdx.x % a.kv_heads;
    const int items = gridDim.x / a.kv_heads, item = items - 1 - static_cast<int>(blockIdx.x / a.kv_heads);
    __shared__ int s_sum[kThreads / 32], s_request, s_tile;
    if (threadIdx.x == 0) s_request = -1;
    int before = 0;
    for (int first = 0; first < a.batch && (before <= item || blockIdx.x == 0); first += kThreads) {
        const int r = first + threadIdx.x;
        int mine = 0;
        if (r < a.batch) {
            const int rows = range_of(a, r).rows;
            if (rows > a.most_rows) mine = (rows + kCtaRows - 1) / kCtaRows;
        }
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int start = before + incl - mine;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) start += s_sum[w];
            before += s_sum[w];
        }
        if (start <= item && item < start + mine) {
            s_request = r;
            s_tile = item - start;
        }
    }
    __syncthreads();
    // more queries than the call said: some rows are not computed
    if (blockIdx.x == 0 && threadIdx.x == 0 && before > items) raise_status(a.status, ECQ_STATUS_BADARG);
    const int b = s_request, tile = s_tile;
    const bool work = b >= 0;
    const Range rq = range_of(a, max(b, 0));
    if (!work) {
        ecq_dev::pdl_launch_dependents();
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init((bars + offsetof(Control, packed_full) + 8 * (i)), kTileBlocks);
            mbar_init((bars + offsetof(Control, packed_empty) + 8 * (i)), kDecodeWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init((bars + offsetof(Control, k_full) + 8 * (i)), kDecodeWarps * 16);
            mbar_init((bars + offsetof(Control, v_full) + 8 * (i)), kDecodeWarps * 16);
            mbar_init((bars + offsetof(Control, k_empty) + 8 * (i)), 1);
            mbar_init((bars + offsetof(Control, v_empty) + 8 * (i)), 1);
            mbar_init((bars + offsetof(Control, q_full) + 8 * (i)), 2 * kRows);
            mbar_init((bars + offsetof(Control, s_full) + 8 * (i)), 1);
            mbar_init((bars + offsetof(Control, s_read) + 8 * (i)), 2 * kRows);
            mbar_init((bars + offsetof(Control, p_full) + 8 * (i)), 2 * kRows);
            mbar_init((bars + offsetof(Control, p_read) + 8 * (i)), 1);
        }
        mbar_init(bars + offsetof(Control, drained), 1);
        for (int i = 0; i < 2; ++i) mbar_init(bars + offsetof(Control, rows) + 8 * i, kSoftmaxWarps / 2);
        for (int i = 0; i < 8; ++i) mbar_init((bars + offsetof(Control, pair) + 8 * (i)), 2);
        ctl.gave_up = 0u;
        for (int g = 0; g < 4; ++g) ctl.poison[g] = INT32_MAX;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&ctl.tmem)),
                     "r"(kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, ctl.tmem, 0);
    ecq_dev::pdl_launch_dependents();  // after the allocation: the next kernel may want tensor memory too

    // steps of the two tiles
    int n[2] = {0, 0};
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int first = tile * kCtaRows + x * kRows, last = min(rq.rows, first + kRows) - 1;
        if (first < rq.rows) n[x] = (max(rq.len - rq.queries + last / a.share + 1, 0) + kKeys - 1) / kKeys;
    }
    // one for the warp, as the compiler can see: the products' operands stay in uniform registers
    n[0] = __shfl_sync(0xffffffffu, n[0], 0);
    n[1] = __shfl_sync(0xffffffffu, n[1], 0);
    const int steps = max(n[0], n[1]);
    const uint32_t base = smem_addr(smem);

    if (warp < kSoftmaxWarps) {
        // ---------------------------------------------------------------- softmax: two threads per row
        const int x = warp / 8, h = warp / 4 & 1, here = x * kRows + (warp & 3) * 32 + lane, row = tile * kCtaRows + x * kRows + (warp & 3) * 32 + lane;
        const bool in = row < rq.rows;
        const int i = row / a.share;
        const uint32_t mine = tmem + ((warp & 3) << 21);  // lanes 32 (warp % 4) ..
        const int limit = in ? rq.len - rq.queries + i + 1 : 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, int parity) {
            ok = __all_sync(0xffffffffu, wait_for(bar, parity, gave_up, a.status));
            return ok;
        };
        // q: a group of D / 8 lanes takes a row (all loads at once), brings it to its power of two and writes it to shared
        // memory in the order of a K row's decoded nibbles: of 8 channels 0 4 1 5 2 6 3 7
        {
            constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kLoads = 16 / kAtOnce;  // 16 rows a warp
            const int c = lane % kLanes;
            uint4 u[kLoads];
#pragma unroll
            for (int e = 0; e < kLoads; ++e) {
                const int at = (warp & 7) * 16 + e * kAtOnce + lane / kLanes, qr = tile * kCtaRows + x * kRows + at;
                u[e] = make_uint4(0, 0, 0, 0);
                if (qr < rq.rows) {
                    const int qi = qr / a.share;
                    const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(rq.first_q + qi) * a.q_token +
                                   static_cast<int64_t>(head * a.share + qr - qi * a.share) * a.q_head;
                    u[e] = __ldg(reinterpret_cast<const uint4*>(src) + c);
                }
            }
#pragma unroll
            for (int e = 0; e < kLoads; ++e) {
                const int at = (warp & 7) * 16 + e * kAtOnce + lane / kLanes;
                const float2 f0 = cvt2(u[e].x, T()), f1 = cvt2(u[e].y, T()), f2 = cvt2(u[e].z, T()), f3 = cvt2(u[e].w, T());
                float top = fmaxf(fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y))),
                                  fmaxf(fmaxf(fabsf(f2.x), fabsf(f2.y)), fmaxf(fabsf(f3.x), fabsf(f3.y))));
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const int ex = top == 0.f ? 0 : max((__float_as_int(top) >> 23) - 127, -100);
                float up = __int_as_float((10 - ex + 127) << 23);
                float f = fabsf(a.scale) * 1.4426950408889634f * __int_as_float((ex - 10 + 127) << 23);
                // the products reach 2^34 (128 channels of 65504 times 2^11): a factor of up to 2^93 keeps scores
                // finite, and tells apart all that a larger one would (nonzero differences are 2^-48 and more)
                constexpr float kMostFactor = 9.903520314283042e27f;
                if (f > kMostFactor) f = kMostFactor;
                if (a.scale < 0.f) up = -up;
                if (f == 0.f) {
                    up = 0.f;
                    f = 1.f;
                }
                if (c == 0) ctl.factor[x * kRows + at] = f;
                sts4(base + S::kAtQ + x * S::kBytesQ + c * S::kLboQ + at * 16, pack2(f0.x * up, f2.x * up, __half()),
                     pack2(f0.y * up, f2.y * up, __half()), pack2(f1.x * up, f3.x * up, __half()),
                     pack2(f1.y * up, f3.y * up, __half()));
            }
            if (x == 1) {
                fence_proxy_async();
                mbar_arrive(bars + offsetof(Control, q_full) + 8);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + offsetof(Control, rows) + 8 * x);
            wait(bars + offsetof(Control, rows) + 8 * x, 0);
        }
        float factor = *reinterpret_cast<volatile float*>(&ctl.factor[here]);
        if (x == 0 && ok) {  // this thread's half of the row's channels to tensor memory
#pragma unroll
            for (int part = 0; part < D / 64; ++part) {
                if (part != h % (D / 64)) continue;
                uint32_t v[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 u = lds4(base + S::kAtQ + (8 * part + c) * S::kLboQ + here * 16);
                    v[4 * c] = u.x, v[4 * c + 1] = u.y, v[4 * c + 2] = u.z, v[4 * c + 3] = u.w;
                }
                tmem_st(mine + M::kQ + 32 * part, v);
            }
            wait_st();
            before_sync();
            mbar_arrive(bars + offsetof(Control, q_full));
        }
        float m = kNoMax;
        uint64_t l[2] = {0ull, 0ull};  // two pairs of sums
        const uint32_t pair = (bars + offsetof(Control, pair) + 8 * (x * 4 + (warp & 3)));
        int j = 0;
#pragma unroll 1
        for (; ok && j < n[x]; ++j) {
            if (!wait((bars + offsetof(Control, s_full) + 8 * (x)), j & 1)) break;
            after_sync();
            uint32_t s[kHalf];
            tmem_ld(mine + M::s(x) + kHalf * h, s);
            wait_ld();
            before_sync();
            mbar_arrive((bars + offsetof(Control, s_read) + 8 * (x)));
            const uint32_t hidden = *reinterpret_cast<volatile uint32_t*>(&ctl.hidden[j & 7]) >> (h * kTileBlocks / 2);
            const int left = limit - j * kKeys - h * kHalf;  // of this thread's keys those that the row sees
            if (__any_sync(0xffffffffu, left < kHalf) || hidden) {
#pragma unroll
                for (int k = 0; k < kHalf; ++k)
                    if (k >= left || (hidden >> (k / kBlockTokens) & 1u)) s[k] = 0xff800000u;
            }
            float t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = __uint_as_float(s[k]);
#pragma unroll
            for (int k = 4; k < kHalf; ++k) t[k & 3] = fmaxf(t[k & 3], __uint_as_float(s[k]));
            float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
            volatile float* tops = &ctl.top[j & 1][0][0];
            tops[h * 2 * kRows + here] = top;
            __syncwarp();
            if (lane == 0) mbar_arrive(pair);
            if (!wait(pair, j & 1)) break;
            top = fmaxf(top, tops[(h ^ 1) * 2 * kRows + here]);
            bool emptied = j == 0;  // P and O are not in use by the last step's product
            if (__any_sync(0xffffffffu, fmaf(top, factor, -m) > kSlack + kLift)) {
                float held = m;
                m = fmaxf(fmaf(top, factor, -kLift), held);
                const bool far = (fabsf(m) > kNear && m != kNoMax) || (fabsf(held) > kNear && held != kNoMax);
                if (__any_sync(0xffffffffu, far) && m > held)
                    raise_far(m, held, factor, top, *reinterpret_cast<volatile float*>(&ctl.factor[here]), kLift);
                const float keep = exp2_fast(held - m);
                const uint64_t k2 = ecq_dev::pack2(__float_as_uint(keep), __float_as_uint(keep));
#pragma unroll
                for (int u = 0; u < 2; ++u) l[u] = ecq_dev::fma2(l[u], k2, 0ull);
                if (j) {
                    if (!wait((bars + offsetof(Control, p_read) + 8 * (x)), (j - 1) & 1)) break;
                    after_sync();
                    emptied = true;
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 16) {  // this thread's half of the channels
                        uint32_t o[16];
                        tmem_ld16(mine + M::o(x) + h * (D / 2) + c, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_st16(mine + M::o(x) + h * (D / 2) + c, o);
                    }
                }
            }
            const uint64_t f2x = ecq_dev::pack2(__float_as_uint(factor), __float_as_uint(factor));
            const uint64_t m2 = ecq_dev::pack2(__float_as_uint(-m), __float_as_uint(-m));
#pragma unroll
            for (int k = 0; k < kHalf; k += 2) {
                float e0, e1;
                ecq_dev::unpack2(ecq_dev::fma2(ecq_dev::pack2(s[k], s[k + 1]), f2x, m2), e0, e1);
                e0 = exp2_fast(e0);
                e1 = exp2_fast(e1);
                l[k / 2 % 2] = ecq_dev::add2(l[k / 2 % 2], ecq_dev::pack2(__float_as_uint(e0), __float_as_uint(e1)));
                s[k / 2] = pack2(e0, e1, __half());
            }
            if (!emptied) {
                if (!wait((bars + offsetof(Control, p_read) + 8 * (x)), (j - 1) & 1)) break;
                after_sync();
            }
            tmem_st16(mine + M::p(x) + kHalf / 2 * h, s);
            wait_st();
            before_sync();
            mbar_arrive((bars + offsetof(Control, p_full) + 8 * (x)));
        }
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float e0, e1;
            ecq_dev::unpack2(l[u], e0, e1);
            sum += e0 + e1;
        }
        if (ok && n[x]) {
            volatile float* sums = &ctl.sum[0][0];
            sums[h * 2 * kRows + here] = sum;
            __syncwarp();
            if (lane == 0) mbar_arrive(pair);
            if (wait(pair, j & 1)) {
                sum += sums[(h ^ 1) * 2 * kRows + here];
                wait((bars + offsetof(Control, p_read) + 8 * (x)), (j - 1) & 1);
            }
            after_sync();
        }
        if (ok) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            // this warp's 32 rows and half of the channels through its part of the tile's q (no product reads that any
            // more), so that rows are stored together
            constexpr int kBytesRow = D, kChunks = kBytesRow / 16;
            const uint32_t mem = base + S::kAtQ + x * S::kBytesQ + (warp & 7) * 32 * kBytesRow;
            auto chunk = [&](int r, int c) { return mem + r * kBytesRow + ((c ^ (r * kBytesRow / 128)) & (kChunks - 1)) * 16; };
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
                uint32_t o[16];
                if (n[x]) {
                    tmem_ld16(mine + M::o(x) + h * (D / 2) + c, o);
                    wait_ld();
                }
                if (limit > ctl.poison[(h * (D / 2) + c) * G / D]) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = 0x7fc00000u;
                }
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = sum == 0.f ? 0u : pack2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv, T());
                sts4(chunk(lane, c / 8), v[0], v[1], v[2], v[3]);
                sts4(chunk(lane, c / 8 + 1), v[4], v[5], v[6], v[7]);
            }
            __syncwarp();
            constexpr int kLanes = kBytesRow / 8, kAtOnce = 32 / kLanes;  // 8 bytes a lane
            const int e = lane % kLanes, row0 = tile * kCtaRows + x * kRows + (warp & 3) * 32;
#pragma unroll 4
            for (int r = lane / kLanes; r < 32; r += kAtOnce) {
                const uint2 v = lds2(chunk(r, e / 2) + (e & 1) * 8);
                if (row0 + r < rq.rows)
                    *reinterpret_cast<uint2*>(out_row<T>(a, rq.first_q, head, row0 + r) + h * (D / 2) + 4 * e) = v;
            }
        }
    } else if (warp < kMmaWarp) {
        // ---------------------------------------------------------------- decoders
        const int tid = threadIdx.x - kSoftmaxWarps * 32;
        if (warp < kSoftmaxWarps + kDecodeWarps / 2) {
            // K: key tid / 4 (and 32 more), a quarter of its channels
            const int t = tid & 3;
            const uint32_t from = base + S::kRingAt + (tid / 64) * BB + (tid / 4 % kBlockTokens) * (D / 2) + t * (D / 8);
            const uint32_t from_p = base + S::kRingAt + (tid / 64) * BB + k_params_at(D) + (tid / 4 % kBlockTokens) * 4 * G;
            const uint32_t to = base + S::kAtK + (tid / 32) * 128 + (tid / 4 % 8) * 16 + t * S::kLboK;
#pragma unroll 1
            for (int j = 0; j < steps; ++j) {
                const int slot = j % kRing, stage = j & 1;
                if (!__all_sync(0xffffffffu, wait_for((bars + offsetof(Control, packed_full) + 8 * (slot)), (j / kRing) & 1, gave_up, a.status))) break;
                // all that this thread needs of the step, then the slot is free
                const uint32_t off = slot * S::kPacked;
                uint32_t w[2][D / 32], p[2][G];
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // 32 keys on: two blocks on
                    if constexpr (D == 128) {
                        const uint4 u = lds4(from + off + half * 2 * BB);
                        w[half][0] = u.x, w[half][1] = u.y, w[half][2] = u.z, w[half][3] = u.w;
                    } else {
                        const uint2 u = lds2(from + off + half * 2 * BB);
                        w[half][0] = u.x, w[half][1] = u.y;
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) p[half][g] = lds1(from_p + off + half * 2 * BB + 4 * g);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive((bars + offsetof(Control, packed_empty) + 8 * (slot)));
                if (j >= 2 && !__all_sync(0xffffffffu, wait_for((bars + offsetof(Control, k_empty) + 8 * (stage)), ((j >> 1) - 1) & 1, gave_up, a.status)))
                    break;
                uint32_t probe = 0u;
#pragma unroll
                for (int g = 0; g < G; ++g)
                    probe = not_finite(hfma(__byte_perm(p[0][g], p[1][g], 0x5410), kTop, __byte_perm(p[0][g], p[1][g], 0x7632)), probe);
                auto store = [&](auto held) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t dst = to + stage * S::kBytesK + half * 512;
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) {
                            const uint32_t pg = p[half][q * 32 * G / D], sc = __byte_perm(pg, pg, 0x1010), z = __byte_perm(pg, pg, 0x3232);
                            const uint32_t u = w[half][q], y = u >> 8;
                            uint32_t v[4] = {value_low(u, sc, z), value_high(u, sc, z), value_low(y, sc, z), value_high(y, sc, z)};
                            if (decltype(held)::value && !any_nan(not_finite(pg, 0u))) {  // what is not finite itself stays so
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[i] = hold(v[i]);
                            }
                            sts4(dst + 4 * q * S::kLboK, v[0], v[1], v[2], v[3]);
                        }
                    }
                };
                if (any_nan(probe)) store(std::true_type());
                else store(std::false_type());
                fence_proxy_async();
                mbar_arrive((bars + offsetof(Control, k_full) + 8 * (stage)));
            }
        } else {
            // V: eight keys (a core column) of chunk r, one word (8 channels) of each
            constexpr int kWords = D / 64;                            // words of a V chunk
            constexpr int kGroups = G * 64 / D > 0 ? G * 64 / D : 1;  // groups that a word's channels lie in
            const int id = tid - kDecodeWarps / 2 * 32;
            const int wd = id % kWords, r = id / kWords % 8, kc = id / kWords / 8, g0 = wd * 64 * G / D;
            const bool has = kc < kKeys / 8;
            const uint32_t blk = base + S::kRingAt + (has ? kc / 2 : 0) * BB, tok = (kc & 1) * 8;
            const uint32_t from = blk + v_codes_at(D) + tok * (D / 2) + r * (D / 16) + 4 * wd;
            const uint32_t from_p = blk + v_params_at(D, G) + tok * 4 * G + 4 * g0;
            const uint32_t to = base + S::kAtV + kc * S::kLboV + wd * 1024 + r * 16;
#pragma unroll 1
            for (int j = 0; j < steps; ++j) {
                const int slot = j % kRing, stage = j & 1;
                if (!__all_sync(0xffffffffu, wait_for((bars + offsetof(Control, packed_full) + 8 * (slot)), (j / kRing) & 1, gave_up, a.status))) break;
                const uint32_t off = slot * S::kPacked;
                uint32_t w[8], p[kGroups][8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    w[k] = lds1(from + off + k * (D / 2));
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) p[g][k] = lds1(from_p + off + k * 4 * G + 4 * g);
                }
                const uint32_t hidden = *reinterpret_cast<volatile uint32_t*>(&ctl.hidden[j & 7]);
                __syncwarp();
                if (lane == 0) mbar_arrive((bars + offsetof(Control, packed_empty) + 8 * (slot)));
                if (j >= 2 && !__all_sync(0xffffffffu, wait_for((bars + offsetof(Control, v_empty) + 8 * (stage)), ((j >> 1) - 1) & 1, gave_up, a.status)))
                    break;
                const bool ragged = (j + 1) * kKeys > rq.len || hidden;
                if (has) {
                    uint32_t sc[kGroups][4], z[kGroups][4];
                    bool past = false;  // values past fp16's end
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        if (ragged) {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (j * kKeys + kc * 8 + k >= rq.len || (hidden >> (kc / 2) & 1u)) p[g][k] = 0u;
                        }
                        uint32_t probe = 0u;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            sc[g][k] = __byte_perm(p[g][2 * k], p[g][2 * k + 1], 0x5410);
                            z[g][k] = __byte_perm(p[g][2 * k], p[g][2 * k + 1], 0x7632);
                            probe = not_finite(hfma(sc[g][k], kTop, z[g][k]), probe);
                        }
                        if (any_nan(probe)) {
                            past = true;
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (any_nan(not_finite(p[g][k], 0u))) {
                                    sc[g][k / 2] &= k & 1 ? 0xffffu : 0xffff0000u;
                                    z[g][k / 2] &= k & 1 ? 0xffffu : 0xffff0000u;
                                    atomicMin(&ctl.poison[g0 + g], j * kKeys + kc * 8 + k);
                                }
                        }
                    }
                    const uint32_t dst = to + stage * S::kBytesV;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // nibbles 4 h .. 4 h + 3: channels 8 (8 wd + 4 h + i) + r
                        uint32_t v[4][4];
                        const int g = kGroups == 1 ? 0 : h * kGroups / 2;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t both = __byte_perm(w[2 * k], w[2 * k + 1], h ? 0x7632 : 0x5410), y = both >> 8;
                            v[0][k] = value_low(both, sc[g][k], z[g][k]);
                            v[1][k] = value_high(both, sc[g][k], z[g][k]);
                            v[2][k] = value_low(y, sc[g][k], z[g][k]);
                            v[3][k] = value_high(y, sc[g][k], z[g][k]);
                        }
                        if (past) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) v[e / 4][e % 4] = hold(v[e / 4][e % 4]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) sts4(dst + (4 * h + e) * 128, v[e][0], v[e][1], v[e][2], v[e][3]);
                    }
                }
                fence_proxy_async();
                mbar_arrive((bars + offsetof(Control, v_full) + 8 * (stage)));
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------------------------------------------------------- products
        if (steps) {
            // D fp32, A and B fp16, both K-major; N >> 3 at bit 17, M = 128 >> 4 at bit 24
            constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(kKeys >> 3) << 17) | (8u << 24);
            constexpr uint32_t kIdescO = (1u << 4) | (static_cast<uint32_t>(D >> 3) << 17) | (8u << 24);
            const uint64_t k0 = kmajor(base + S::kAtK, S::kLboK, 128), v0 = kmajor(base + S::kAtV, S::kLboV, 128),
                           q0 = kmajor(base + S::kAtQ + S::kBytesQ, S::kLboQ, 128);
            auto wait = [&](uint32_t bar, int parity) {
                return __all_sync(0xffffffffu, wait_for(bar, parity, gave_up, a.status)) != 0;
            };
            bool ok = true;
#pragma unroll 1
            for (int j = -1; j < steps && ok; ++j) {
                // scores of step j + 1, as soon as those of step j are in registers
                const int next = (j + 1) & 1;
                if (j + 1 < steps) ok = wait(bars + offsetof(Control, k_full) + 8 * next, ((j + 1) >> 1) & 1);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!ok || j + 1 >= n[x]) continue;
                    ok = j < 0 ? wait(bars + offsetof(Control, q_full) + 8 * x, 0) : wait(bars + offsetof(Control, s_read) + 8 * x, j & 1);
                    if (!ok) continue;
                    after_sync();
                    const uint64_t k = k0 + next * (S::kBytesK / 16);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        if (x == 0) mma_ts(tmem + M::s(0), tmem + M::kQ + 8 * i, k + 2 * i * (S::kLboK / 16), kIdescS, i != 0);
                        else mma_ss(tmem + M::s(1), q0 + 2 * i * (S::kLboQ / 16), k + 2 * i * (S::kLboK / 16), kIdescS, i != 0);
                    }
                    commit((bars + offsetof(Control, s_full) + 8 * (x)));
                }
                if (!ok) break;
                if (j + 1 < steps) commit((bars + offsetof(Control, k_empty) + 8 * (next)));
                if (j < 0) continue;
                ok = wait(bars + offsetof(Control, v_full) + 8 * (j & 1), (j >> 1) & 1);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!ok || j >= n[x]) continue;
                    ok = wait(bars + offsetof(Control, p_full) + 8 * x, j & 1);
                    if (!ok) continue;
                    after_sync();
                    const uint64_t v = v0 + (j & 1) * (S::kBytesV / 16);
#pragma unroll
                    for (int i = 0; i < kKeys / 16; ++i)
                        mma_ts(tmem + M::o(x), tmem + M::p(x) + 8 * i, v + 2 * i * (S::kLboV / 16), kIdescO, (j | i) != 0);
                    commit((bars + offsetof(Control, p_read) + 8 * (x)));
                }
                if (ok) commit((bars + offsetof(Control, v_empty) + 8 * (j & 1)));
            }
            // nothing is in flight when tensor memory is given back
            commit((bars + offsetof(Control, drained)));
            ecq_dev::mbar_wait((bars + offsetof(Control, drained)), 0);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- loader: a lane per block of the step
        if (lane < kTileBlocks) {
            const int shift = a.page_shift - 4;
            const int64_t page_bytes = static_cast<int64_t>(BB) << shift;
            const int32_t* row = a.table + b * a.table_stride;
            auto page_of = [&](int j) {  // -1: no such tokens
                const int blk = j * kTileBlocks + lane;
                return j < steps && blk * kBlockTokens < rq.len ? page_at(row + (blk >> shift)) : -1;
            };
            constexpr uint32_t kLanes = (1u << kTileBlocks) - 1u;
            int page = page_of(0), j = 0;
#pragma unroll 1
            for (; j < steps; ++j) {
                const int slot = j % kRing;
                const uint32_t bar = (bars + offsetof(Control, packed_full) + 8 * (slot));
                bool ok = true;
                if (j >= kRing) ok = wait_for((bars + offsetof(Control, packed_empty) + 8 * (slot)), (j / kRing - 1) & 1, gave_up, a.status);
                if (!__all_sync(kLanes, ok)) break;
                const bool there = page >= 0 && page < a.n_pages;
                if (page >= a.n_pages) raise_status(a.status, ECQ_STATUS_BADARG);
                const uint32_t hidden = __ballot_sync(kLanes, !there);
                if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&ctl.hidden[j & 7]) = hidden;
                __syncwarp(kLanes);
                if (there) {
                    const int blk = j * kTileBlocks + lane;
                    mbar_expect_tx(bar, BB);
                    bulk_copy_g2s(base + S::kRingAt + slot * S::kPacked + lane * BB,
                                  a.pages + (static_cast<int64_t>(page) * a.kv_heads + head) * page_bytes +
                                      (blk & ((1 << shift) - 1)) * BB,
                                  BB, bar);
                } else {
                    mbar_expect_tx(bar, 0);
                }
                page = page_of(j + 1);
            }
            // no copy is in flight when the shared memory is given back
            for (int i = max(j - kRing, 0); i < j; ++i) ecq_dev::mbar_wait((bars + offsetof(Control, packed_full) + 8 * (i % kRing)), (i / kRing) & 1);
        }
        __syncwarp();
    }
    before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
    }
}

}  // namespace

namespace ecq_kv4 {

int32_t launch_prompt(const Args& a, int dtype, int head_dim, int groups, int max_q, cudaStream_t stream) {
    // tiles of a request: its rows / 256, rounded up; of all requests at most so many
    const int64_t each = (static_cast<int64_t>(a.share) * max_q + kCtaRows - 1) / kCtaRows * a.batch;
    const int64_t all = static_cast<int64_t>(a.share) * a.total_q / kCtaRows + a.batch;
    const int64_t ctas = (each < all ? each : all) * a.kv_heads;
    if (ctas > INT32_MAX) return ECQ_ERR_UNSUPPORTED;
    return by_layout(dtype, head_dim, groups, [&](auto layout) {
        using L = decltype(layout);
        const auto kernel = prompt_kernel<typename L::T, L::D, L::G>;
        // more than half of the shared memory, whatever is used: one CTA per SM, as tensor memory has room for one
        const int smem = Smem<L::D, L::G>::kBytes > 120 * 1024 ? Smem<L::D, L::G>::kBytes : 120 * 1024;
        if (!ecq_dev::ensure_smem_limit(reinterpret_cast<const void*>(kernel), smem)) return ECQ_ERR_CUDA;
        return result(ecq_dev::launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), smem, stream, a));
    });
}

}  // namespace ecq_kv4

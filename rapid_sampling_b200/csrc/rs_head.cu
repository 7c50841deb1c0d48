// The lm_head in 8-bit floating point: logits = hidden times weights, both held as e4m3 codes with a 32-bit scale for each
// block of 128 (hidden states: a row's 128 columns; weights: 128 x 128).  sm_100a only.
//
//     y[m, v] = sum over blocks b of 128 columns:  sa[m, b] sw[v / 128, b] * (sum over k in b of a[m, k] w[v, k])
//
// The inner sums are tcgen05 products; the two scales differ from block to block, so every block's sum leaves the tensor core
// and is added in fp32 registers.  Products of e4m3 values are exact, a block's 128 of them are summed in the tensor core's fp32
// (measured against 64 bits: 1e-7 relative for K = 4096, where a plain fp32 product is 1e-6 off).
//
// What bounds it (B200, K = 4096, us): few tokens, the weights' bytes: V = 151936, 1 token 103 to 107 of 95 at the measured copy
// rate, 64 tokens 126 of 101 (133 to 149 in a loop of seconds, under the power cap).  Many tokens, the adding of the blocks' sums:
// V = 65536, 2048 tokens 515 to 523 for a short while (2.1 PFLOP/s), 575 to 615 under the cap, by the GPU.
//
// The product of a block's two scales is one fp32 number: where it is subnormal (scales of 2^-63 both, say) results lose digits.
#include "rs_common.cuh"
#include "rs_head_drain.cuh"
#include "rs_host.cuh"
#include "../../include/rapid_sampling_b200.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstring>
#include <mutex>

namespace rs {

constexpr int kHeadBlock = 128;
constexpr float kE4m3Max = 448.f;

// ---- elements of 32 or 16 bits --------------------------------------------------------------------------------------
template <int DT> struct HeadIn;
template <> struct HeadIn<RS_DTYPE_F32> { using T = float; };
template <> struct HeadIn<RS_DTYPE_F16> { using T = __half; };
template <> struct HeadIn<RS_DTYPE_BF16> { using T = __nv_bfloat16; };
__device__ __forceinline__ float head_f(float x) { return x; }
__device__ __forceinline__ float head_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float head_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void head_to(float& o, float x) { o = x; }
__device__ __forceinline__ void head_to(__half& o, float x) { o = __float2half_rn(x); }
__device__ __forceinline__ void head_to(__nv_bfloat16& o, float x) { o = __float2bfloat16_rn(x); }

// Four neighbours: one load where the rows start at multiples of it (VEC), else one by one.
template <bool VEC, class T>
__device__ __forceinline__ void head_ld4(const T* p, float (&x)[4]) {
    if constexpr (VEC && sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else if constexpr (VEC) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = head_f(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = head_f(p[i]);
    }
}

// ---- codes and scales -------------------------------------------------------------------------------------------------
// scale = max(amax / 448, 2^-126); code = the e4m3 value nearest to x / scale, quotient and scale in 32 bits.  amax comes as
// the largest bit pattern of |x|, in which NaN lies above infinity: a block with either has codes or a scale that are NaN.
__device__ __forceinline__ float head_scale(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits), s = __fdiv_rn(a, kE4m3Max);
    return a != a ? a : fmaxf(s, 1.1754943508222875e-38f);
}
// x / s in 32 bits from r, the rounded 1/s.  Quotients of 2^-10 and more matter (smaller ones are code 0), and for those the
// remainders of the short division are multiples of 2^-116 as long as s >= 2^-60: exact.  Other scales divide.
__device__ __forceinline__ float head_quotient(float x, float s, float r) {
    return s >= 8.6736174e-19f && s <= 1e30f ? div_by(x, s, r) : __fdiv_rn(x, s);
}
__device__ __forceinline__ uint32_t head_codes4(const float (&x)[4], float s, float r) {
    uint16_t lo, hi;
    const float a = head_quotient(x[0], s, r), b = head_quotient(x[1], s, r), c = head_quotient(x[2], s, r), d = head_quotient(x[3], s, r);
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ uint32_t head_amax4(const float (&x)[4]) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    return m;
}

// One warp per row and block of 128 columns.  scales: (blocks, pitch), a column per row, as the product reads them.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) head_quantize_rows_kernel(const void* src, long long stride, int M, int K, int blocks, uint8_t* codes,
                                                                 float* scales, int pitch, int* arrived, int counters) {
    using T = typename HeadIn<DT>::T;
    grid_dependents_may_launch();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < counters; i += 256) arrived[i] = 0;      // the product's
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, m = (int)(item / blocks), b = (int)(item - (long long)m * blocks);
    if (m >= M) return;
    const int k = b * kHeadBlock + lane * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (k < K) head_ld4<VEC>((const T*)src + m * stride + k, x);       // K is a multiple of 16
    const float s = head_scale(__reduce_max_sync(0xffffffffu, head_amax4(x)));
    if (k < K) *reinterpret_cast<uint32_t*>(codes + (long long)m * K + k) = head_codes4(x, s, __frcp_rn(s));
    if (lane == 0) scales[(long long)b * pitch + m] = s;
}

// Codes of a pair by div_by's steps (a + b r with -s for the remainders).
__device__ __forceinline__ uint32_t head_codes2(float a, float b, uint64_t minus_s, uint64_t r) {
    const uint64_t x = f2_pack(a, b);
    uint64_t q = f2_mul(x, r);
    q = f2_fma(f2_fma(q, minus_s, x), r, q);
    q = f2_fma(f2_fma(q, minus_s, x), r, q);
    f2_unpack(q, a, b);
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(b), "f"(a));
    return c;
}

// 16 bytes of weights, as they lie in memory.
template <int DT, bool VEC>
__device__ __forceinline__ uint4 head_ld16(const typename HeadIn<DT>::T* p) {
    using T = typename HeadIn<DT>::T;
    uint4 v;
    if constexpr (VEC) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    } else {
        T* e = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int i = 0; i < 16 / (int)sizeof(T); i++) e[i] = p[i];
    }
    return v;
}
// The bits of the largest |x| of a word (fp32), or of either half (bf16, fp16: positive patterns compare as integers, NaN
// above infinity).
template <int DT>
__device__ __forceinline__ uint32_t head_abs_max(uint32_t m, uint32_t w) {
    if constexpr (DT == RS_DTYPE_F32) return max(m, w & 0x7FFFFFFFu);
    else return __vmaxu2(m, w & 0x7FFF7FFFu);
}
template <int DT>
__device__ __forceinline__ uint32_t head_abs_bits(uint32_t m) {      // as the bits of a float
    if constexpr (DT == RS_DTYPE_F32) return m;
    const uint32_t h = max(m & 0xFFFFu, m >> 16);
    if constexpr (DT == RS_DTYPE_BF16) return h << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h))) & 0x7FFFFFFFu;
}
template <int DT>
__device__ __forceinline__ void head_pair(uint32_t w, float& a, float& b) {      // both halves of a 16-bit pair
    if constexpr (DT == RS_DTYPE_BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = f.x;
        b = f.y;
    }
}

// One CTA per block of 128 x 128 weights, which stays in registers as it was read (16-bit: 32 a thread, four CTAs an SM): 16
// bytes a load, a warp's lanes along the rows.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256, DT == RS_DTYPE_F32 ? 2 : 4)
    head_quantize_blocks_kernel(const void* src, long long stride, int V, int K, int blocks, uint8_t* codes, float* scales) {
    using T = typename HeadIn<DT>::T;
    constexpr int E = 16 / (int)sizeof(T), PER_ROW = 128 / E, ROWS = 256 / PER_ROW, N = 128 / ROWS;
    __shared__ uint32_t sh[8];
    const int t = threadIdx.x;
    const int vb = (int)(blockIdx.x / (unsigned)blocks), b = (int)(blockIdx.x - (unsigned)vb * (unsigned)blocks);
    const int k = b * kHeadBlock + (t % PER_ROW) * E, v0 = vb * kHeadBlock + t / PER_ROW;
    const T* p = (const T*)src + v0 * stride + k;
    uint4 x[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = make_uint4(0u, 0u, 0u, 0u);
        if (v0 + i * ROWS < V && k < K) x[i] = head_ld16<DT, VEC>(p + i * ROWS * stride);
    }
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < N; i++) m = head_abs_max<DT>(head_abs_max<DT>(head_abs_max<DT>(head_abs_max<DT>(m, x[i].x), x[i].y), x[i].z), x[i].w);
    m = __reduce_max_sync(0xffffffffu, head_abs_bits<DT>(m));
    if ((t & 31) == 0) sh[t >> 5] = m;
    __syncthreads();
    m = sh[0];
#pragma unroll
    for (int i = 1; i < 8; i++) m = max(m, sh[i]);
    const float s = head_scale(m), r = __frcp_rn(s);
    const uint64_t minus_s = f2_pack(-s, -s), rr = f2_pack(r, r);
    const bool quick = s >= 8.6736174e-19f && s <= 1e30f;       // as in head_quotient
    uint8_t* out = codes + (long long)v0 * K + k;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (v0 + i * ROWS < V && k < K) {
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            if constexpr (E == 4) {
                float f[4];
#pragma unroll
                for (int j = 0; j < 4; j++) f[j] = __uint_as_float(w[j]);
                *reinterpret_cast<uint32_t*>(out + (long long)i * ROWS * K) =
                    quick ? head_codes2(f[0], f[1], minus_s, rr) | (head_codes2(f[2], f[3], minus_s, rr) << 16) : head_codes4(f, s, r);
            } else {
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; j++) head_pair<DT>(w[j], f[2 * j], f[2 * j + 1]);
                uint2 c;
                if (quick) {
                    c.x = head_codes2(f[0], f[1], minus_s, rr) | (head_codes2(f[2], f[3], minus_s, rr) << 16);
                    c.y = head_codes2(f[4], f[5], minus_s, rr) | (head_codes2(f[6], f[7], minus_s, rr) << 16);
                } else {
                    const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
                    c = make_uint2(head_codes4(lo, s, r), head_codes4(hi, s, r));
                }
                *reinterpret_cast<uint2*>(out + (long long)i * ROWS * K) = c;
            }
        }
    }
    if (t == 0) scales[(long long)vb * blocks + b] = s;
}

// ---- tcgen05 ------------------------------------------------------------------------------------------------------------
// Operand tile in shared memory: rows of 128 bytes (128 codes along K), 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t head_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// e4m3 by e4m3, both along K, fp32 sums; m lanes (128 a CTA), n columns
__device__ __forceinline__ uint32_t head_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void head_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void head_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 lanes (a warp's quarter of the accumulator) by 16 or 32 columns; valid after tmem_ld_wait.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}

// ---- how the work is split ----------------------------------------------------------------------------------------------
// A unit is one tile of the result and one block of 128 columns of K; unit u = tile * blocks + block.  Either every worker (a
// CTA, or a pair of them) takes whole tiles in turn, or the units are cut into equal runs of neighbours (`split`), so that all
// workers end together however many tiles there are; head_split decides.  In runs a tile may lie with several workers: each
// leaves its sums in the workspace, and the one that is done last adds them up in a fixed order.
struct HeadWork {
    long long units;
    int workers, blocks, tiles, split;
    __host__ __device__ __forceinline__ long long start(int w) const { return units * w / workers; }
    __device__ __forceinline__ int owner(long long u) const { return (int)(((u + 1) * workers - 1) / units); }
};
struct HeadWalk {      // one worker's segments, in order
    const HeadWork& k;
    const int worker;
    long long u, u1;
    int tile, b0, b1;
    __device__ __forceinline__ HeadWalk(const HeadWork& kk, int w) : k(kk), worker(w), tile(w - kk.workers), b0(0), b1(0) {
        u = k.start(w);
        u1 = k.start(w + 1);
    }
    __device__ __forceinline__ bool next() {
        if (!k.split) {
            tile += k.workers;
            b1 = k.blocks;
            return tile < k.tiles;
        }
        if (u >= u1) return false;
        tile = (int)(u / k.blocks);
        b0 = (int)(u - (long long)tile * k.blocks);
        b1 = (int)min((long long)k.blocks, b0 + (u1 - u));
        u += b1 - b0;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return b1 - b0 == k.blocks; }
};

struct HeadParams {
    const float* sa;         // (blocks, pitch): the tokens' scales
    const float* sw;         // (V blocks, blocks): the weights'
    void* out;               // (M, V), rows ldo elements apart
    long long ldo;
    HeadWork work;
    int M, V, pitch;
    int n;                   // rows of tokens that a CTA brings, a multiple of 16 and at most 128
    int token_tiles;         // more tokens: tiles of 128, or of 256 for pairs (few: 1)
    int stages;
    int boxes;               // pairs: the copy engine stores the result
    int wide_store;          // more tokens, else: bytes of a store that the result's rows allow (32, 16, or 0)
    int turn_at;             // offset in shared memory of what head_store_turned needs
    float* partial;          // split work: two slots a CTA
    int* arrived;            // split work: workers done with the tile that begins in a worker's run
    uint32_t polls;
    int *status, *mirror;
};

constexpr int kHeadMaxWorkers = 160;      // CTAs that the workspace has slots for
constexpr int kHeadMaxStages = 12;
constexpr uint32_t kHeadDrainPolls = 1u << 16;      // limit of the waits for what is in flight after a wait ran out, whatever its own limit

// One lane of a converged warp.  The copying and the multiplying warp run their loops with all lanes and only issue with one:
// uniform control flow keeps descriptors and coordinates in uniform registers (a loop of one lane alone took 1200 cycles a unit).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Bounded waits: the first that runs out reports, and everyone stops at the next wait.
struct HeadWait {
    const HeadParams& p;
    volatile int* gave_up;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
        for (uint32_t i = 0; i < p.polls; i++) {
            if (mbar_try_wait(bar, parity)) return true;
            if (*gave_up) return false;
        }
        *gave_up = 1;
        atomicExch(p.status, RS_ERR_TIMEOUT);
        if (p.mirror) *reinterpret_cast<volatile int*>(p.mirror) = RS_ERR_TIMEOUT;
        return false;
    }
    // For a converged warp.  What is ready costs 73 cycles so, and 104 by way of the loop (155 with one lane waiting for all).
    __device__ __forceinline__ bool warp(uint32_t bar, uint32_t parity) const {
        return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || __all_sync(0xffffffffu, (*this)(bar, parity));
    }
};
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// After a wait that ran out, by one warp once all others have stopped: waits for the copies, products and arrivals that the steps
// so far left on their way into this CTA.  A pair's copies count on the first CTA's barriers (`copies`: this one's), those of a step
// that only one of the two had begun by an arrival of the other's copying warp here (drain_owed).
__device__ __noinline__ void head_drain(uint32_t full, uint32_t empty, uint32_t sfull, uint32_t stages, uint32_t bufs, uint32_t issued,
                                        uint32_t products, bool copies) {
    DrainSteps d = drain_recent(products, stages);
    for (uint32_t k = d.from; k < d.to; k++) mbar_wait_bounded(empty + 8 * drain_slot(k, stages), drain_parity(k, stages), kHeadDrainPolls);
    d = drain_recent(products, bufs);
    for (uint32_t k = d.from; k < d.to; k++) mbar_wait_bounded(sfull + 8 * drain_slot(k, bufs), drain_parity(k, bufs), kHeadDrainPolls);
    d = drain_recent(issued, stages);
    for (uint32_t k = d.from; copies && k < d.to; k++)
        mbar_wait_bounded(full + 8 * drain_slot(k, stages), drain_parity(k, stages), kHeadDrainPolls);
}
// A thread's sums of one row and `cols` tokens in a slot of the workspace: four tokens of 128 rows together, so that both the
// threads' 16 bytes and a warp's 512 are contiguous.
template <int COLS>
__device__ __forceinline__ void head_leave(float* slot, int row, int col0, int cols, const uint64_t (&acc)[COLS / 2]) {
#pragma unroll
    for (int i = 0; i < COLS; i += 4) {
        float4 v;
        f2_unpack(acc[i / 2], v.x, v.y);
        f2_unpack(acc[i / 2 + 1], v.z, v.w);
        if (i < cols) __stcg(reinterpret_cast<float4*>(slot + ((col0 + i) / 4 * 128 + row) * 4), v);
    }
}
template <int COLS>
__device__ __forceinline__ void head_fetch(const float* slot, int row, int col0, int cols, uint64_t (&acc)[COLS / 2]) {      // adds
#pragma unroll
    for (int i = 0; i < COLS; i += 4) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < cols) v = __ldcg(reinterpret_cast<const float4*>(slot + ((col0 + i) / 4 * 128 + row) * 4));
        acc[i / 2] = f2_add(acc[i / 2], f2_pack(v.x, v.y));
        acc[i / 2 + 1] = f2_add(acc[i / 2 + 1], f2_pack(v.z, v.w));
    }
}
// Ends a shared tile's segment (few tokens), called by all adding threads (THREADS of them, barrier 1): returns whether this
// worker was the tile's last, and then its sums are the whole tile's.  Slot 1 of a worker is for the tile that begins in its
// run, slot 0 for the one that began in an earlier one.  Of two workers the last keeps its own sums in registers, and does not
// write them if the other's are there already, as they nearly always are (64 tokens: 152 -> 145 us); of more than two, all are
// added in their order.  (Not inlined: the loop around it needs the registers.)
template <int THREADS, int COLS>
__device__ __noinline__ bool head_share(const HeadParams& p, int slot_floats, int tile, int worker, bool begins, int row, int col0, int cols,
                                        uint64_t (&acc)[COLS / 2], int* flag) {
    const long long u = (long long)tile * p.work.blocks;
    const int first = p.work.owner(u), last = p.work.owner(u + p.work.blocks - 1), needed = last - first + 1;
    int* const counter = p.arrived + first;
    auto slot = [&](int w) { return p.partial + (long long)(2 * w + (w == first)) * slot_floats; };
    auto vote = [&](bool mine) {                  // thread 0's word, to all
        if (threadIdx.x == 0) *flag = mine;
        asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
        const bool v = *(volatile int*)flag;
        asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
        return v;
    };
    bool end = needed == 2 && vote(threadIdx.x == 0 && atomicAdd(counter, 0) == 1);
    if (!end) {
        head_leave<COLS>(p.partial + (long long)(2 * worker + begins) * slot_floats, row, col0, cols, acc);
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
        end = vote(threadIdx.x == 0 && atomicAdd(counter, 1) == needed - 1);
        if (!end) return false;
    }
    __threadfence();
    if (needed == 2) {
        head_fetch<COLS>(slot(worker == first ? last : first), row, col0, cols, acc);
    } else {
#pragma unroll
        for (int i = 0; i < COLS / 2; i++) acc[i] = 0ull;
        for (int w = first; w <= last; w++) head_fetch<COLS>(slot(w), row, col0, cols, acc);
    }
    return true;
}

// Called by the adding threads (THREADS of them, barrier 1) after they have written their sums of a tile they share.
// Returns whether this CTA is the last, and then sees the others' sums.
template <int THREADS>
__device__ __forceinline__ bool head_last(const HeadParams& p, int counter, int needed, int* flag) {
    __threadfence();
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    if (threadIdx.x == 0) *flag = atomicAdd(p.arrived + counter, 1) == needed - 1;
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    const bool last = *(volatile int*)flag;
    __threadfence();
    return last;
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------
// 128 rows of weights are the accumulator's lanes and all tokens (at most 64) its columns, so that the tensor core's work is
// small; the time is that of the weights' bytes.  Warps 0 .. W-1 add the blocks' sums up, each thread one row by 32 tokens; then
// one warp that copies and one that multiplies.  A ring of stages and four accumulators keep the three apart.  A step is two
// blocks: waits and arrivals, about 150 cycles each between products, are paid once for both.
constexpr int kFewTokens = 64, kFewBufs = 4;
// weights of both blocks, tokens of both, the tokens' scales of both
__host__ __device__ constexpr int head_few_stage(int n) { return 2 * 128 * 128 + 2 * n * 128 + 1024; }

template <int NT, typename OUT>
__global__ void __launch_bounds__(NT * 4 + 64, 1)
    head_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ HeadParams p) {
    constexpr int W = NT / 8, COLS = 32, BUFS = kFewBufs;
    constexpr uint32_t kTmemCols = BUFS * 2 * NT;
    extern __shared__ uint8_t raw_smem[];
    __shared__ uint64_t full_[kHeadMaxStages], empty_[kHeadMaxStages], sfull_[BUFS], sempty_[BUFS];
    __shared__ uint32_t tmem_at, issued, products;
    __shared__ int gave_up, flag;
    const uint32_t base = (smem_addr(raw_smem) + 1023u) & ~1023u;
    const uint8_t* const base_p = raw_smem + (base - smem_addr(raw_smem));
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t stage_bytes = (uint32_t)head_few_stage(p.n), stages = (uint32_t)p.stages, x_bytes = (uint32_t)p.n * 128u;
    const uint32_t full = smem_addr(full_), empty = smem_addr(empty_), sfull = smem_addr(sfull_), sempty = smem_addr(sempty_);
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < stages; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1 + W);
        }
        for (int i = 0; i < BUFS; i++) {
            mbar_init(sfull + 8 * i, 1);
            mbar_init(sempty + 8 * i, W);
        }
        gave_up = 0;
        fence_mbar_init();
    }
    if (w == W + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_at)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_at;
    grid_dependency_wait();                       // the tokens' codes and scales are another kernel's
    const HeadWait wait = {p, &gave_up};
    HeadWalk walk(p.work, blockIdx.x);
    if (w == W) {
        uint32_t it = 0, s = 0, ph = 0;           // steps so far, their stage, its phase
        bool ok = true;
        while (ok && walk.next())
            for (int b = walk.b0; b < walk.b1; b += 2, it++) {
                if (it >= stages && !wait.warp(empty + 8 * s, ph ^ 1u)) { ok = false; break; }
                if (elect_one()) {
                    const uint32_t at = base + s * stage_bytes, bar = full + 8 * s, n = (uint32_t)min(2, walk.b1 - b);
                    mbar_expect_tx(bar, n * (128u * 128u + (uint32_t)p.n * 132u));
                    for (uint32_t i = 0; i < n; i++) {
                        tma_2d(at + i * 16384u, &map_w, (b + (int)i) * kHeadBlock, walk.tile * 128, bar);
                        tma_2d(at + 32768u + i * x_bytes, &map_x, (b + (int)i) * kHeadBlock, 0, bar);
                        bulk_g2s(at + 32768u + 2 * x_bytes + i * (uint32_t)p.n * 4u, p.sa + (long long)(b + i) * p.pitch, (uint32_t)p.n * 4u, bar);
                    }
                }
                __syncwarp();
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
        // nothing may still be on its way into shared memory when the CTA ends: neither a copy nor the arrival that frees a stage
        const DrainSteps last = drain_recent(it, stages);
        for (uint32_t k = last.from; ok && k < last.to; k++) ok = wait.warp(empty + 8 * drain_slot(k, stages), drain_parity(k, stages));
        if (lane == 0) issued = it;
    } else if (w == W + 1) {
        const uint32_t idesc = head_idesc(128, p.n);
        const uint64_t desc = head_desc(base);
        uint32_t it = 0, s = 0, ph = 0;
        bool ok = true;
        while (ok && walk.next())
            for (int b = walk.b0; b < walk.b1; b += 2, it++) {
                const uint32_t buf = it % BUFS;
                if (!wait.warp(full + 8 * s, ph)) { ok = false; break; }
                if (it >= BUFS && !wait.warp(sempty + 8 * buf, ((it / BUFS) & 1u) ^ 1u)) { ok = false; break; }
                tmem_fence_after();
                if (elect_one()) {
                    const uint64_t da = desc + ((s * stage_bytes) >> 4), db = da + (32768u >> 4);
#pragma unroll
                    for (int k = 0; k < 4; k++) head_mma(tmem + buf * 2 * NT, da + 2 * k, db + 2 * k, idesc, k > 0);
                    if (b + 1 < walk.b1) {
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            head_mma(tmem + buf * 2 * NT + NT, da + (16384u >> 4) + 2 * k, db + (x_bytes >> 4) + 2 * k, idesc, k > 0);
                    }
                    head_commit(sfull + 8 * buf);
                    head_commit(empty + 8 * s);
                }
                __syncwarp();
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
        if (lane == 0) products = it;
    } else {
        const int quad = w & 3, row = quad * 32 + lane, col0 = (w >> 2) * COLS, cols = p.M - col0;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)col0;
        uint32_t it = 0, s = 0;
        bool dead = false;                        // after a wait that ran out: no more waits, but every barrier of the adding warps
        float scale[2] = {0.f, 0.f};              // of the weights' blocks: these 32 and the next, one a lane
        while (walk.next()) {
            const float* sw = p.sw + (long long)walk.tile * p.work.blocks;
            scale[0] = walk.b0 + lane < walk.b1 ? __ldg(sw + walk.b0 + lane) : 0.f;
            uint64_t acc[COLS / 2];
#pragma unroll
            for (int i = 0; i < COLS / 2; i++) acc[i] = 0ull;
            for (int b = walk.b0; b < walk.b1; b += 2, it++) {
                const uint32_t buf = it % BUFS;
                const int q = (b - walk.b0) & 31;
                if (q == 0) {
                    if (b > walk.b0) scale[0] = scale[1];
                    scale[1] = b + 32 + lane < walk.b1 ? __ldg(sw + b + 32 + lane) : 0.f;
                }
                const float f0 = __shfl_sync(0xffffffffu, scale[0], q), f1 = __shfl_sync(0xffffffffu, scale[0], q + 1);
                if (!dead) dead = !wait.warp(sfull + 8 * buf, (it / BUFS) & 1u);
                if (dead) break;
                tmem_fence_after();
                const ulonglong2* sa = reinterpret_cast<const ulonglong2*>(base_p + s * stage_bytes + 32768u + 2 * x_bytes);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (b + h < walk.b1) {
                        const uint64_t ff = h ? f2_pack(f1, f1) : f2_pack(f0, f0);
                        uint32_t v[COLS];
                        tmem_ld32(lanes + buf * 2 * NT + h * NT, v);      // (columns behind the last token: not looked at)
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < COLS; c += 16)
                            if (col0 + c < p.n) {
#pragma unroll
                                for (int i = c; i < c + 16; i += 4) {
                                    const ulonglong2 g = sa[(h * p.n + col0 + i) / 4];
                                    acc[i / 2] = f2_fma(f2_pack(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), f2_mul(g.x, ff), acc[i / 2]);
                                    acc[i / 2 + 1] = f2_fma(f2_pack(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), f2_mul(g.y, ff), acc[i / 2 + 1]);
                                }
                            }
                    }
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(sempty + 8 * buf);
                    mbar_arrive(empty + 8 * s);
                }
                if (++s == stages) s = 0;
            }
            if (!walk.whole()) {
                uint64_t sums[COLS / 2];
#pragma unroll
                for (int i = 0; i < COLS / 2; i++) sums[i] = acc[i];
                if (!head_share<W * 32, COLS>(p, 128 * NT, walk.tile, blockIdx.x, walk.b0 == 0, row, col0, cols, sums, &flag)) continue;
#pragma unroll
                for (int i = 0; i < COLS / 2; i++) acc[i] = sums[i];
            }
            float y[COLS];
#pragma unroll
            for (int i = 0; i < COLS / 2; i++) f2_unpack(acc[i], y[2 * i], y[2 * i + 1]);
            const int v = walk.tile * 128 + row;
            if (v < p.V && !dead) {
                OUT* o = (OUT*)p.out + (long long)col0 * p.ldo + v;
#pragma unroll
                for (int i = 0; i < COLS; i++) {
                    OUT z;
                    head_to(z, y[i]);
                    if (i < cols) __stcs(o + i * p.ldo, z);
                }
            }
        }
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    if (gave_up) {
        if (w == W) head_drain(full, empty, sfull, stages, BUFS, issued, products, true);
        __syncthreads();
    }
    tmem_fence_after();
    if (w == W + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// ---- more tokens ------------------------------------------------------------------------------------------------------------
// The tokens are the accumulator's lanes and 256 rows of weights its columns: a thread's sums of a block then share one scale,
// its token's times the block's, where weights on the lanes need one of each token.  Up to 128 tokens a CTA has a tile to itself
// and the time is that of the weights' bytes.  Beyond, a pair of CTAs shares a tile of 256 tokens by 256 weight rows (but see
// head_by_pairs): each CTA brings 128 tokens and 128 weight rows, its accumulator holds its 128 tokens by all 256 weight rows,
// and one thread of the first CTA issues the products of both; the pair reads 64 KB for a unit where two CTAs of their own
// read 96 KB.  What bounds it is the adding: 2048 tokens, K = 4096, V = 65536 take 515 to 523 us, and in copies of the kernel 402 without
// the adding, 371 without scales and stores too; with the reading of the accumulators but not the additions 443, the other way
// round 449: the sums leave too few registers to keep both going at once.
constexpr int kMoreAdders = 8, kMoreThreads = kMoreAdders * 32 + 64;      // warps that add, threads of a CTA
// weights, then tokens; a CTA by itself brings only the `n` rows of tokens that there are (in steps of 16): what the other lanes
// multiply is whatever lies behind, and nobody looks at their sums.  (The products read 128 rows all the same: behind the last
// stage lies as much shared memory as they reach beyond it, head_more_tail.)
__host__ __device__ constexpr int head_more_stage(bool pair, int n) { return (pair ? 128 + 128 : 256 + n) * 128; }
__host__ __device__ constexpr int head_more_tail(bool pair, int n) { return pair ? 0 : (128 - n) * 128; }

__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void head_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// arrives at the barrier of the same address in both CTAs once the products issued so far are done
__device__ __forceinline__ void head_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
}
// (nothing in ordinary memory is handed over with these two: releasing it to the cluster would cost each arrival a fence)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx_cluster(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

template <typename OUT>
__device__ __forceinline__ uint32_t head_word(float a, float b);
template <> __device__ __forceinline__ uint32_t head_word<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t head_word<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// COLS neighbours of a row, or the first `cols` of them, 32 or 16 bytes a store.
template <int COLS, typename OUT>
__device__ __forceinline__ void head_store(OUT* o, const uint64_t (&acc)[COLS / 2], int cols, int wide) {
    constexpr int PER32 = 32 / (int)sizeof(OUT);
#pragma unroll
    for (int i = 0; i < COLS; i += PER32) {
        uint32_t x[8];
        if constexpr (sizeof(OUT) == 4) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float a, b;
                f2_unpack(acc[i / 2 + j], a, b);
                x[2 * j] = __float_as_uint(a);
                x[2 * j + 1] = __float_as_uint(b);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float a, b;
                f2_unpack(acc[i / 2 + j], a, b);
                x[j] = head_word<OUT>(a, b);
            }
        }
        if (i + PER32 > cols) {
#pragma unroll
            for (int j = 0; j < PER32; j++) {
                float a, b;
                f2_unpack(acc[(i + j) / 2], a, b);
                OUT z;
                head_to(z, j & 1 ? b : a);
                if (i + j < cols) o[i + j] = z;
            }
        } else if (wide == 32) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o + i), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]),
                         "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                         : "memory");
        } else {
            *reinterpret_cast<uint4*>(o + i) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(o + i + PER32 / 2) = make_uint4(x[4], x[5], x[6], x[7]);
        }
    }
}
// A warp's 32 rows by COLS columns where the rows allow no wide stores (a store of one element a row each took 50 us for 1293
// rows of 2931 fp16, the products 5): 32 columns at a time by way of shared memory (rows of 33 words: no bank twice), then row by row, neighbours of a row from neighbouring lanes.
constexpr int kTurnBytes = 32 * 33 * 4;
template <int COLS, typename OUT>
__device__ __forceinline__ void head_store_turned(OUT* o, long long ldo, float* buf, const uint64_t (&acc)[COLS / 2], int lane, int rows, int cols) {
#pragma unroll
    for (int c0 = 0; c0 < COLS; c0 += 32) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float a, b;
            f2_unpack(acc[c0 / 2 + i], a, b);
            buf[lane * 33 + 2 * i] = a;
            buf[lane * 33 + 2 * i + 1] = b;
        }
        __syncwarp();
        if (c0 + lane < cols)
#pragma unroll 8
            for (int r = 0; r < min(rows, 32); r++) {
                OUT z;
                head_to(z, buf[r * 33 + lane]);
                __stcs(o + r * ldo + c0 + lane, z);
            }
        __syncwarp();
    }
}

// The same by way of shared memory, 8 KB a warp, for the warp's 32 rows: two boxes of 128 bytes by 32 rows at a time, which the
// copy engine stores (and cuts off behind the last row and the last whole 16 bytes of a row: it writes no less, so that the few
// columns behind, from `whole` on, are stored one by one) while the warp goes on with the next tile.  All CTAs end
// their tiles at about the same time: stores by the threads themselves waited 3.6 us a tile for one another (16 % of the time at
// 2048 tokens).  128-byte swizzle: the 16-byte column c of row r lies at c ^ (r % 8).
constexpr int kStoreBytes = 8192;
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
template <int COLS, typename OUT>
__device__ __forceinline__ void head_store_box(const CUtensorMap* map, uint32_t buf, const uint64_t (&acc)[COLS / 2], int lane, int m, int v0,
                                               const HeadParams& p) {
    constexpr int PER16 = 16 / (int)sizeof(OUT);
    const int whole = p.V / PER16 * PER16;    constexpr int PER = 128 / (int)sizeof(OUT);       // columns of a box
#pragma unroll
    for (int c0 = 0; c0 < COLS; c0 += 2 * PER) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the boxes before have been read
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; i++) {                // 16 bytes each
            const int col = c0 + i * (16 / (int)sizeof(OUT));
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float a, b;
                if constexpr (sizeof(OUT) == 4) {
                    f2_unpack(acc[(col + j) / 2], a, b);
                    x[j] = __float_as_uint(j & 1 ? b : a);
                } else {
                    f2_unpack(acc[col / 2 + j], a, b);
                    x[j] = head_word<OUT>(a, b);
                }
            }
            const uint32_t at = buf + (uint32_t)(i / 8) * 4096u + (uint32_t)lane * 128u + (uint32_t)(((i & 7) ^ (lane & 7)) * 16);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
        }
        if (whole < p.V && whole >= v0 + c0 && whole < v0 + c0 + 2 * PER && m + lane < p.M) {      // what this lane has just written
            const uint32_t i = (uint32_t)(whole - v0 - c0) / PER16;
            const uint32_t at = buf + (i / 8u) * 4096u + (uint32_t)lane * 128u + ((i & 7u) ^ (uint32_t)(lane & 7)) * 16u;
            OUT* o = (OUT*)p.out + (long long)(m + lane) * p.ldo + whole;
            for (int k = 0; k < p.V - whole; k++) {
                if constexpr (sizeof(OUT) == 4) {
                    uint32_t x;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at + 4u * (uint32_t)k) : "memory");
                    *reinterpret_cast<uint32_t*>(o + k) = x;
                } else {
                    uint16_t x;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at + 2u * (uint32_t)k) : "memory");
                    *reinterpret_cast<uint16_t*>(o + k) = x;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            if (v0 + c0 < whole) tma_store_2d(map, buf, v0 + c0, m);
            if (v0 + c0 + PER < whole) tma_store_2d(map, buf + 4096u, v0 + c0 + PER, m);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}

template <bool PAIR, typename OUT>
__global__ void __launch_bounds__(kMoreThreads, 1)
    head_more_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_out,
                     const __grid_constant__ HeadParams p) {
    constexpr int W = kMoreAdders, COLS = 256 / (W / 4), NT = 256, CTAS = PAIR ? 2 : 1;
    constexpr uint32_t kTmemCols = 512, kWeights = (PAIR ? 128 : 256) * 128;
    const uint32_t stage_bytes = (uint32_t)head_more_stage(PAIR, p.n);
    extern __shared__ uint8_t raw_smem[];
    __shared__ uint64_t full_[kHeadMaxStages], empty_[kHeadMaxStages], sfull_[2], sempty_[2];
    __shared__ uint32_t tmem_at, issued, products;
    __shared__ int gave_up, flag, other_gave_up;
    const uint32_t base = (smem_addr(raw_smem) + 1023u) & ~1023u;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_ctarank() : 0, worker = (int)blockIdx.x / CTAS;
    const uint32_t stages = (uint32_t)p.stages;
    const uint32_t full = smem_addr(full_), empty = smem_addr(empty_), sfull = smem_addr(sfull_), sempty = smem_addr(sempty_);
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < stages; i++) {
            mbar_init(full + 8 * i, CTAS);            // a pair's: those of the first CTA, both copying warps
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(sfull + 8 * i, 1);
            mbar_init(sempty + 8 * i, CTAS * W);      // a pair's: those of the first CTA, both CTAs' adding warps
        }
        gave_up = other_gave_up = 0;
        fence_mbar_init();
    }
    if (w == W + 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_at)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_at)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    tmem_fence_before();
    __syncthreads();
    if constexpr (PAIR) {
        cluster_arrive();
        cluster_wait();                               // the other CTA's barriers are there
    }
    tmem_fence_after();
    const uint32_t tmem = tmem_at;
    grid_dependency_wait();
    const HeadWait wait = {p, &gave_up};
    HeadWalk walk(p.work, worker);
    if (w == W) {
        const uint32_t first_full = PAIR ? map_to_cta(full, 0) : full;
        uint32_t it = 0, s = 0, ph = 0;
        bool ok = true;
        while (ok && walk.next()) {
            const int vt = walk.tile / p.token_tiles, mt = walk.tile - vt * p.token_tiles;
            const int v0 = vt * 256 + rank * 128, m0 = mt * 128 * CTAS + rank * 128;
            for (int b = walk.b0; b < walk.b1; b++, it++) {
                if (it >= stages && !wait.warp(empty + 8 * s, ph ^ 1u)) { ok = false; break; }
                if (elect_one()) {
                    const uint32_t at = base + s * stage_bytes, bar = first_full + 8 * s;
                    if constexpr (PAIR) {
                        mbar_expect_tx_cluster(bar, stage_bytes);
                        tma_2d_pair(at, &map_w, b * kHeadBlock, v0, bar);
                        tma_2d_pair(at + kWeights, &map_x, b * kHeadBlock, m0, bar);
                    } else {
                        mbar_expect_tx(bar, stage_bytes);
                        tma_2d(at, &map_w, b * kHeadBlock, v0, bar);
                        tma_2d(at + kWeights, &map_x, b * kHeadBlock, m0, bar);
                    }
                }
                __syncwarp();
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
        }
        const DrainSteps last = drain_recent(it, stages);      // as in head_few_kernel
        for (uint32_t k = last.from; ok && k < last.to; k++) ok = wait.warp(empty + 8 * drain_slot(k, stages), drain_parity(k, stages));
        if (lane == 0) issued = it;
    } else if (w == W + 1) {
        if (rank == 0) {
            const uint32_t idesc = head_idesc(128 * CTAS, NT);
            const uint64_t desc = head_desc(base);
            uint32_t it = 0, s = 0, ph = 0;
            bool ok = true;
            while (ok && walk.next())
                for (int b = walk.b0; b < walk.b1; b++, it++) {
                    const uint32_t buf = it & 1u;
                    if (!wait.warp(full + 8 * s, ph)) { ok = false; break; }
                    if (it >= 2 && !wait.warp(sempty + 8 * buf, ((it >> 1) & 1u) ^ 1u)) { ok = false; break; }
                    tmem_fence_after();
                    if (elect_one()) {
                        const uint64_t db = desc + ((s * stage_bytes) >> 4), da = db + (kWeights >> 4);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if constexpr (PAIR) head_mma_pair(tmem + buf * NT, da + 2 * k, db + 2 * k, idesc, k > 0);
                            else head_mma(tmem + buf * NT, da + 2 * k, db + 2 * k, idesc, k > 0);
                        }
                        if constexpr (PAIR) {
                            head_commit_pair(sfull + 8 * buf);
                            head_commit_pair(empty + 8 * s);
                        } else {
                            head_commit(sfull + 8 * buf);
                            head_commit(empty + 8 * s);
                        }
                    }
                    __syncwarp();
                    if (++s == stages) { s = 0; ph ^= 1u; }
                }
            if (lane == 0) products = it;
        }
    } else {
        const int quad = w & 3, col0 = (w >> 2) * COLS, row = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)col0;
        const uint32_t first_sempty = PAIR ? map_to_cta(sempty, 0) : sempty;
        uint32_t it = 0;
        bool dead = false;                            // as in head_few_kernel
        while (walk.next()) {
            const int vt = walk.tile / p.token_tiles, mt = walk.tile - vt * p.token_tiles;
            const int m = mt * 128 * CTAS + rank * 128 + row, v0 = vt * 256 + col0;
            // (weight rows and tokens behind the last one: any scale, their sums are not stored)
            const float* sw = p.sw + (long long)(min(v0, p.V - 1) / 128) * p.work.blocks;
            const float* sa = p.sa + m;
            // two blocks ahead: a load from L2 takes longer than a block's products
            float a1 = __ldcg(sa + (long long)walk.b0 * p.pitch), w1 = __ldg(sw + walk.b0), a2 = 0.f, w2 = 0.f;
            if (walk.b0 + 1 < walk.b1) {
                a2 = __ldcg(sa + (long long)(walk.b0 + 1) * p.pitch);
                w2 = __ldg(sw + walk.b0 + 1);
            }
            uint64_t acc[COLS / 2];
#pragma unroll
            for (int i = 0; i < COLS / 2; i++) acc[i] = 0ull;
            for (int b = walk.b0; b < walk.b1; b++, it++) {
                const uint32_t buf = it & 1u;
                const float f = a1 * w1;
                a1 = a2;
                w1 = w2;
                if (b + 2 < walk.b1) {
                    a2 = __ldcg(sa + (long long)(b + 2) * p.pitch);
                    w2 = __ldg(sw + b + 2);
                }
                const uint64_t ff = f2_pack(f, f);
                if (!dead) dead = !wait.warp(sfull + 8 * buf, (it >> 1) & 1u);
                if (dead) break;
                tmem_fence_after();
#pragma unroll
                for (int c = 0; c < COLS; c += 16) {
                    uint32_t v[16];
                    tmem_ld16(lanes + buf * NT + c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        acc[c / 2 + i] = f2_fma(f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ff, acc[c / 2 + i]);
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_cluster(first_sempty + 8 * buf);
                    else mbar_arrive(sempty + 8 * buf);
                }
            }
            if (!walk.whole()) {
                float* mine = p.partial + (long long)(2 * (int)blockIdx.x + (walk.b0 == 0)) * 128 * 256 + (long long)col0 * 128 + row;
                if (m < p.M) {
#pragma unroll
                    for (int i = 0; i < COLS / 2; i++) {
                        float a, b;
                        f2_unpack(acc[i], a, b);
                        mine[(2 * i) * 128] = a;
                        mine[(2 * i + 1) * 128] = b;
                    }
                }
                const long long u = (long long)walk.tile * p.work.blocks;
                const int c0 = p.work.owner(u), c1 = p.work.owner(u + p.work.blocks - 1);
                // counted for each CTA of a pair apart: they share no row
                if (!head_last<W * 32>(p, CTAS * c0 + rank, c1 - c0 + 1, &flag)) continue;
#pragma unroll
                for (int i = 0; i < COLS / 2; i++) acc[i] = 0ull;
                for (int c = c0; c <= c1 && m < p.M; c++) {
                    const float* from = p.partial + (long long)(2 * (CTAS * c + rank) + (c == c0)) * 128 * 256 + (long long)col0 * 128 + row;
#pragma unroll
                    for (int i = 0; i < COLS / 2; i++) {
                        float a, b;
                        f2_unpack(acc[i], a, b);
                        acc[i] = f2_pack(a + __ldcg(from + (2 * i) * 128), b + __ldcg(from + (2 * i + 1) * 128));
                    }
                }
            }
            // the place once more, from what the compiler cannot keep in registers through the loop above (us for pairs, 2048 x 4096 x
            // 65536 bf16 / 32768 f32: 524 / 288, with the places kept 529 / 290)
            uint32_t tile = (uint32_t)walk.tile, tid;
            asm volatile("" : "+r"(tile));
            asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
            const int here = (int)(tid >> 5), vt1 = (int)tile / p.token_tiles;
            const int m0 = ((int)tile - vt1 * p.token_tiles) * 128 * CTAS + rank * 128 + (here & 3) * 32, v1 = vt1 * 256 + (here >> 2) * COLS;
            if (PAIR && p.boxes) {
                if (!dead && m0 < p.M && v1 < p.V)
                    head_store_box<COLS, OUT>(&map_out, base + stages * stage_bytes + (uint32_t)(here * kStoreBytes), acc, lane, m0, v1, p);
            } else if (!dead && m0 < p.M && v1 < p.V) {
                OUT* o = (OUT*)p.out + (long long)m0 * p.ldo + v1;
                if (!PAIR && p.wide_store) {               // (a pair's wide stores are boxes)
                    if (m0 + lane < p.M) head_store<COLS, OUT>(o + lane * p.ldo, acc, p.V - v1, p.wide_store);
                } else {
                    float* buf = reinterpret_cast<float*>(raw_smem + (base - smem_addr(raw_smem)) + p.turn_at + (uint32_t)(here * kTurnBytes));
                    head_store_turned<COLS, OUT>(o, p.ldo, buf, acc, lane, p.M - m0, p.V - v1);
                }
            }
        }
        if (PAIR && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    if constexpr (PAIR) {
        if (threadIdx.x == 0 && gave_up) st_cluster_u32(map_to_cta(smem_addr(&other_gave_up), (uint32_t)rank ^ 1u), 1u);
        __syncwarp();
        cluster_arrive();
        cluster_wait();                               // neither CTA leaves while the other's products, copies or arrivals may reach it
        if (gave_up || other_gave_up) {               // the same in both: and none of its own either
            if (w == W) {
                const uint32_t other = ld_cluster_u32(map_to_cta(smem_addr(&issued), (uint32_t)rank ^ 1u));
                const uint32_t multiplied = ld_cluster_u32(map_to_cta(smem_addr(&products), 0)), first_full = map_to_cta(full, 0);
                const DrainSteps owed = drain_owed(issued, other);
                for (uint32_t k = owed.from; k < owed.to; k++)
                    if (lane == 0) mbar_arrive_cluster(first_full + 8 * drain_slot(k, stages));
                head_drain(full, empty, sfull, stages, 2, max(issued, other), multiplied, rank == 0);
                __syncwarp();
            }
            cluster_arrive();
            cluster_wait();
        }
    } else if (gave_up) {
        if (w == W) head_drain(full, empty, sfull, stages, 2, issued, products, true);
        __syncthreads();
    }
    tmem_fence_after();
    if (w == W + 1) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled head_encoder() {
    static EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (EncodeTiled)f;
    }();
    return fn;
}
// (rows, cols) elements, rows `pitch` bytes apart, in boxes of box_rows rows by 128 bytes; what lies outside reads as zero
static int head_map(CUtensorMap* m, CUtensorMapDataType type, int size, const void* at, long long rows, long long cols, long long pitch, int box_rows) {
    EncodeTiled enc = head_encoder();
    if (!enc) return host_cuda_fail(cudaErrorSymbolNotFound, "cuTensorMapEncodeTiled");
    const cuuint64_t dim[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult e = enc(m, type, 2, const_cast<void*>(at), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? RS_OK : host_cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
}

template <typename KERN, typename... ARGS>
static int head_launch(KERN kern, int threads, int smem, int grid, int cluster, cudaStream_t stream, bool (&done)[64], const ARGS&... args) {
    {
        static std::mutex mu;
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return host_cuda_fail(e, "cudaGetDevice");
        std::lock_guard<std::mutex> lk(mu);
        if (!done[dev & 63]) {
            HostDevice d;
            const int rc = host_device(&d);
            if (rc) return rc;
            cudaFuncAttributes fa;
            e = cudaFuncGetAttributes(&fa, kern);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, d.smem_optin - (int)fa.sharedSizeBytes);
            if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(head)");
            done[dev & 63] = true;
        }
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    // starts while the tokens are still being quantized and waits for them itself
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaLaunchKernelEx(head)");
    host_count_launch();
    return RS_OK;
}
template <typename OUT>
static int head_run(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& out, const HeadParams& p, bool pair, int smem, cudaStream_t stream) {
    static bool done[4][64] = {};      // per device
    const int n = p.work.workers;
    if (p.M <= 32) return head_launch(head_few_kernel<32, OUT>, 192, smem, n, 1, stream, done[0], w, x, p);
    if (p.M <= kFewTokens) return head_launch(head_few_kernel<64, OUT>, 320, smem, n, 1, stream, done[1], w, x, p);
    if (!pair) return head_launch(head_more_kernel<false, OUT>, kMoreThreads, smem, n, 1, stream, done[3], w, x, out, p);
    return head_launch(head_more_kernel<true, OUT>, kMoreThreads, smem, 2 * n, 2, stream, done[2], w, x, out, p);
}

// More than 128 tokens: pairs, unless the last one's second half would have no tokens and that costs more than pairs gain, a
// tenth.  us for pairs / single CTAs, K = 4096, V = 32768: 384 tokens 89 / 79, 640 127 / 122, 896 146 / 164, 1408 221 / 239.
static bool head_by_pairs(long long M) {
    const long long tiles = (M + 127) / 128;
    return M > 128 && tiles != 3 && tiles != 5;
}
// How the units are given out: whole tiles in turn, every tile in equal runs of its own, or equal runs throughout, where most
// workers share two tiles.  Each way's time is estimated in that of a unit when all workers are busy; with few of them a unit
// takes `alone` of it.  Sharing a tile costs what its sums take through L2 (from 65 tokens on 128 KB a CTA, below that 16 or
// 32): `first` for two workers, `next` for each more, `runs` for equal runs.  With 65 to 128 tokens whole tiles in turn leave
// HBM idle whenever all workers store theirs.  us for whole tiles / the best number of runs each / equal runs:
//   64 tokens, K = 4096, V = 151936: 141 / - / 135;   64, 2048, 50304: 31 / - / 38;      64, 4096, 19000: 35 / - / 31;
//   33 tokens, K = 4992, V = 2000: 24 / 22 (2) / 28;  8, 6976, 11215: 25 / - / 28;       1, 4096, 151936: 104 / - / 103;
//   128 tokens, K = 4096, V = 151936: 160 / - / 137;  80, 2048, 65536: 37 / - / 50;      128, 8192, 1000: 48 / 33 (3) / 53;
//   467 tokens, K = 4192, V = 3565: 34 / 40 (2) / 56; 757, 960, 5863: 19 / - / 38;       251, 6112, 114533: 241 / - / 222.
static void head_split(HeadWork& k, long long M) {
    struct Costs { float alone, first, next, runs; };
    const Costs c = M <= kFewTokens ? Costs{0.55f, 6.f, 1.f, 10.f} : head_by_pairs(M) ? Costs{0.8f, 19.f, 8.f, 25.f} : Costs{0.65f, 9.5f, 4.f, 27.f};
    const int W = k.workers, rest = k.tiles % W;
    auto busy = [&](long long workers) { return fmaxf((float)workers / (float)W, c.alone); };
    float best = (float)k.blocks * ((float)(k.tiles / W) + (rest ? busy(rest) : 0.f));
    if (M > kFewTokens && M <= 128 && k.tiles > W) best *= 1.25f;
    int workers = k.tiles < W ? k.tiles : W, split = 0;
    for (int parts = 2; (long long)parts * k.tiles <= W && parts * 4 <= k.blocks; parts++) {
        const float cost = (float)((k.blocks + parts - 1) / parts) * busy(parts * k.tiles) + c.first + c.next * (float)(parts - 2);
        if (cost < best) { best = cost; workers = parts * k.tiles; split = 1; }
    }
    const float cost = (float)k.units / (float)W + c.runs + (k.tiles < W ? c.next * (float)(W / k.tiles) : 0.f);
    if (cost < best && k.units >= 4LL * W) { workers = W; split = 1; }
    k.workers = workers;
    k.split = split;
}

// Pairs of CTAs that the device runs at once.
static int head_pairs(int* out) {
    static std::mutex mu;
    static int known[64] = {};         // per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaGetDevice");
    std::lock_guard<std::mutex> lk(mu);
    if (!known[dev & 63]) {
        auto kern = head_more_kernel<true, float>;
        const int smem = 6 * head_more_stage(true, 128) + 1024;
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof cfg);
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(kMoreThreads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 2;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        int n = 0;
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
        if (e != cudaSuccess) return host_cuda_fail(e, "cudaOccupancyMaxActiveClusters");
        known[dev & 63] = n < 1 ? 1 : n;
    }
    *out = known[dev & 63];
    return RS_OK;
}

template <bool ROWS>
static int head_quantize(const void* src, int dtype, long long stride, long long rows, long long K, uint8_t* codes, float* scales, int pitch,
                         int* arrived, cudaStream_t st) {
    const int blocks = (int)((K + kHeadBlock - 1) / kHeadBlock);
    const uintptr_t size = dtype == RS_DTYPE_F32 ? 4 : 2;
    const bool vec = ROWS ? ((uintptr_t)src & (4 * size - 1)) == 0 && stride % 4 == 0 : ((uintptr_t)src & 15) == 0 && stride * size % 16 == 0;
    const long long ctas = ROWS ? (rows * blocks + 7) / 8 : (rows + kHeadBlock - 1) / kHeadBlock * blocks;
    if (ctas > 0x7fffffffLL) return RS_ERR_LIMIT;
    const unsigned grid = (unsigned)ctas;
#define RS_HEAD_Q(DT, VEC)                                                                                                          \
    if constexpr (ROWS) head_quantize_rows_kernel<DT, VEC><<<grid, 256, 0, st>>>(src, stride, (int)rows, (int)K, blocks, codes, scales, pitch, arrived, \
                                                                                2 * kHeadMaxWorkers); \
    else head_quantize_blocks_kernel<DT, VEC><<<grid, 256, 0, st>>>(src, stride, (int)rows, (int)K, blocks, codes, scales)
    if (dtype == RS_DTYPE_F32) { if (vec) { RS_HEAD_Q(RS_DTYPE_F32, true); } else { RS_HEAD_Q(RS_DTYPE_F32, false); } }
    else if (dtype == RS_DTYPE_F16) { if (vec) { RS_HEAD_Q(RS_DTYPE_F16, true); } else { RS_HEAD_Q(RS_DTYPE_F16, false); } }
    else { if (vec) { RS_HEAD_Q(RS_DTYPE_BF16, true); } else { RS_HEAD_Q(RS_DTYPE_BF16, false); } }
#undef RS_HEAD_Q
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return host_cuda_fail(e, "launch(head quantize)");
    host_count_launch();
    return RS_OK;
}

static bool head_dtype(int d) { return d == RS_DTYPE_F32 || d == RS_DTYPE_F16 || d == RS_DTYPE_BF16; }
static int head_pitch(long long M) { return (int)((M + 255) / 256 * 256) + 256; }      // a multiple of a tile: its scales never end behind a row
struct HeadLayout { size_t scales, arrived, partial, total; };
static HeadLayout head_layout(long long M, long long K) {
    HeadLayout l;
    const size_t blocks = (size_t)((K + 127) / 128), n = M <= 32 ? 32 : M <= kFewTokens ? 64 : 256;
    l.scales = ((size_t)M * (size_t)K + 255) / 256 * 256;
    l.arrived = l.scales + blocks * (size_t)head_pitch(M) * 4;
    l.partial = l.arrived + 2 * kHeadMaxWorkers * 4;
    l.total = l.partial + (size_t)kHeadMaxWorkers * 2 * 128 * n * 4;
    return l;
}
static int head_check(int64_t rows, int64_t K) {
    if (rows <= 0) return RS_ERR_BATCH;
    if (K <= 0 || K % 16 != 0 || K > RS_HEAD_MAX_K || rows > RS_HEAD_MAX_ROWS) return RS_ERR_LIMIT;
    return RS_OK;
}

}  // namespace rs

extern "C" {

int rs_head_quantize(const void* weight, int32_t dtype, int64_t V, int64_t K, int64_t row_stride, void* codes_device, float* scales_device,
                     void* stream) {
    using namespace rs;
    if (!head_dtype(dtype)) return RS_ERR_DTYPE;
    const int rc = head_check(V, K);
    if (rc) return rc;
    const uintptr_t size = dtype == RS_DTYPE_F32 ? 4 : 2;
    if (!weight || !codes_device || !scales_device || ((uintptr_t)weight & (size - 1)) || ((uintptr_t)codes_device & 15) || ((uintptr_t)scales_device & 3))
        return RS_ERR_POINTER;
    if (row_stride < 0) return RS_ERR_LIMIT;
    return head_quantize<false>(weight, dtype, row_stride, V, K, (uint8_t*)codes_device, scales_device, 0, nullptr, (cudaStream_t)stream);
}

size_t rs_head_workspace_bytes(int64_t M, int64_t K) {
    if (rs::head_check(M, K)) return 0;
    return rs::head_layout(M, K).total;
}

int rs_head_logits(const void* hidden, int32_t hidden_dtype, int64_t M, int64_t K, int64_t hidden_stride, const void* codes_device,
                   const float* scales_device, int64_t V, void* out_device, int32_t out_dtype, int64_t out_stride, void* workspace_device,
                   size_t workspace_bytes, void* stream) {
    using namespace rs;
    if (!head_dtype(hidden_dtype) || !head_dtype(out_dtype)) return RS_ERR_DTYPE;
    int rc = head_check(M, K);
    if (rc) return rc;
    if ((rc = head_check(V, K))) return rc;
    const uintptr_t hs = hidden_dtype == RS_DTYPE_F32 ? 4 : 2, os = out_dtype == RS_DTYPE_F32 ? 4 : 2;
    if (!hidden || !codes_device || !scales_device || !out_device || !workspace_device || ((uintptr_t)hidden & (hs - 1)) ||
        ((uintptr_t)codes_device & 15) || ((uintptr_t)scales_device & 3) || ((uintptr_t)out_device & (os - 1)) || ((uintptr_t)workspace_device & 255))
        return RS_ERR_POINTER;
    if (hidden_stride < 0 || out_stride < V) return RS_ERR_LIMIT;
    if (workspace_bytes < rs_head_workspace_bytes(M, K)) return RS_ERR_WORKSPACE;
    HostDevice dev;
    if ((rc = host_device(&dev))) return rc;
    HeadParams p;
    memset(&p, 0, sizeof p);
    if ((rc = host_status_word(&p.status))) return rc;
    const HeadLayout l = head_layout(M, K);
    uint8_t* ws = (uint8_t*)workspace_device;
    float* sa = (float*)(ws + l.scales);
    p.sa = sa;
    p.sw = scales_device;
    p.out = out_device;
    p.ldo = out_stride;
    p.M = (int)M;
    p.V = (int)V;
    p.pitch = head_pitch(M);
    p.partial = (float*)(ws + l.partial);
    p.arrived = (int*)(ws + l.arrived);
    p.polls = host_wait_polls();
    p.mirror = dev.mirror;
    const bool few = M <= kFewTokens, pair = head_by_pairs(M);
    p.n = M >= 128 ? 128 : (int)((M + 15) / 16 * 16);
    p.token_tiles = (int)(pair ? (M + 255) / 256 : (M + 127) / 128);
    const int tile_v = few ? 128 : 256;
    HeadWork& k = p.work;
    k.blocks = (int)((K + 127) / 128);
    const long long tiles = (V + tile_v - 1) / tile_v * p.token_tiles;
    if (tiles > 0x7fffffffLL) return RS_ERR_LIMIT;
    k.tiles = (int)tiles;
    k.units = tiles * k.blocks;
    k.workers = dev.sms < kHeadMaxWorkers ? dev.sms : kHeadMaxWorkers;
    if (pair) {
        int pairs = 0;
        if ((rc = head_pairs(&pairs))) return rc;
        k.workers = k.workers / 2 < pairs ? k.workers / 2 : pairs;
    }
    head_split(k, M);
    const int per = few ? head_few_stage(p.n) : head_more_stage(pair, p.n);
    const uintptr_t step = (uintptr_t)out_device | (uintptr_t)out_stride * os;
    p.wide_store = step % 32 == 0 ? 32 : step % 16 == 0 ? 16 : 0;
    const long long whole = V / (long long)(16 / os) * (long long)(16 / os);      // columns of a row that boxes store
    if (pair && whole == 0) p.wide_store = 0;
    p.boxes = pair && p.wide_store;
    // behind the stages: the boxes to store, or what the products read beyond the last stage and the rows to turn
    const int tail = few ? 0 : p.boxes ? kMoreAdders * kStoreBytes : head_more_tail(pair, p.n) + (p.wide_store ? 0 : kMoreAdders * kTurnBytes);
    const int room = dev.smem_optin - 2048 - 1024 - tail;
    p.stages = room / per > kHeadMaxStages ? kHeadMaxStages : room / per;
    CUtensorMap w, x, out;
    if ((rc = head_map(&w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes_device, V, K, K, few || pair ? 128 : 256)) ||
        (rc = head_map(&x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, ws, M, K, K, p.n)))
        return rc;
    memset(&out, 0, sizeof out);
    if (p.boxes) {
        const CUtensorMapDataType type = out_dtype == RS_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : out_dtype == RS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if ((rc = head_map(&out, type, (int)os, out_device, M, whole, (long long)(out_stride * (int64_t)os), 32))) return rc;
    }
    if ((rc = head_quantize<true>(hidden, hidden_dtype, hidden_stride, M, K, ws, sa, p.pitch, p.arrived, (cudaStream_t)stream))) return rc;
    p.turn_at = p.stages * per + (few ? 0 : head_more_tail(pair, p.n));
    const int smem = p.stages * per + tail + 1024;
    switch (out_dtype) {
        case RS_DTYPE_F32: return head_run<float>(w, x, out, p, pair, smem, (cudaStream_t)stream);
        case RS_DTYPE_F16: return head_run<__half>(w, x, out, p, pair, smem, (cudaStream_t)stream);
        default: return head_run<__nv_bfloat16>(w, x, out, p, pair, smem, (cudaStream_t)stream);
    }
}

}  // extern "C"

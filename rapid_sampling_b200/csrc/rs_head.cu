// The lm_head in 8-bit floating point: logits = hidden times weights, both held as e4m3 codes with a 32-bit scale for each
// block of 128 (hidden states: a row's 128 columns; weights: 128 x 128).  sm_100a only.
//
//     y[m, v] = sum over blocks b of 128 columns:  sa[m, b] sw[v / 128, b] * (sum over k in b of a[m, k] w[v, k])
//
// The inner sums are tcgen05 products of 128 weights rows (the accumulator's lanes) by up to 256 tokens (its columns); the
// two scales differ from block to block, so every block's sum leaves the tensor core and is added in fp32 registers.
#include "rs_common.cuh"
#include "rs_host.cuh"
#include "../../include/rapid_sampling_b200.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
                                                                 float* scales, int pitch) {
    using T = typename HeadIn<DT>::T;
    grid_dependents_may_launch();
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

// One CTA per block of 128 x 128 weights: a warp's lanes are 128 columns, a warp takes every eighth row.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) head_quantize_blocks_kernel(const void* src, long long stride, int V, int K, int blocks, uint8_t* codes,
                                                                   float* scales) {
    using T = typename HeadIn<DT>::T;
    __shared__ uint32_t sh[8];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int vb = (int)(blockIdx.x / (unsigned)blocks), b = (int)(blockIdx.x - (unsigned)vb * (unsigned)blocks);
    const int k = b * kHeadBlock + lane * 4;
    float x[16][4];
    uint32_t amax = 0u;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int v = vb * kHeadBlock + i * 8 + w;
        x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
        if (v < V && k < K) head_ld4<VEC>((const T*)src + v * stride + k, x[i]);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) amax = max(amax, head_amax4(x[i]));
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (lane == 0) sh[w] = amax;
    __syncthreads();
    amax = sh[0];
#pragma unroll
    for (int i = 1; i < 8; i++) amax = max(amax, sh[i]);
    const float s = head_scale(amax), r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int v = vb * kHeadBlock + i * 8 + w;
        if (v < V && k < K) *reinterpret_cast<uint32_t*>(codes + (long long)v * K + k) = head_codes4(x[i], s, r);
    }
    if (threadIdx.x == 0) scales[(long long)vb * blocks + b] = s;
}

// ---- tcgen05 ------------------------------------------------------------------------------------------------------------
// Operand tile in shared memory: rows of 128 bytes (128 codes along K), 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t head_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// e4m3 by e4m3, both along K, fp32 sums; M = 128 lanes, N columns
__device__ __forceinline__ uint32_t head_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24); }
__device__ __forceinline__ void head_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void head_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
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

// ---- the product --------------------------------------------------------------------------------------------------------
struct HeadParams {
    const float* sa;         // (blocks, pitch): the tokens' scales
    const float* sw;         // (V blocks, blocks): the weights'
    void* out;               // (M, V), rows ldo elements apart
    long long ldo;
    int M, V, blocks, pitch;
    int n;                   // tokens of a tile, a multiple of 16
    int token_tiles, tiles;
    int stages;
    uint32_t polls;
    int *status, *mirror;
};

constexpr int kHeadMaxStages = 12;
__host__ __device__ constexpr int head_stage_bytes(int n) { return 128 * 128 + n * 128 + ((n * 4 + 1023) / 1024) * 1024; }

struct HeadShared {
    uint64_t full[kHeadMaxStages], empty[kHeadMaxStages], sum_full[2], sum_empty[2];
    uint32_t tmem;
    int gave_up;
};

// NT: most tokens of a tile (32, 64, 128, 256).  Warps 0 .. W-1 add the blocks' sums up, each thread one row of weights by
// NT tokens (half of them at NT = 256); then one warp that copies and one that multiplies.
template <int NT, typename OUT>
__global__ void __launch_bounds__((NT > 128 ? 8 : 4) * 32 + 64, 1)
    head_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ HeadParams p) {
    constexpr int W = NT > 128 ? 8 : 4, COLS = NT > 128 ? NT / 2 : NT;
    constexpr uint32_t kTmemCols = 2 * NT;
    extern __shared__ uint8_t raw_smem[];
    __shared__ HeadShared sh;
    const uint32_t base = (smem_addr(raw_smem) + 1023u) & ~1023u;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t stage_bytes = (uint32_t)head_stage_bytes(p.n);
    const uint32_t full = smem_addr(sh.full), empty = smem_addr(sh.empty), sfull = smem_addr(sh.sum_full), sempty = smem_addr(sh.sum_empty);
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1 + W);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(sfull + 8 * i, 1);
            mbar_init(sempty + 8 * i, W);
        }
        sh.gave_up = 0;
        fence_mbar_init();
    }
    if (w == W + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sh.tmem;
    grid_dependency_wait();                       // the tokens' codes and scales are another kernel's
    const volatile int* gave_up = &sh.gave_up;
    // A wait that runs out is reported; everyone stops at the next wait, and the copies in flight are waited for below.
    auto wait = [&](uint32_t bar, uint32_t parity) {
        for (uint32_t i = 0; i < p.polls; i++) {
            if (mbar_try_wait(bar, parity)) return true;
            if (*gave_up) return false;
        }
        sh.gave_up = 1;
        atomicExch(p.status, RS_ERR_TIMEOUT);
        if (p.mirror) *reinterpret_cast<volatile int*>(p.mirror) = RS_ERR_TIMEOUT;
        return false;
    };
    if (w == W) {
        if (lane == 0) {
            uint32_t it = 0, s = 0, ph = 0;      // blocks so far, their stage, its phase
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
                const int vb = tile / p.token_tiles, m0 = (tile - vb * p.token_tiles) * p.n;
                for (int b = 0; b < p.blocks; b++, it++) {
                    if (it >= (uint32_t)p.stages && !wait(empty + 8 * s, ph ^ 1u)) { ok = false; break; }
                    const uint32_t at = base + s * stage_bytes, bar = full + 8 * s;
                    mbar_expect_tx(bar, 128u * 128u + (uint32_t)p.n * 132u);
                    tma_2d(at, &map_w, b * kHeadBlock, vb * 128, bar);
                    tma_2d(at + 16384u, &map_x, b * kHeadBlock, m0, bar);
                    bulk_g2s(at + 16384u + (uint32_t)p.n * 128u, p.sa + (long long)b * p.pitch + m0, (uint32_t)p.n * 4u, bar);
                    if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1u; }
                }
            }
            // nothing may still be on its way into shared memory when the CTA ends: neither a copy nor, in the ordinary
            // case, the arrival that frees a stage
            const uint32_t n = min(it, (uint32_t)p.stages);
            for (uint32_t i = 0; i < n; i++) {
                const uint32_t k = it - 1 - i, st = k % (uint32_t)p.stages, parity = (k / (uint32_t)p.stages) & 1u;
                if (!ok || !wait(empty + 8 * st, parity)) {
                    ok = false;
                    mbar_wait_bounded(full + 8 * st, parity, p.polls);
                }
            }
        }
    } else if (w == W + 1) {
        if (lane == 0) {
            const uint32_t idesc = head_idesc(p.n);
            uint32_t it = 0, s = 0, ph = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x)
                for (int b = 0; b < p.blocks; b++, it++) {
                    const uint32_t buf = it & 1u;
                    if (it >= 2 && !wait(sempty + 8 * buf, ((it >> 1) & 1u) ^ 1u)) { ok = false; break; }
                    if (!wait(full + 8 * s, ph)) { ok = false; break; }
                    tmem_fence_after();
                    const uint64_t da = head_desc(base + s * stage_bytes), db = head_desc(base + s * stage_bytes + 16384u);
#pragma unroll
                    for (int k = 0; k < 4; k++) head_mma(tmem + buf * NT, da + 2 * k, db + 2 * k, idesc, k > 0);
                    head_commit(empty + 8 * s);
                    head_commit(sfull + 8 * buf);
                    if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1u; }
                }
            // (after a wait that ran out: the products in flight end by themselves)
            if (!ok && it > 0) mbar_wait_bounded(sfull + 8 * ((it - 1) & 1u), ((it - 1) >> 1) & 1u, p.polls);
        }
    } else {
        const int quad = w & 3, half = w >> 2, row = quad * 32 + lane, col0 = half * COLS;
        uint32_t it = 0, s = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
            const int vb = tile / p.token_tiles, m0 = (tile - vb * p.token_tiles) * p.n;
            const float* sw = p.sw + (long long)vb * p.blocks;
            float acc[COLS];
#pragma unroll
            for (int i = 0; i < COLS; i++) acc[i] = 0.f;
            for (int b = 0; b < p.blocks; b++, it++) {
                const uint32_t buf = it & 1u;
                const float f = __ldg(sw + b);
                ok = wait(sfull + 8 * buf, (it >> 1) & 1u);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tmem_fence_after();
                const float* sa = reinterpret_cast<const float*>(raw_smem + (base - smem_addr(raw_smem)) + s * stage_bytes + 16384u + (uint32_t)p.n * 128u) + col0;
#pragma unroll
                for (int q = 0; q < COLS; q += 16) {
                    if (col0 + q < p.n) {
                        float v[16];
                        tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + buf * NT + col0 + q, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 g = *reinterpret_cast<const float4*>(sa + q + i);
                            acc[q + i] = fmaf(v[i], g.x * f, acc[q + i]);
                            acc[q + i + 1] = fmaf(v[i + 1], g.y * f, acc[q + i + 1]);
                            acc[q + i + 2] = fmaf(v[i + 2], g.z * f, acc[q + i + 2]);
                            acc[q + i + 3] = fmaf(v[i + 3], g.w * f, acc[q + i + 3]);
                        }
                    }
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(sempty + 8 * buf);
                    mbar_arrive(empty + 8 * s);
                }
                if (++s == (uint32_t)p.stages) s = 0;
            }
            if (!ok) break;
            const int v = vb * 128 + row;
            if (v < p.V) {
                OUT* o = (OUT*)p.out + (long long)(m0 + col0) * p.ldo + v;
                const int cols = min(p.n, p.M - m0) - col0;
#pragma unroll
                for (int i = 0; i < COLS; i++) {
                    OUT y;
                    head_to(y, acc[i]);
                    if (i < cols) __stcs(o + i * p.ldo, y);
                }
            }
        }
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (w == W + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
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
// (rows, K) codes in tiles of box_rows x 128; what lies outside reads as zero
static int head_map(CUtensorMap* m, const void* codes, long long rows, long long K, int box_rows) {
    EncodeTiled enc = head_encoder();
    if (!enc) return host_cuda_fail(cudaErrorSymbolNotFound, "cuTensorMapEncodeTiled");
    const cuuint64_t dim[2] = {(cuuint64_t)K, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)K};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult e = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? RS_OK : host_cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
}

template <int NT, typename OUT>
static int head_launch(const CUtensorMap& w, const CUtensorMap& x, const HeadParams& p, int smem, int grid, cudaStream_t stream) {
    auto kern = head_product_kernel<NT, OUT>;
    {
        static std::mutex mu;
        static bool done[64] = {};      // per device
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
    cfg.blockDim = dim3((NT > 128 ? 8 : 4) * 32 + 64);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    // starts while the tokens are still being quantized and waits for them itself
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, w, x, p);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaLaunchKernelEx(head)");
    host_count_launch();
    return RS_OK;
}
template <typename OUT>
static int head_launch_n(const CUtensorMap& w, const CUtensorMap& x, const HeadParams& p, int smem, int grid, cudaStream_t stream) {
    if (p.n <= 32) return head_launch<32, OUT>(w, x, p, smem, grid, stream);
    if (p.n <= 64) return head_launch<64, OUT>(w, x, p, smem, grid, stream);
    if (p.n <= 128) return head_launch<128, OUT>(w, x, p, smem, grid, stream);
    return head_launch<256, OUT>(w, x, p, smem, grid, stream);
}

template <bool ROWS>
static int head_quantize(const void* src, int dtype, long long stride, long long rows, long long K, uint8_t* codes, float* scales, int pitch,
                         cudaStream_t st) {
    const int blocks = (int)((K + kHeadBlock - 1) / kHeadBlock);
    const uintptr_t size = dtype == RS_DTYPE_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)src & (4 * size - 1)) == 0 && stride % 4 == 0;
    const long long ctas = ROWS ? (rows * blocks + 7) / 8 : (rows + kHeadBlock - 1) / kHeadBlock * blocks;
    if (ctas > 0x7fffffffLL) return RS_ERR_LIMIT;
    const unsigned grid = (unsigned)ctas;
#define RS_HEAD_Q(DT, VEC)                                                                                                          \
    if constexpr (ROWS) head_quantize_rows_kernel<DT, VEC><<<grid, 256, 0, st>>>(src, stride, (int)rows, (int)K, blocks, codes, scales, pitch); \
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
static int head_pitch(long long M) { return (int)((M + 255) / 256 * 256) + 256; }      // a tile's scales never end behind a row
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
    return head_quantize<false>(weight, dtype, row_stride, V, K, (uint8_t*)codes_device, scales_device, 0, (cudaStream_t)stream);
}

size_t rs_head_workspace_bytes(int64_t M, int64_t K) {
    if (rs::head_check(M, K)) return 0;
    const size_t blocks = (size_t)((K + 127) / 128), codes = ((size_t)M * (size_t)K + 255) / 256 * 256;
    return codes + blocks * (size_t)rs::head_pitch(M) * 4;
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
    const size_t code_bytes = ((size_t)M * (size_t)K + 255) / 256 * 256;
    uint8_t* a = (uint8_t*)workspace_device;
    float* sa = (float*)(a + code_bytes);
    p.sa = sa;
    p.sw = scales_device;
    p.out = out_device;
    p.ldo = out_stride;
    p.M = (int)M;
    p.V = (int)V;
    p.blocks = (int)((K + 127) / 128);
    p.pitch = head_pitch(M);
    // tiles of at most 256 tokens, as equal as multiples of 16 allow
    const long long most = (M + 255) / 256;
    p.n = (int)(((M + most - 1) / most + 15) / 16 * 16);
    p.token_tiles = (int)((M + p.n - 1) / p.n);
    const long long tiles = (V + 127) / 128 * p.token_tiles;
    if (tiles > 0x7fffffffLL) return RS_ERR_LIMIT;
    p.tiles = (int)tiles;
    const int room = dev.smem_optin - 2048 - 1024, per = head_stage_bytes(p.n);
    p.stages = room / per > kHeadMaxStages ? kHeadMaxStages : room / per;
    p.polls = host_wait_polls();
    p.mirror = dev.mirror;
    CUtensorMap w, x;
    if ((rc = head_map(&w, codes_device, V, K, 128)) || (rc = head_map(&x, a, M, K, p.n))) return rc;
    if ((rc = head_quantize<true>(hidden, hidden_dtype, hidden_stride, M, K, a, sa, p.pitch, (cudaStream_t)stream))) return rc;
    const int smem = p.stages * per + 1024, grid = p.tiles < dev.sms ? p.tiles : dev.sms;
    switch (out_dtype) {
        case RS_DTYPE_F32: return head_launch_n<float>(w, x, p, smem, grid, (cudaStream_t)stream);
        case RS_DTYPE_F16: return head_launch_n<__half>(w, x, p, smem, grid, (cudaStream_t)stream);
        default: return head_launch_n<__nv_bfloat16>(w, x, p, smem, grid, (cudaStream_t)stream);
    }
}

}  // extern "C"

// Log probabilities of given tokens, their entropy, rank and alternatives, and the gradient with respect to the logits.
// sm_100a only.
//
// With z = x / T, m = max z, s = sum exp(z - m):
//     log p_t = z_t - m - ln s          H = ln s - sum (z - m) exp(z - m) / s
//     d/dx_j (g log p_t + h H) = 1/T (g [j = t] - p_j (g + h (ln p_j + H)))
// A row is read once: every thread keeps the maximum it has seen, and the two sums relative to it.  Maxima are compared on
// the logits as they are; exponents are taken as ((x - m) log2(e)/T) so that neither masks of the type's lowest value nor a
// row made of nothing else overflow.  log p of a token of probability nearly one is -log1p(excess), the excess being s without
// the maximum's own 1.  What the other threads hold is added up apart from that 1.  The maximum's own thread adds to it and loses
// what lies below 2^-24 there; where the excess is small, its elements are read again and added by themselves (lp_rest).
#include "rs_device.cuh"
#include "rs_host.cuh"
#include "../../include/rapid_sampling_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <mutex>
#include <type_traits>

namespace rs {

constexpr int kLpAhead = 4;            // 16-byte loads in flight per thread
constexpr int kTopMax = 64;            // longest list of alternatives
constexpr int kTopHot = 256;           // most pieces of a part that are looked at again (a list of 64 has about 100)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFloor = -160.f;       // exponent from which on exp2f is zero; keeps 0 * inf out of the second sum
// Excess below which the maximum's thread is read again.  Its own sum is off by 2^-24 for each of its additions at most (17, and one
// a step, of which a row of 151936 has up to 37), so the excess keeps its digits to 2^-12 from here on, and to 2^-16 as a rule.
constexpr float kSmallExcess = 0.015625f;

__device__ int g_lp_status;            // status word of these calls on this device (rs_logprobs_status)

struct LpParams {
    const void* logits;
    long long sb, st;                  // elements between sequences, between positions
    long long rows;                    // B * T
    int T, V;
    const void* tokens;                // int32 or int64, or null
    int wide_tokens;
    long long tok_sb, tok_st;
    float temperature;
    const float* row_temperature;      // or null
    long long tmp_sb, tmp_st;
    float *logprob, *entropy;          // rows
    float2* stats;                     // rows: largest logit, log2 of the sum
    int* rank;                         // rows
    float* top;                        // rows * top_n
    int* top_ids;
    int top_n;
    int* mirror;
    // backward
    const float *g_logprob, *g_entropy;
    long long gl_sb, gl_st, ge_sb, ge_st;
    void* grad;                        // (rows, V) contiguous
    int chunks, piece;                 // CTAs per row, vectors of each
};

// ---- elements -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 16 bytes of logits: E elements, widened pair by pair.
template <int DT> struct Elem;
template <> struct Elem<RS_DTYPE_F32> {
    using T = float;
    static constexpr int E = 4;
    static __device__ __forceinline__ void pairs(const uint4& v, uint64_t (&x)[2]) {
        x[0] = f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
        x[1] = f2_pack(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    template <int U> static __device__ __forceinline__ float largest(const uint4 (&v)[U]) {      // NaN if any element is
        float m = __uint_as_float(v[0].x);
#pragma unroll
        for (int i = 0; i < U; i++) {
            m = max3_nan(m, __uint_as_float(v[i].x), __uint_as_float(v[i].y));
            m = max3_nan(m, __uint_as_float(v[i].z), __uint_as_float(v[i].w));
        }
        return m;
    }
    // counts the elements of at least `from`, a value of the type
    using Count = int;
    static __device__ __forceinline__ Count none() { return 0; }
    static __device__ __forceinline__ void reach(Count& n, const uint4& v, float from) {
        n += (__uint_as_float(v.x) >= from) + (__uint_as_float(v.y) >= from) + (__uint_as_float(v.z) >= from) + (__uint_as_float(v.w) >= from);
    }
    static __device__ __forceinline__ int whole(Count n) { return n; }
    static __device__ __forceinline__ float one(const T* p) { return *p; }
    static __device__ __forceinline__ uint4 narrow(const uint64_t (&x)[2]) {
        float a, b, c, d;
        f2_unpack(x[0], a, b);
        f2_unpack(x[1], c, d);
        return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
    }
    static __device__ __forceinline__ T to(float x) { return x; }
};
template <> struct Elem<RS_DTYPE_F16> {
    using T = __half;
    static constexpr int E = 8;
    static __device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
    static __device__ __forceinline__ void pairs(const uint4& v, uint64_t (&x)[4]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h2(w[i]));
            x[i] = f2_pack(f.x, f.y);
        }
    }
    template <int U> static __device__ __forceinline__ float largest(const uint4 (&v)[U]) {
        __half2 m = h2(v[0].x);
#pragma unroll
        for (int i = 0; i < U; i++) m = __hmax2_nan(__hmax2_nan(__hmax2_nan(__hmax2_nan(m, h2(v[i].x)), h2(v[i].y)), h2(v[i].z)), h2(v[i].w));
        const float2 f = __half22float2(m);
        return max_nan(f.x, f.y);
    }
    using Count = __half2;             // exact up to 2048 in each half
    static __device__ __forceinline__ Count none() { return __float2half2_rn(0.f); }
    static __device__ __forceinline__ void reach(Count& n, const uint4& v, float from) {
        const __half2 f = __float2half2_rn(from);
        n = __hadd2(__hadd2(__hadd2(__hge2(h2(v.x), f), __hge2(h2(v.y), f)), __hadd2(__hge2(h2(v.z), f), __hge2(h2(v.w), f))), n);
    }
    static __device__ __forceinline__ int whole(Count n) { return (int)(__low2float(n) + __high2float(n)); }
    static __device__ __forceinline__ float one(const T* p) { return __half2float(*p); }
    static __device__ __forceinline__ uint4 narrow(const uint64_t (&x)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float a, b;
            f2_unpack(x[i], a, b);
            const __half2 h = __floats2half2_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ T to(float x) { return __float2half_rn(x); }
};
template <> struct Elem<RS_DTYPE_BF16> {
    using T = __nv_bfloat16;
    static constexpr int E = 8;
    static __device__ __forceinline__ __nv_bfloat162 h2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    static __device__ __forceinline__ void pairs(const uint4& v, uint64_t (&x)[4]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
    template <int U> static __device__ __forceinline__ float largest(const uint4 (&v)[U]) {
        __nv_bfloat162 m = h2(v[0].x);
#pragma unroll
        for (int i = 0; i < U; i++) m = __hmax2_nan(__hmax2_nan(__hmax2_nan(__hmax2_nan(m, h2(v[i].x)), h2(v[i].y)), h2(v[i].z)), h2(v[i].w));
        return max_nan(__low2float(m), __high2float(m));
    }
    using Count = __nv_bfloat162;      // exact up to 256 in each half
    static __device__ __forceinline__ Count none() { return __float2bfloat162_rn(0.f); }
    static __device__ __forceinline__ void reach(Count& n, const uint4& v, float from) {
        const __nv_bfloat162 f = __float2bfloat162_rn(from);
        n = __hadd2(__hadd2(__hadd2(__hge2(h2(v.x), f), __hge2(h2(v.y), f)), __hadd2(__hge2(h2(v.z), f), __hge2(h2(v.w), f))), n);
    }
    static __device__ __forceinline__ int whole(Count n) { return (int)(__low2float(n) + __high2float(n)); }
    static __device__ __forceinline__ float one(const T* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ uint4 narrow(const uint64_t (&x)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float a, b;
            f2_unpack(x[i], a, b);
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ T to(float x) { return __float2bfloat16_rn(x); }
};
template <int DT>
__device__ __forceinline__ void widen(const uint4& v, float (&x)[Elem<DT>::E]) {
    uint64_t p[Elem<DT>::E / 2];
    Elem<DT>::pairs(v, p);
#pragma unroll
    for (int i = 0; i < Elem<DT>::E / 2; i++) f2_unpack(p[i], x[2 * i], x[2 * i + 1]);
}

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Order of floats as unsigned integers, -0 equal to +0; NaN above everything or below, which no caller relies on.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kKeyNone = 0x007FFFFFu;      // key of -inf
// The next larger value of the logits' type; of +inf a NaN, which nothing reaches.
template <int DT>
__device__ __forceinline__ float next_above(float x) {
    constexpr uint32_t kStep = DT == RS_DTYPE_F32 ? 1u : DT == RS_DTYPE_F16 ? 0u : 0x10000u;
    if constexpr (DT == RS_DTYPE_F16) {
        const uint32_t u = __half_as_ushort(__float2half_rn(x + 0.0f));
        return __half2float(__ushort_as_half((unsigned short)(u & 0x8000u ? (u == 0x8001u ? 0u : u - 1u) : u + 1u)));
    } else {
        const uint32_t u = __float_as_uint(x + 0.0f);
        return __uint_as_float(u >> 31 ? (u == 0x80000000u + kStep ? 0u : u - kStep) : u + kStep);
    }
}

// ---- one row's position, token and temperature --------------------------------------------------------------------
struct LpRow {
    long long b, t, token;      // token: < 0 where the position is not scored
    float inv_t, c;             // 1 / T, log2(e) / T
    bool bad_token, bad_temperature;
};
__device__ __forceinline__ LpRow lp_row(const LpParams& p, uint32_t r) {
    LpRow o;
    const uint32_t b = r / (uint32_t)p.T;
    o.b = b;
    o.t = r - b * (uint32_t)p.T;
    o.token = 0;
    if (p.tokens) {
        const long long at = o.b * p.tok_sb + o.t * p.tok_st;
        o.token = p.wide_tokens ? ((const long long*)p.tokens)[at] : (long long)((const int*)p.tokens)[at];
    }
    o.bad_token = o.token >= p.V;
    float t = p.row_temperature ? p.row_temperature[o.b * p.tmp_sb + o.t * p.tmp_st] : p.temperature;
    o.bad_temperature = !(t >= 0.001f && t <= 1000.f);
    if (o.bad_temperature) t = 1.f;
    o.inv_t = __fdiv_rn(1.f, t);
    o.c = __fdiv_rn(kLog2e, t);
    return o;
}
// (x - m) / T; by way of halves, whose difference is finite however far apart the two lie
__device__ __forceinline__ float lp_scaled(float x, float m, float inv_t) { return (0.5f * x - 0.5f * m) * (2.f * inv_t); }
__device__ __forceinline__ void lp_report(const LpParams& p, int code) {
    atomicExch(&g_lp_status, code);
    if (p.mirror) *reinterpret_cast<volatile int*>(p.mirror) = code;
}

// ---- running statistics -------------------------------------------------------------------------------------------
struct Stat {
    float mx;      // largest logit seen (NaN if any is); -inf: none but -inf
    float s, u;    // sums of e and of e (x - m) c with e = exp2((x - m) c), m = max(mx, -FLT_MAX)
};
__device__ __forceinline__ float ref_of(float mx) { return max_nan(mx, -FLT_MAX); }
__device__ __forceinline__ void stat_raise(Stat& a, float bm, float c) {
    const float m0 = ref_of(a.mx);
    a.mx = max_nan(a.mx, bm);
    const float d = fmaxf((m0 - ref_of(a.mx)) * c, kFloor), f = ex2(d);
    a.u = f * fmaf(d, a.s, a.u);
    a.s *= f;
}
__device__ __forceinline__ void stat_one(Stat& a, float x, float c) {
    stat_raise(a, x, c);
    const float d = fmaxf((x - ref_of(a.mx)) * c, kFloor), e = ex2(d);
    a.s += e;
    a.u = fmaf(d, e, a.u);
}
// U vectors; the products and sums two at a time.
template <int DT, int U>
__device__ __forceinline__ float stat_add(Stat& a, const uint4 (&v)[U], float c) {      // returns their maximum
    const float most = Elem<DT>::largest(v);
    stat_raise(a, most, c);
    const float m = -ref_of(a.mx);
    const uint64_t mm = f2_pack(m, m), cc = f2_pack(c, c);
    uint64_t s = 0ull, u = 0ull;
#pragma unroll
    for (int i = 0; i < U; i++) {
        uint64_t x[Elem<DT>::E / 2];
        Elem<DT>::pairs(v[i], x);
#pragma unroll
        for (int k = 0; k < Elem<DT>::E / 2; k++) {
            float d0, d1;
            f2_unpack(f2_mul(f2_add(x[k], mm), cc), d0, d1);
            d0 = fmaxf(d0, kFloor);
            d1 = fmaxf(d1, kFloor);
            const uint64_t e = f2_pack(ex2(d0), ex2(d1));
            s = f2_add(s, e);
            u = f2_fma(f2_pack(d0, d1), e, u);
        }
    }
    float s0, s1, u0, u1;
    f2_unpack(s, s0, s1);
    f2_unpack(u, u0, u1);
    a.s += s0 + s1;
    a.u += u0 + u1;
    return most;
}
// Statistics of many threads.  The sum is w = 1 + own + s: own is the excess of the thread `who`, which has the maximum (-1: no
// element above -inf), s what all others add.
struct Group {
    float mx, s, u, own;
    int who;
    __device__ __forceinline__ float excess() const { return s + own; }
};
__device__ __forceinline__ Group group_none() { return {-INFINITY, 0.f, 0.f, -1.f, 0}; }
// The lanes' statistics as one, in every lane.  Terms are added in a fixed order.
__device__ __forceinline__ Group group_warp(const Group& a, float c) {
    Group r;
    r.mx = warp_max_nan(a.mx);
    const float d = fmaxf((ref_of(a.mx) - ref_of(r.mx)) * c, kFloor), f = ex2(d), w = (1.f + a.own) + a.s;
    const int owner = __ffs(__ballot_sync(0xffffffffu, a.mx == r.mx)) - 1;
    r.s = (int)(threadIdx.x & 31) == owner ? a.s : f * w;
    r.u = f * fmaf(d, w, a.u);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
        r.u += __shfl_xor_sync(0xffffffffu, r.u, o);
    }
    r.own = __shfl_sync(0xffffffffu, a.own, owner);      // (a NaN has no owner, and its sums are not used)
    r.who = __shfl_sync(0xffffffffu, a.who, owner);
    return r;
}

// ---- the part of a row that a CTA reads ----------------------------------------------------------------------------
// Elements up to the first 16-byte boundary and behind the last whole vector are single ones, taken by the first and the
// last CTA of the row; the vectors between are split evenly.  Vector v of the CTA belongs to thread v % NT.
template <int DT>
struct Span {
    using T = typename Elem<DT>::T;
    const T* row;
    const uint4* vec;
    int head, nvec, V;       // of the row
    int v0, v1;              // this CTA's vectors
    bool first, last;
    __device__ __forceinline__ Span(const LpParams& p, const LpRow& w) : Span((const T*)p.logits + w.b * p.sb + w.t * p.st, p.V) {}
    __device__ __forceinline__ Span(const T* at, int n) : row(at), V(n) {
        constexpr int E = Elem<DT>::E;
        head = (int)((16u - ((uint32_t)(uintptr_t)row & 15u)) & 15u) / (int)sizeof(T);
        if (head > V) head = V;
        nvec = (V - head) / E;
        vec = reinterpret_cast<const uint4*>(row + head);
    }
    __device__ __forceinline__ void share(int part, int log_parts) {      // one of 2^log_parts equal parts
        v0 = (int)(((long long)nvec * part) >> log_parts);
        v1 = (int)(((long long)nvec * (part + 1)) >> log_parts);
        first = part == 0;
        last = part == (1 << log_parts) - 1;
    }
    __device__ __forceinline__ void piece(int part, int size, int parts) {      // `size` vectors, the last part the rest
        v0 = min(part * size, nvec);
        v1 = part == parts - 1 ? nvec : min(v0 + size, nvec);
        first = part == 0;
        last = part == parts - 1;
    }
    __device__ __forceinline__ int tail() const { return head + nvec * Elem<DT>::E; }      // index of the first element behind
    __device__ __forceinline__ int index(int v) const { return head + v * Elem<DT>::E; }
    // calls f(index, value) for the single elements of thread h
    template <class F> __device__ __forceinline__ void singles(int h, F&& f) const {
        if (first && h < head) f(h, Elem<DT>::one(row + h));
        const int j = tail() + h;
        if (last && h < Elem<DT>::E && j < V) f(j, Elem<DT>::one(row + j));
    }
};

// The excess of thread `th`, which has the row's maximum `mx`, by one warp: its vectors and single elements are read again and
// what lies below the maximum is added by itself; every further element equal to the maximum counts 1.  It costs such a row the
// latency of its loads, 1.3 us, which the other rows on the multiprocessor hide in part.  us without and with, every row of such
// logits: statistics of 4088 rows of 151936 bf16 195 / 201, 16384 of 4096 43 / 53; with a list of 20 249 / 258 and 105 / 112.
template <int DT, int NT>
__device__ __forceinline__ float lp_rest(const typename Elem<DT>::T* row, int V, int v0, int v1, bool first, bool last, int th, float mx, float c) {
    constexpr int E = Elem<DT>::E;
    Span<DT> sp(row, V);
    sp.v0 = v0; sp.v1 = v1; sp.first = first; sp.last = last;
    const int lane = threadIdx.x & 31;
    float rest = 0.f;
    int equal = 0;
    auto add = [&](float x) {
        const float e = ex2(fmaxf((x - mx) * c, kFloor));
        equal += x == mx;
        rest += x == mx ? 0.f : e;
    };
    if (lane == 0) sp.singles(th, [&](int, float x) { add(x); });
    for (int v = v0 + th + lane * NT; v < v1; v += 4 * 32 * NT) {
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (v + i * 32 * NT < v1) raw[i] = ld_stream(sp.vec + v + i * 32 * NT);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (v + i * 32 * NT < v1) {
                float x[E];
                widen<DT>(raw[i], x);
#pragma unroll
                for (int k = 0; k < E; k++) add(x[k]);
            }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
    return rest + (float)((int)warp_sum_u32((uint32_t)equal) - 1);
}

// A call of its own leaves the statistics' loop the registers it had (inlined: 196 -> 203 us for the 4088 rows, nothing small about
// their excess); with a list inlining is as good or better (252 -> 250).
template <int DT, int NT>
__device__ __noinline__ float lp_rest_called(const typename Elem<DT>::T* row, int V, int v0, int v1, bool first, bool last, int th, float mx, float c) {
    return lp_rest<DT, NT>(row, V, v0, v1, first, last, th, mx, c);
}

// ---- statistics, rank and alternatives of rows ---------------------------------------------------------------------
struct LpShared {
    float mx[8], s[8], u[8], own[8];                     // the CTA's warps
    int who[8], cnt[8];
    float c_mx[16], c_s[16], c_u[16], c_own[16];         // the cluster's CTAs
    int c_who[16], c_cnt[16];
    float r_mx, r_logs;
};
// SHARED: the row is a cluster's.  Small, because what it takes is lost to the loads in flight, which pass through L1.
template <int NT, bool SHARED>
struct TopShared {
    static constexpr int kThreads = NT;
    static constexpr int kCap = 640;                               // candidates for a list
    static constexpr int kPieces = NT == 64 ? 2 : 16;              // steps that the maxima of pieces are kept of
    alignas(16) uint32_t key[NT];
    unsigned long long cand[kCap];
    unsigned long long list[(SHARED ? 16 : 1) * kTopMax];          // the cluster's lists of top_n entries, in the first CTA; 0: none
    alignas(16) uint16_t piece[kPieces * NT];                      // upper halves of keys
    short hot[kTopHot];
    int nhot, nfinite, ncand, count;
    uint32_t tau;
};

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) { st_cluster_u32(addr, __float_as_uint(v)); }
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// The maxima of pieces, a thread's vectors of a step or, in long parts, of 2^shift steps: where a list's entries are.  The
// upper half of a key is kept: all of a 16-bit logit's, and of a 32-bit one's enough.
template <class TS>
__device__ __forceinline__ int top_shift_of(int steps) {
    return steps <= TS::kPieces ? 0 : 32 - __clz((steps - 1) / TS::kPieces);
}
template <class TS>
__device__ __forceinline__ void top_note(TS& sh, int step, int shift, float most) {
    uint16_t* at = sh.piece + (step >> shift) * TS::kThreads + threadIdx.x;
    const uint32_t k = key_of(most) >> 16;
    *at = (uint16_t)((step & ((1 << shift) - 1)) ? max((uint32_t)*at, k) : k);
}
template <class TS>
__device__ __forceinline__ void top_push(TS& sh, uint32_t key, int j) {
    const int at = atomicAdd(&sh.ncand, 1);
    if (at < TS::kCap) sh.cand[at] = ((unsigned long long)key << 32) | (uint32_t)~j;
}
// Elements of the CTA's part with a key of at least `at_least`.
template <int DT, class TS>
__device__ int top_count(const Span<DT>& sp, TS& sh, uint32_t at_least) {
    constexpr int NT = TS::kThreads;
    constexpr int E = Elem<DT>::E;
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    int n = 0;
    for (int v = sp.v0 + (int)threadIdx.x; v < sp.v1; v += NT) {
        float x[E];
        widen<DT>(ld_stream(sp.vec + v), x);
#pragma unroll
        for (int i = 0; i < E; i++) n += key_of(x[i]) >= at_least;
    }
    sp.singles(threadIdx.x, [&](int, float x) { n += key_of(x) >= at_least; });
    atomicAdd(&sh.count, n);
    __syncthreads();
    return sh.count;
}
// The n-th largest key is bisected, what lies above it collected, and the rest filled up with elements equal to it in the
// order of their indices.  For parts whose n largest elements are not told apart by the threads' maxima: long runs of equal
// logits, or large ones that crowd in few threads.  About 32 passes over the part at worst, 2 where the threads' n-th
// largest maximum is the key, as with a mask of the type's lowest value.
template <int DT, class TS>
__device__ void top_exact(const Span<DT>& sp, TS& sh, int n) {
    constexpr int NT = TS::kThreads;
    constexpr int E = Elem<DT>::E;
    const int t = threadIdx.x;
    uint32_t lo = sh.tau, hi = 0xFF800001u;        // count(lo) >= n > count(hi): nothing lies above +inf's key
    for (uint32_t mid = lo + 1; hi - lo > 1; mid = lo + (hi - lo) / 2) {
        if (top_count(sp, sh, mid) >= n) lo = mid; else hi = mid;
    }
    __syncthreads();
    if (t == 0) sh.ncand = 0;
    __syncthreads();
    for (int v = sp.v0 + t; v < sp.v1; v += NT) {
        float x[E];
        widen<DT>(ld_stream(sp.vec + v), x);
#pragma unroll
        for (int i = 0; i < E; i++)
            if (key_of(x[i]) > lo) top_push(sh, key_of(x[i]), sp.index(v) + i);
    }
    sp.singles(t, [&](int j, float x) { if (key_of(x) > lo) top_push(sh, key_of(x), j); });
    __syncthreads();
    if (sp.first) {
        if (t < sp.head && key_of(Elem<DT>::one(sp.row + t)) == lo) top_push(sh, lo, t);
        __syncthreads();
    }
    constexpr int kStep = 64;                      // vectors at a time: at most 512 entries more than the list needs
    for (int v = sp.v0; v < sp.v1; v += kStep) {
        const int have = sh.ncand;
        __syncthreads();
        if (have >= n) break;
        if (t < kStep && v + t < sp.v1) {
            float x[E];
            widen<DT>(ld_stream(sp.vec + v + t), x);
#pragma unroll
            for (int i = 0; i < E; i++)
                if (key_of(x[i]) == lo) top_push(sh, lo, sp.index(v + t) + i);
        }
        __syncthreads();
    }
    if (sp.last && sh.ncand < n) {
        const int j = sp.tail() + t;
        __syncthreads();
        if (t < E && j < sp.V && key_of(Elem<DT>::one(sp.row + j)) == lo) top_push(sh, lo, j);
    }
    __syncthreads();
}
// The n largest elements of the CTA's part (larger key first, then lower index), unordered, among sh.cand[0 .. result).
// At least n threads have a maximum that reaches the n-th largest maximum of the groups, so the list lies within the elements
// that reach it too, and those are in the few pieces whose maximum does: only they are read again.
template <int DT, class TS>
__device__ int top_collect(const Span<DT>& sp, TS& sh, float mx, int n) {
    constexpr int NT = TS::kThreads;
    constexpr int E = Elem<DT>::E;
    const int t = threadIdx.x;
    const uint32_t mine = key_of(mx);
    // the n-th largest of the maxima of equal groups of threads, at least 1.6 n of them: exact enough (about 1.5 n threads
    // reach it) and a quarter of the time that the n-th largest of all threads' takes
    const int busy = min(NT, sp.v1 - sp.v0);      // threads that have vectors
    int lg = 0;
    while (lg < 5 && NT >> (lg + 1) >= 4 && (busy >> (lg + 1)) * 5 >= n * 8) lg++;      // (four keys are read at a time)
    const int groups = NT >> lg;
    uint32_t of_group = mine;
    for (int step = 1; step < (1 << lg); step *= 2) of_group = max(of_group, __shfl_xor_sync(0xffffffffu, of_group, step));
    if ((t & ((1 << lg) - 1)) == 0) sh.key[t >> lg] = of_group;
    if (t == 0) { sh.nhot = 0; sh.ncand = 0; sh.tau = kKeyNone + 1u; }      // (fewer than n groups with a logit left: all those logits)
    __syncthreads();
    if (t < groups) {
        const uint32_t k = sh.key[t];
        int rank = 0;
#pragma unroll 4
        for (int i = 0; i < groups; i += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(sh.key + i);
            rank += (o.x > k || (o.x == k && i < t)) + (o.y > k || (o.y == k && i + 1 < t)) + (o.z > k || (o.z == k && i + 2 < t)) +
                    (o.w > k || (o.w == k && i + 3 < t));
        }
        if (rank == n - 1) sh.tau = max(k, kKeyNone + 1u);                   // one thread
    }
    __syncthreads();
    const uint32_t tau = sh.tau;
    constexpr int kStep = kLpAhead * NT;
    const int steps = (sp.v1 - sp.v0 + kStep - 1) / kStep, shift = top_shift_of<TS>(steps), pieces = ((steps + (1 << shift) - 1) >> shift) * NT;
    if (mine >= tau)                               // a thread's own pieces
        for (int i = t; i < pieces; i += NT)
            if (sh.piece[i] >= tau >> 16) {
                const int at = atomicAdd(&sh.nhot, 1);
                if (at < kTopHot) sh.hot[at] = (short)i;
            }
    sp.singles(t, [&](int j, float x) { if (key_of(x) >= tau) top_push(sh, key_of(x), j); });
    __syncthreads();
    const int nhot = sh.nhot;
    if (nhot <= kTopHot) {
        // the hot pieces' vectors spread over the CTA, four loads ahead
        static_assert(kLpAhead == 4, "vectors of a piece");
        const int le = 2 + shift, all = nhot << le;
        for (int i0 = t; i0 < all; i0 += 4 * NT) {
            uint4 raw[4];
            int at[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int i = i0 + q * NT;
                at[q] = sp.v1;
                if (i < all) {
                    const int piece = sh.hot[i >> le], k = i & ((1 << le) - 1), step = ((piece / NT) << shift) + (k >> 2);
                    at[q] = sp.v0 + step * kStep + (k & 3) * NT + piece % NT;
                }
                if (at[q] < sp.v1) raw[q] = ld_stream(sp.vec + at[q]);
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (at[q] >= sp.v1) continue;
                float x[E];
                widen<DT>(raw[q], x);
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (key_of(x[e]) >= tau) top_push(sh, key_of(x[e]), sp.index(at[q]) + e);
            }
        }
        __syncthreads();
    }
    if (nhot > kTopHot || sh.ncand > TS::kCap) top_exact(sp, sh, n);
    return min(sh.ncand, TS::kCap);      // (a row with NaN may offer more; its list is not used)
}

// One cluster of 2^log_parts CTAs per row (SHARED), or one CTA.  Many rows: bound by HBM, and by the exponentials as soon as the
// power cap lowers the clock (a bf16 logit takes one of 16 a cycle and multiprocessor, 7 instructions in all): 4088 rows of
// 151936 bf16 188 us for a short while (6.6 TB/s), 215 to 230 under the cap; f32 half as many 190 and 200.  With a list of 20: 250
// and 216.  Few rows: bound by latency, of the token's and the first logits' loads (1.6 us), the reduction (1), the list's bound
// (0.7), its second look (1.3), the cluster's barrier (1.2) and its end (1): 64 rows of 151936 bf16 with a list of 5, 15 us.
template <int DT, bool TOP, int NT, bool SHARED>
__global__ void __launch_bounds__(NT, 1024 / NT) lp_rows_kernel(const __grid_constant__ LpParams p, int log_parts) {
    constexpr int E = Elem<DT>::E;
    __shared__ LpShared sh;
    using TS = TopShared<NT, SHARED>;
    __shared__ typename std::conditional<TOP, TS, int>::type top;
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    if (!SHARED) log_parts = 0;
    const int parts = 1 << log_parts, part = SHARED ? (int)cluster_ctarank() : 0;
    const long long r = blockIdx.x >> log_parts;
    const LpRow row = lp_row(p, (uint32_t)r);
    Span<DT> sp(p, row);
    sp.share(part, log_parts);
    // steps of kLpAhead vectors a thread, the next step's on their way while one is added; the last one may be a part of one.
    // The first is asked for before the token is known, whose load takes as long.
    constexpr int kStep = kLpAhead * NT;
    uint4 raw[2][kLpAhead];
    auto load = [&](uint4 (&to)[kLpAhead], int v) {
#pragma unroll
        for (int i = 0; i < kLpAhead; i++)
            if (v + i * NT + t < sp.v1) to[i] = ld_stream(sp.vec + v + i * NT + t);
    };
    load(raw[0], sp.v0);
    if (row.token < 0 || row.bad_token) {         // not scored: the same for the whole cluster
        if (part == 0) {
            const float v = row.bad_token ? __int_as_float(0x7FC00000) : 0.f;
            if (t == 0) {
                if (row.bad_token) lp_report(p, RS_ERR_TOKEN);
                if (p.logprob) p.logprob[r] = v;
                if (p.entropy) p.entropy[r] = v;
                if (p.stats) p.stats[r] = make_float2(0.f, 0.f);
                if (p.rank) p.rank[r] = 0;
            }
            if (TOP && t < p.top_n) {
                p.top[r * p.top_n + t] = row.bad_token ? v : -INFINITY;
                p.top_ids[r * p.top_n + t] = -1;
            }
        }
        return;
    }
    if (parts > 1) cluster_arrive();
    const float c = row.c;
    const int token = (int)row.token;
    const float xt = Elem<DT>::one(sp.row + token);
    // rank: an element before the token counts from xt on, one behind it only from the type's next value on
    const float xt_above = next_above<DT>(xt);
    int cnt = 0;

    Stat a = {-INFINITY, 0.f, 0.f};
    sp.singles(t, [&](int j, float x) {
        stat_one(a, x, c);
        if (TOP) cnt += j < token ? x >= xt : x > xt;
    });
    const int top_shift = TOP ? top_shift_of<TS>((sp.v1 - sp.v0 + kStep - 1) / kStep) : 0;
    auto from = [&](int v) { return sp.index(v) < token ? xt : xt_above; };
    auto add = [&](const uint4 (&x)[kLpAhead], int v) {
        float most = -INFINITY;
        if (v + kStep <= sp.v1) {
            most = stat_add<DT>(a, x, c);
            if (TOP && most >= xt) {      // nothing to count otherwise: nearly always, where the token is a likely one
                typename Elem<DT>::Count n = Elem<DT>::none();
#pragma unroll
                for (int i = 0; i < kLpAhead; i++) Elem<DT>::reach(n, x[i], from(v + i * NT + t));
                cnt += Elem<DT>::whole(n);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLpAhead; i++)
                if (v + i * NT + t < sp.v1) {
                    const uint4 one[1] = {x[i]};
                    const float here = stat_add<DT>(a, one, c);
                    most = fmaxf(most, here);
                    if (TOP && here >= xt) {
                        typename Elem<DT>::Count n = Elem<DT>::none();
                        Elem<DT>::reach(n, x[i], from(v + i * NT + t));
                        cnt += Elem<DT>::whole(n);
                    }
                }
        }
        if constexpr (TOP) top_note(top, (v - sp.v0) / kStep, top_shift, most);
    };
    int v = sp.v0;
    if (TOP && p.tokens) {             // the token's own vector, if it begins before the token, is counted from xt on throughout
        const int own = token >= sp.head && token < sp.tail() ? (token - sp.head) / E : -1;
        if (own >= sp.v0 && own < sp.v1 && (own - sp.v0) % NT == t && sp.index(own) < token) {
            float x[E];
            widen<DT>(ld_stream(sp.vec + own), x);
#pragma unroll
            for (int i = 0; i < E; i++) cnt -= sp.index(own) + i >= token && x[i] == xt;
        }
    }
    while (v < sp.v1) {
        if (v + kStep < sp.v1) load(raw[1], v + kStep);
        add(raw[0], v);
        v += kStep;
        if (v >= sp.v1) break;
        if (v + kStep < sp.v1) load(raw[0], v + kStep);
        add(raw[1], v);
        v += kStep;
    }
    const float my_mx = a.mx;
    const Group of_warp = group_warp({a.mx, 0.f, a.u, a.s - 1.f, t}, c);
    if (TOP) cnt = (int)warp_sum_u32((uint32_t)cnt);
    if (lane == 0) {
        sh.mx[w] = of_warp.mx; sh.s[w] = of_warp.s; sh.u[w] = of_warp.u; sh.own[w] = of_warp.own; sh.who[w] = of_warp.who;
        if (TOP) sh.cnt[w] = cnt;
    }
    __syncthreads();
    if (parts > 1) cluster_wait();                // every CTA of the cluster runs: its shared memory may be written
    if (w == 0) {
        Group b = group_none();
        if (lane < NT / 32) b = {sh.mx[lane], sh.s[lane], sh.u[lane], sh.own[lane], sh.who[lane]};
        b = group_warp(b, c);
        int n = TOP ? (int)warp_sum_u32(lane < NT / 32 ? (uint32_t)sh.cnt[lane] : 0u) : 0;
        if (parts > 1) {
            if (lane == 0) {
                st_cluster_f32(map_to_cta(smem_addr(&sh.c_mx[part]), 0), b.mx);
                st_cluster_f32(map_to_cta(smem_addr(&sh.c_s[part]), 0), b.s);
                st_cluster_f32(map_to_cta(smem_addr(&sh.c_u[part]), 0), b.u);
                st_cluster_f32(map_to_cta(smem_addr(&sh.c_own[part]), 0), b.own);
                st_cluster_u32(map_to_cta(smem_addr(&sh.c_who[part]), 0), (uint32_t)b.who);
                if (TOP) st_cluster_u32(map_to_cta(smem_addr(&sh.c_cnt[part]), 0), (uint32_t)n);
            }
        } else if (lane == 0) {
            sh.c_mx[0] = b.mx; sh.c_s[0] = b.s; sh.c_u[0] = b.u; sh.c_own[0] = b.own; sh.c_who[0] = b.who;
            if (TOP) sh.c_cnt[0] = n;
        }
    }
    if constexpr (TOP) {
        const int n = p.top_n;
        const int nc = top_collect(sp, top, my_mx, n);
        for (int i = t; i < nc; i += NT) {
            const unsigned long long e = top.cand[i];
            int at = 0;
#pragma unroll 8
            for (int q = 0; q < nc; q++) at += top.cand[q] > e;
            if (at < n) st_cluster_u64(map_to_cta(smem_addr(&top.list[part * n + at]), 0), e);
        }
        if (t >= nc && t < n) st_cluster_u64(map_to_cta(smem_addr(&top.list[part * n + t]), 0), 0ull);      // no entry
    }
    if (parts > 1) {
        cluster_arrive();
        cluster_wait();
        if (part) return;
    } else {
        __syncthreads();
    }
    // the first CTA has everything
    if (w == 0) {
        const int from = SHARED ? lane : 0;
        Group b = group_none();
        if (from < parts) b = {sh.c_mx[from], sh.c_s[from], sh.c_u[from], sh.c_own[from], from * NT + sh.c_who[from]};
        int above = TOP && from < parts ? sh.c_cnt[from] : 0;
        if (SHARED) {
            b = group_warp(b, c);
            if (TOP) above = (int)warp_sum_u32((uint32_t)above);
        }
        const bool bad = !(b.mx < INFINITY), none = b.mx == -INFINITY;
        if (!bad && !none && b.excess() < kSmallExcess) {
            const int of = b.who / NT;
            sp.share(of, log_parts);
            if constexpr (TOP) b.own = lp_rest<DT, NT>(sp.row, sp.V, sp.v0, sp.v1, sp.first, sp.last, b.who % NT, b.mx, c);
            else b.own = lp_rest_called<DT, NT>(sp.row, sp.V, sp.v0, sp.v1, sp.first, sp.last, b.who % NT, b.mx, c);
        }
        if (lane == 0) {
            const float nan = __int_as_float(0x7FC00000);
            const float excess = b.excess(), logs = log1pf(excess);
            const float lp = bad ? nan : none ? -INFINITY : lp_scaled(xt, b.mx, row.inv_t) - logs;
            const float ent = bad ? nan : none ? 0.f : logs - b.u / (1.f + excess) * 0.6931471805599453f;
            if (p.logprob) p.logprob[r] = lp;
            if (p.entropy) p.entropy[r] = ent;
            if (p.stats) p.stats[r] = make_float2(b.mx, logs * kLog2e);
            if (row.bad_temperature) lp_report(p, RS_ERR_TEMPERATURE);
            if (TOP) {
                if (p.rank) p.rank[r] = bad ? 0 : above + 1;
                sh.r_mx = b.mx;
                sh.r_logs = logs;
            }
        }
    }
    if constexpr (TOP) {
        __syncthreads();
        const int n = p.top_n;
        const float mx = sh.r_mx, logs = sh.r_logs;
        const bool bad = !(mx < INFINITY);
        auto put = [&](unsigned long long e, int at) {      // e = 0: a slot that stays empty
            p.top[r * n + at] = bad ? __int_as_float(0x7FC00000) : e ? lp_scaled(of_key((uint32_t)(e >> 32)), mx, row.inv_t) - logs : -INFINITY;
            p.top_ids[r * n + at] = bad || !e ? -1 : (int)~(uint32_t)e;
        };
        const int all = parts * n;
        if (parts == 1) {
            if (t < n) put(top.list[t], t);          // in order already
        } else if (all <= NT / 2) {
            if (t < all) {
                const unsigned long long e = top.list[t];
                int at = 0;
#pragma unroll 8
                for (int q = 0; q < all; q++) at += top.list[q] > e || (top.list[q] == e && q < t);      // (equal: both empty)
                if (at < n) put(e, at);
            }
        } else {
            // every list's first ceil(n / parts) entries are n in all: what lies below the least of those is not among the n largest
            const int share = (n + parts - 1) >> log_parts;
            unsigned long long* left = reinterpret_cast<unsigned long long*>(top.piece);      // up to parts * top_n; the pieces have served
            unsigned long long least = ~0ull;
            for (int q = 0; q < parts; q++) least = min(least, top.list[q * n + share - 1]);
            if (t == 0) top.ncand = 0;
            __syncthreads();
            for (int i = t; i < all; i += NT)
                if (top.list[i] && top.list[i] >= least) left[atomicAdd(&top.ncand, 1)] = top.list[i];
            __syncthreads();
            const int nc = top.ncand;
            for (int i = t; i < nc; i += NT) {
                const unsigned long long e = left[i];
                int at = 0;
#pragma unroll 8
                for (int q = 0; q < nc; q++) at += left[q] > e;
                if (at < n) put(e, at);
            }
            if (t >= nc && t < n) put(0ull, t);
        }
    }
}

// ---- gradient -------------------------------------------------------------------------------------------------------
// With d = (x - m) c - log2 s, p = 2^d, every element is p (A + D d); the token's own also has g/T, and the two are taken together
// as -expm1(log p) so that a token of probability nearly one keeps its digits.  Logits and gradient pass once: bound by HBM, 4088 rows
// of 151936 bf16 395 us (6.3 TB/s; 415 to 430 under the power cap), f32 half as many 374 (6.6 TB/s).
template <int DT, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) lp_backward_kernel(const __grid_constant__ LpParams p) {
    constexpr int E = Elem<DT>::E;
    using T = typename Elem<DT>::T;
    const uint32_t r32 = blockIdx.x / (unsigned)p.chunks;
    const int part = (int)(blockIdx.x - r32 * (unsigned)p.chunks), t = threadIdx.x;
    const long long r = r32;
    const LpRow row = lp_row(p, r32);
    Span<DT> sp(p, row);
    sp.piece(part, p.piece, p.chunks);
    T* const out = (T*)p.grad + r * p.V;
    const bool together = (((uintptr_t)(out + sp.head)) & 15) == 0;      // logits and gradient: 16-byte boundaries at the same elements
    const float2 st = p.stats[r];
    uint4* const vec = reinterpret_cast<uint4*>(out + sp.head);
    if (row.token < 0 || row.bad_token || st.x == -INFINITY) {
        const T zero = Elem<DT>::to(0.f);
        sp.singles(t, [&](int j, float) { out[j] = zero; });
        if (together) {
            for (int v = sp.v0 + t; v < sp.v1; v += NT) __stcs(vec + v, make_uint4(0u, 0u, 0u, 0u));
        } else {
            for (int j = sp.index(sp.v0) + t, j1 = sp.index(sp.v1); j < j1; j += NT) out[j] = zero;
        }
        return;
    }
    const float g = p.g_logprob ? p.g_logprob[row.b * p.gl_sb + row.t * p.gl_st] : 0.f;
    const float h = p.g_entropy ? p.g_entropy[row.b * p.ge_sb + row.t * p.ge_st] : 0.f;
    const float nan = __int_as_float(0x7FC00000), m = ref_of(st.x), c = row.c, H = p.entropy[r], kLn2 = 0.6931471805599453f;
    const float A = st.x < INFINITY ? -(g + h * H) * row.inv_t : nan, D = -h * row.inv_t * kLn2;
    const int token = (int)row.token;
    auto grad = [&](float x) {
        const float d = fmaxf(fmaf(x - m, c, -st.y), kFloor);
        return ex2(d) * fmaf(D, d, A);
    };
    auto grad_at = [&](float x) {      // the token's own
        const float d = fmaxf(fmaf(x - m, c, -st.y), kFloor);
        const float q = -expm1f(fmaxf((x - m) * row.inv_t - st.y * kLn2, -1e4f));
        const float v = g * row.inv_t * q + ex2(d) * fmaf(D, d, -h * H * row.inv_t);
        return st.x < INFINITY ? v : nan;
    };
    sp.singles(t, [&](int j, float x) { out[j] = Elem<DT>::to(j == token ? grad_at(x) : grad(x)); });
    if (together) {
        const uint64_t mm = f2_pack(-m, -m), cc = f2_pack(c, c), ll = f2_pack(-st.y, -st.y), AA = f2_pack(A, A), DD = f2_pack(D, D);
        auto one = [&](const uint4& from, int at) {
            uint64_t x[E / 2];
            Elem<DT>::pairs(from, x);
#pragma unroll
            for (int k = 0; k < E / 2; k++) {
                float d0, d1;
                f2_unpack(f2_fma(f2_add(x[k], mm), cc, ll), d0, d1);
                d0 = fmaxf(d0, kFloor);
                d1 = fmaxf(d1, kFloor);
                x[k] = f2_mul(f2_pack(ex2(d0), ex2(d1)), f2_fma(DD, f2_pack(d0, d1), AA));
            }
            __stcs(vec + at, Elem<DT>::narrow(x));
        };
        // as in the forward pass: the next step's loads are on their way while one is computed and stored
        constexpr int kStep = kLpAhead * NT;
        uint4 raw[2][kLpAhead];
        auto load = [&](uint4 (&to)[kLpAhead], int v) {
#pragma unroll
            for (int i = 0; i < kLpAhead; i++)
                if (v + i * NT + t < sp.v1) to[i] = ld_stream(sp.vec + v + i * NT + t);
        };
        auto step = [&](const uint4 (&x)[kLpAhead], int v) {
#pragma unroll
            for (int i = 0; i < kLpAhead; i++)
                if (v + i * NT + t < sp.v1) one(x[i], v + i * NT + t);
        };
        int v = sp.v0;
        load(raw[0], v);
        while (v < sp.v1) {
            if (v + kStep < sp.v1) load(raw[1], v + kStep);
            step(raw[0], v);
            v += kStep;
            if (v >= sp.v1) break;
            if (v + kStep < sp.v1) load(raw[0], v + kStep);
            step(raw[1], v);
            v += kStep;
        }
        // the token's own, behind the store of its vector by the same thread
        const int own = token >= sp.head && token < sp.tail() ? (token - sp.head) / E : -1;
        if (own >= sp.v0 && own < sp.v1 && (own - sp.v0) % NT == t) out[token] = Elem<DT>::to(grad_at(Elem<DT>::one(sp.row + token)));
    } else {                           // they start at different places of their 16 bytes: element by element
        for (int j = sp.index(sp.v0) + t, j1 = sp.index(sp.v1); j < j1; j += NT) {
            const float x = Elem<DT>::one(sp.row + j);
            out[j] = Elem<DT>::to(j == token ? grad_at(x) : grad(x));
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
static int lp_params(const rs_logprob_call* k, bool needs_tokens, LpParams* p, HostDevice* dev) {
    if (!k) return RS_ERR_POINTER;
    if (k->dtype != RS_DTYPE_F32 && k->dtype != RS_DTYPE_F16 && k->dtype != RS_DTYPE_BF16) return RS_ERR_DTYPE;
    if (k->V <= 0 || k->V > RS_LOGPROB_MAX_V) return RS_ERR_LIMIT;
    if (k->B <= 0 || k->T <= 0) return RS_ERR_BATCH;
    if (k->T > 0x7fffffff || k->B > 0x7fffffff / k->T) return RS_ERR_LIMIT;
    if (!(k->temperature >= 0.001 && k->temperature <= 1000)) return RS_ERR_TEMPERATURE;
    const uintptr_t size = k->dtype == RS_DTYPE_F32 ? 4 : 2;
    if (!k->logits || ((uintptr_t)k->logits & (size - 1))) return RS_ERR_POINTER;
    if (k->token_bits != 32 && k->token_bits != 64) return RS_ERR_DTYPE;
    if ((needs_tokens && !k->tokens) || ((uintptr_t)k->tokens & (uintptr_t)(k->token_bits / 8 - 1))) return RS_ERR_POINTER;
    if ((uintptr_t)k->row_temperature & 3) return RS_ERR_POINTER;
    memset(p, 0, sizeof *p);
    p->logits = k->logits;
    p->sb = k->stride_b;
    p->st = k->stride_t;
    p->rows = k->B * k->T;
    p->T = (int)k->T;
    p->V = (int)k->V;
    p->tokens = k->tokens;
    p->wide_tokens = k->token_bits == 64;
    p->tok_sb = k->token_stride_b;
    p->tok_st = k->token_stride_t;
    p->temperature = (float)k->temperature;
    p->row_temperature = k->row_temperature;
    p->tmp_sb = k->temperature_stride_b;
    p->tmp_st = k->temperature_stride_t;
    const int rc = host_device(dev);
    if (rc) return rc;
    p->mirror = dev->mirror;
    return RS_OK;
}

template <int DT, bool TOP, int NT, bool SHARED>
static int lp_launch(const LpParams& p, int parts, cudaStream_t stream) {
    auto kern = lp_rows_kernel<DT, TOP, NT, SHARED>;
    if (parts > 8) {
        static std::mutex mu;
        static bool done[64] = {};      // per device
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return host_cuda_fail(e, "cudaGetDevice");
        std::lock_guard<std::mutex> lk(mu);
        if (!done[dev & 63]) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(cluster)");
            done[dev & 63] = true;
        }
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    const int log_parts = 31 - __builtin_clz((unsigned)parts);
    cfg.gridDim = dim3((unsigned)(p.rows * parts));
    cfg.blockDim = dim3(NT);
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;      // a cluster of one too: its shared memory is addressed as the cluster's
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, log_parts);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaLaunchKernelEx(logprobs)");
    host_count_launch();
    return RS_OK;
}

// CTAs per row: enough of them that every multiprocessor has two, as long as each keeps 4096 logits to read; clusters of 16, which
// the device places less freely, only for up to 18 rows.  us for statistics / a list of 20, V = 151936, f32, at 1, 2, 4, 8 CTAs:
// 100 rows 34 / 44, 22 / 31, 16 / 24, 19 / 29; 300 rows 40 / 52, 42 / 57; 32 rows bf16 at 1, 8, 16: 16 / 30, 8 / 15, 11 / 19.
static int lp_parts(long long rows, int V, int sms) {
    const int most = rows * 16 <= 2LL * sms ? 16 : 8;
    int parts = 1;
    while (parts < most && rows * parts < 2LL * sms && V / (2 * parts) >= 4096) parts *= 2;
    return parts;
}
// Threads of a CTA that has a row to itself.  A row's fixed costs, about 3 us, are hidden by the other rows on its
// multiprocessor, and the fewer threads a row has the more of them there are (16 of 64, 8 of 128, 4 of 256); long rows need
// the loads in flight of many threads.  us at 64 / 128 / 256 threads, bf16, statistics and a list of 20:
//   16384 rows of 1024: 35 / 37 / 64 and 113 / 124 / more;  of 4096: 46 / 43 / 74 and 159 / 134 / 217;
//   7629 of 65536: 175 / 153 / 158 and 426 / 283 / 287;  3290 of 151936: 179 / 155 / 155 and 489 / 297 / 249.
static int lp_threads(int V, int size, int top_n) {
    const int bytes = V * size;
    if (bytes <= 4096) return top_n > 40 ? 128 : 64;
    return bytes <= 131072 ? 128 : 256;
}

template <bool TOP, int NT, bool SHARED>
static int lp_typed(const LpParams& p, int dtype, int parts, cudaStream_t stream) {
    switch (dtype) {
        case RS_DTYPE_F32: return lp_launch<RS_DTYPE_F32, TOP, NT, SHARED>(p, parts, stream);
        case RS_DTYPE_F16: return lp_launch<RS_DTYPE_F16, TOP, NT, SHARED>(p, parts, stream);
        default: return lp_launch<RS_DTYPE_BF16, TOP, NT, SHARED>(p, parts, stream);
    }
}
template <bool TOP>
static int lp_dispatch(const LpParams& p, int dtype, int sms, cudaStream_t stream) {
    const int parts = lp_parts(p.rows, p.V, sms);
    if (parts > 1) return lp_typed<TOP, 256, true>(p, dtype, parts, stream);
    const int threads = lp_threads(p.V, dtype == RS_DTYPE_F32 ? 4 : 2, TOP ? p.top_n : 0);
    if (threads == 64) return lp_typed<TOP, 64, false>(p, dtype, 1, stream);
    if (threads == 128) return lp_typed<TOP, 128, false>(p, dtype, 1, stream);
    return lp_typed<TOP, 256, false>(p, dtype, 1, stream);
}
template <int DT>
static void lp_backward(const LpParams& p, int threads, unsigned grid, cudaStream_t st) {
    if (threads == 64) lp_backward_kernel<DT, 64><<<grid, 64, 0, st>>>(p);
    else if (threads == 128) lp_backward_kernel<DT, 128><<<grid, 128, 0, st>>>(p);
    else lp_backward_kernel<DT, 256><<<grid, 256, 0, st>>>(p);
}

int host_status_word(int** out) {
    static std::mutex mu;
    static int* at[64] = {};      // per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaGetDevice");
    std::lock_guard<std::mutex> lk(mu);
    if (!at[dev & 63]) {
        void* a = nullptr;
        e = cudaGetSymbolAddress(&a, g_lp_status);
        if (e != cudaSuccess) return host_cuda_fail(e, "cudaGetSymbolAddress(status)");
        at[dev & 63] = (int*)a;
    }
    *out = at[dev & 63];
    return RS_OK;
}

}  // namespace rs

extern "C" {

int rs_token_logprobs(const rs_logprob_call* call, float* logprob_device, float* entropy_device, float* stats_device) {
    rs::LpParams p;
    rs::HostDevice dev;
    const int rc = rs::lp_params(call, true, &p, &dev);
    if (rc) return rc;
    if (!logprob_device || !entropy_device || ((uintptr_t)logprob_device & 3) || ((uintptr_t)entropy_device & 3) || ((uintptr_t)stats_device & 7))
        return RS_ERR_POINTER;
    p.logprob = logprob_device;
    p.entropy = entropy_device;
    p.stats = (float2*)stats_device;
    return rs::lp_dispatch<false>(p, call->dtype, dev.sms, (cudaStream_t)call->stream);
}

int rs_token_logprobs_backward(const rs_logprob_call* call, const float* entropy_device, const float* stats_device,
                               const float* grad_logprob_device, int64_t gl_stride_b, int64_t gl_stride_t,
                               const float* grad_entropy_device, int64_t ge_stride_b, int64_t ge_stride_t, void* grad_device) {
    rs::LpParams p;
    rs::HostDevice dev;
    const int rc = rs::lp_params(call, true, &p, &dev);
    if (rc) return rc;
    const uintptr_t size = call->dtype == RS_DTYPE_F32 ? 4 : 2;
    if (!entropy_device || !stats_device || !grad_device || ((uintptr_t)entropy_device & 3) || ((uintptr_t)stats_device & 7) ||
        ((uintptr_t)grad_device & (size - 1)) || ((uintptr_t)grad_logprob_device & 3) || ((uintptr_t)grad_entropy_device & 3))
        return RS_ERR_POINTER;
    p.entropy = const_cast<float*>(entropy_device);
    p.stats = (float2*)const_cast<float*>(stats_device);
    p.g_logprob = grad_logprob_device;
    p.gl_sb = gl_stride_b;
    p.gl_st = gl_stride_t;
    p.g_entropy = grad_entropy_device;
    p.ge_sb = ge_stride_b;
    p.ge_st = ge_stride_t;
    p.grad = grad_device;
    // 64 KB of logits a CTA, so that its row's few numbers cost little; down to 8 KB where that leaves multiprocessors idle
    const long long vectors = p.V * (long long)size / 16 + 1;
    long long piece = 4096;
    while (piece > 512 && p.rows * ((vectors + piece - 1) / piece) < 4LL * dev.sms) piece /= 2;
    while (p.rows * ((vectors + piece - 1) / piece) > 0x7fffffffLL) piece *= 2;
    const long long chunks = (vectors + piece - 1) / piece;
    p.piece = (int)piece;
    p.chunks = (int)chunks;
    const int threads = rs::lp_threads((int)call->V, (int)size, 0);
    const unsigned grid = (unsigned)(p.rows * chunks);
    cudaStream_t st = (cudaStream_t)call->stream;
    switch (call->dtype) {
        case RS_DTYPE_F32: rs::lp_backward<RS_DTYPE_F32>(p, threads, grid, st); break;
        case RS_DTYPE_F16: rs::lp_backward<RS_DTYPE_F16>(p, threads, grid, st); break;
        default: rs::lp_backward<RS_DTYPE_BF16>(p, threads, grid, st);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return rs::host_cuda_fail(e, "launch(logprobs backward)");
    rs::host_count_launch();
    return RS_OK;
}

int rs_top_logprobs(const rs_logprob_call* call, int32_t top_n, float* logprob_device, int32_t* rank_device, float* entropy_device,
                    float* top_device, int32_t* top_ids_device) {
    rs::LpParams p;
    rs::HostDevice dev;
    const int rc = rs::lp_params(call, false, &p, &dev);
    if (rc) return rc;
    if (top_n < 1 || top_n > RS_LOGPROB_MAX_TOP) return RS_ERR_LIMIT;
    if (!entropy_device || !top_device || !top_ids_device || ((uintptr_t)logprob_device & 3) || ((uintptr_t)rank_device & 3) ||
        ((uintptr_t)entropy_device & 3) || ((uintptr_t)top_device & 3) || ((uintptr_t)top_ids_device & 3))
        return RS_ERR_POINTER;
    if (!call->tokens && (logprob_device || rank_device)) return RS_ERR_POINTER;
    p.logprob = logprob_device;
    p.rank = rank_device;
    p.entropy = entropy_device;
    p.top = top_device;
    p.top_ids = top_ids_device;
    p.top_n = top_n;
    return rs::lp_dispatch<true>(p, call->dtype, dev.sms, (cudaStream_t)call->stream);
}

int rs_logprobs_status(void* stream) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&v, rs::g_lp_status, sizeof v, 0, cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e == cudaSuccess && v) {
        const int zero = 0;
        e = cudaMemcpyToSymbolAsync(rs::g_lp_status, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, (cudaStream_t)stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    }
    if (e != cudaSuccess) return rs::host_cuda_fail(e, "status read");
    return v;
}

}  // extern "C"

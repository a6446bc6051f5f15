// RMS norm of every query and key head with the position rotation, one pass over the heads:
//   x' = x / sqrt(mean x^2 + eps) * w over the D elements of a head, then for the pairs (a, b) of
//   its first R elements, i = 0 .. R/2 - 1, with the angle t = pos freq_i:
//   (a, b) <- (a cos t - b sin t, b cos t + a sin t)      (Su et al. 2021, equation 15)
// Pairs are (i, i + R/2), or (2 i, 2 i + 1) where interleaved. Norm and rotation are in fp32, the
// result is rounded once.
//
// The angle is formed in double in units of whole turns, reduced to half a turn there, and only
// then rounded: a position of 10^6 would lose 0.06 rad in fp32.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr double kTurn = 0.15915494309189535;   // 1 / (2 pi)
constexpr int kMaxD = 512;

struct HeadArgs {
    const void* q; long ldq;
    const void* k; long ldk;
    const float* wq; const float* wk;
    const int* pos;
    const double* freq;
    void* qo; long ldqo;
    void* ko; long ldko;
    int T, H, G, D, R, tokens;   // tokens of a workgroup
    float eps;
};

__device__ __forceinline__ float2 turn(int pos, double freq) {
    const double t = (double)pos * (freq * kTurn);
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    return make_float2(c, s);
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load4(const __bf16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return make_float4(__builtin_bit_cast(float, u.x << 16), __builtin_bit_cast(float, u.x & 0xffff0000u),
                       __builtin_bit_cast(float, u.y << 16), __builtin_bit_cast(float, u.y & 0xffff0000u));
}

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__bf16* p, float4 v) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<bf16x4*>(p) = bf16x4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
}

// Memory bound: 36 heads of 128 bf16 of 16384 tokens (302 MB) take 64 us, 4.7 TB/s, where a copy of 1 GiB
// reaches 5.1. A lane holds eight elements of a head as two 4-element pieces, both of every pair (PAIR 0: 4 p ..
// + 3 and R/2 on; 1: 8 p .. + 7), LPR lanes a head (D <= 8 LPR). The workgroup forms the cosines
// and sines of its tokens once, in LDS, for all their heads; its heads' loads are issued U at a
// time.
template <typename T, int LPR, bool BESIDE>
__global__ __launch_bounds__(256) void head_kernel(HeadArgs a) {
    constexpr int RPB = 256 / LPR, U = 4;
    extern __shared__ float2 cs[];   // [token][R / 2]
    const int tid = threadIdx.x;
    const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.T - t0);
    const int half = a.R / 2, HG = a.H + a.G, rows = nt * HG;
    const int p = tid % LPR, rb = tid / LPR;
    const bool live = 8 * p < a.D, rot = 8 * p < a.R;
    const int e0 = BESIDE ? 8 * p : (rot ? 4 * p : a.R + 8 * (p - a.R / 8));
    const int e1 = BESIDE || !rot ? e0 + 4 : e0 + half;

    float4 x0[U], x1[U];
    auto src = [&](int r, bool out) -> T* {
        const int tok = r / HG, hd = r - tok * HG;
        const long t = t0 + tok;
        if (hd < a.H)
            return out ? static_cast<T*>(a.qo) + t * a.ldqo + (long)hd * a.D
                       : const_cast<T*>(static_cast<const T*>(a.q)) + t * a.ldq + (long)hd * a.D;
        return out ? static_cast<T*>(a.ko) + t * a.ldko + (long)(hd - a.H) * a.D
                   : const_cast<T*>(static_cast<const T*>(a.k)) + t * a.ldk + (long)(hd - a.H) * a.D;
    };
    auto fetch = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * RPB;
            x0[u] = x1[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (live && r < rows) {
                const T* s = src(r, false);
                x0[u] = load4(s + e0);
                x1[u] = load4(s + e1);
            }
        }
    };
    fetch(rb);
    for (int i = tid; i < nt * half; i += 256) {
        const int tok = i / half;
        cs[i] = turn(a.pos[t0 + tok], a.freq[i - tok * half]);
    }
    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
    const float4 q0 = a.wq && live ? load4(a.wq + e0) : one, q1 = a.wq && live ? load4(a.wq + e1) : one;
    const float4 k0 = a.wk && live ? load4(a.wk + e0) : one, k1 = a.wk && live ? load4(a.wk + e1) : one;
    __syncthreads();
    const float inv = 1.f / (float)a.D;
    for (int r0 = rb; r0 < rows; r0 += U * RPB) {
        if (r0 != rb) fetch(r0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * RPB;
            const float4 s0 = x0[u], s1 = x1[u];
            float ss = s0.x * s0.x + s0.y * s0.y + s0.z * s0.z + s0.w * s0.w;
            ss += s1.x * s1.x + s1.y * s1.y + s1.z * s1.z + s1.w * s1.w;
#pragma unroll
            for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, LPR);
            if (!live || r >= rows) continue;
            const float n = rsqrtf(fmaf(ss, inv, a.eps));
            const int tok = r / HG, hd = r - tok * HG;
            const float4 w0 = hd < a.H ? q0 : k0, w1 = hd < a.H ? q1 : k1;
            float4 a0 = make_float4(s0.x * n * w0.x, s0.y * n * w0.y, s0.z * n * w0.z, s0.w * n * w0.w);
            float4 a1 = make_float4(s1.x * n * w1.x, s1.y * n * w1.y, s1.z * n * w1.z, s1.w * n * w1.w);
            if (rot) {
                const float2* c = cs + tok * half + 4 * p;
                auto spin = [](float& x, float& y, float2 c) {
                    const float u = x * c.x - y * c.y;
                    y = y * c.x + x * c.y;
                    x = u;
                };
                if constexpr (BESIDE) {
                    spin(a0.x, a0.y, c[0]);
                    spin(a0.z, a0.w, c[1]);
                    spin(a1.x, a1.y, c[2]);
                    spin(a1.z, a1.w, c[3]);
                } else {
                    spin(a0.x, a1.x, c[0]);
                    spin(a0.y, a1.y, c[1]);
                    spin(a0.z, a1.z, c[2]);
                    spin(a0.w, a1.w, c[3]);
                }
            }
            T* d = src(r, true);
            store4(d + e0, a0);
            store4(d + e1, a1);
        }
    }
}

// Any D up to 512 and any alignment: a wave a head, one element at a time. Every element and its
// partner are loaded before anything is stored (in and out may be the same).
template <typename T, bool BESIDE>
__global__ __launch_bounds__(256) void head_any_kernel(HeadArgs a) {
    constexpr int U = kMaxD / 64;
    const int lane = threadIdx.x & 63;
    const int HG = a.H + a.G;
    const long r = ((long)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (r >= (long)a.T * HG) return;
    const long t = r / HG;
    const int hd = (int)(r - t * HG);
    const bool isq = hd < a.H;
    const T* s = isq ? static_cast<const T*>(a.q) + t * a.ldq + (long)hd * a.D
                     : static_cast<const T*>(a.k) + t * a.ldk + (long)(hd - a.H) * a.D;
    T* d = isq ? static_cast<T*>(a.qo) + t * a.ldqo + (long)hd * a.D
               : static_cast<T*>(a.ko) + t * a.ldko + (long)(hd - a.H) * a.D;
    const float* w = isq ? a.wq : a.wk;
    const int half = a.R / 2;
    float x[U], y[U];
    float ss = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = lane + 64 * u;
        x[u] = y[u] = 0.f;
        if (e < a.D) {
            x[u] = (float)s[e];
            ss = fmaf(x[u], x[u], ss);
            if (e < a.R) {
                const int o = BESIDE ? e ^ 1 : (e < half ? e + half : e - half);
                y[u] = (float)s[o] * (w ? w[o] : 1.f);
            }
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off);
    const float n = rsqrtf(fmaf(ss, 1.f / (float)a.D, a.eps));
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = lane + 64 * u;
        if (e >= a.D) continue;
        float o = x[u] * n * (w ? w[e] : 1.f);
        if (e < a.R) {
            const bool second = BESIDE ? e & 1 : e >= half;
            const float2 c = turn(a.pos[t], a.freq[BESIDE ? e >> 1 : (second ? e - half : e)]);
            o = o * c.x + (second ? y[u] * n : -(y[u] * n)) * c.y;
        }
        d[e] = (T)o;
    }
}

template <typename T, int LPR>
void launch_heads(const HeadArgs& a, bool beside, unsigned n, size_t lds, hipStream_t st) {
    if (beside) head_kernel<T, LPR, true><<<n, 256, lds, st>>>(a);
    else head_kernel<T, LPR, false><<<n, 256, lds, st>>>(a);
}

template <typename T>
ssm_status run_heads(HeadArgs a, bool beside, bool vec, hipStream_t st) {
    if (!vec) {
        const long wgs = ssm::cdiv((long)a.T * (a.H + a.G), 4);
        const dim3 n((unsigned)std::min(wgs, 1L << 20), (unsigned)ssm::cdiv(wgs, 1L << 20));
        if (beside) head_any_kernel<T, true><<<n, 256, 0, st>>>(a);
        else head_any_kernel<T, false><<<n, 256, 0, st>>>(a);
        return ssm::check_launch("ssm_qk_norm_rope");
    }
    // four tokens a workgroup where that leaves four workgroups a CU: their angles' cost is one sine and
    // cosine a thread (36 heads of 128, bf16: 16384 tokens 62 us, 76 with one token, 69 with eight; 64
    // tokens 4.6 us with one, 9.2 with four)
    a.tokens = a.T >= 4096 ? 4 : 1;
    const unsigned n = (unsigned)ssm::cdiv(a.T, a.tokens);
    const size_t lds = sizeof(float2) * (size_t)a.tokens * (a.R / 2);
    if (a.D <= 64) launch_heads<T, 8>(a, beside, n, lds, st);
    else if (a.D <= 128) launch_heads<T, 16>(a, beside, n, lds, st);
    else if (a.D <= 256) launch_heads<T, 32>(a, beside, n, lds, st);
    else launch_heads<T, 64>(a, beside, n, lds, st);
    return ssm::check_launch("ssm_qk_norm_rope");
}

}  // namespace

extern "C" ssm_status ssm_qk_norm_rope(int dtype, const void* q, long ldq, const void* k, long ldk,
                                       const float* wq, const float* wk, const int* pos,
                                       const double* freq, int interleaved, float eps, void* qo,
                                       long ldqo, void* ko, long ldko, int T, int H, int G, int D,
                                       int R, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_qk_norm_rope: bad dtype");
    SSM_REQUIRE(T >= 0 && H >= 0 && G >= 0 && D > 0, "ssm_qk_norm_rope: bad shape");
    SSM_REQUIRE(R >= 0 && R <= D && R % 2 == 0,
                "ssm_qk_norm_rope: %d rotated elements of %d (an even number up to all)", R, D);
    if (D > kMaxD)
        return ssm::fail(SSM_ERR_UNSUPPORTED, "ssm_qk_norm_rope: head dim %d above %d", D, kMaxD);
    if (T == 0 || (H == 0 && G == 0)) return SSM_OK;
    SSM_REQUIRE((H == 0 || (q && qo)) && (G == 0 || (k && ko)) && (R == 0 || (pos && freq)),
                "ssm_qk_norm_rope: null input");
    const long wide_q = (long)H * D, wide_k = (long)G * D;
    SSM_REQUIRE(T == 1 || (ldq >= wide_q && ldqo >= wide_q && ldk >= wide_k && ldko >= wide_k),
                "ssm_qk_norm_rope: row stride below row width");
    const long heads = (long)H + G;
    SSM_REQUIRE(heads <= ssm::kMaxSteps && T * heads < (1L << 32), "ssm_qk_norm_rope: too many heads");
    const long es = dtype == SSM_F32 ? 4 : 2;
    auto rows = [&](const void* x, long ld, long wide) { return ssm::Rows{x, ld * es, wide * es, T}; };
    const ssm::Rows rq = rows(q, ldq, wide_q), rk = rows(k, ldk, wide_k), rqo = rows(qo, ldqo, wide_q),
                    rko = rows(ko, ldko, wide_k);
    SSM_REQUIRE(((q == qo && (ldq == ldqo || T == 1)) || !ssm::meet(rq, rqo)) &&
                    ((k == ko && (ldk == ldko || T == 1)) || !ssm::meet(rk, rko)) &&
                    !ssm::meet(rq, rko) && !ssm::meet(rk, rqo) && !ssm::meet(rqo, rko),
                "ssm_qk_norm_rope: an output overlaps an input that it is not, or the other output");
    const ssm::Rows gq = ssm::block(wq, 4L * D), gk = ssm::block(wk, 4L * D),
                    at = ssm::block(R ? pos : nullptr, 4L * T), turns = ssm::block(R ? freq : nullptr, 4L * R);
    SSM_REQUIRE(!ssm::meets(rqo, gq, gk, at, turns) && !ssm::meets(rko, gq, gk, at, turns),
                "ssm_qk_norm_rope: an output overlaps the weights, positions or frequencies");
    HeadArgs a{q, ldq, k, ldk, wq, wk, pos, freq, qo, ldqo, ko, ldko, T, H, G, D, R, 1, eps};
    // pieces of four elements: 16 bytes in fp32 (and of the weights), 8 in bf16
    const uintptr_t piece = dtype == SSM_F32 ? 15 : 7;
    const bool vec = D % 8 == 0 && R % 8 == 0 && T <= ssm::kMaxGroups && (ldq | ldk | ldqo | ldko) % 4 == 0 &&
                     (((uintptr_t)q | (uintptr_t)k | (uintptr_t)qo | (uintptr_t)ko) & piece) == 0 &&
                     (((uintptr_t)wq | (uintptr_t)wk) & 15) == 0;
    return dtype == SSM_F32 ? run_heads<float>(a, interleaved != 0, vec, (hipStream_t)stream)
                            : run_heads<__bf16>(a, interleaved != 0, vec, (hipStream_t)stream);
}

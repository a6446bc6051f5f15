// Products of 8-bit integers with a scale for each row of x (token) and of W (output channel):
//   quantised rows    s_m = max_k |x_mk| / 127 (fp32),  q_mk = x_mk / s_m to the nearest integer,
//                     ties to even (from the exact quotient), held to -127 .. 127
//   y_mn = beta y_mn + s_m s_n sum_k q_mk w_nk (+ bias_n)
// The sums are exact 32-bit integers (|q|, |w| <= 128: K up to 131071).
//
// Three kernels share the work by rows:
//   - up to 64 rows (one per decoded sequence): the weights' bytes bound it. i8_rows_kernel reads
//     every weight row once, straight into registers, the k of a row shared by its waves
//     (v_mfma_i32_16x16x64_i8).
//   - more rows: the matrix cores bound it. i8_gemm_kernel and, where every CU has a tile of 256 x 256,
//     i8_gemm_big_kernel are tiled products out of LDS (v_mfma_i32_32x32x32_i8).
// Rows that these cannot read in place (not 16-byte aligned, x's of few rows in the operands' order) are laid
// out in the workspace first, in every call (lay_rows_kernel): weights kept at a stride of 16 bytes save that.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr unsigned kOut = 0x80000000u;   // a buffer offset past any descriptor
constexpr int kMaxK = 131071;
constexpr int kPad = 256;          // rows of the workspace are whole blocks of 256 bytes, zeros past K
constexpr int kCUs = 256;          // workgroups of the large tiles' kernel: one a CU
constexpr int kRowsMax = 64;       // rows of the few-row kernel (64 x 2048 x 2048: 9.3 us, 11.9 in tiles)
inline long up(long n, long to) { return (n + to - 1) / to * to; }

// ---------------------------------------------------------------- rows to integers
// x / s to the nearest integer. t = x inv is within 127 * 2^-23 of the quotient, so its nearest integer
// is the quotient's unless t is that near to a half; then the exact remainder decides (x - q s has 24
// bits). Adding 1.5 * 2^23 leaves the integer in the sum's low bits, two's complement.
struct Quant {
    float f, s, inv;   // x f / (s f), s f in the normal range
    static constexpr float kMagic = 12582912.f, kSure = 0.4999f;
    __device__ __forceinline__ explicit Quant(float scale) {
        f = scale < 0x1p-100f ? 0x1p120f : 1.f;
        s = scale * f;
        inv = 1.f / s;
    }
    __device__ __forceinline__ unsigned exact(float x) const {
        x *= f;
        float q = rintf(x * inv);
        const float r = fmaf(-q, s, x), d = 2.f * fabsf(r);
        if (d > s || (d == s && ((int)q & 1))) q += copysignf(1.f, r);
        return (unsigned)(int)fminf(fmaxf(q, -127.f), 127.f);
    }
    __device__ __forceinline__ unsigned near(float x, float& off) const {
        const float u = fmaf(x, inv, kMagic);
        off = fmaxf(off, fabsf(fmaf(x, inv, kMagic - u)));
        return __builtin_bit_cast(unsigned, u);
    }
    static __device__ __forceinline__ unsigned bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
        // (v_perm_b32: the low bytes of two words side by side)
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u),
                                     __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
    }
    __device__ __forceinline__ unsigned pack(float4 v) const {
        float off = 0.f;
        const unsigned b = bytes(near(v.x, off), near(v.y, off), near(v.z, off), near(v.w, off));
        if (off <= kSure && f == 1.f) return b;
        return bytes(exact(v.x), exact(v.y), exact(v.z), exact(v.w));
    }
};

// A value that the compiler forms again here: registers for it are not held over a loop.
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

// The largest magnitude's scale: 0 where all are zero, inf or NaN where one is (such rows hold
// zeros, so that their products are NaN).
__device__ __forceinline__ float scale_of(unsigned most) {
    return __fdiv_rn(__builtin_bit_cast(float, most), 127.f);
}

__device__ __forceinline__ bool usable(float scale) { return scale > 0.f && scale < INFINITY; }

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

struct Eight { float4 a, b; };
__device__ __forceinline__ Eight load8(const float* p) { return Eight{load4(p), load4(p + 4)}; }
__device__ __forceinline__ Eight load8(const __bf16* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    auto two = [](unsigned x, unsigned y) {
        return make_float4(__builtin_bit_cast(float, x << 16), __builtin_bit_cast(float, x & 0xffff0000u),
                           __builtin_bit_cast(float, y << 16), __builtin_bit_cast(float, y & 0xffff0000u));
    };
    return Eight{two(u.x, u.y), two(u.z, u.w)};
}

// Four consecutive elements from k on, zeros past K.
template <typename T, bool VEC>
__device__ __forceinline__ float4 some4(const T* row, int k, int K) {
    if constexpr (VEC) {
        return k < K ? load4(row + k) : make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
        return make_float4(k < K ? (float)row[k] : 0.f, k + 1 < K ? (float)row[k + 1] : 0.f,
                           k + 2 < K ? (float)row[k + 2] : 0.f, k + 3 < K ? (float)row[k + 3] : 0.f);
    }
}

__device__ __forceinline__ unsigned max4(unsigned m, float4 v) {
    return max(max(m, max(abs_bits(v.x), abs_bits(v.y))), max(abs_bits(v.z), abs_bits(v.w)));
}

// The largest of a wave's values, in every lane: four steps inside each 16 lanes (quad_perm, half_mirror,
// mirror), then the four rows.
__device__ __forceinline__ unsigned wave_max(unsigned v) {
    auto step = [&](auto ctrl) {
        v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true));
    };
    step(std::integral_constant<int, 0xb1>{});
    step(std::integral_constant<int, 0x4e>{});
    step(std::integral_constant<int, 0x141>{});
    step(std::integral_constant<int, 0x140>{});
    auto row = [&](int l) { return (unsigned)__builtin_amdgcn_readlane((int)v, l); };
    return max(max(row(0), row(16)), max(row(32), row(48)));
}

struct QuantArgs {
    const void* x; long ldx;
    signed char* q; long ldq;
    float* scale;
    int M, K, Kq;   // Kq: bytes written per row (zeros past K)
    int frag;       // in the order of the few-row kernel's operand
};

// Byte k of row m in the order of the few-row kernel's operand: the 16-row block m / 16 and the block
// of 256 k hold four operands of 1 KB, of which lane (g, i) has 16 bytes, row i's from 64 g + 16 u on.
// (k's 16-byte pieces stay whole.)
__device__ __forceinline__ long frag_at(long m, int k, int Kp) {
    return ((m >> 4) * (Kp >> 8) + (k >> 8)) * 4096L + (k >> 4 & 3) * 1024 + (k >> 6 & 3) * 256 +
           (m & 15) * 16 + (k & 15);
}

// TPR threads a row, 256 / TPR rows a workgroup: U pieces of eight elements a thread are held between
// the two passes (further ones are read again). VEC: elements of an aligned load, 8 (K a multiple of it
// too), 4 or 1. Memory bound; at 8192 x 2048 bf16 (50 MB) 13.5 us, 3.7 TB/s.
template <typename T, int TPR, int VEC>
__global__ __launch_bounds__(256) void quant_kernel(QuantArgs a) {
    constexpr int U = 4, RPB = 256 / TPR, NW = TPR / 64;
    __shared__ unsigned red[4];
    const int tid = threadIdx.x % TPR, rw = threadIdx.x / TPR;
    const long m = (long)blockIdx.x * RPB + rw;
    const bool live = m < a.M;
    const T* row = static_cast<const T*>(a.x) + (live ? m : 0) * a.ldx;
    auto get = [&](int k) {
        if constexpr (VEC == 8) {
            const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            return k < a.K ? load8(row + k) : Eight{z, z};
        } else {
            return Eight{some4<T, VEC == 4>(row, k, a.K), some4<T, VEC == 4>(row, k + 4, a.K)};
        }
    };
    Eight v[U];
    unsigned most = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = get(8 * (tid + TPR * u));
#pragma unroll
    for (int u = 0; u < U; ++u) most = max4(max4(most, v[u].a), v[u].b);
    for (int k = 8 * (tid + TPR * U); k < a.K; k += 8 * TPR) {
        const Eight e = get(k);
        most = max4(max4(most, e.a), e.b);
    }
    most = wave_max(most);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
        __syncthreads();
        most = red[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) most = max(most, red[i]);
    }
    if (!live) return;
    const float s = scale_of(most);
    if (tid == 0) a.scale[m] = s;
    const bool ok = usable(s);
    const Quant z(ok ? s : 1.f);
    signed char* out = a.q + (a.frag ? 0 : m * a.ldq);
    auto put = [&](int k, const Eight& e) {
        if (k >= a.Kq) return;
        const uint2 b = ok ? make_uint2(z.pack(e.a), z.pack(e.b)) : make_uint2(0u, 0u);
        if (a.frag) {   // (Kq is a whole number of pieces)
            *reinterpret_cast<uint2*>(out + frag_at(m, k, (int)a.ldq)) = b;
        } else if constexpr (VEC > 1) {
            *reinterpret_cast<uint2*>(out + k) = b;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < a.Kq) out[k + e] = (signed char)((e < 4 ? b.x : b.y) >> 8 * (e & 3));
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) put(8 * (tid + TPR * u), v[u]);
    for (int k = 8 * (tid + TPR * U); k < a.Kq; k += 8 * TPR) put(k, get(k));
}

template <typename T, int VEC>
void quant_launch(const QuantArgs& a, hipStream_t st) {
    // a wave a row up to 2048 elements (its four pieces a lane) where there are more rows than
    // elements (bf16, 8192 x 2048: 13.5 us, 15.0 with a workgroup a row; 8192 x 768: 7.1, 12.0), a
    // workgroup a row else (1000 x 2048: 4.4 us, 6.0 with waves)
    if (a.K <= 2048 && a.M >= std::max(a.K, 1000)) quant_kernel<T, 64, VEC><<<(unsigned)ssm::cdiv(a.M, 4), 256, 0, st>>>(a);
    else quant_kernel<T, 256, VEC><<<a.M, 256, 0, st>>>(a);
}

ssm_status quantize(int dtype, const void* x, long ldx, signed char* q, long ldq, float* scale,
                    int M, int K, int Kq, bool frag, hipStream_t st) {
    const QuantArgs a{x, ldx, q, ldq, scale, M, K, Kq, frag};
    const bool out8 = Kq % 8 == 0 && ldq % 8 == 0 && ((uintptr_t)q & 7) == 0;
    auto aligned = [&](int n) {   // n elements, 16 bytes at most
        const uintptr_t b = std::min(16, n * (dtype == SSM_F32 ? 4 : 2));
        return out8 && K % n == 0 && ldx % n == 0 && ((uintptr_t)x & (b - 1)) == 0;
    };
    const int vec = aligned(8) ? 8 : aligned(4) ? 4 : 1;
    if (dtype == SSM_F32) {
        if (vec == 8) quant_launch<float, 8>(a, st);
        else if (vec == 4) quant_launch<float, 4>(a, st);
        else quant_launch<float, 1>(a, st);
    } else {
        if (vec == 8) quant_launch<__bf16, 8>(a, st);
        else if (vec == 4) quant_launch<__bf16, 4>(a, st);
        else quant_launch<__bf16, 1>(a, st);
    }
    return ssm::check_launch("ssm_quantize_rows");
}

// Rows of K bytes at any alignment -> rows of Kp bytes, zeros past K (or the few-row operand's order).
template <bool FRAG>
__global__ __launch_bounds__(256) void lay_rows_kernel(const signed char* __restrict__ x, long ldx,
                                                       int K, signed char* __restrict__ o, int Kp) {
    const signed char* row = x + (long)blockIdx.x * ldx;
    for (int k = 4 * threadIdx.x; k < Kp; k += 1024) {
        unsigned b = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < K) b |= (unsigned)(unsigned char)row[k + e] << 8 * e;
        *reinterpret_cast<unsigned*>(o + (FRAG ? frag_at(blockIdx.x, k, Kp) : (long)blockIdx.x * Kp + k)) = b;
    }
}

// ---------------------------------------------------------------- epilogue
struct I8Args {
    const signed char* X; long ldx; const float* sx;   // x as integers (null: from Xf)
    const void* Xf; long ldxf; int x_dtype;            // x to be rounded in the kernel
    const signed char* W; long ldw; const float* sw;
    const float* bias;
    void* y; long ldy;
    int M, N, K;
    float beta;
    int vec;      // outputs in aligned pieces of 16 bytes
    int mt, nt, gn;
};

// The outputs of a tile, rows m0 .. and columns n0 ..: a descriptor that ends with the last of them.
template <typename TO>
struct Out {
    __amdgpu_buffer_rsrc_t d;
    unsigned ld;
    int cols;
    __device__ __forceinline__ Out(const I8Args& a, int m0, int rows, int n0, int cols_)
        : d(ssm::rsrc(static_cast<TO*>(a.y) + (long)m0 * a.ldy + n0,
                      (unsigned)(((long)(rows - 1) * a.ldy + cols_) * (long)sizeof(TO)))),
          ld((unsigned)a.ldy), cols(cols_) {}
};

// A scale of which a product with another one could leave the normal numbers.
__device__ __forceinline__ bool far(float scale) {
    const float m = fabsf(scale);
    return m != 0.f && !(m >= 0x1p-60f && m <= 0x1p60f);
}

// The sum times both scales. FAR: where one is far, times the smaller one first: what that leaves is as large
// as an integer or has all its digits, so the second product is out of range only where the result is.
template <bool FAR>
__device__ __forceinline__ float scaled(int sum, float row, float channel) {
    const float c = (float)sum;
    if constexpr (FAR)
        if (far(row) || far(channel))
            return fabsf(row) < fabsf(channel) ? c * row * channel : c * channel * row;
    return c * (row * channel);
}

// One output, n of row m of the tile.
template <typename TO, bool BETA>
__device__ __forceinline__ void put1(const Out<TO>& o, float beta, int m, int n, float x) {
    const unsigned off = n < o.cols ? ((unsigned)m * o.ld + (unsigned)n) * (unsigned)sizeof(TO) : kOut;
    if constexpr (sizeof(TO) == 4) {
        if constexpr (BETA) x += beta * ssm::bload4(o.d, off);
        ssm::bstore4(x, o.d, off);
    } else {
        if constexpr (BETA) {
            const unsigned p = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(o.d, off, 0, 0);
            x += beta * __builtin_bit_cast(float, p << 16);
        }
        const __bf16 y = (__bf16)x;
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, y), o.d, off, 0, 0);
    }
}

// 16 bytes of outputs, n .. of row m, aligned to their size.
template <typename TO, bool BETA>
__device__ __forceinline__ void put(const Out<TO>& o, float beta, int m, int n, float* v) {
    constexpr int E = 16 / sizeof(TO);
    const unsigned off = n < o.cols ? ((unsigned)m * o.ld + (unsigned)n) * (unsigned)sizeof(TO) : kOut;
    if constexpr (sizeof(TO) == 4) {
        if constexpr (BETA) {
            const floatx4 y = ssm::bload16<floatx4>(o.d, off);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += beta * y[e];
        }
        ssm::bstore16(make_float4(v[0], v[1], v[2], v[3]), o.d, off);
    } else {
        bf16x8 y;
        if constexpr (BETA) {
            y = ssm::bload16<bf16x8>(o.d, off);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += beta * (float)y[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = (__bf16)v[e];
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(ssm::u32x4, y), o.d, off, 0, 0);
    }
}

// Four outputs, n .. of row m, aligned to their size.
template <typename TO, bool BETA>
__device__ __forceinline__ void put4(const Out<TO>& o, float beta, int m, int n, float* v) {
    if constexpr (sizeof(TO) == 4) {
        put<TO, BETA>(o, beta, m, n, v);
    } else {
        const unsigned off = n < o.cols ? ((unsigned)m * o.ld + (unsigned)n) * 2u : kOut;
        bf16x4 y;
        if constexpr (BETA) {
            y = __builtin_bit_cast(bf16x4, __builtin_amdgcn_raw_buffer_load_b64(o.d, off, 0, 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += beta * (float)y[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (__bf16)v[e];
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, y), o.d, off, 0, 0);
    }
}

// A row's bytes in whole dwords: one that a descriptor ends inside reads as zeros. (Rows that are
// read in place have a multiple of four, the workspace's are longer.)
__device__ __forceinline__ int whole(int K) { return (K + 3) & ~3; }

__device__ __forceinline__ intx4 mfma8(intx4 w, intx4 x, intx4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
}

// ---------------------------------------------------------------- up to 64 rows
// A workgroup owns 16 output channels; its NW waves take the blocks of 256 k in turn, two blocks' weights in
// flight a wave. Lane (g, i) = (lane / 16, lane % 16) reads W row i's bytes 64 g + 16 u .. of the block for
// u = 0 .. 3, which is the operand of MFMA u with the block's k in another order, the same for x. So a
// lane reads 64 consecutive bytes of its row, and x lies in the workspace in the operands' own order (a
// row-major x took 3 times as long at 64 rows: 16 lines an instruction). The waves' sums meet in
// LDS (integers: their order changes nothing).
//
// FUSED: up to four rows of x of at most kFusedX elements in all are rounded by every workgroup for
// itself, into LDS, while its weights are on their way: one launch instead of two (N 8512, K 2048, bf16:
// one row 6.0 us, 8.5 in two launches; two rows 7.3, 8.3; four rows, past kFusedX, would take 10.4).
constexpr int kFusedX = 4096, kFusedRows = 4;

template <int MB, typename TX, typename TO, bool BETA, int NW>
__global__ __launch_bounds__(64 * NW) void i8_rows_kernel(I8Args a) {
    constexpr bool FUSED = !std::is_void<TX>::value;
    static_assert(!FUSED || NW == 4, "256 threads round x");
    constexpr int kPieces = kFusedX / 1024;
    __shared__ intx4 red[NW][MB][64];
    __shared__ __attribute__((aligned(16))) signed char xs[FUSED ? kFusedX + kFusedRows * kPad : 16];
    __shared__ unsigned most[FUSED ? 4 : 1][kPieces];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int n0 = blockIdx.x * 16;
    const int rows = min(16, a.N - n0);
    const auto rw = ssm::rsrc(a.W + (long)n0 * a.ldw, (unsigned)((long)(rows - 1) * a.ldw + whole(a.K)));
    const unsigned wo = (unsigned)(i * a.ldw) + 64u * g;
    const int steps = (a.K + 255) / 256, Kp = steps * 256;
    intx4 wv[2][4];
    auto fetch = [&](intx4 (&v)[4], int s) {
        if (s >= steps) return;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            v[u] = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(rw, wo + 16u * u + 256u * s, 0, 0));
    };
    intx4 acc[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[m] = intx4{0, 0, 0, 0};
    float sm[MB];
    if constexpr (FUSED) {
        // piece p: 1024 elements of row p >> sh, from 1024 (p & (per - 1)) on
        const int sh = a.K > 2048 ? 2 : a.K > 1024 ? 1 : 0, pieces = a.M << sh;
        float4 v[kPieces];
        auto row = [&](int p) { return p >> sh; };
        auto col = [&](int p) { return 4 * ((int)threadIdx.x + 256 * (p & ((1 << sh) - 1))); };
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
            if (p < pieces) v[p] = some4<TX, true>(static_cast<const TX*>(a.Xf) + (long)row(p) * a.ldxf, col(p), a.K);
        fetch(wv[0], w);   // (behind x: loads come back in order)
        fetch(wv[1], w + NW);
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
            if (p < pieces) {
                const unsigned t = wave_max(max4(0, v[p]));
                if (lane == 0) most[w][p] = t;
            }
        __syncthreads();
        auto scale = [&](int m) {
            unsigned t = 0;
            for (int p = m << sh; p < (m + 1) << sh; ++p)
                t = max(max(t, max(most[0][p], most[1][p])), max(most[2][p], most[3][p]));
            return scale_of(t);
        };
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
            if (p < pieces && col(p) < Kp) {
                const float s = scale(row(p));
                const bool ok = usable(s);
                *reinterpret_cast<unsigned*>(xs + row(p) * Kp + col(p)) = ok ? Quant(ok ? s : 1.f).pack(v[p]) : 0u;
            }
        sm[0] = scale(min(i, a.M - 1));
        __syncthreads();
    } else {
        fetch(wv[0], w);
        fetch(wv[1], w + NW);
#pragma unroll
        for (int m = 0; m < MB; ++m) sm[m] = a.sx[min(16 * m + i, a.M - 1)];
    }
    auto operands = [&](intx4 (&x)[MB][4], int s) {
        if (s >= steps) return;
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (FUSED) {
                    x[m][u] = intx4{0, 0, 0, 0};
                    if (i < a.M) x[m][u] = *reinterpret_cast<const intx4*>(xs + i * Kp + 256 * s + 64 * g + 16 * u);
                } else {
                    x[m][u] = *reinterpret_cast<const intx4*>(a.X + ((long)m * steps + s) * 4096 + u * 1024 + lane * 16);
                }
            }
    };
    auto step = [&](const intx4 (&v)[4], const intx4 (&x)[MB][4], int s) {
        if (s >= steps) return;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int m = 0; m < MB; ++m) acc[m] = mfma8(v[u], x[m][u], acc[m]);
    };
    // (one workgroup a CU: x's operands a block ahead, too; 64 x 2048 x 4096 11.3 -> 10.3 us. With more of them
    // the registers cost as much: 48 x 8512 x 2048 11.4 -> 11.6.)
    if constexpr (NW == 8) {
        intx4 xv[2][MB][4];
        operands(xv[0], w);
        for (int s = w; s < steps; s += 2 * NW) {
            operands(xv[1], s + NW);
            step(wv[0], xv[0], s);
            fetch(wv[0], s + 2 * NW);
            operands(xv[0], s + 2 * NW);
            step(wv[1], xv[1], s + NW);
            fetch(wv[1], s + 3 * NW);
        }
    } else {
        auto both = [&](const intx4 (&v)[4], int s) {
            if (s >= steps) return;
            intx4 x[MB][4];
            operands(x, s);
            step(v, x, s);
        };
        for (int s = w; s < steps; s += 2 * NW) {
            both(wv[0], s);
            fetch(wv[0], s + 2 * NW);
            both(wv[1], s + NW);
            fetch(wv[1], s + 3 * NW);
        }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) red[w][m][lane] = acc[m];
    __syncthreads();
    // rows 16 t .. are finished by wave t
    const Out<TO> out(a, 0, a.M, n0, rows);
#pragma unroll
    for (int t = 0; t < MB; ++t) {
        if (t != w) continue;
        const int n = 4 * g, row = 16 * t + i;
        intx4 c = red[0][t][lane];
#pragma unroll
        for (int o = 1; o < NW; ++o) c += red[o][t][lane];
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = min(n0 + n + r, a.N - 1);
            v[r] = scaled<true>(c[r], sm[t], a.sw[k]) + (a.bias ? a.bias[k] : 0.f);
        }
        const int rr = row < a.M ? row : 0, nn = row < a.M ? n : 1 << 30;
        if (a.vec) put4<TO, BETA>(out, a.beta, rr, nn, v);
        else {
#pragma unroll
            for (int r = 0; r < 4; ++r) put1<TO, BETA>(out, a.beta, rr, nn + r, v[r]);
        }
    }
}

// ---------------------------------------------------------------- tiles
__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t r, char* lds, unsigned voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, voff, 0, 0, 0);
}

// WN x WM waves, each with TN x TM tiles of 32 x 32 (v_mfma_i32_32x32x32_i8): a workgroup owns 32 TN
// WN output channels of 32 TM WM rows and walks k in blocks of 64 through four LDS stages. The loads
// go straight from memory to LDS, sixteen rows of 64 bytes an instruction. A row's 64 bytes lie as
// four 16-byte pieces, piece c at place c ^ (row / 4 % 4): any 16 consecutive rows of a piece then
// fall on all banks.
//
// A block's k are two steps of 32 (one MFMA deep). While a step multiplies, the operands of the next
// one are read; so a stage is free once its second step is in registers, a step before its products
// end. There the wave waits for its loads of the next stage and for the workgroup, issues the loads
// of the fourth block on into the stage that came free, and goes on: one barrier a block, with
// products behind and ahead of it, and a load has three blocks' time to land. At a tile's end these
// are the next tile's first blocks: its operands land while the outputs are written.
//
// Bound by the matrix cores and the LDS reads that feed them: 8192 x 8512 x 2048 to bf16 takes 152 to 164 us
// on different cards, 1.74 POP/s and more (a library's product of the integers alone 164 us), 8192 x 8192 x 8192 477 us, 2.3 POP/s (457).
//
// The outputs go through LDS, so that they are written 128 bytes of a row at a time: as they lie in the
// accumulators (16 bytes of 32 rows an instruction) they took 17 us of a tile's 40 at K 2048.
struct Tiles {        // tile ids first, first + step, .. below end; id -> place
    int first, step, end;
};

template <int WN, int WM, int TN, int TM, bool ONE, typename TO, bool BETA, int SB, typename Place>
__device__ __forceinline__ void i8_tiles(const I8Args& a, Tiles tiles, Place place_of, char* s0, char* s1,
                                         char* s2, char* s3, float* chs, float* chb, float* rows_s,
                                         float* outs) {
    constexpr int NW = WN * WM, BN = 32 * TN * WN, BM = 32 * TM * WM;
    constexpr int PW = BN / 16 / NW, PX = BM / 16 / NW, PER = PW + PX;
    static_assert(BN % (16 * NW) == 0 && BM % (16 * NW) == 0 && (BN + BM) * 64 <= SB, "loads shared out evenly");
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 5, i32 = lane & 31;
    const int wn = w % WN, wm = w / WN;
    // a wave loads PW groups of sixteen rows of W and PX of x
    const unsigned piece = 16u * ((lane & 3) ^ (lane >> 4));
    const unsigned downw = 16u * (unsigned)a.ldw, downx = 16u * (unsigned)a.ldx;
    const unsigned atw = (unsigned)((lane >> 2) * a.ldw) + piece + PW * w * downw;
    const unsigned atx = (unsigned)((lane >> 2) * a.ldx) + piece + PX * w * downx;
    const int KB = (a.K + 63) / 64, KR = (KB + 3) & ~3;   // (blocks past the last multiply zeros)

    struct Where { int n0, m0, nrows, mrows; };
    auto where = [&](int id) {
        int tn, tm;
        place_of(id, tn, tm);
        return Where{tn * BN, tm * BM, min(BN, a.N - tn * BN), min(BM, a.M - tm * BM)};
    };
    auto rsrc_w = [&](const Where& t) {
        return ssm::rsrc(a.W + (long)t.n0 * a.ldw, (unsigned)((long)(t.nrows - 1) * a.ldw + whole(a.K)));
    };
    auto rsrc_x = [&](const Where& t) {
        return ssm::rsrc(a.X + (long)t.m0 * a.ldx, (unsigned)((long)(t.mrows - 1) * a.ldx + whole(a.K)));
    };
    auto load = [&](char* s, __amdgpu_buffer_rsrc_t rw, __amdgpu_buffer_rsrc_t rx, int kb) {
        // (a block past the last reads zeros: past the descriptors)
        const unsigned k = kb < KB ? 64u * (unsigned)kb : kOut;
#pragma unroll
        for (int u = 0; u < PW; ++u) to_lds16(rw, s + (PW * w + u) * 1024, atw + (k + u * downw));
#pragma unroll
        for (int u = 0; u < PX; ++u) to_lds16(rx, s + BN * 64 + (PX * w + u) * 1024, atx + (k + u * downx));
    };
    struct Frags { intx4 w[TN], x[TM]; };
    const int swz = i32 >> 2 & 3;
    const int wrow = (32 * TN * wn + i32) * 64, xrow = (BN + 32 * TM * wm + i32) * 64;
    auto read = [&](Frags& f, const char* s, int step) {
        const int c = 16 * ((2 * step + g) ^ swz);
#pragma unroll
        for (int j = 0; j < TM; ++j) f.x[j] = *reinterpret_cast<const intx4*>(s + xrow + c + 32 * j * 64);
#pragma unroll
        for (int i = 0; i < TN; ++i) f.w[i] = *reinterpret_cast<const intx4*>(s + wrow + c + 32 * i * 64);
    };
    intx16 acc[TN][TM];
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
    };
    // the reads (and L loads) of a step spread over the products of the one before
    constexpr int NF = TN + TM, NP = TN * TM;
    auto spread = [&](auto loads) {
        constexpr int L = decltype(loads)::value;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i < NF) __builtin_amdgcn_sched_group_barrier(0x100, (NF + NP - 1) / NP, 0);
            if (L && i >= NP / 2) __builtin_amdgcn_sched_group_barrier(0x020, (2 * L + NP - 1) / NP, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // at most KEEP of the wave's loads (and stores) in flight, its LDS reads done, then the workgroup
    auto meet = [&](auto keep) {
        constexpr int KEEP = decltype(keep)::value;
        static_assert(KEEP < 64, "vmcnt has six bits");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0070 | (KEEP & 15) | ((KEEP >> 4) << 14));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, 2 * PER> two{};
    constexpr std::integral_constant<int, 3 * PER> three{};

    int id = tiles.first;
    if (id >= tiles.end) return;
    Where t = where(id);
    auto rw = rsrc_w(t), rx = rsrc_x(t);
    load(s0, rw, rx, 0);
    load(s1, rw, rx, 1);
    load(s2, rw, rx, 2);
    load(s3, rw, rx, 3);
    Frags f0, f1;
    for (;;) {
        const int after = id + tiles.step;
        const bool more = !ONE && after < tiles.end;
        const Where tn = more ? where(after) : t;
        const auto nw = rsrc_w(tn), nx = rsrc_x(tn);
        // one block out of stage s, its first step in f0; leaves the next block's first step there
        auto block = [&](char* s, char* next, int kb) {
            read(f1, s, 1);
            multiply(f0);
            spread(std::integral_constant<int, 0>{});
            meet(two);
            read(f0, next, 0);
            if (kb + 4 < KR) load(s, rw, rx, kb + 4);
            else load(s, nw, nx, more ? kb + 4 - KR : KB);
            multiply(f1);
            spread(std::integral_constant<int, PER>{});
        };
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                acc[i][j] = intx16{};
                asm volatile("" : "+a"(acc[i][j]));   // (in accumulation registers from the start)
            }
        meet(three);
        read(f0, s0, 0);
        // the tile's scales, for its end (the last tile's were read before the barrier)
        for (int i = threadIdx.x; i < BN + BM; i += 64 * NW) {
            if (i < BN) {
                const int n = min(t.n0 + i, a.N - 1);
                chs[i] = a.sw[n];
                chb[i] = a.bias ? a.bias[n] : 0.f;
            } else {
                rows_s[i - BN] = a.sx[min(t.m0 + i - BN, a.M - 1)];
            }
        }
        for (int kb = 0; kb < KR; kb += 4) {
            block(s0, s1, kb);
            block(s1, s2, kb + 1);
            block(s2, s3, kb + 2);
            block(s3, s0, kb + 3);
        }

        if constexpr (ONE) {   // (the outputs take a stage)
            __builtin_amdgcn_s_waitcnt(0x0070);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
        // ---- outputs, 32 rows of 128 bytes at a time through the wave's own 4 KB of LDS: bf16 as they are
        // written (two tiles of columns), fp32 and what beta y is added to as fp32 (one). The 16-byte piece
        // u of row r lies at u ^ (r % 8), so that the rows of a piece fall on all banks.
        using TL = typename std::conditional<BETA, float, TO>::type;
        constexpr int UI = 4 / sizeof(TL), CP = 32 * UI;   // tiles and columns a time
        const int li = fresh(i32), lg = fresh(g), ll = fresh(lane);
        char* tile = reinterpret_cast<char*>(outs) + w * 4096;
        auto place = [&](int r, int u) { return tile + r * 128 + 16 * (u ^ (r & 7)); };
        const Out<TO> out(a, t.m0, t.mrows, t.n0, t.nrows);
        bool any_far = false;   // (of the wave's channels and rows)
#pragma unroll
        for (int c = 0; c < 32 * TN; c += 64) any_far |= far(chs[32 * TN * wn + c + ll % (32 * TN)]);
#pragma unroll
        for (int r = 0; r < 32 * TM; r += 64) any_far |= far(rows_s[32 * TM * wm + r + ll % (32 * TM)]);
        auto finish = [&](auto vec, auto fars) {
            constexpr bool VEC = decltype(vec)::value, FAR = decltype(fars)::value;
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const int mw = 32 * (TM * wm + j);
                const float sm = rows_s[mw + li];
#pragma unroll
                for (int i0 = 0; i0 < TN; i0 += UI) {
                    const int nw = 32 * (TN * wn + i0);
#pragma unroll
                    for (int i = 0; i < UI; ++i)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {   // channels 8 q + 4 g .. + 3 of the tile, row i32
                            const int c = 32 * i + 8 * q + 4 * lg;
                            const floatx4 s4 = *reinterpret_cast<const floatx4*>(&chs[nw + c]);
                            const floatx4 b4 = *reinterpret_cast<const floatx4*>(&chb[nw + c]);
                            floatx4 v;
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[r] = scaled<FAR>(acc[i0 + i][j][4 * q + r], sm, s4[r]) + b4[r];
                            if constexpr (sizeof(TL) == 4) {
                                *reinterpret_cast<floatx4*>(place(li, c / 4)) = v;
                            } else {
                                bf16x4 y;
#pragma unroll
                                for (int r = 0; r < 4; ++r) y[r] = (__bf16)v[r];
                                *reinterpret_cast<bf16x4*>(place(li, c / 8) + 2 * (c & 4)) = y;
                            }
                        }
                    __builtin_amdgcn_wave_barrier();
                    if constexpr (VEC) {
                        constexpr int E = 16 / sizeof(TO), LR = CP / E, RR = 64 / LR;   // lanes a row, rows a time
#pragma unroll
                        for (int r0 = 0; r0 < 32; r0 += RR) {
                            const int r = r0 + ll / LR, c = ll % LR * E;
                            if constexpr (BETA || sizeof(TO) == 4) {
                                float v[E];
#pragma unroll
                                for (int p = 0; p < E / 4; ++p) {
                                    const floatx4 x = *reinterpret_cast<const floatx4*>(place(r, c / 4 + p));
#pragma unroll
                                    for (int e = 0; e < 4; ++e) v[4 * p + e] = x[e];
                                }
                                put<TO, BETA>(out, a.beta, mw + r, nw + c, v);
                            } else {
                                const unsigned off = nw + c < out.cols ? ((unsigned)(mw + r) * out.ld + (unsigned)(nw + c)) * 2u : kOut;
                                __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const ssm::u32x4*>(place(r, c / 8)), out.d, off, 0, 0);
                            }
                        }
                    } else {
#pragma unroll 4
                        for (int k = 0; k < 32 * CP; k += 64) {
                            const int r = (k + ll) / CP, c = (k + ll) % CP;
                            const TL y = reinterpret_cast<const TL*>(place(r, c * (int)sizeof(TL) / 16))[c % (16 / (int)sizeof(TL))];
                            put1<TO, BETA>(out, a.beta, mw + r, nw + c, (float)y);
                        }
                    }
                    __builtin_amdgcn_wave_barrier();
                }
            }
        };
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        if (__any(any_far)) {
            if (a.vec) finish(yes, yes);
            else finish(no, yes);
        } else {
            if (a.vec) finish(yes, no);
            else finish(no, no);
        }
        if (ONE || !more) break;
        id = after;
        t = tn;
        rw = nw;
        rx = nx;
    }
    // no load is in flight into LDS, and no wave reads from it, when it is used otherwise
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
}

// One tile of 128 channels and 64 TM rows a workgroup, several workgroups a CU.
template <int TM, typename TO, bool BETA>
__global__ __launch_bounds__(256, 2) void i8_gemm_kernel(I8Args a) {
    constexpr int SB = (128 + 64 * TM) * 64;
    // (the stages are objects of their own: a read of one does not wait for the loads into the others;
    // the first takes the outputs too, 4 KB a wave)
    constexpr int S0 = SB < 4 * 4096 ? 4 * 4096 : SB;
    __shared__ __attribute__((aligned(16))) char s0[S0], s1[SB], s2[SB], s3[SB];
    __shared__ __attribute__((aligned(16))) float chs[128], chb[128], rows_s[64 * TM];
    // consecutive ids on one XCD, in groups of gn channel tiles
    const int T = a.mt * a.nt, xcd = blockIdx.x & 7, per = T >> 3, rem = T & 7;
    const int id = xcd * per + min(xcd, rem) + (blockIdx.x >> 3);
    auto place = [&](int id, int& tn, int& tm) {
        const int gsz = a.gn * a.mt, grp = id / gsz, gr = id - grp * gsz;
        const int gn = min(a.gn, a.nt - grp * a.gn);
        tn = grp * a.gn + gr % gn;
        tm = gr / gn;
    };
    i8_tiles<2, 2, 2, TM, true, TO, BETA, SB>(a, Tiles{id, 1, id + 1}, place, s0, s1, s2, s3, chs, chb, rows_s,
                                              reinterpret_cast<float*>(s0));
}

// 256 x 256 tiles, one workgroup a CU that walks its share of them: XCD x's 32 workgroups take its
// tiles in turn. Tiles of a last turn that would leave three quarters of the CUs idle are shared out
// in quarters, 128 x 128 a workgroup (8192 x 8512: 1088 tiles are 4.25 turns).
template <typename TO, bool BETA>
__global__ __launch_bounds__(256, 1) void i8_gemm_big_kernel(I8Args a) {
    constexpr int SB = 512 * 64;
    __shared__ __attribute__((aligned(16))) char s0[SB], s1[SB], s2[SB], s3[SB];
    __shared__ __attribute__((aligned(16))) float chs[256], chb[256], rows_s[256], outs[4096];
    const int T = a.mt * a.nt, xcd = blockIdx.x & 7, local = blockIdx.x >> 3, wgs = gridDim.x >> 3;
    const int per = T >> 3, rem = T & 7;
    const int lo = xcd * per + min(xcd, rem), n = per + (xcd < rem), tail = n % wgs;
    const bool quarters = 4 * tail <= wgs;
    auto place = [&](int id, int& tn, int& tm) {
        const int gsz = a.gn * a.mt, grp = id / gsz, gr = id - grp * gsz;
        const int gn = min(a.gn, a.nt - grp * a.gn);
        tn = grp * a.gn + gr % gn;
        tm = gr / gn;
    };
    const int whole_end = lo + n - (quarters ? tail : 0);
    i8_tiles<2, 2, 4, 4, false, TO, BETA, SB>(a, Tiles{lo + local, wgs, whole_end}, place, s0, s1, s2, s3, chs, chb,
                                       rows_s, outs);
    if (!quarters) return;
    auto quarter = [&](int id, int& tn, int& tm) {
        place(whole_end + (id >> 2), tn, tm);
        tn = 2 * tn + (id & 1);
        tm = 2 * tm + (id >> 1 & 1);
    };
    // (a quarter that lies past the matrix is not begun)
    int id = local;
    if (id < 4 * tail) {
        int tn, tm;
        quarter(id, tn, tm);
        if (tn * 128 >= a.N || tm * 128 >= a.M) id = 4 * tail;
    }
    i8_tiles<2, 2, 2, 2, true, TO, BETA, SB>(a, Tiles{id, wgs, min(4 * tail, id + 1)}, quarter, s0, s1, s2, s3,
                                             chs, chb, rows_s, outs);
}

// ---------------------------------------------------------------- plan
template <int MB, typename TX, typename TO, int NW>
void rows_launch(const I8Args& a, hipStream_t st) {
    const unsigned n = (unsigned)ssm::cdiv(a.N, 16);
    if (a.beta != 0.f) i8_rows_kernel<MB, TX, TO, true, NW><<<n, 64 * NW, 0, st>>>(a);
    else i8_rows_kernel<MB, TX, TO, false, NW><<<n, 64 * NW, 0, st>>>(a);
}

// Eight waves a workgroup where there is at most one a CU (rounding and product of 64 rows, N 2048, K 4096: 10.3
// us, 13.1 with four; N 6144: 15.0, 14.7).
template <int MB, typename TO>
void rows_of(const I8Args& a, hipStream_t st) {
    if (a.N <= 16 * kCUs) rows_launch<MB, void, TO, 8>(a, st);
    else rows_launch<MB, void, TO, 4>(a, st);
}

template <int TM, typename TO>
void tile_launch(I8Args a, hipStream_t st) {
    a.nt = (int)ssm::cdiv(a.N, 128);
    a.mt = (int)ssm::cdiv(a.M, 64 * TM);
    a.gn = std::min(a.nt, 8);
    const unsigned n = (unsigned)(a.nt * a.mt);
    if (a.beta != 0.f) i8_gemm_kernel<TM, TO, true><<<n, 256, 0, st>>>(a);
    else i8_gemm_kernel<TM, TO, false><<<n, 256, 0, st>>>(a);
}

template <typename TO>
void gemm_launch(I8Args a, hipStream_t st) {
    // tiles of 256 where every CU has one (4096 x 4096 x 4096: 68 us, 80 in tiles of 128; with half as many,
    // 2048 x 4096 x 2048: 36 us, 26). gn: 4, 8 and 16 are within 3%.
    const long big = ssm::cdiv(a.N, 256) * ssm::cdiv(a.M, 256);
    if (big >= kCUs) {
        a.nt = (int)ssm::cdiv(a.N, 256);
        a.mt = (int)ssm::cdiv(a.M, 256);
        a.gn = std::min(a.nt, 8);
        if (a.beta != 0.f) i8_gemm_big_kernel<TO, true><<<kCUs, 256, 0, st>>>(a);
        else i8_gemm_big_kernel<TO, false><<<kCUs, 256, 0, st>>>(a);
        return;
    }
    // tiles of 64 rows where those of 128 would leave CUs idle (512 x 4096 x 4096: 16.0 us, 19.7; a tile
    // for every CU, 1000 x 4096 x 2048: 15.0 us with 64 rows, 12.1 with 128)
    if (ssm::cdiv(a.N, 128) * ssm::cdiv(a.M, 128) < kCUs) tile_launch<1, TO>(a, st);
    else tile_launch<2, TO>(a, st);
}

template <typename TO>
ssm_status product(const I8Args& a, hipStream_t st) {
    if (a.Xf && a.x_dtype == SSM_F32) rows_launch<1, float, TO, 4>(a, st);
    else if (a.Xf) rows_launch<1, __bf16, TO, 4>(a, st);
    else if (a.M <= 16) rows_of<1, TO>(a, st);
    else if (a.M <= 32) rows_of<2, TO>(a, st);
    else if (a.M <= kRowsMax) rows_of<4, TO>(a, st);
    else gemm_launch<TO>(a, st);
    return ssm::check_launch("ssm_linear_i8");
}

bool direct_w(const void* p, long ld, int K) { return ((uintptr_t)p & 15) == 0 && ld % 16 == 0 && K % 4 == 0; }
// (x's bytes past K must be zeros; W's do not matter then)
bool direct_x(const void* p, long ld, int M, int K) {
    return M > kRowsMax && ((uintptr_t)p & 15) == 0 && ld % 16 == 0 && K % kPad == 0;
}

// Rows of x that a product reads: the few-row kernel whole blocks of 16 (what the last of them holds
// past M goes into sums that are not kept).
long rows_read(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= kRowsMax ? kRowsMax : M; }

// Workspace: x's rows as integers (Kp bytes each) with their scales, then W's where they have to be
// laid out.
struct Layout { size_t x, sx, w, all; long Kp; };
Layout layout(int M, int N, int K, bool x, bool scales, bool w) {
    Layout l{};
    l.Kp = up(K, kPad);
    size_t o = 0;
    l.x = o;
    if (x) o += (size_t)rows_read(M) * l.Kp;
    l.sx = o;
    if (scales) o += (size_t)up(4L * M, 256);
    l.w = o;
    if (w) o += (size_t)N * l.Kp;
    l.all = o;
    return l;
}

ssm_status check_product(const char* who, const void* x, long ldx, const int8_t* W, long ldw,
                         const float* sw, int out_dtype, const void* y, long ldy, int M, int N, int K) {
    SSM_REQUIRE(out_dtype == SSM_F32 || out_dtype == SSM_BF16, "%s: bad output dtype", who);
    SSM_REQUIRE(M >= 0 && N > 0 && K > 0, "%s: bad shape", who);
    if (K > kMaxK)
        return ssm::fail(SSM_ERR_UNSUPPORTED, "%s: K %d above %d (32-bit sums)", who, K, kMaxK);
    if (M == 0) return SSM_OK;
    SSM_REQUIRE(x && W && sw && y, "%s: null input", who);
    SSM_REQUIRE(ldx >= K && ldw >= K && ldy >= N, "%s: row stride below row width", who);
    SSM_REQUIRE(M <= ssm::kMaxGroups && N <= ssm::kMaxGroups, "%s: too many rows", who);
    SSM_REQUIRE(ldw < (1L << 22) && ldx < (1L << 22) && ldy < (1L << 21), "%s: row stride too large", who);
    return SSM_OK;
}

// y apart from what is read while it is written, the workspace from everything.
ssm_status check_overlaps(const char* who, const ssm::Rows& y, const int8_t* W, long ldw, const float* sw,
                          const float* bias, int N, int K, const ssm::Rows& workspace, const ssm::Rows& x,
                          const ssm::Rows& sx) {
    const ssm::Rows w{W, ldw, K, N}, s = ssm::block(sw, 4L * N), b = ssm::block(bias, 4L * N);
    SSM_REQUIRE(!ssm::meets(y, w, s, b), "%s: y overlaps the weights, their scales or the bias", who);
    SSM_REQUIRE(!ssm::meets(workspace, w, s, b, y, x, sx),
                "%s: the workspace overlaps another operand", who);
    return SSM_OK;
}

ssm_status launch_product(I8Args a, int out_dtype, const Layout& l, bool lay_w, char* ws,
                          hipStream_t st) {
    if (lay_w) {
        signed char* o = (signed char*)ws + l.w;
        lay_rows_kernel<false><<<a.N, 256, 0, st>>>(a.W, a.ldw, a.K, o, (int)l.Kp);
        if (ssm_status e = ssm::check_launch("ssm_linear_i8 (weight rows)")) return e;
        a.W = o;
        a.ldw = l.Kp;
    }
    const int e = out_dtype == SSM_F32 ? 4 : 8;
    a.vec = a.N % e == 0 && a.ldy % e == 0 && ((uintptr_t)a.y & 15) == 0;
    return out_dtype == SSM_F32 ? product<float>(a, st) : product<__bf16>(a, st);
}

}  // namespace

extern "C" ssm_status ssm_quantize_rows(int dtype, const void* x, long ldx, int8_t* q, long ldq,
                                        float* scale, int M, int K, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_quantize_rows: bad dtype");
    SSM_REQUIRE(M >= 0 && K > 0, "ssm_quantize_rows: bad shape");
    if (M == 0) return SSM_OK;
    SSM_REQUIRE(x && q && scale, "ssm_quantize_rows: null input");
    SSM_REQUIRE(ldx >= K && ldq >= K, "ssm_quantize_rows: row stride below row width");
    SSM_REQUIRE(M <= ssm::kMaxGroups, "ssm_quantize_rows: too many rows");
    SSM_REQUIRE(K <= ssm::kMaxSteps, "ssm_quantize_rows: too long");
    const long es = dtype == SSM_F32 ? 4 : 2;
    const ssm::Rows rx{x, ldx * es, K * es, M}, rq{q, ldq, K, M};
    SSM_REQUIRE(!ssm::meet(rx, rq), "ssm_quantize_rows: q overlaps x");
    SSM_REQUIRE(!ssm::meets(ssm::block(scale, 4L * M), rx, rq), "ssm_quantize_rows: the scales overlap x or q");
    return quantize(dtype, x, ldx, (signed char*)q, ldq, scale, M, K, K, false, (hipStream_t)stream);
}

extern "C" size_t ssm_linear_i8_workspace(const int8_t* x, long ldx, const int8_t* W, long ldw, int M,
                                          int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return layout(M, N, K, !direct_x(x, ldx, M, K), false, !direct_w(W, ldw, K)).all;
}

extern "C" ssm_status ssm_linear_i8(const int8_t* x, long ldx, const float* sx, const int8_t* W,
                                    long ldw, const float* sw, const float* bias, int out_dtype,
                                    void* y, long ldy, int M, int N, int K, float beta,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    if (ssm_status e = check_product("ssm_linear_i8", x, ldx, W, ldw, sw, out_dtype, y, ldy, M, N, K))
        return e;
    if (M == 0) return SSM_OK;
    SSM_REQUIRE(sx, "ssm_linear_i8: null input");
    const bool lay_x = !direct_x(x, ldx, M, K), lay_w = !direct_w(W, ldw, K);
    const Layout l = layout(M, N, K, lay_x, false, lay_w);
    SSM_REQUIRE(l.all == 0 || (workspace && workspace_bytes >= l.all && ((uintptr_t)workspace & 15) == 0),
                "ssm_linear_i8: 16-byte aligned workspace of %zu bytes needed", l.all);
    const long es = out_dtype == SSM_F32 ? 4 : 2;
    const ssm::Rows rx{x, ldx, K, M}, rs = ssm::block(sx, 4L * M), ry{y, ldy * es, N * es, M};
    SSM_REQUIRE(!ssm::meets(ry, rx, rs), "ssm_linear_i8: y overlaps x or its scales");
    if (ssm_status e = check_overlaps("ssm_linear_i8", ry, W, ldw, sw, bias, N, K, ssm::block(workspace, l.all),
                                      rx, rs))
        return e;
    I8Args a{(const signed char*)x, ldx, sx, nullptr, 0, 0, (const signed char*)W, ldw, sw, bias, y, ldy,
             M, N, K, beta, 0, 0, 0, 0};
    if (lay_x) {
        signed char* o = (signed char*)workspace + l.x;
        if (M <= kRowsMax)
            lay_rows_kernel<true><<<M, 256, 0, (hipStream_t)stream>>>(a.X, ldx, K, o, (int)l.Kp);
        else
            lay_rows_kernel<false><<<M, 256, 0, (hipStream_t)stream>>>(a.X, ldx, K, o, (int)l.Kp);
        if (ssm_status e = ssm::check_launch("ssm_linear_i8 (rows)")) return e;
        a.X = o;
        a.ldx = l.Kp;
    }
    return launch_product(a, out_dtype, l, lay_w, (char*)workspace, (hipStream_t)stream);
}

extern "C" size_t ssm_linear_q8_workspace(const int8_t* W, long ldw, int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return layout(M, N, K, true, true, !direct_w(W, ldw, K)).all;
}

extern "C" ssm_status ssm_linear_q8(int in_dtype, const void* x, long ldx, const int8_t* W, long ldw,
                                    const float* sw, const float* bias, int out_dtype, void* y,
                                    long ldy, int M, int N, int K, float beta, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(in_dtype == SSM_F32 || in_dtype == SSM_BF16, "ssm_linear_q8: bad dtype");
    if (ssm_status e = check_product("ssm_linear_q8", x, ldx, W, ldw, sw, out_dtype, y, ldy, M, N, K))
        return e;
    if (M == 0) return SSM_OK;
    const bool lay_w = !direct_w(W, ldw, K);
    const Layout l = layout(M, N, K, true, true, lay_w);
    SSM_REQUIRE(workspace && workspace_bytes >= l.all && ((uintptr_t)workspace & 15) == 0,
                "ssm_linear_q8: 16-byte aligned workspace of %zu bytes needed", l.all);
    signed char* q = (signed char*)workspace + l.x;
    float* sx = (float*)((char*)workspace + l.sx);
    I8Args a{q, l.Kp, sx, nullptr, ldx, in_dtype, (const signed char*)W, ldw, sw, bias, y, ldy,
             M, N, K, beta, 0, 0, 0, 0};
    const bool vec = K % 4 == 0 && ldx % 4 == 0 && ((uintptr_t)x & (in_dtype == SSM_F32 ? 15 : 7)) == 0;
    const int per = K > 2048 ? 4 : K > 1024 ? 2 : 1;
    const long ei = in_dtype == SSM_F32 ? 4 : 2, eo = out_dtype == SSM_F32 ? 4 : 2;
    const ssm::Rows rx{x, ldx * ei, K * ei, M}, ry{y, ldy * eo, N * eo, M};
    if (ssm_status e = check_overlaps("ssm_linear_q8", ry, W, ldw, sw, bias, N, K, ssm::block(workspace, l.all),
                                      rx, ssm::block(nullptr, 0)))
        return e;
    // (each workgroup reads all of x there while others write: y has to be elsewhere)
    if (vec && !ssm::meet(rx, ry) && K <= kFusedX && M <= kFusedRows && M * per <= kFusedX / 1024)
        a.Xf = x;
    else if (ssm_status e = quantize(in_dtype, x, ldx, q, l.Kp, sx, M, K, (int)l.Kp, M <= kRowsMax,
                                     (hipStream_t)stream))
        return e;
    return launch_product(a, out_dtype, l, lay_w, (char*)workspace, (hipStream_t)stream);
}

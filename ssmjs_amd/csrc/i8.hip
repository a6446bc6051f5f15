// Products of 8-bit integers with a scale for each row of x (token) and of W (output channel):
//   quantised rows    s_m = max_k |x_mk| / 127 (fp32),  q_mk = x_mk / s_m to the nearest integer,
//                     ties to even (from the exact quotient), held to -127 .. 127
//   y_mn = beta y_mn + s_m s_n sum_k q_mk w_nk (+ bias_n)
// The sums are exact 32-bit integers (|q|, |w| <= 128: K up to 131071), on v_mfma_i32_16x16x64_i8.
//
// Three kernels share the work by rows:
//   - up to 64 rows (one per decoded sequence): the weights' bytes bound it. i8_rows_kernel reads
//     every weight row once, straight into registers, the k of a row shared by the four waves.
//   - more rows: the matrix cores bound it. i8_gemm_kernel is a tiled product out of LDS.
//   - rows that are not 16-byte aligned are laid out in the workspace first (pad_rows_kernel).
#include <algorithm>

#include "common.hpp"

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kMaxK = 131071;
constexpr int kPad = 256;          // rows of the workspace are whole blocks of 256 bytes, zeros past K
constexpr int kRowsMax = 64;       // rows of the few-row kernel
inline long up(long n, long to) { return (n + to - 1) / to * to; }

// ---------------------------------------------------------------- rows to integers
struct Quant {
    float f, s, inv;   // x f / (s f), s f in the normal range
    __device__ __forceinline__ explicit Quant(float scale) {
        f = scale < 0x1p-100f ? 0x1p120f : 1.f;
        s = scale * f;
        inv = 1.f / s;
    }
    // nearest integer to x / s: a first guess, then the exact remainder (x - q s has 24 bits)
    __device__ __forceinline__ int operator()(float x) const {
        x *= f;
        float q = rintf(x * inv);
        const float r = fmaf(-q, s, x), d = 2.f * fabsf(r);
        if (d > s || (d == s && ((int)q & 1))) q += copysignf(1.f, r);
        return (int)fminf(fmaxf(q, -127.f), 127.f);
    }
};

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

__device__ __forceinline__ unsigned pack4(const Quant& z, float4 v) {
    return (z(v.x) & 255) | (z(v.y) & 255) << 8 | (z(v.z) & 255) << 16 | (unsigned)z(v.w) << 24;
}

struct QuantArgs {
    const void* x; long ldx;
    signed char* q; long ldq;
    float* scale;
    int M, K, Kq;   // Kq: bytes written per row (zeros past K)
};

// A row per workgroup of TPR threads' share: 256 / TPR rows a workgroup, U pieces of four held
// between the two passes (further ones are read again).
template <typename T, int TPR, bool VEC>
__global__ __launch_bounds__(256) void quant_kernel(QuantArgs a) {
    constexpr int U = 8, RPB = 256 / TPR, NW = TPR / 64;
    __shared__ unsigned red[4];
    const int tid = threadIdx.x % TPR, rw = threadIdx.x / TPR;
    const long m = (long)blockIdx.x * RPB + rw;
    const bool live = m < a.M;
    const T* row = static_cast<const T*>(a.x) + (live ? m : 0) * a.ldx;
    float4 v[U];
    unsigned most = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        v[u] = some4<T, VEC>(row, 4 * (tid + TPR * u), a.K);
        most = max4(most, v[u]);
    }
    for (int k = 4 * (tid + TPR * U); k < a.K; k += 4 * TPR) most = max4(most, some4<T, VEC>(row, k, a.K));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, off));
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
    signed char* out = a.q + m * a.ldq;
    auto put = [&](int k, float4 x) {
        if (k >= a.Kq) return;
        const unsigned b = ok ? pack4(z, x) : 0u;
        if constexpr (VEC) {
            *reinterpret_cast<unsigned*>(out + k) = b;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k + e < a.Kq) out[k + e] = (signed char)(b >> 8 * e);
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) put(4 * (tid + TPR * u), v[u]);
    for (int k = 4 * (tid + TPR * U); k < a.Kq; k += 4 * TPR) put(k, some4<T, VEC>(row, k, a.K));
}

template <typename T>
ssm_status run_quant(const QuantArgs& a, bool vec, hipStream_t st) {
    // a wave a row up to 2048 elements (its eight pieces a lane), a workgroup beyond
    if (a.K <= 2048 && a.M >= 1024) {
        const unsigned n = (unsigned)ssm::cdiv(a.M, 4);
        if (vec) quant_kernel<T, 64, true><<<n, 256, 0, st>>>(a);
        else quant_kernel<T, 64, false><<<n, 256, 0, st>>>(a);
    } else {
        if (vec) quant_kernel<T, 256, true><<<a.M, 256, 0, st>>>(a);
        else quant_kernel<T, 256, false><<<a.M, 256, 0, st>>>(a);
    }
    return ssm::check_launch("ssm_quantize_rows");
}

ssm_status quantize(int dtype, const void* x, long ldx, signed char* q, long ldq, float* scale,
                    int M, int K, int Kq, hipStream_t st) {
    const QuantArgs a{x, ldx, q, ldq, scale, M, K, Kq};
    const bool vec = K % 4 == 0 && Kq % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 &&
                     ((uintptr_t)x & (dtype == SSM_F32 ? 15 : 7)) == 0 && ((uintptr_t)q & 3) == 0;
    return dtype == SSM_F32 ? run_quant<float>(a, vec, st) : run_quant<__bf16>(a, vec, st);
}

// Rows of K bytes at any alignment -> rows of Kp bytes, zeros past K.
__global__ __launch_bounds__(256) void pad_rows_kernel(const signed char* __restrict__ x, long ldx,
                                                       int K, signed char* __restrict__ o, int Kp) {
    const signed char* row = x + (long)blockIdx.x * ldx;
    for (int k = 4 * threadIdx.x; k < Kp; k += 1024) {
        unsigned b = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < K) b |= (unsigned)(unsigned char)row[k + e] << 8 * e;
        *reinterpret_cast<unsigned*>(o + (long)blockIdx.x * Kp + k) = b;
    }
}

// ---------------------------------------------------------------- epilogue
struct I8Args {
    const signed char* X; long ldx; const float* sx;   // x as integers (null: from Xf)
    const void* Xf; long ldxf;                         // x to be rounded in the kernel
    const signed char* W; long ldw; const float* sw;
    const float* bias;
    void* y; long ldy;
    int M, N, K;
    float beta;
    int mt, nt, gn;
};

// Four outputs n .. n + 3 of row m.
template <typename TO, bool BETA>
__device__ __forceinline__ void put4(const I8Args& a, int m, int n, intx4 c, float sm, bool vec) {
    if (m >= a.M || n >= a.N) return;
    TO* y = static_cast<TO*>(a.y) + (long)m * a.ldy + n;
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int nn = min(n + r, a.N - 1);
        o[r] = (float)c[r] * (sm * a.sw[nn]);
        if (a.bias) o[r] += a.bias[nn];
    }
    if (vec && n + 3 < a.N) {
        if constexpr (sizeof(TO) == 4) {
            floatx4 v = {o[0], o[1], o[2], o[3]};
            if constexpr (BETA) v += a.beta * *reinterpret_cast<const floatx4*>(y);
            *reinterpret_cast<floatx4*>(y) = v;
        } else {
            bf16x4 v;
            if constexpr (BETA) {
                const bf16x4 p = *reinterpret_cast<const bf16x4*>(y);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] += a.beta * (float)p[r];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (__bf16)o[r];
            *reinterpret_cast<bf16x4*>(y) = v;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < a.N) {
                if constexpr (BETA) o[r] += a.beta * (float)y[r];
                y[r] = (TO)o[r];
            }
    }
}

template <typename TO>
__device__ __forceinline__ bool vec_out(const I8Args& a) {
    return a.ldy % 4 == 0 && ((uintptr_t)a.y & (4 * sizeof(TO) - 1)) == 0;
}

// A row's bytes in whole dwords: one that a descriptor ends inside reads as zeros. (Rows that are
// read in place have a multiple of four, the workspace's are longer.)
__device__ __forceinline__ int whole(int K) { return (K + 3) & ~3; }

__device__ __forceinline__ intx4 mfma8(intx4 w, intx4 x, intx4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
}

// ---------------------------------------------------------------- up to 64 rows
// A workgroup owns NB blocks of 16 output channels; its four waves take the blocks of 256 k in
// turn. Lane (g, i) = (lane / 16, lane % 16) holds row i's bytes 64 g + 16 u .. of the block for
// u = 0 .. 3, which is the operand of MFMA u with the block's k in another order, the same for both
// operands; so a lane reads 64 consecutive bytes. The waves' sums meet in LDS (integers: their order
// changes nothing).
template <int MB, int NB, typename TO, bool BETA>
__global__ __launch_bounds__(256) void i8_rows_kernel(I8Args a) {
    __shared__ intx4 red[3][NB * MB][64];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int n0 = blockIdx.x * 16 * NB;
    const int rows = min(16 * NB, a.N - n0);
    const auto rw = ssm::rsrc(a.W + (long)n0 * a.ldw, (unsigned)((long)(rows - 1) * a.ldw + whole(a.K)));
    const auto rx = ssm::rsrc(a.X, (unsigned)((long)(a.M - 1) * a.ldx + whole(a.K)));
    const unsigned wo = (unsigned)(i * a.ldw) + 64u * g, xo = (unsigned)(i * a.ldx) + 64u * g;
    intx4 acc[NB][MB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[b][m] = intx4{0, 0, 0, 0};
    const int steps = (a.K + 255) / 256;
    for (int s = w; s < steps; s += 4) {
        intx4 wv[NB][4], xv[MB][4];
        const unsigned k = 256u * s;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                wv[b][u] = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(
                    rw, wo + (unsigned)(16 * b * a.ldw) + 16u * u + k, 0, 0));
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                xv[m][u] = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(
                    rx, xo + (unsigned)(16 * m * a.ldx) + 16u * u + k, 0, 0));
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < MB; ++m) acc[b][m] = mfma8(wv[b][u], xv[m][u], acc[b][m]);
    }
    if (w > 0) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int m = 0; m < MB; ++m) red[w - 1][b * MB + m][lane] = acc[b][m];
    }
    __syncthreads();
    if (w > 0) return;
    const bool vec = vec_out<TO>(a);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int row = 16 * m + i;
        const float sm = row < a.M ? a.sx[row] : 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            intx4 c = acc[b][m];
#pragma unroll
            for (int o = 0; o < 3; ++o) c += red[o][b * MB + m][lane];
            put4<TO, BETA>(a, row, n0 + 16 * b + 4 * g, c, sm, vec);
        }
    }
}

// ---------------------------------------------------------------- tiles
__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t r, char* lds, unsigned voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, voff, 0, 0, 0);
}

// All of the wave's loads, then the workgroup barrier: the next stage is whole, and every wave has
// finished with the stage read before.
__device__ __forceinline__ void stage_step() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// WN x WM waves, each with TN x TM tiles of 16 x 16: a workgroup owns 16 TN WN output channels of
// 16 TM WM rows and walks k in blocks of 128 bytes through two LDS stages, the next block's loads in
// flight while one multiplies. A row's 128 bytes lie as eight 16-byte pieces, piece c at place
// c ^ (row / 2 % 8): the 16 rows of an operand read then fall on all banks. The loads go straight
// from memory to LDS (eight rows of 128 bytes an instruction), the order of the pieces being that
// of their addresses.
template <int WN, int WM, int TN, int TM, typename TO, bool BETA>
__global__ __launch_bounds__(64 * WN * WM, 2) void i8_gemm_kernel(I8Args a) {
    constexpr int NW = WN * WM, BN = 16 * TN * WN, BM = 16 * TM * WM;
    constexpr int NL = (BN + BM) / 8, PER = NL / NW, SB = (BN + BM) * 128;
    static_assert(NL % NW == 0 && BN % 8 == 0, "loads shared out evenly");
    __shared__ __attribute__((aligned(16))) char s0[SB];
    __shared__ __attribute__((aligned(16))) char s1[SB];

    // consecutive ids on one XCD, in groups of gn channel tiles
    const int T = a.mt * a.nt, bid = blockIdx.x;
    const int xcd = bid & 7, per = T >> 3, rem = T & 7;
    const int id = xcd * per + min(xcd, rem) + (bid >> 3);
    const int gsz = a.gn * a.mt, grp = id / gsz, gr = id - grp * gsz;
    const int gn = min(a.gn, a.nt - grp * a.gn);
    const int tn = grp * a.gn + gr % gn, tm = gr / gn;

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i16 = lane & 15;
    const int wn = w % WN, wm = w / WN;
    const int n0 = tn * BN, m0 = tm * BM;
    const int nrows = min(BN, a.N - n0), mrows = min(BM, a.M - m0);
    const auto rw = ssm::rsrc(a.W + (long)n0 * a.ldw, (unsigned)((long)(nrows - 1) * a.ldw + whole(a.K)));
    const auto rx = ssm::rsrc(a.X + (long)m0 * a.ldx, (unsigned)((long)(mrows - 1) * a.ldx + whole(a.K)));

    unsigned off[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int r = 8 * (PER * w + u) + (lane >> 3);   // row of the stage: W's, then x's
        const int c = (lane & 7) ^ (r >> 1 & 7);
        off[u] = 8 * (PER * w + u) < BN ? (unsigned)(r * a.ldw) + 16u * c
                                        : (unsigned)((r - BN) * a.ldx) + 16u * c;
    }
    const int KB = (a.K + 127) / 128;
    auto load = [&](char* s, int kb) {
        const unsigned k = 128u * (unsigned)kb;
        if (kb >= KB) return;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int f = PER * w + u;
            to_lds16(8 * f < BN ? rw : rx, s + f * 1024, off[u] + k);
        }
    };
    intx4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = intx4{0, 0, 0, 0};
    const int l0 = i16 * 128 + 16 * (g ^ (i16 >> 1)), l1 = i16 * 128 + 16 * ((4 + g) ^ (i16 >> 1));
    auto compute = [&](const char* s) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* p = s + (h ? l1 : l0);
            intx4 wf[TN], xf[TM];
#pragma unroll
            for (int j = 0; j < TM; ++j)
                xf[j] = *reinterpret_cast<const intx4*>(p + (BN + 16 * (TM * wm + j)) * 128);
#pragma unroll
            for (int i = 0; i < TN; ++i)
                wf[i] = *reinterpret_cast<const intx4*>(p + 16 * (TN * wn + i) * 128);
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = mfma8(wf[i], xf[j], acc[i][j]);
        }
    };
    load(s0, 0);
    for (int kb = 0; kb < KB; kb += 2) {
        stage_step();
        load(s1, kb + 1);
        compute(s0);
        stage_step();
        load(s0, kb + 2);
        if (kb + 1 < KB) compute(s1);
    }
    const bool vec = vec_out<TO>(a);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int m = m0 + 16 * (TM * wm + j) + i16;
        const float sm = m < a.M ? a.sx[m] : 0.f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
            put4<TO, BETA>(a, m, n0 + 16 * (TN * wn + i) + 4 * g, acc[i][j], sm, vec);
    }
}

// ---------------------------------------------------------------- plan
template <int MB, int NB, typename TO>
void rows_launch(const I8Args& a, hipStream_t st) {
    const unsigned n = (unsigned)ssm::cdiv(a.N, 16 * NB);
    if (a.beta != 0.f) i8_rows_kernel<MB, NB, TO, true><<<n, 256, 0, st>>>(a);
    else i8_rows_kernel<MB, NB, TO, false><<<n, 256, 0, st>>>(a);
}

template <int WN, int WM, int TN, int TM, typename TO>
void gemm_launch(I8Args a, hipStream_t st) {
    a.nt = (int)ssm::cdiv(a.N, 16 * TN * WN);
    a.mt = (int)ssm::cdiv(a.M, 16 * TM * WM);
    a.gn = std::min(a.nt, 8);
    const unsigned n = (unsigned)(a.nt * a.mt);
    if (a.beta != 0.f) i8_gemm_kernel<WN, WM, TN, TM, TO, true><<<n, 64 * WN * WM, 0, st>>>(a);
    else i8_gemm_kernel<WN, WM, TN, TM, TO, false><<<n, 64 * WN * WM, 0, st>>>(a);
}

template <typename TO>
ssm_status product(const I8Args& a, hipStream_t st) {
    if (a.M <= 16) rows_launch<1, 1, TO>(a, st);
    else if (a.M <= 32) rows_launch<2, 1, TO>(a, st);
    else if (a.M <= kRowsMax) rows_launch<4, 2, TO>(a, st);
    else if (ssm::cdiv(a.N, 256) * ssm::cdiv(a.M, 256) >= 256) gemm_launch<4, 2, 4, 8, TO>(a, st);
    else gemm_launch<2, 2, 4, 4, TO>(a, st);
    return ssm::check_launch("ssm_linear_i8");
}

bool direct(const void* p, long ld, int K, bool x) {
    // x's bytes past K must be zeros (W's then do not matter)
    return ((uintptr_t)p & 15) == 0 && ld % 16 == 0 && K % (x ? kPad : 4) == 0;
}

// Workspace: x's rows as integers (Kp bytes each) with their scales, then W's where they have to
// be laid out.
struct Layout { size_t x, sx, w, all; long Kp; };
Layout layout(int M, int N, int K, bool x, bool scales, bool w) {
    Layout l{};
    l.Kp = up(K, kPad);
    size_t o = 0;
    l.x = o;
    if (x) o += (size_t)M * l.Kp;
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
    SSM_REQUIRE(ldw < (1L << 22) && ldx < (1L << 22), "%s: row stride too large", who);
    return SSM_OK;
}

ssm_status launch_product(I8Args a, int out_dtype, const Layout& l, bool lay_w, char* ws,
                          hipStream_t st) {
    if (lay_w) {
        signed char* o = (signed char*)ws + l.w;
        pad_rows_kernel<<<a.N, 256, 0, st>>>(a.W, a.ldw, a.K, o, (int)l.Kp);
        if (ssm_status e = ssm::check_launch("ssm_linear_i8 (weight rows)")) return e;
        a.W = o;
        a.ldw = l.Kp;
    }
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
    return quantize(dtype, x, ldx, (signed char*)q, ldq, scale, M, K, K, (hipStream_t)stream);
}

extern "C" size_t ssm_linear_i8_workspace(const int8_t* x, long ldx, const int8_t* W, long ldw, int M,
                                          int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return layout(M, N, K, !direct(x, ldx, K, true), false, !direct(W, ldw, K, false)).all;
}

extern "C" ssm_status ssm_linear_i8(const int8_t* x, long ldx, const float* sx, const int8_t* W,
                                    long ldw, const float* sw, const float* bias, int out_dtype,
                                    void* y, long ldy, int M, int N, int K, float beta,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    if (ssm_status e = check_product("ssm_linear_i8", x, ldx, W, ldw, sw, out_dtype, y, ldy, M, N, K))
        return e;
    if (M == 0) return SSM_OK;
    SSM_REQUIRE(sx, "ssm_linear_i8: null input");
    const bool lay_x = !direct(x, ldx, K, true), lay_w = !direct(W, ldw, K, false);
    const Layout l = layout(M, N, K, lay_x, false, lay_w);
    SSM_REQUIRE(l.all == 0 || (workspace && workspace_bytes >= l.all && ((uintptr_t)workspace & 15) == 0),
                "ssm_linear_i8: 16-byte aligned workspace of %zu bytes needed", l.all);
    I8Args a{(const signed char*)x, ldx, sx, nullptr, 0, (const signed char*)W, ldw, sw, bias, y, ldy,
             M, N, K, beta, 0, 0, 0};
    if (lay_x) {
        signed char* o = (signed char*)workspace + l.x;
        pad_rows_kernel<<<M, 256, 0, (hipStream_t)stream>>>(a.X, ldx, K, o, (int)l.Kp);
        if (ssm_status e = ssm::check_launch("ssm_linear_i8 (rows)")) return e;
        a.X = o;
        a.ldx = l.Kp;
    }
    return launch_product(a, out_dtype, l, lay_w, (char*)workspace, (hipStream_t)stream);
}

extern "C" size_t ssm_linear_q8_workspace(const int8_t* W, long ldw, int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return layout(M, N, K, true, true, !direct(W, ldw, K, false)).all;
}

extern "C" ssm_status ssm_linear_q8(int in_dtype, const void* x, long ldx, const int8_t* W, long ldw,
                                    const float* sw, const float* bias, int out_dtype, void* y,
                                    long ldy, int M, int N, int K, float beta, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(in_dtype == SSM_F32 || in_dtype == SSM_BF16, "ssm_linear_q8: bad dtype");
    if (ssm_status e = check_product("ssm_linear_q8", x, ldx, W, ldw, sw, out_dtype, y, ldy, M, N, K))
        return e;
    if (M == 0) return SSM_OK;
    const bool lay_w = !direct(W, ldw, K, false);
    const Layout l = layout(M, N, K, true, true, lay_w);
    SSM_REQUIRE(workspace && workspace_bytes >= l.all && ((uintptr_t)workspace & 15) == 0,
                "ssm_linear_q8: 16-byte aligned workspace of %zu bytes needed", l.all);
    signed char* q = (signed char*)workspace + l.x;
    float* sx = (float*)((char*)workspace + l.sx);
    if (ssm_status e = quantize(in_dtype, x, ldx, q, l.Kp, sx, M, K, (int)l.Kp, (hipStream_t)stream))
        return e;
    const I8Args a{q, l.Kp, sx, nullptr, 0, (const signed char*)W, ldw, sw, bias, y, ldy,
                   M, N, K, beta, 0, 0, 0};
    return launch_product(a, out_dtype, l, lay_w, (char*)workspace, (hipStream_t)stream);
}

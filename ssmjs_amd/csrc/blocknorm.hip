// The norms around a block, one pass over its rows: with y the block's output, x the residual stream and z its gate,
//   w = y / sqrt(mean y^2 + eps),  u = w post,  v = u silu(z),  x' = x + scale v,  n = x' / sqrt(mean x'^2 + eps) pre
// and the gradients of all of it: with g that of x' (its own and the one through n),
//   d = dn pre,  g = dx' + (d - n^ mean(d n^)) / rms(x')   (n^ = x' / rms(x'))
//   dx = g,  t = g scale,  dz = t u s (1 + z (1 - s)),  s = sigmoid(z),  c = t silu(z) post
//   dy = (c - w mean(c w)) / rms(y);  dscale = sum g v,  dpre = sum dn n^,  dpost = sum t silu(z) w  over the rows.
// Sums and everything between the loads and the stores are in fp32; x' enters n before its own rounding.
//
// Memory bound. A row lies in the registers of one wave, or of a few where it is long: each element is read once and
// written once (gradients of rows above 8192 elements read some again), and the sums over a row are lane exchanges. Rows
// need no alignment: vector loads and stores of eight elements are made at the elements' own alignment, which the hardware
// splits where it must. Measured: 16384 x 2048 bf16 63 us (5.3 TB/s) and its gradients 137 (3.9 TB/s), 8192 x 768 fp32 without
// gate 24 us (4.2 TB/s) and its gradients 40 (3.7 TB/s) and 5 for the columns' sums; 64 x 2048 3.4 us, two trips to memory
// and a launch.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int kMaxD = 16384;

// Eight elements of a row, as they lie in memory; `left` of them exist. WHOLE: at least eight, or none, which keeps the
// code short.
template <typename T, bool WHOLE> struct Eight;
template <bool WHOLE> struct Eight<float, WHOLE> {
    float v[8];
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    __device__ __forceinline__ void load(const float* p, int left) {
        if (left >= 8) {
            const f4 a = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p)),
                     b = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p) + 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = !WHOLE && j < left ? p[j] : 0.f;
        }
    }
    __device__ __forceinline__ float operator[](int j) const { return v[j]; }
    static __device__ __forceinline__ void store(const float (&f)[8], float* p, int left) {
        if (left >= 8) {
            reinterpret_cast<f4*>(p)[0] = f4{f[0], f[1], f[2], f[3]};
            reinterpret_cast<f4*>(p)[1] = f4{f[4], f[5], f[6], f[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!WHOLE && j < left) p[j] = f[j];
        }
    }
};
template <bool WHOLE> struct Eight<__bf16, WHOLE> {
    typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    unsigned v[4];
    __device__ __forceinline__ void load(const __bf16* p, int left) {
        if (left >= 8) {
            const u4 a = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j];
        } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = (!WHOLE && 2 * j < left ? h[2 * j] : 0u) | (!WHOLE && 2 * j + 1 < left ? (unsigned)h[2 * j + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ float operator[](int j) const {
        return __builtin_bit_cast(float, j % 2 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
    }
    static __device__ __forceinline__ void store(const float (&f)[8], __bf16* p, int left) {
        if (left >= 8) {
            b8 b;
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = (__bf16)f[j];
            *reinterpret_cast<u4*>(p) = __builtin_bit_cast(u4, b);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!WHOLE && j < left) p[j] = (__bf16)f[j];
        }
    }
};

// Eight weights (none: ones).
template <bool WHOLE>
__device__ __forceinline__ void weights(const float* w, int e, int left, float (&f)[8]) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    if (!w) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 1.f;
    } else if (left >= 8) {
        const f4 a = *reinterpret_cast<const f4*>(w + e), b = *reinterpret_cast<const f4*>(w + e + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = a[j], f[4 + j] = b[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = !WHOLE && j < left ? w[e + j] : 0.f;
    }
}

// Keeps loads through `p` where they are: the backward pass needs its registers for rows, and the weights lie in
// the caches.
__device__ __forceinline__ const float* again(const float* p) {
    asm volatile("" : "+s"(p));
    return p;
}

struct NormArgs {
    const void* x; long ldx;
    const void* y; long ldy;
    const void* z; long ldz;      // (null: no gate)
    const float* post; const float* scale; const float* pre;
    void* x1; long ldx1;          // x', or dx
    void* n; long ldn;            // n, or dy
    const void* dx1; long lddx1;  // (null: zeros)
    const void* dn; long lddn;
    void* dz; long lddz;
    float* part;                  // the workgroups' column sums: dpost, dscale, dpre of D each
    int T, D;
    float eps;
};

// Sum over a wave: rotations within its rows of 16 lanes, then two exchanges between them.
template <int N>
__device__ __forceinline__ float rotated(float v) {   // by N lanes of 16 (row_ror)
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float s) {
    s += rotated<8>(s);
    s += rotated<4>(s);
    s += rotated<2>(s);
    s += rotated<1>(s);
    s += __shfl_xor(s, 16);
    return s + __shfl_xor(s, 32);
}

// Sum over the lanes of a row: one wave, or WPR waves (the workgroup's waves are W, its rows W / WPR) through `red`
// (two buffers in turn: one barrier a sum).
template <int WPR, int W>
__device__ __forceinline__ float row_sum(float s, float (&red)[2][W], int& turn) {
    s = wave_sum(s);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = s;
        __syncthreads();
        s = 0.f;
        const int first = (threadIdx.x >> 6) / WPR * WPR;
#pragma unroll
        for (int w = 0; w < WPR; ++w) s += red[turn][first + w];
        turn ^= 1;
    }
    return s;
}

template <typename T> __device__ __forceinline__ const T* row_of(const void* p, long ld, long t) {
    return static_cast<const T*>(p) + t * ld;
}
template <typename T> __device__ __forceinline__ T* row_of(void* p, long ld, long t) { return static_cast<T*>(p) + t * ld; }

// 512 NC WPR elements a row at most; four rows a workgroup where a row is one wave's.
template <typename T, int NC, int WPR, bool GATE, bool WHOLE>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void norm_kernel(NormArgs a) {
    __shared__ float red[2][WPR];
    int turn = 0;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long t = WPR == 1 ? (long)blockIdx.x * 4 + w : blockIdx.x;
    if (t >= a.T) return;
    const int e0 = ((WPR == 1 ? 0 : w * NC) * 64 + lane) * 8;   // chunk c begins at e0 + 512 c
    const T* px = row_of<T>(a.x, a.ldx, t) + e0;
    const T* py = row_of<T>(a.y, a.ldy, t) + e0;
    const T* pz = GATE ? row_of<T>(a.z, a.ldz, t) + e0 : nullptr;
    Eight<T, WHOLE> x[NC], y[NC], z[NC];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        y[c].load(py + 512 * c, a.D - e0 - 512 * c);
        x[c].load(px + 512 * c, a.D - e0 - 512 * c);
        if constexpr (GATE) z[c].load(pz + 512 * c, a.D - e0 - 512 * c);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(y[c][j], y[c][j], ss);
    // (the weights with the row where there is one piece of each: one trip to memory)
    float post[8], scale[8], pre[8];
    if constexpr (NC == 1) {
        weights<WHOLE>(a.post, e0, a.D - e0, post);
        weights<WHOLE>(a.scale, e0, a.D - e0, scale);
        weights<WHOLE>(a.pre, e0, a.D - e0, pre);
    }
    const float inv = 1.f / (float)a.D;
    const float ry = __builtin_amdgcn_rsqf(fmaf(row_sum<WPR, WPR>(ss, red, turn), inv, a.eps));
    float x1[NC][8];
    ss = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int e = e0 + 512 * c;
        if constexpr (NC > 1) {
            weights<WHOLE>(a.post, e, a.D - e, post);
            weights<WHOLE>(a.scale, e, a.D - e, scale);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float u = y[c][j] * ry * post[j];
            if constexpr (GATE) u *= ssm::silu_fast(z[c][j]);
            x1[c][j] = fmaf(scale[j], u, x[c][j]);
            ss = fmaf(x1[c][j], x1[c][j], ss);
        }
    }
    const float rx = __builtin_amdgcn_rsqf(fmaf(row_sum<WPR, WPR>(ss, red, turn), inv, a.eps));
    T* p1 = row_of<T>(a.x1, a.ldx1, t);
    T* pn = row_of<T>(a.n, a.ldn, t);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int e = e0 + 512 * c;
        float n[8];
        if constexpr (NC > 1) weights<WHOLE>(a.pre, e, a.D - e, pre);
#pragma unroll
        for (int j = 0; j < 8; ++j) n[j] = x1[c][j] * rx * pre[j];
        Eight<T, WHOLE>::store(x1[c], p1 + e, a.D - e);
        Eight<T, WHOLE>::store(n, pn + e, a.D - e);
    }
}

// Keeps what follows, and what is formed from `e`, in its place: moved up over it, it would take registers.
__device__ __forceinline__ int apart(int e) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(e)::"memory");
    return e;
}

// W = 8 waves a workgroup and one workgroup a CU, which walks its rows and keeps the column sums of
// its lanes' elements: few partial sums, and they go to memory once.
template <typename T, int NC, int WPR, bool GATE, bool WHOLE>
__global__ __launch_bounds__(512, 2) void norm_backward(NormArgs a) {
    constexpr int W = 8, RPG = W / WPR;   // rows at a time
    // Rows above 8192 elements have more than fits in registers: two of the column sums stay in LDS, and of a row's operands
    // y alone is held, the others read again from the cache where they are wanted (1024 x 16384, all held by 16 waves / this:
    // bf16 311 / 177 us, fp32 325 / 260)
    constexpr bool kHeld = NC > 2;
    __shared__ float red[2][W];
    __shared__ alignas(16) float cols[kHeld ? 2 : RPG][512 * NC * WPR];
    int turn = 0;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int e0 = (w % WPR * NC * 64 + lane) * 8;
    const float inv = 1.f / (float)a.D;
    float spost[NC][8] = {}, sscale[NC][8] = {}, spre[NC][8] = {};
    if constexpr (kHeld)   // (its own lane's alone, up to the end)
        for (int c = 0; c < NC; ++c)
            for (int j = 0; j < 8; ++j) cols[0][e0 + 512 * c + j] = cols[1][e0 + 512 * c + j] = 0.f;
    const long step = (long)RPG * gridDim.x;
    // The next row is on its way where registers hold it too (fp32 rows of whole eights in one wave: 8192 x 768 42.6 / 41.4 us
    // without / with; in two waves 4096 x 2048 51.6 / 53.7, which spills).
    constexpr bool kAhead = NC == 1 || (!GATE && !kHeld && (sizeof(T) == 2 || (WPR == 1 && WHOLE)));
    Eight<T, WHOLE> x[NC], y[NC], z[NC], dn[NC], g0[NC], nx[NC], ny[NC], nz[NC], ndn[NC], ng0[NC];
    auto fetch_y = [&](int c, int e, long t, int left) { ny[c].load(row_of<T>(a.y, a.ldy, t) + e, left); };
    auto fetch_x = [&](int c, int e, long t, int left) { nx[c].load(row_of<T>(a.x, a.ldx, t) + e, left); };
    auto fetch_z = [&](int c, int e, long t, int left) {
        if constexpr (GATE) nz[c].load(row_of<T>(a.z, a.ldz, t) + e, left);
    };
    auto fetch_n = [&](int c, int e, long t, int left) { ndn[c].load(row_of<T>(a.dn, a.lddn, t) + e, left); };
    auto fetch_g = [&](int c, int e, long t, int left) {
        ng0[c].load(a.dx1 ? row_of<T>(a.dx1, a.lddx1, t) + e : nullptr, a.dx1 ? left : 0);
    };
    auto fetch = [&](long t) {   // the next row, on its way while this one is worked on
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int e = e0 + 512 * c, left = t < a.T ? a.D - e : 0;
            fetch_y(c, e, t, left);
            if constexpr (kHeld) continue;
            fetch_x(c, e, t, left);
            fetch_z(c, e, t, left);
            fetch_n(c, e, t, left);
            fetch_g(c, e, t, left);
        }
    };
    long t = (long)blockIdx.x * RPG + w / WPR;
    if constexpr (kAhead) fetch(t);
    for (long group = (long)blockIdx.x * RPG; group < a.T; group += step, t += step) {
        const bool on = t < a.T;   // (all waves take part in the sums)
        if constexpr (!kAhead) fetch(t);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            y[c] = ny[c];
            if constexpr (kHeld) continue;
            x[c] = nx[c], dn[c] = ndn[c], g0[c] = ng0[c];
            if constexpr (GATE) z[c] = nz[c];
        }
        if constexpr (kAhead) fetch(t + step);
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(y[c][j], y[c][j], ss);
        const float sy = row_sum<WPR, W>(ss, red, turn), ry = on ? __builtin_amdgcn_rsqf(fmaf(sy, inv, a.eps)) : 0.f;
        float x1[NC][8];
        float s1 = 0.f, sd = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int e = kHeld ? apart(e0 + 512 * c) : e0 + 512 * c;
            if constexpr (kHeld) {
                const int left = on ? a.D - e : 0;
                fetch_x(c, e, t, left), fetch_z(c, e, t, left), fetch_n(c, e, t, left);
                x[c] = nx[c], z[c] = nz[c], dn[c] = ndn[c];
            }
            float post[8], scale[8], pre[8];
            weights<WHOLE>(again(a.post), e, a.D - e, post);
            weights<WHOLE>(again(a.scale), e, a.D - e, scale);
            weights<WHOLE>(again(a.pre), e, a.D - e, pre);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float u = y[c][j] * ry * post[j];
                if constexpr (GATE) u *= ssm::silu_fast(z[c][j]);
                x1[c][j] = fmaf(scale[j], u, x[c][j]);
                s1 = fmaf(x1[c][j], x1[c][j], s1);
                sd = fmaf(dn[c][j] * pre[j], x1[c][j], sd);
            }
        }
        const float sx = row_sum<WPR, W>(s1, red, turn), rx = on ? __builtin_amdgcn_rsqf(fmaf(sx, inv, a.eps)) : 0.f;
        const float m1 = row_sum<WPR, W>(sd, red, turn) * rx * inv;   // mean of d n^
        float s2 = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int e = kHeld ? apart(e0 + 512 * c) : e0 + 512 * c;
            float post[8], scale[8], pre[8], dz[8];
            weights<WHOLE>(again(a.post), e, a.D - e, post);
            weights<WHOLE>(again(a.scale), e, a.D - e, scale);
            weights<WHOLE>(again(a.pre), e, a.D - e, pre);
            if constexpr (kHeld) {
                const int left = on ? a.D - e : 0;
                fetch_z(c, e, t, left), fetch_n(c, e, t, left), fetch_g(c, e, t, left);
                z[c] = nz[c], dn[c] = ndn[c], g0[c] = ng0[c];
#pragma unroll
                for (int j = 0; j < 8; ++j) spost[c][j] = cols[0][e + j], sscale[c][j] = cols[1][e + j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float nh = x1[c][j] * rx, g = fmaf(rx, dn[c][j] * pre[j] - nh * m1, g0[c][j]);
                const float wv = y[c][j] * ry, u = wv * post[j];
                spre[c][j] = fmaf(dn[c][j], nh, spre[c][j]);
                float t1 = g * scale[j], v = u;
                if constexpr (GATE) {
                    const float zj = z[c][j], s = __builtin_amdgcn_rcpf(1.f + __expf(-zj)), sl = zj * s;
                    dz[j] = t1 * u * (s * fmaf(zj, 1.f - s, 1.f));
                    v = u * sl;
                    t1 *= sl;
                }
                sscale[c][j] = fmaf(g, v, sscale[c][j]);
                spost[c][j] = fmaf(t1, wv, spost[c][j]);
                s2 = fmaf(t1 * post[j], wv, s2);
                x1[c][j] = g;
            }
            if constexpr (kHeld) {
#pragma unroll
                for (int j = 0; j < 8; ++j) cols[0][e + j] = spost[c][j], cols[1][e + j] = sscale[c][j];
            }
            const int left = on ? a.D - e : 0;
            Eight<T, WHOLE>::store(x1[c], row_of<T>(a.x1, a.ldx1, t) + e, left);
            if constexpr (GATE) Eight<T, WHOLE>::store(dz, row_of<T>(a.dz, a.lddz, t) + e, left);
        }
        const float m2 = row_sum<WPR, W>(s2, red, turn) * inv;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int e = kHeld ? apart(e0 + 512 * c) : e0 + 512 * c;
            if constexpr (kHeld) {
                fetch_z(c, e, t, on ? a.D - e : 0);
                z[c] = nz[c];
            }
            float post[8], scale[8], dy[8];
            weights<WHOLE>(again(a.post), e, a.D - e, post);
            weights<WHOLE>(again(a.scale), e, a.D - e, scale);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float t1 = x1[c][j] * scale[j];
                if constexpr (GATE) t1 *= ssm::silu_fast(z[c][j]);
                dy[j] = ry * (t1 * post[j] - y[c][j] * ry * m2);
            }
            Eight<T, WHOLE>::store(dy, row_of<T>(a.n, a.ldn, t) + e, on ? a.D - e : 0);
        }
    }
    // the workgroup's column sums
    float* part = a.part + (long)blockIdx.x * 3 * a.D;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        float (&s)[NC][8] = k == 0 ? spost : k == 1 ? sscale : spre;
        const bool there = kHeld && k < 2;
        if (!there) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) cols[w / WPR][e0 + 512 * c + j] = s[c][j];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
            float t = cols[kHeld ? k % 2 : 0][e];
#pragma unroll
            for (int r = 1; r < RPG; ++r) t += cols[r][e];
            part[(long)k * a.D + e] = t;
        }
    }
}

// Column sums of n rows of 3 D partial sums, in one order: dpost, dscale, dpre (null: not wanted).
__global__ __launch_bounds__(1024) void norm_columns(const float* __restrict__ part, int n, int D, float* dpost,
                                                     float* dscale, float* dpre) {
    __shared__ float sum[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, k = blockIdx.y, e = blockIdx.x * 64 + lane;
    float* out = k == 0 ? dpost : k == 1 ? dscale : dpre;
    if (!out) return;
    float s = 0.f;
    if (e < D)
#pragma unroll 4
        for (int r = w; r < n; r += 16) s += part[((long)r * 3 + k) * D + e];
    sum[w][lane] = s;
    __syncthreads();
    if (w || e >= D) return;
#pragma unroll
    for (int r = 8; r > 0; r /= 2)
        for (int q = 0; q < r; ++q) sum[q][lane] += sum[q + r][lane];
    out[e] = sum[0][lane];
}

template <typename T, int NC, int WPR>
void go_forward(const NormArgs& a, hipStream_t st) {
    const unsigned n = (unsigned)(WPR == 1 ? ssm::cdiv(a.T, 4) : a.T), threads = WPR == 1 ? 256 : 64 * WPR;
    if (a.D % 8) a.z ? norm_kernel<T, NC, WPR, true, false><<<n, threads, 0, st>>>(a) : norm_kernel<T, NC, WPR, false, false><<<n, threads, 0, st>>>(a);
    else a.z ? norm_kernel<T, NC, WPR, true, true><<<n, threads, 0, st>>>(a) : norm_kernel<T, NC, WPR, false, true><<<n, threads, 0, st>>>(a);
}
template <typename T>
void forward_of(const NormArgs& a, hipStream_t st) {
    // eight elements a lane, as many waves as that takes (us, against four times the elements and a quarter of the
    // waves: 64 x 2048 bf16 3.4 / 5.8, 16384 x 2048 62.9 / 64.6, 4096 x 8192 63.8 / 69.0)
    if (a.D <= 512) go_forward<T, 1, 1>(a, st);
    else if (a.D <= 1024) go_forward<T, 1, 2>(a, st);
    else if (a.D <= 2048) go_forward<T, 1, 4>(a, st);
    else if (a.D <= 4096) go_forward<T, 1, 8>(a, st);
    else if (a.D <= 8192) go_forward<T, 1, 16>(a, st);
    else go_forward<T, 2, 16>(a, st);
}

// Workgroups of the backward pass: one a CU.
int rows_at_a_time(int D) { return D <= 1024 ? 8 : D <= 2048 ? 4 : D <= 4096 ? 2 : 1; }
int groups_back(int T, int D) { return (int)std::min(ssm::cdiv(T, rows_at_a_time(D)), 256L); }

template <typename T, int NC, int WPR>
void go_backward(const NormArgs& a, hipStream_t st) {
    const unsigned n = (unsigned)groups_back(a.T, a.D), threads = 512;
    if (a.D % 8) a.z ? norm_backward<T, NC, WPR, true, false><<<n, threads, 0, st>>>(a) : norm_backward<T, NC, WPR, false, false><<<n, threads, 0, st>>>(a);
    else a.z ? norm_backward<T, NC, WPR, true, true><<<n, threads, 0, st>>>(a) : norm_backward<T, NC, WPR, false, true><<<n, threads, 0, st>>>(a);
}
template <typename T>
void backward_of(const NormArgs& a, hipStream_t st) {
    if (a.D <= 512) go_backward<T, 1, 1>(a, st);
    else if (a.D <= 1024) go_backward<T, 2, 1>(a, st);
    else if (a.D <= 2048) go_backward<T, 2, 2>(a, st);
    else if (a.D <= 4096) go_backward<T, 2, 4>(a, st);
    else if (a.D <= 8192) go_backward<T, 2, 8>(a, st);
    else go_backward<T, 4, 8>(a, st);
}

}  // namespace

extern "C" ssm_status ssm_block_norm(int dtype, const void* x, long ldx, const void* y, long ldy, const void* z,
                                     long ldz, const float* post, const float* scale, const float* pre, float eps,
                                     void* x1, long ldx1, void* n, long ldn, int T, int D, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_block_norm: bad dtype");
    SSM_REQUIRE(T >= 0 && D > 0, "ssm_block_norm: bad shape");
    SSM_REQUIRE(eps >= 0.f, "ssm_block_norm: eps below 0");
    if (D > kMaxD) return ssm::fail(SSM_ERR_UNSUPPORTED, "ssm_block_norm: rows of %d elements, at most %d", D, kMaxD);
    if (T == 0) return SSM_OK;
    SSM_REQUIRE(x && y && x1 && n, "ssm_block_norm: null input");
    if (T == 1) ldx = ldy = ldz = ldx1 = ldn = D;
    SSM_REQUIRE(ldx >= D && ldy >= D && (!z || ldz >= D) && ldx1 >= D && ldn >= D, "ssm_block_norm: row stride below row width");
    SSM_REQUIRE(T <= ssm::kMaxGroups / 4, "ssm_block_norm: too many rows");
    const long es = dtype == SSM_F32 ? 4 : 2;
    auto op = [&](const void* p, long ld) { return ssm::Rows{p, ld * es, D * es, T}; };
    const ssm::Rows rx = op(x, ldx), ry = op(y, ldy), rz = op(z, ldz), o1 = op(x1, ldx1), on = op(n, ldn),
                    w0 = ssm::block(post, 4L * D), w1 = ssm::block(scale, 4L * D), w2 = ssm::block(pre, 4L * D);
    // a row is read before it is written: x' may be x, n may be y
    SSM_REQUIRE(!ssm::meets(o1, ry, rz, on, w0, w1, w2) && !ssm::meets(on, rx, rz, w0, w1, w2) &&
                    ((x1 == x && ldx1 == ldx) || !ssm::meet(o1, rx)) && ((n == y && ldn == ldy) || !ssm::meet(on, ry)),
                "ssm_block_norm: an output overlaps an operand that it is not");
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy; a.z = z; a.ldz = ldz; a.post = post; a.scale = scale; a.pre = pre;
    a.x1 = x1; a.ldx1 = ldx1; a.n = n; a.ldn = ldn; a.T = T; a.D = D; a.eps = eps;
    if (dtype == SSM_F32) forward_of<float>(a, (hipStream_t)stream);
    else forward_of<__bf16>(a, (hipStream_t)stream);
    return ssm::check_launch("ssm_block_norm");
}

extern "C" size_t ssm_block_norm_backward_workspace(int T, int D) {
    return T > 0 && D > 0 ? (size_t)groups_back(T, D) * 3 * D * sizeof(float) : 0;
}

extern "C" ssm_status ssm_block_norm_backward(int dtype, const void* dx1, long lddx1, const void* dn, long lddn,
                                              const void* x, long ldx, const void* y, long ldy, const void* z, long ldz,
                                              const float* post, const float* scale, const float* pre, float eps, void* dx,
                                              long lddx, void* dy, long lddy, void* dz, long lddz, float* dpost,
                                              float* dscale, float* dpre, int T, int D, void* workspace,
                                              size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_block_norm_backward: bad dtype");
    SSM_REQUIRE(T > 0 && D > 0, "ssm_block_norm_backward: bad shape");
    SSM_REQUIRE(eps >= 0.f, "ssm_block_norm_backward: eps below 0");
    if (D > kMaxD)
        return ssm::fail(SSM_ERR_UNSUPPORTED, "ssm_block_norm_backward: rows of %d elements, at most %d", D, kMaxD);
    SSM_REQUIRE(dn && x && y && dx && dy && (!z || dz), "ssm_block_norm_backward: null input");
    if (!z) dz = nullptr;
    if (T == 1) lddx1 = lddn = ldx = ldy = ldz = lddx = lddy = lddz = D;
    SSM_REQUIRE((!dx1 || lddx1 >= D) && lddn >= D && ldx >= D && ldy >= D && (!z || (ldz >= D && lddz >= D)) &&
                    lddx >= D && lddy >= D, "ssm_block_norm_backward: row stride below row width");
    SSM_REQUIRE(T <= ssm::kMaxGroups / 4, "ssm_block_norm_backward: too many rows");
    const size_t need = ssm_block_norm_backward_workspace(T, D);
    SSM_REQUIRE(workspace && workspace_bytes >= need, "ssm_block_norm_backward: needs a workspace of %zu bytes", need);
    SSM_REQUIRE(((uintptr_t)workspace & 15) == 0, "ssm_block_norm_backward: workspace must be 16-byte aligned");
    const long es = dtype == SSM_F32 ? 4 : 2;
    auto op = [&](const void* p, long ld) { return ssm::Rows{p, ld * es, D * es, T}; };
    const ssm::Rows g1 = op(dx1, lddx1), gn = op(dn, lddn), rx = op(x, ldx), ry = op(y, ldy), rz = op(z, ldz),
                    ox = op(dx, lddx), oy = op(dy, lddy), oz = op(dz, lddz), w0 = ssm::block(post, 4L * D),
                    w1 = ssm::block(scale, 4L * D), w2 = ssm::block(pre, 4L * D), s0 = ssm::block(dpost, 4L * D),
                    s1 = ssm::block(dscale, 4L * D), s2 = ssm::block(dpre, 4L * D), ws = ssm::block(workspace, need);
    auto clear = [&](const ssm::Rows& o) { return !ssm::meets(o, gn, rx, ry, rz, w0, w1, w2); };
    // a row's gradient dx' is read before dx is written: they may be one
    SSM_REQUIRE(clear(ox) && clear(oy) && clear(oz) && clear(s0) && clear(s1) && clear(s2) && clear(ws) &&
                    ((dx == dx1 && lddx == lddx1) || !ssm::meet(ox, g1)) && !ssm::meets(g1, oy, oz, s0, s1, s2, ws) &&
                    !ssm::meets(ox, oy, oz, s0, s1, s2, ws) && !ssm::meets(oy, oz, s0, s1, s2, ws) &&
                    !ssm::meets(oz, s0, s1, s2, ws) && !ssm::meets(s0, s1, s2, ws) && !ssm::meets(s1, s2, ws) &&
                    !ssm::meet(s2, ws),
                "ssm_block_norm_backward: an output or the workspace overlaps an operand that it is not");
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy; a.z = z; a.ldz = ldz; a.post = post; a.scale = scale; a.pre = pre;
    a.dx1 = dx1; a.lddx1 = lddx1; a.dn = dn; a.lddn = lddn;
    a.x1 = dx; a.ldx1 = lddx; a.n = dy; a.ldn = lddy; a.dz = dz; a.lddz = lddz;
    a.part = static_cast<float*>(workspace); a.T = T; a.D = D; a.eps = eps;
    if (dtype == SSM_F32) backward_of<float>(a, (hipStream_t)stream);
    else backward_of<__bf16>(a, (hipStream_t)stream);
    if (dpost || dscale || dpre)
        norm_columns<<<dim3((unsigned)ssm::cdiv(D, 64), 3), 1024, 0, (hipStream_t)stream>>>(a.part, groups_back(T, D), D,
                                                                                          dpost, dscale, dpre);
    return ssm::check_launch("ssm_block_norm_backward");
}

// Gated linear recurrence (De et al. 2024, equations 1-4): per channel d and step t
//   z_t = c softplus(lam_d) sigmoid(r_t),  a_t = e^{-z_t},  b_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t
//   h_t = a_t h_{t-1} + b_t,  y_t = h_t
// over whole prompts, its gradients, and one token of it.
//
// The recurrence is associative: a run of steps maps its entering state h to A h + H with A the product
// of its decays and H its result from a zero state. A workgroup of W waves walks one sequence's 64
// channels in blocks of kBlock steps: a lane holds 16 (step, channel) elements of consecutive steps,
// forms their a and b once, in registers, and its run's (A, H); runs are composed over the lanes of a
// wave (lane exchanges) and over the waves (LDS, one barrier a block), and each lane then walks its steps
// from its true entering state, as the formula says.
//
// 1 - a^2 from a rounded a would lose its digits where a is near 1 (0.999 and more in use): with
// q = 1 - e^{-z} by its series below z = 1/4, a = 1 - q and 1 - a^2 = q (1 + a).
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int kCh = 64;          // channels of a workgroup
constexpr int kKept = 64;        // steps between the states that a backward pass needs
constexpr float kSeries = 0.25f; // z up to which 1 - e^-z is summed as a series
constexpr float kTiny = 1.17549435e-38f;

// ---------------------------------------------------------------- elements
template <typename T, int VEC> struct Raw;
template <> struct Raw<float, 4> {
    float4 v;
    __device__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = ssm::bload16<float4>(r, o); }
    __device__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
};
template <> struct Raw<float, 1> {
    float v;
    __device__ void load(const float* p) { v = *p; }
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = ssm::bload4(r, o); }
    __device__ void get(float (&f)[1]) const { f[0] = v; }
};
template <> struct Raw<__bf16, 4> {
    uint2 v;
    __device__ void load(const __bf16* p) { v = *reinterpret_cast<const uint2*>(p); }
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) {
        v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, o, 0, 0));
    }
    __device__ void get(float (&f)[4]) const {
        f[0] = __builtin_bit_cast(float, v.x << 16);
        f[1] = __builtin_bit_cast(float, v.x & 0xffff0000u);
        f[2] = __builtin_bit_cast(float, v.y << 16);
        f[3] = __builtin_bit_cast(float, v.y & 0xffff0000u);
    }
};
template <> struct Raw<__bf16, 1> {
    unsigned short v;
    __device__ void load(const __bf16* p) { v = *reinterpret_cast<const unsigned short*>(p); }
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = __builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0); }
    __device__ void get(float (&f)[1]) const { f[0] = __builtin_bit_cast(float, (unsigned)v << 16); }
};

__device__ __forceinline__ void put(const float (&f)[4], __amdgpu_buffer_rsrc_t r, unsigned o, float) {
    ssm::bstore16(make_float4(f[0], f[1], f[2], f[3]), r, o);
}
__device__ __forceinline__ void put(const float (&f)[1], __amdgpu_buffer_rsrc_t r, unsigned o, float) {
    ssm::bstore4(f[0], r, o);
}
__device__ __forceinline__ void put(const float (&f)[4], __amdgpu_buffer_rsrc_t r, unsigned o, __bf16) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const bf16x4 b{(__bf16)f[0], (__bf16)f[1], (__bf16)f[2], (__bf16)f[3]};
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, b), r, o, 0, 0);
}
__device__ __forceinline__ void put(const float (&f)[1], __amdgpu_buffer_rsrc_t r, unsigned o, __bf16) {
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, (__bf16)f[0]), r, o, 0, 0);
}

// ---------------------------------------------------------------- gates
// e^-v; held to 2^126 where its product with 1 / (1 + e^-v) is wanted (a NaN stays one).
__device__ __forceinline__ float fall(float v) { return ssm::ex2(-ssm::kLog2e * v); }
__device__ __forceinline__ float fall_held(float v) {
    const float t = -ssm::kLog2e * v;
    return ssm::ex2(t > 126.f ? 126.f : t);
}
__device__ __forceinline__ float open(float e) { return __builtin_amdgcn_rcpf(1.f + e); }   // sigmoid of e = e^-v

// 1 - e^-z for z <= kSeries, to 2e-8 of its value: z (1 - z/2 (1 - z/3 (... (1 - z/7)))).
__device__ __forceinline__ float lost_small(float z) {
    float p = fmaf(z, -1.f / 7, 1.f);
    p = fmaf(z * p, -1.f / 6, 1.f);
    p = fmaf(z * p, -1.f / 5, 1.f);
    p = fmaf(z * p, -1.f / 4, 1.f);
    p = fmaf(z * p, -1.f / 3, 1.f);
    p = fmaf(z * p, -1.f / 2, 1.f);
    return z * p;
}

// a = e^-z and q = 1 - a of one element; `near` where no channel of the wave goes beyond the series.
__device__ __forceinline__ void decay(float z, bool near, float& a, float& q) {
    q = lost_small(z);
    a = 1.f - q;
    if (!near) {
        const float e = fall(z);
        const bool far = !(z <= kSeries);
        q = far ? 1.f - e : q;
        a = far ? e : a;
    }
}

// A run's result from entering state h. An infinite state stays infinite: its decay is positive, however
// far below fp32's range.
__device__ __forceinline__ float onto(float A, float H, float h) {
    return fmaf(__builtin_isinf(h) ? fmaxf(A, kTiny) : A, h, H);
}

struct RecArgs {
    const void* x; long ldx;
    const void* r; long ldr;
    const void* i; long ldi;
    const void* dy; long lddy;
    const float* lam;
    const int* lengths;
    void* y; long ldy;          // y, or dx
    void* dr; long lddr;
    void* di; long lddi;
    const float* h0; float* hT; // (backward: the gradients of hT and of h0)
    float* states;
    float2* seg;                // (A, H) of each segment but the last, and h0; h0 and (A, G) of each but the first
    float* sums;
    int B, L, D, span, nseg;    // span: steps of a segment
    int pad;                    // rows behind a sequence become zeros
    float c;
};

// A lane's place: VEC channels of 64 / LC rows of a wave, S consecutive steps a row; W waves.
template <typename T, int VEC, int W_>
struct Place {
    static constexpr int LC = kCh / VEC, R = 64 / LC, S = 16 / VEC, W = W_, TB = W * R * S;
    int lane, w, col, row, ch, cg, b, seg, n;
    bool live;
    float kd[VEC];   // c softplus(lam)
    bool near;
    __device__ Place(const RecArgs& a) {
        lane = threadIdx.x & 63;
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        col = lane % LC;
        row = lane / LC;
        const int groups = (a.D + kCh - 1) / kCh;
        cg = blockIdx.x % groups;
        const int rest = blockIdx.x / groups;
        b = rest % a.B;
        seg = rest / a.B;
        ch = cg * kCh + col * VEC;
        live = ch < a.D;
        n = a.L;
        if (a.lengths) n = min(max(a.lengths[b], 0), a.L);
    }
    __device__ void channels(const RecArgs& a) {
        float most = 0.f;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            kd[v] = live ? a.c * ssm::softplus(a.lam[ch + v]) : 0.f;
            most = kd[v] <= most ? most : kd[v];   // (NaN goes the general way)
        }
        near = __all(most <= kSeries);
    }
    // rows t0 .. t0 + rows - 1 of this group's channels
    template <typename P>
    __device__ __amdgpu_buffer_rsrc_t rows(P* p, long ld, long t0, int L, int D, int rows) const {
        const char* base = (const char*)p + (((long)b * L + t0) * ld + cg * kCh) * sizeof(T);
        const int wide = min(kCh, D - cg * kCh);
        return ssm::rsrc(base, rows > 0 ? (unsigned)(((long)(rows - 1) * ld + wide) * sizeof(T)) : 0u);
    }
    __device__ unsigned at(long ld, int step) const {   // (dead lanes: past every end)
        return live ? (unsigned)((step * ld + col * VEC) * sizeof(T)) : 0x80000000u;
    }
};

// Zeros for the rows of a segment that lie behind its sequence's end.
template <typename T, int VEC, int W>
__device__ void clear_rows(const Place<T, VEC, W>& p, const RecArgs& a, void* y, long ldy) {
    using P = Place<T, VEC, W>;
    const int s0 = p.seg * a.span, s1 = min(a.L, s0 + a.span), from = max(p.n, s0);
    const float none[VEC] = {};
    for (int t = from; t < s1; t += P::TB) {
        const auto ry = p.rows(y, ldy, t, a.L, a.D, min(P::TB, s1 - t));
        for (int s = 0; s < P::S; ++s) put(none, ry, p.at(ldy, (p.w * P::S + s) * P::R + p.row), T());
    }
}

// Keeps what is formed from `v` inside the loop: the offsets of a lane's steps, one addition each, would
// otherwise wait in registers for all of it.
__device__ __forceinline__ unsigned here(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// ---------------------------------------------------------------- a segment's (A, H)
// Without outputs no order binds the lanes: each walks a run of span / (R W) steps of its own, and runs
// are composed once, at the end. BACK: the adjoint e_{t-1} = a_t (dy_t + e_t), walked from the end.
template <typename T, int VEC, int W, bool BACK>
__global__ __launch_bounds__(64 * W) void rec_segment(RecArgs a) {
    using P = Place<T, VEC, W>;
    constexpr int S = P::S, R = P::R;
    P p(a);
    const int seg = BACK ? p.seg + 1 : p.seg;
    const int last = p.n > 0 ? (p.n - 1) / a.span : 0;
    const int ch = threadIdx.x;
    const bool mine = ch < kCh && p.cg * kCh + ch < a.D;
    // the entering state goes on from here: the one of the caller may be where the final one is written
    if (p.seg == 0 && mine) {
        const float h0 = a.h0 ? a.h0[(long)p.b * a.D + p.cg * kCh + ch] : 0.f;
        a.seg[((long)p.b * a.nseg + (BACK ? 0 : a.nseg - 1)) * a.D + p.cg * kCh + ch] = make_float2(h0, 0.f);
    }
    if (BACK ? seg > last : seg >= last) return;
    p.channels(a);
    const long t0 = (long)p.b * a.L + (long)seg * a.span;
    const int steps = min(a.span, p.n - seg * a.span);
    const int run = a.span / (R * W);   // a multiple of S
    const int first = (p.w * R + p.row) * run;
    const long ldx = BACK ? a.lddy : a.ldx;
    const T* px = static_cast<const T*>(BACK ? a.dy : a.x) + t0 * ldx + p.ch;
    const T* pr = static_cast<const T*>(a.r) + t0 * a.ldr + p.ch;
    const T* pi = static_cast<const T*>(a.i) + t0 * a.ldi + p.ch;
    float A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
    for (int k = 0; k < run; k += S) {
        const int at = first + (BACK ? run - S - k : k);
        Raw<T, VEC> qx[S] = {}, qr[S] = {}, qi[S] = {};
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (p.live && at + s < steps) {
                qr[s].load(pr + (at + s) * a.ldr);
                qx[s].load(px + (at + s) * ldx);
                if constexpr (!BACK) qi[s].load(pi + (at + s) * a.ldi);
            }
#pragma unroll
        for (int u = 0; u < S; ++u) {
            const int s = BACK ? S - 1 - u : u;
            float x[VEC], r[VEC], i[VEC];
            qx[s].get(x);
            qr[s].get(r);
            if constexpr (!BACK) qi[s].get(i);
            const bool on = at + s < steps;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float d, q;
                decay(p.kd[v] * open(fall(r[v])), p.near, d, q);
                if (BACK) {
                    H[v] = on ? d * (x[v] + H[v]) : H[v];
                } else {
                    const float bt = __builtin_amdgcn_sqrtf(fmaf(q, d, q)) * (open(fall(i[v])) * x[v]);
                    H[v] = on ? onto(d, bt, H[v]) : H[v];
                }
                A[v] = on ? A[v] * d : A[v];
            }
        }
    }
    __shared__ float sa[R * W][kCh], sh[R * W][kCh];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        sa[p.w * R + p.row][p.col * VEC + v] = A[v];
        sh[p.w * R + p.row][p.col * VEC + v] = H[v];
    }
    __syncthreads();
    if (mine) {
        float At = 1.f, Ht = 0.f;
        for (int u = 0; u < R * W; ++u) {
            const int k = BACK ? R * W - 1 - u : u;
            Ht = onto(sa[k][ch], sh[k][ch], Ht);
            At *= sa[k][ch];
        }
        a.seg[((long)p.b * a.nseg + seg) * a.D + p.cg * kCh + ch] = make_float2(At, Ht);
    }
}

// The value of a lane (modulo 64).
__device__ __forceinline__ float of_lane(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(lane * 4, __builtin_bit_cast(int, v)));
}

// Composition over the rows of a wave: (A, H) becomes the run of all rows up to this one, (Ae, He) that of
// the rows before it. BACK: of the rows from this one on, and after it.
template <int VEC, int LC, bool BACK>
__device__ __forceinline__ void compose(int lane, int row, float (&A)[VEC], float (&H)[VEC], float (&Ae)[VEC],
                                        float (&He)[VEC]) {
    constexpr int R = 64 / LC;
    const int left = BACK ? R - 1 - row : row;   // rows that come before in the walk
#pragma unroll
    for (int k = 1; k < R; k *= 2) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float A1 = of_lane(A[v], lane + (BACK ? k : -k) * LC), H1 = of_lane(H[v], lane + (BACK ? k : -k) * LC);
            if (left < k) A1 = 1.f, H1 = 0.f;
            H[v] = BACK ? fmaf(A[v], H1, H[v]) : onto(A[v], H[v], H1);
            A[v] *= A1;
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Ae[v] = 1.f;
        He[v] = 0.f;
        if constexpr (R > 1) {
            const float A1 = of_lane(A[v], lane + (BACK ? LC : -LC)), H1 = of_lane(H[v], lane + (BACK ? LC : -LC));
            Ae[v] = left ? A1 : 1.f;
            He[v] = left ? H1 : 0.f;
        }
    }
}

template <int VEC>
__device__ __forceinline__ bool any_nan(const float (&h)[VEC]) {
    bool no = false;
#pragma unroll
    for (int v = 0; v < VEC; ++v) no |= h[v] != h[v];
    return __any(no);
}

// ---------------------------------------------------------------- prompts
template <typename T, int VEC, int W>
__global__ __launch_bounds__(64 * W) void rec_kernel(RecArgs a) {
    using P = Place<T, VEC, W>;
    constexpr int S = P::S, R = P::R, LC = P::LC, TB = P::TB;
    __shared__ float aggA[2][W][kCh], aggH[2][W][kCh];
    P p(a);
    const int last = p.n > 0 ? (p.n - 1) / a.span : 0;
    if (a.pad) clear_rows(p, a, a.y, a.ldy);
    if (p.seg > last) return;
    p.channels(a);
    // the state entering a block, of channel `lane`
    const int chl = p.cg * kCh + p.lane;
    const bool has = chl < a.D;
    float st = 0.f;
    if (has && a.nseg > 1) st = a.seg[((long)p.b * a.nseg + a.nseg - 1) * a.D + chl].x;
    else if (has && a.h0) st = a.h0[(long)p.b * a.D + chl];
    for (int q = 0; q < p.seg; ++q)
        if (has) {
            const float2 e = a.seg[((long)p.b * a.nseg + q) * a.D + chl];
            st = onto(e.x, e.y, st);
        }
    const int s0 = p.seg * a.span, s1 = min(p.n, s0 + a.span);
    const int mine = (p.w * R + p.row) * S;   // this lane's first step of a block
    const unsigned ox = p.at(a.ldx, mine), orr = p.at(a.ldr, mine), oi = p.at(a.ldi, mine), oy = p.at(a.ldy, mine);
    const unsigned sx = (unsigned)(a.ldx * sizeof(T)), sr = (unsigned)(a.ldr * sizeof(T)),
                   si = (unsigned)(a.ldi * sizeof(T)), sy = (unsigned)(a.ldy * sizeof(T));
    Raw<T, VEC> qx[S], qr[S], qi[S];
    auto fetch = [&](int t0) {
        const int rows = min(TB, s1 - t0);   // (none past the end: zeros)
        const auto rx = p.rows(a.x, a.ldx, t0, a.L, a.D, rows), rr = p.rows(a.r, a.ldr, t0, a.L, a.D, rows),
                   ri = p.rows(a.i, a.ldi, t0, a.L, a.D, rows);
        unsigned vx = here(ox), vr = here(orr), vi = here(oi);
#pragma unroll
        for (int s = 0; s < S; ++s, vx += sx, vr += sr, vi += si) {
            qr[s].load(rr, vr);
            qi[s].load(ri, vi);
            qx[s].load(rx, vx);
        }
    };
    fetch(s0);
    int buf = 0;
    for (int t0 = s0; t0 < s1; t0 += TB, buf ^= 1) {
        float d[S][VEC], bt[S][VEC];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
            qx[s].get(x);
            qr[s].get(r);
            qi[s].get(i);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float q;
                decay(p.kd[v] * open(fall(r[v])), p.near, d[s][v], q);
                bt[s][v] = __builtin_amdgcn_sqrtf(fmaf(q, d[s][v], q)) * (open(fall(i[v])) * x[v]);
            }
            if ((s + 1) * VEC % 4 == 0) __builtin_amdgcn_sched_barrier(0);   // (four elements at a time)
        }
        if (t0 + TB > s1) {   // past the end the state stays
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (t0 + mine + s >= s1)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) d[s][v] = 1.f, bt[s][v] = 0.f;
        }
        fetch(min(t0 + TB, s1));
        float A[VEC], H[VEC], Ae[VEC], He[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            A[v] = d[0][v];
            H[v] = bt[0][v];
#pragma unroll
            for (int s = 1; s < S; ++s) {
                H[v] = fmaf(d[s][v], H[v], bt[s][v]);
                A[v] *= d[s][v];
            }
        }
        if (any_nan<VEC>(H)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                H[v] = bt[0][v];
#pragma unroll
                for (int s = 1; s < S; ++s) H[v] = onto(d[s][v], bt[s][v], H[v]);
            }
        }
        compose<VEC, LC, false>(p.lane, p.row, A, H, Ae, He);
        if (p.row == R - 1) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                aggA[buf][p.w][p.col * VEC + v] = A[v];
                aggH[buf][p.w][p.col * VEC + v] = H[v];
            }
        }
        __syncthreads();
        float enter = st, next = st;
#pragma unroll 4
        for (int w = 0; w < W; ++w) {
            if (w == p.w) enter = next;
            next = fmaf(aggA[buf][w][p.lane], next, aggH[buf][w][p.lane]);
        }
        if (__any(next != next)) {
            next = st;
            for (int w = 0; w < W; ++w) {
                if (w == p.w) enter = next;
                next = onto(aggA[buf][w][p.lane], aggH[buf][w][p.lane], next);
            }
        }
        st = next;
        float h[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = onto(Ae[v], He[v], VEC == 1 ? enter : of_lane(enter, p.col * VEC + v));
        if (a.states && (t0 + mine) % kKept == 0 && t0 + mine < s1 && p.live) {
            float* o = a.states + ((long)p.b * ((a.L + kKept - 1) / kKept) + (t0 + mine) / kKept) * a.D + p.ch;
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = h[v];
        }
        float y[S][VEC], g[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            g[v] = h[v];
#pragma unroll
            for (int s = 0; s < S; ++s) y[s][v] = g[v] = fmaf(d[s][v], g[v], bt[s][v]);
        }
        if (any_nan<VEC>(g)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                g[v] = h[v];
#pragma unroll
                for (int s = 0; s < S; ++s) y[s][v] = g[v] = onto(d[s][v], bt[s][v], g[v]);
            }
        }
        const auto ry = p.rows(a.y, a.ldy, t0, a.L, a.D, min(TB, s1 - t0));
        unsigned vy = here(oy);
#pragma unroll
        for (int s = 0; s < S; ++s, vy += sy) put(y[s], ry, vy, T());
    }
    if (a.hT && p.seg == last && p.w == 0 && has) a.hT[(long)p.b * a.D + chl] = st;
}

// ---------------------------------------------------------------- gradients
// With g_t the gradient of h_t, walked from the last step: g_t = dy_t + a_{t+1} g_{t+1}, and from
// log a = -z, d sqrt(1 - a^2) / d log a = -a^2 / sqrt(1 - a^2):
//   dx = g sqrt(1 - a^2) i,  di = g b (1 - i)   (i: the open gate)
//   q = z dL/dz = g (i x a^2 z / sqrt(1 - a^2) - a z h_{t-1}),  dr = q (1 - sigmoid r)
//   dlam = sum q sigmoid(lam) / softplus(lam),  dh0 = a_1 g_1
// z / sqrt(1 - a^2) goes to 0 with z. The states h_{t-1} are walked again from those that the forward
// pass kept; runs compose forwards for h and backwards for the adjoint with the same A.
template <typename T, int VEC, int W>
__global__ __launch_bounds__(64 * W) void rec_backward(RecArgs a) {
    using P = Place<T, VEC, W>;
    constexpr int S = P::S, R = P::R, LC = P::LC, TB = P::TB;
    constexpr int WK = kKept / (R * S);   // waves of a kept state
    static_assert(TB % kKept == 0 && WK >= 1 && W % WK == 0, "whole kept spans");
    __shared__ float aggA[2][W][kCh], aggH[2][W][kCh], aggG[2][W][kCh];
    P p(a);
    const int last = p.n > 0 ? (p.n - 1) / a.span : 0;
    const int kept = (a.L + kKept - 1) / kKept;
    if (a.pad) {
        clear_rows(p, a, a.y, a.ldy);
        clear_rows(p, a, a.dr, a.lddr);
        clear_rows(p, a, a.di, a.lddi);
    }
    float sum[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) sum[v] = 0.f;
    // the adjoint that leaves a block's first step, of channel `lane`
    const int chl = p.cg * kCh + p.lane;
    const bool has = chl < a.D;
    float e = 0.f;
    if (has && a.nseg > 1) e = a.seg[(long)p.b * a.nseg * a.D + chl].x;
    else if (has && a.h0) e = a.h0[(long)p.b * a.D + chl];
    const int s0 = p.seg * a.span, s1 = min(p.n, s0 + a.span);
    if (p.seg <= last) {
        p.channels(a);
        for (int q = last; q > p.seg; --q)
            if (has) {
                const float2 f = a.seg[((long)p.b * a.nseg + q) * a.D + chl];
                e = fmaf(f.x, e, f.y);
            }
    }
    const int mine = (p.w * R + p.row) * S;
    Raw<T, VEC> qx[S], qr[S], qi[S], qg[S];
    float ks = 0.f;   // the kept state of this wave's span, of channel `lane`
    auto fetch = [&](int t0) {
        const int rows = t0 < s0 ? 0 : min(TB, s1 - t0);
        const int at = max(t0, s0);
        const auto rx = p.rows(a.x, a.ldx, at, a.L, a.D, rows), rr = p.rows(a.r, a.ldr, at, a.L, a.D, rows),
                   ri = p.rows(a.i, a.ldi, at, a.L, a.D, rows), rg = p.rows(a.dy, a.lddy, at, a.L, a.D, rows);
        unsigned vx = here(p.at(a.ldx, mine)), vr = here(p.at(a.ldr, mine)), vi = here(p.at(a.ldi, mine)),
                 vg = here(p.at(a.lddy, mine));
#pragma unroll
        for (int s = 0; s < S; ++s) {
            qr[s].load(rr, vr);
            qi[s].load(ri, vi);
            qx[s].load(rx, vx);
            qg[s].load(rg, vg);
            vx += (unsigned)(a.ldx * sizeof(T));
            vr += (unsigned)(a.ldr * sizeof(T));
            vi += (unsigned)(a.ldi * sizeof(T));
            vg += (unsigned)(a.lddy * sizeof(T));
        }
        const int k = (at + p.w / WK * kKept) / kKept;
        ks = has && rows > 0 && at + p.w / WK * kKept < s1 ? a.states[((long)p.b * kept + k) * a.D + chl] : 0.f;
    };
    int buf = 0;
    const int t1 = s1 > s0 ? s0 + (s1 - s0 - 1) / TB * TB : s0 - TB;
    if (t1 >= s0) fetch(t1);
    for (int t0 = t1; t0 >= s0; t0 -= TB, buf ^= 1) {
        float d[S][VEC], bt[S][VEC], bi[S][VEC], bj[S][VEC], k1[S][VEC], k2[S][VEC], cr[S][VEC], gy[S][VEC];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
            qx[s].get(x);
            qr[s].get(r);
            qi[s].get(i);
            qg[s].get(gy[s]);
            const bool on = t0 + mine + s < s1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float er = fall_held(r[v]), ei = fall_held(i[v]);
                const float gr = open(er), gi = open(ei), z = p.kd[v] * gr;
                float q;
                decay(z, p.near, d[s][v], q);
                const float b2 = fmaf(q, d[s][v], q), inv = __builtin_amdgcn_rsqf(fmaxf(b2, kTiny)), be = b2 * inv;
                const float u = gi * x[v];
                bi[s][v] = be * gi;
                bt[s][v] = be * u;
                bj[s][v] = bt[s][v] * (ei * gi);
                k2[s][v] = d[s][v] * z;
                k1[s][v] = u * d[s][v] * d[s][v] * (z * inv);
                cr[s][v] = er * gr;
                if (!on) d[s][v] = 1.f, bt[s][v] = k1[s][v] = k2[s][v] = gy[s][v] = 0.f;
            }
            if ((s + 1) * VEC % 4 == 0) __builtin_amdgcn_sched_barrier(0);   // (four elements at a time)
        }
        float hl = ks;
        fetch(t0 - TB);
        float A[VEC], H[VEC], G[VEC], Ab[VEC], Ae[VEC], He[VEC], Ax[VEC], Gx[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            A[v] = d[0][v];
            H[v] = bt[0][v];
            G[v] = d[S - 1][v] * gy[S - 1][v];
#pragma unroll
            for (int s = 1; s < S; ++s) {
                H[v] = fmaf(d[s][v], H[v], bt[s][v]);
                A[v] *= d[s][v];
                G[v] = d[S - 1 - s][v] * (gy[S - 1 - s][v] + G[v]);
            }
            Ab[v] = A[v];
        }
        compose<VEC, LC, false>(p.lane, p.row, A, H, Ae, He);
        compose<VEC, LC, true>(p.lane, p.row, Ab, G, Ax, Gx);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (p.row == R - 1) {
                aggA[buf][p.w][p.col * VEC + v] = A[v];
                aggH[buf][p.w][p.col * VEC + v] = H[v];
            }
            if (p.row == 0) aggG[buf][p.w][p.col * VEC + v] = G[v];
        }
        __syncthreads();
        const int w0 = p.w / WK * WK;
        for (int w = w0; w < p.w; ++w) hl = fmaf(aggA[buf][w][p.lane], hl, aggH[buf][w][p.lane]);
        float el = e;
#pragma unroll 4
        for (int w = W - 1; w >= 0; --w) {
            if (w == p.w) el = e;
            e = fmaf(aggA[buf][w][p.lane], e, aggG[buf][w][p.lane]);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float hv = fmaf(Ae[v], VEC == 1 ? hl : of_lane(hl, p.col * VEC + v), He[v]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float before = hv;
                hv = fmaf(d[s][v], hv, bt[s][v]);
                bt[s][v] = before;
            }
            float ev = fmaf(Ax[v], VEC == 1 ? el : of_lane(el, p.col * VEC + v), Gx[v]);
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const float g = gy[s][v] + ev;
                ev = d[s][v] * g;
                const float q = g * fmaf(-k2[s][v], bt[s][v], k1[s][v]);
                sum[v] += q;
                bi[s][v] *= g;
                bj[s][v] *= g;
                cr[s][v] *= q;
            }
        }
        const int rows = min(TB, s1 - t0);
        const auto ox = p.rows(a.y, a.ldy, t0, a.L, a.D, rows), orr = p.rows(a.dr, a.lddr, t0, a.L, a.D, rows),
                   oi = p.rows(a.di, a.lddi, t0, a.L, a.D, rows);
        unsigned vx = here(p.at(a.ldy, mine)), vr = here(p.at(a.lddr, mine)), vi = here(p.at(a.lddi, mine));
#pragma unroll
        for (int s = 0; s < S; ++s) {
            put(bi[s], ox, vx, T());
            put(cr[s], orr, vr, T());
            put(bj[s], oi, vi, T());
            vx += (unsigned)(a.ldy * sizeof(T));
            vr += (unsigned)(a.lddr * sizeof(T));
            vi += (unsigned)(a.lddi * sizeof(T));
        }
    }
    if (a.hT && p.seg == 0 && p.w == 0 && has) a.hT[(long)p.b * a.D + chl] = e;
    // the workgroup's sums of q, in the order of rows and waves
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
#pragma unroll
        for (int k = LC; k < 64; k *= 2) sum[v] += __shfl_xor(sum[v], k);
        if (p.row == 0) aggA[0][p.w][p.col * VEC + v] = sum[v];
    }
    __syncthreads();
    const int ch = threadIdx.x;
    if (ch < kCh && p.cg * kCh + ch < a.D) {
        float t = 0.f;
        for (int w = 0; w < W; ++w) t += aggA[0][w][ch];
        a.sums[((long)p.b * a.nseg + p.seg) * a.D + p.cg * kCh + ch] = t;
    }
}

// dlam from the workgroups' sums, in double and in one order.
__global__ __launch_bounds__(256) void rec_dlam(const float* __restrict__ sums, const float* __restrict__ lam, int n,
                                                int D, float* __restrict__ dlam) {
    __shared__ double part[4][64];
    const int ch = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + ch;
    double t = 0.;
    if (d < D)
        for (int k = w; k < n; k += 4) t += (double)sums[(long)k * D + d];
    part[w][ch] = t;
    __syncthreads();
    if (w || d >= D) return;
    t = part[0][ch] + part[1][ch] + part[2][ch] + part[3][ch];
    const float l = lam[d];
    // sigmoid(lam) / softplus(lam), which is 1 - e^lam / 2 where e^lam is below fp32's half step
    const float f = l < -17.f ? 1.f : (1.f / (1.f + expf(-l))) / ssm::softplus(l);
    dlam[d] = (float)(t * (double)f);
}

// ---------------------------------------------------------------- one token
template <typename T, int VEC>
__global__ __launch_bounds__(256) void rec_step(RecArgs a) {
    const int per = a.D / VEC;
    const long k = (long)blockIdx.x * 256 + threadIdx.x;
    if (k >= (long)a.B * per) return;
    const int b = (int)(k / per), ch = (int)(k - (long)b * per) * VEC;
    const T* px = static_cast<const T*>(a.x) + b * a.ldx + ch;
    const T* pr = static_cast<const T*>(a.r) + b * a.ldr + ch;
    const T* pi = static_cast<const T*>(a.i) + b * a.ldi + ch;
    T* py = static_cast<T*>(a.y) + b * a.ldy + ch;
    float* ph = a.hT + (long)b * a.D + ch;
    typedef T Tv __attribute__((ext_vector_type(VEC)));
    typedef float Fv __attribute__((ext_vector_type(VEC)));
    const Tv x = *reinterpret_cast<const Tv*>(px), r = *reinterpret_cast<const Tv*>(pr),
             i = *reinterpret_cast<const Tv*>(pi);
    Fv h = *reinterpret_cast<const Fv*>(ph);
    const Fv lam = *reinterpret_cast<const Fv*>(a.lam + ch);
    Tv y;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float d, q;
        decay(a.c * ssm::softplus(lam[v]) * open(fall((float)r[v])), false, d, q);
        const float bt = __builtin_amdgcn_sqrtf(fmaf(q, d, q)) * (open(fall((float)i[v])) * (float)x[v]);
        h[v] = onto(d, bt, h[v]);
        y[v] = (T)h[v];
    }
    *reinterpret_cast<Fv*>(ph) = h;
    *reinterpret_cast<Tv*>(py) = y;
}

// ---------------------------------------------------------------- plans
constexpr int kWaves = 16, kWavesBack = 8;

struct Plan {
    long groups;
    int nseg, span;
};

// Segments where the sequences' channel groups alone leave compute units idle: enough for one workgroup a CU
// (two of the backward pass's smaller ones), each of at least four blocks.
Plan plan_of(int B, int L, int D, int block, long want) {
    Plan p{ssm::cdiv(D, kCh) * B, 1, std::max(block, (int)ssm::cdiv(L, block) * block)};
    const long blocks = ssm::cdiv(L, block);
    const long n = std::min(std::min(want / std::max(1L, p.groups), blocks / 4), 64L);
    if (n > 1) {
        const long per = ssm::cdiv(blocks, n);
        p.span = (int)(per * block);
        p.nseg = (int)ssm::cdiv(blocks, per);
    }
    return p;
}
Plan plan_forward(int B, int L, int D) { return plan_of(B, L, D, kWaves * 16, 256); }
Plan plan_backward(int B, int L, int D) { return plan_of(B, L, D, kWavesBack * 16, 256); }

size_t seg_bytes(const Plan& p, int B, int D) {
    return p.nseg > 1 ? ((size_t)B * p.nseg * D * sizeof(float2) + 15) / 16 * 16 : 0;
}
size_t sums_bytes(const Plan& p, int B, int D) { return (size_t)B * p.nseg * D * sizeof(float); }

bool shape_ok(int B, int L, int D) { return B > 0 && L > 0 && D > 0; }

template <typename T, int VEC>
void launch_forward(RecArgs a, const Plan& p, hipStream_t st) {
    if (p.nseg > 1) rec_segment<T, VEC, kWaves, false><<<p.groups * (p.nseg - 1), 64 * kWaves, 0, st>>>(a);
    rec_kernel<T, VEC, kWaves><<<p.groups * p.nseg, 64 * kWaves, 0, st>>>(a);
}
template <typename T, int VEC>
void launch_backward(RecArgs a, const Plan& p, float* dlam, hipStream_t st) {
    if (p.nseg > 1) rec_segment<T, VEC, kWavesBack, true><<<p.groups * (p.nseg - 1), 64 * kWavesBack, 0, st>>>(a);
    rec_backward<T, VEC, kWavesBack><<<p.groups * p.nseg, 64 * kWavesBack, 0, st>>>(a);
    rec_dlam<<<(unsigned)ssm::cdiv(a.D, 64), 256, 0, st>>>(a.sums, a.lam, a.B * a.nseg, a.D, dlam);
}

// Four channels a lane: D and all strides in fours, and rows aligned to that.
bool in_fours(int dtype, int D, std::initializer_list<std::pair<const void*, long>> ops) {
    const uintptr_t piece = dtype == SSM_F32 ? 15 : 7;
    bool ok = D % 4 == 0;
    for (const auto& o : ops) ok = ok && o.second % 4 == 0 && ((uintptr_t)o.first & piece) == 0;
    return ok;
}

constexpr long kMaxLd = 1L << 20;   // a block's rows within 2^31 bytes
}  // namespace

extern "C" size_t ssm_gated_recurrence_workspace(int B, int L, int D) {
    if (!shape_ok(B, L, D)) return 0;
    return seg_bytes(plan_forward(B, L, D), B, D);
}

extern "C" ssm_status ssm_gated_recurrence(int dtype, const void* x, long ldx, const void* r, long ldr, const void* i,
                                           long ldi, const float* lam, float c, const int* lengths, int pad, void* y, long ldy,
                                           int B, int L, int D, const float* h0, float* hT, float* states,
                                           void* workspace, size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_gated_recurrence: bad dtype");
    SSM_REQUIRE(B >= 0 && L >= 0 && D > 0, "ssm_gated_recurrence: bad shape");
    SSM_REQUIRE(c >= 0.f && c < __builtin_inff(), "ssm_gated_recurrence: c is a finite number, not below 0");
    if (B == 0) return SSM_OK;
    SSM_REQUIRE(lam && (L == 0 || (x && r && i && y)), "ssm_gated_recurrence: null input");
    const long rows = (long)B * L, es = dtype == SSM_F32 ? 4 : 2;
    if (rows <= 1) ldx = ldr = ldi = ldy = D;
    SSM_REQUIRE(ldx >= D && ldr >= D && ldi >= D && ldy >= D, "ssm_gated_recurrence: row stride below row width");
    SSM_REQUIRE(ldx < kMaxLd && ldr < kMaxLd && ldi < kMaxLd && ldy < kMaxLd && L <= ssm::kMaxSteps,
                "ssm_gated_recurrence: row strides of %ld elements, or sequences, too large", kMaxLd);
    const Plan p = plan_forward(B, std::max(L, 1), D);
    SSM_REQUIRE(p.groups * p.nseg <= (1L << 22) - 1, "ssm_gated_recurrence: too many sequences and channels");
    const size_t need = L > 0 ? seg_bytes(p, B, D) : 0;
    SSM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
                "ssm_gated_recurrence: needs a workspace of %zu bytes", need);
    SSM_REQUIRE(need == 0 || ((uintptr_t)workspace & 15) == 0, "ssm_gated_recurrence: workspace must be 16-byte aligned");
    auto op = [&](const void* q, long ld) { return ssm::Rows{q, ld * es, D * es, rows}; };
    const ssm::Rows rx = op(x, ldx), rr = op(r, ldr), ri = op(i, ldi), ry = op(y, ldy);
    const long kept = ssm::cdiv(L, kKept);
    const ssm::Rows gl = ssm::block(lam, 4L * D), ln = ssm::block(lengths, 4L * B), s0 = ssm::block(h0, 4L * B * D),
                    sT = ssm::block(hT, 4L * B * D), sk = ssm::block(states, 4L * B * kept * D),
                    ws = ssm::block(need ? workspace : nullptr, need);
    SSM_REQUIRE(!ssm::meets(ry, rx, rr, ri, gl, ln, s0, sT, sk, ws) &&
                    !ssm::meets(sT, rx, rr, ri, gl, ln, sk, ws) && (hT == h0 || !ssm::meet(sT, s0)) &&
                    !ssm::meets(sk, rx, rr, ri, gl, ln, s0, ws) && !ssm::meets(ws, rx, rr, ri, gl, ln, s0),
                "ssm_gated_recurrence: an output or the workspace overlaps another operand");
    RecArgs a{};
    a.x = x; a.ldx = ldx; a.r = r; a.ldr = ldr; a.i = i; a.ldi = ldi; a.y = y; a.ldy = ldy;
    a.lam = lam; a.lengths = lengths; a.pad = lengths && pad; a.h0 = h0; a.hT = hT; a.states = states; a.c = c;
    a.seg = static_cast<float2*>(workspace);
    a.B = B; a.L = L; a.D = D; a.span = p.span; a.nseg = p.nseg;
    const bool four = in_fours(dtype, D, {{x, ldx}, {r, ldr}, {i, ldi}, {y, ldy}});
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SSM_F32) four ? launch_forward<float, 4>(a, p, st) : launch_forward<float, 1>(a, p, st);
    else four ? launch_forward<__bf16, 4>(a, p, st) : launch_forward<__bf16, 1>(a, p, st);
    return ssm::check_launch("ssm_gated_recurrence");
}

extern "C" size_t ssm_gated_recurrence_backward_workspace(int B, int L, int D) {
    if (B <= 0 || L < 0 || D <= 0) return 0;
    const Plan p = plan_backward(B, std::max(L, 1), D);
    return seg_bytes(p, B, D) + sums_bytes(p, B, D);
}

extern "C" ssm_status ssm_gated_recurrence_backward(int dtype, const void* dy, long lddy, const void* x, long ldx,
                                                    const void* r, long ldr, const void* i, long ldi, const float* lam,
                                                    float c, const int* lengths, int pad, const float* states, const float* dhT,
                                                    void* dx, long lddx, void* dr, long lddr, void* di, long lddi,
                                                    float* dlam, float* dh0, int B, int L, int D, void* workspace,
                                                    size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_gated_recurrence_backward: bad dtype");
    SSM_REQUIRE(B > 0 && L >= 0 && D > 0, "ssm_gated_recurrence_backward: bad shape");
    SSM_REQUIRE(c >= 0.f && c < __builtin_inff(), "ssm_gated_recurrence_backward: c is a finite number, not below 0");
    SSM_REQUIRE(lam && dlam && (L == 0 || (dy && x && r && i && states && dx && dr && di)),
                "ssm_gated_recurrence_backward: null input");
    const long rows = (long)B * L, es = dtype == SSM_F32 ? 4 : 2;
    if (rows <= 1) lddy = ldx = ldr = ldi = lddx = lddr = lddi = D;
    for (long ld : {lddy, ldx, ldr, ldi, lddx, lddr, lddi}) {
        SSM_REQUIRE(ld >= D, "ssm_gated_recurrence_backward: row stride below row width");
        SSM_REQUIRE(ld < kMaxLd, "ssm_gated_recurrence_backward: row strides of %ld elements are too large", kMaxLd);
    }
    const Plan p = plan_backward(B, std::max(L, 1), D);
    SSM_REQUIRE(L <= ssm::kMaxSteps && p.groups * p.nseg <= (1L << 22) - 1,
                "ssm_gated_recurrence_backward: too many sequences, steps or channels");
    const size_t segs = seg_bytes(p, B, D), need = segs + sums_bytes(p, B, D);
    SSM_REQUIRE(workspace && workspace_bytes >= need, "ssm_gated_recurrence_backward: needs a workspace of %zu bytes", need);
    SSM_REQUIRE(((uintptr_t)workspace & 15) == 0, "ssm_gated_recurrence_backward: workspace must be 16-byte aligned");
    auto op = [&](const void* q, long ld) { return ssm::Rows{q, ld * es, D * es, rows}; };
    const ssm::Rows rg = op(dy, lddy), rx = op(x, ldx), rr = op(r, ldr), ri = op(i, ldi), ox = op(dx, lddx),
                    orr = op(dr, lddr), oi = op(di, lddi);
    const ssm::Rows gl = ssm::block(lam, 4L * D), ln = ssm::block(lengths, 4L * B),
                    sk = ssm::block(states, 4L * B * ssm::cdiv(L, kKept) * D), gT = ssm::block(dhT, 4L * B * D),
                    ol = ssm::block(dlam, 4L * D), o0 = ssm::block(dh0, 4L * B * D), ws = ssm::block(workspace, need);
    auto clear = [&](const ssm::Rows& o) { return !ssm::meets(o, rg, rx, rr, ri, gl, ln, sk, gT); };
    SSM_REQUIRE(clear(ox) && clear(orr) && clear(oi) && clear(ol) && clear(ws) &&
                    !ssm::meets(o0, rg, rx, rr, ri, gl, ln, sk) && (dh0 == dhT || !ssm::meet(o0, gT)) &&
                    !ssm::meets(ox, orr, oi, ol, o0, ws) && !ssm::meets(orr, oi, ol, o0, ws) &&
                    !ssm::meets(oi, ol, o0, ws) && !ssm::meets(ol, o0, ws) && !ssm::meet(o0, ws),
                "ssm_gated_recurrence_backward: an output or the workspace overlaps another operand");
    RecArgs a{};
    a.dy = dy; a.lddy = lddy; a.x = x; a.ldx = ldx; a.r = r; a.ldr = ldr; a.i = i; a.ldi = ldi;
    a.y = dx; a.ldy = lddx; a.dr = dr; a.lddr = lddr; a.di = di; a.lddi = lddi;
    a.lam = lam; a.lengths = lengths; a.pad = lengths && pad; a.h0 = dhT; a.hT = dh0; a.states = const_cast<float*>(states); a.c = c;
    a.seg = static_cast<float2*>(workspace);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + segs);
    a.B = B; a.L = L; a.D = D; a.span = p.span; a.nseg = p.nseg;
    const bool four = in_fours(dtype, D, {{dy, lddy}, {x, ldx}, {r, ldr}, {i, ldi}, {dx, lddx}, {dr, lddr}, {di, lddi}});
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SSM_F32) four ? launch_backward<float, 4>(a, p, dlam, st) : launch_backward<float, 1>(a, p, dlam, st);
    else four ? launch_backward<__bf16, 4>(a, p, dlam, st) : launch_backward<__bf16, 1>(a, p, dlam, st);
    return ssm::check_launch("ssm_gated_recurrence_backward");
}

extern "C" ssm_status ssm_gated_recurrence_step(int dtype, const void* x, long ldx, const void* r, long ldr,
                                                const void* i, long ldi, const float* lam, float c, void* y, long ldy,
                                                float* h, int B, int D, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_gated_recurrence_step: bad dtype");
    SSM_REQUIRE(B >= 0 && D > 0, "ssm_gated_recurrence_step: bad shape");
    SSM_REQUIRE(c >= 0.f && c < __builtin_inff(), "ssm_gated_recurrence_step: c is a finite number, not below 0");
    if (B == 0) return SSM_OK;
    SSM_REQUIRE(x && r && i && lam && y && h, "ssm_gated_recurrence_step: null input");
    if (B == 1) ldx = ldr = ldi = ldy = D;
    SSM_REQUIRE(ldx >= D && ldr >= D && ldi >= D && ldy >= D, "ssm_gated_recurrence_step: row stride below row width");
    SSM_REQUIRE((long)B * D <= 256 * ssm::kMaxGroups, "ssm_gated_recurrence_step: too many channels");
    const long es = dtype == SSM_F32 ? 4 : 2;
    auto op = [&](const void* q, long ld) { return ssm::Rows{q, ld * es, D * es, B}; };
    const ssm::Rows rx = op(x, ldx), rr = op(r, ldr), ri = op(i, ldi), ry = op(y, ldy), gl = ssm::block(lam, 4L * D),
                    sh = ssm::block(h, 4L * B * D);
    SSM_REQUIRE(!ssm::meets(ry, rx, rr, ri, gl, sh) && !ssm::meets(sh, rx, rr, ri, gl),
                "ssm_gated_recurrence_step: the output or the state overlaps another operand");
    RecArgs a{};
    a.x = x; a.ldx = ldx; a.r = r; a.ldr = ldr; a.i = i; a.ldi = ldi; a.y = y; a.ldy = ldy;
    a.lam = lam; a.hT = h; a.c = c; a.B = B; a.D = D;
    const bool four = in_fours(dtype, D, {{x, ldx}, {r, ldr}, {i, ldi}, {y, ldy}}) &&
                      (((uintptr_t)h | (uintptr_t)lam) & 15) == 0;
    const unsigned n = (unsigned)ssm::cdiv((long)B * (four ? D / 4 : D), 256);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SSM_F32) four ? rec_step<float, 4><<<n, 256, 0, st>>>(a) : rec_step<float, 1><<<n, 256, 0, st>>>(a);
    else four ? rec_step<__bf16, 4><<<n, 256, 0, st>>>(a) : rec_step<__bf16, 1><<<n, 256, 0, st>>>(a);
    return ssm::check_launch("ssm_gated_recurrence_step");
}

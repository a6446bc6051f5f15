// Gated linear recurrence (De et al. 2024, equations 1-4): per channel d and step t
//   z_t = c softplus(lam_d) sigmoid(r_t),  a_t = e^{-z_t},  b_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t
//   h_t = a_t h_{t-1} + b_t,  y_t = h_t
// over whole prompts, its gradients, and one token of it.
//
// The recurrence is associative: a run of steps maps its entering state h to A h + H with A the product
// of its decays and H its result from a zero state. A workgroup of W waves walks 64 channels of one sequence in
// blocks of TB = 16 W steps (32 channels in blocks of 32 W where that fills more of the chip): a lane holds 16 (step,
// channel) elements of consecutive steps, forms their a and b once, in registers, and its run's (A, H); runs are composed
// over the lanes of a wave (lane exchanges) and over the waves (LDS, one barrier a block), and each lane then walks its
// steps from its true entering state, as the formula says. The next block's inputs are on their way meanwhile.
//
// Where the sequences' channels are too few to fill the chip, sequences are cut into segments of whole blocks: a
// first pass forms the (A, H) of every block that others follow, and each segment starts from the composition of
// those before it. (One pass, with workgroups that wait for the results of those before them, read the inputs once
// and took longer, the waiting ones' looks at memory costing more than the second reading. us, two passes / one, when both
// were built: 1 x 32768 x 1024 bf16 100 / 122 to 134, 8 x 4096 x 2048 130 / 155 to 160, 4 x 2048 x 2048 49 / 52.)
//
// Bound by memory where the chip is full, 8 x 4096 x 2048 bf16 131 to 135 us, 4.1 TB/s (rows' pieces of 128 bytes read and
// written with nothing else done take 118, whole rows 106), 256 x 1000 x 1024 fp32 827 us, 5.1 TB/s; with one workgroup a CU as
// much by its instructions, about 60 an element. The gradients of 4 x 2048 x 2048 bf16 take 68 to 73 us (50 to 52 without the
// first pass and the last sum: 4.6 TB/s), of 256 x 1000 x 1024 fp32 1412, 5.2 TB/s. Small calls are launches: 64 tokens of 4096
// channels 4.2 to 4.5 us.
//
// 1 - a^2 from a rounded a would lose its digits where a is near 1 (0.999 and more in use): with
// q = 1 - e^{-z} by its series below z = 0.2, a = 1 - q and 1 - a^2 = q (1 + a).
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace {

constexpr int kCh = 64;          // channels of a workgroup
constexpr int kKept = 64;        // steps between the states that a backward pass needs
constexpr float kSeries = 0.2f;  // z up to which 1 - e^-z is summed as a series
constexpr float kTiny = 1.17549435e-38f;

// ---------------------------------------------------------------- elements
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
template <typename T, int VEC> struct Raw;
template <> struct Raw<float, 2> {
    float2 v;
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) {
        v = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(r, o, 0, 0));
    }
    __device__ void get(float (&f)[2]) const { f[0] = v.x; f[1] = v.y; }
};
template <> struct Raw<float, 1> {
    float v;
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = ssm::bload4(r, o); }
    __device__ void get(float (&f)[1]) const { f[0] = v; }
};
template <> struct Raw<__bf16, 2> {
    unsigned v;
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0); }
    __device__ void get(float (&f)[2]) const {
        f[0] = __builtin_bit_cast(float, v << 16);
        f[1] = __builtin_bit_cast(float, v & 0xffff0000u);
    }
};
template <> struct Raw<float, 4> {
    float4 v;
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = ssm::bload16<float4>(r, o); }
    __device__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
};
template <> struct Raw<__bf16, 4> {
    u32x2 v;
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = __builtin_amdgcn_raw_buffer_load_b64(r, o, 0, 0); }
    __device__ void get(float (&f)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_bit_cast(float, j % 2 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
    }
};
template <> struct Raw<__bf16, 1> {
    unsigned short v;
    __device__ void load(__amdgpu_buffer_rsrc_t r, unsigned o) { v = __builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0); }
    __device__ void get(float (&f)[1]) const { f[0] = __builtin_bit_cast(float, (unsigned)v << 16); }
};

// (stores past the caches: what a second pass reads again stays in them; 1 x 32768 x 1024 113 -> 103 us)
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put(const float (&f)[2], __amdgpu_buffer_rsrc_t r, unsigned o, float) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(f[0], f[1])), r, o, 0, ssm::kPolicyNT);
}
__device__ __forceinline__ void put(const float (&f)[1], __amdgpu_buffer_rsrc_t r, unsigned o, float) {
    ssm::bstore4(f[0], r, o);
}
__device__ __forceinline__ void put(const float (&f)[2], __amdgpu_buffer_rsrc_t r, unsigned o, __bf16) {
    const bf16x2 b{(__bf16)f[0], (__bf16)f[1]};
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, b), r, o, 0, ssm::kPolicyNT);
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

// c softplus(lam), counted up to 2^64: its product with any gate is then finite, and with one below fp32's range (0, or
// 2^-126 by fall_held) next to 0. (A NaN stays one.)
__device__ __forceinline__ float rate(float c, float lam) {
    const float k = c * ssm::softplus(lam);
    return k > 0x1p64f ? 0x1p64f : k;
}

// 1 - e^-z for z <= kSeries: its first six terms, whose rest is below 0.2^6 / 7! = 1.3e-8 of it.
__device__ __forceinline__ float lost_small(float z) {
    float p = fmaf(z, -1.f / 720, 1.f / 120);
    p = fmaf(z, p, -1.f / 24);
    p = fmaf(z, p, 1.f / 6);
    p = fmaf(z, p, -1.f / 2);
    return z * fmaf(z, p, 1.f);
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

// f(std::true_type) where `near`, else f(std::false_type). As selects, the choice takes a sixth of a block's instructions,
// and in the gradients' kernel registers that spill (us, selects / this: 4 x 2048 x 2048 fp32 gradients 165 / 116, bf16
// 72 / 68; 5 x 1500 x 1536 fp32 forward, narrow groups, 29.7 / 27.4).
template <typename F>
__device__ __forceinline__ void by_gates(bool near, F f) {
    if (near) f(std::true_type());
    else f(std::false_type());
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
    float2* runs;               // (A, H) of the sequences' blocks, and their entering states (null: one segment)
    float* sums;                // backward: a segment's sums
    int B, L, D, blocks, seg;   // blocks of a sequence, and of a segment
    int pad;                    // rows behind a sequence become zeros
    float c;
};

// Keeps what is formed from `v` inside the loop: the offsets of a lane's steps, one addition each, would
// otherwise wait in registers for all of it.
__device__ __forceinline__ unsigned here(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A lane's place: VEC of CH channels, in one of R rows of a wave; W waves. A row has S consecutive steps of a block.
template <typename T, int VEC, int W_, int CH = kCh>
struct Place {
    static constexpr int LC = CH / VEC, R = 64 / LC, S = 16 / VEC, W = W_, TB = W * R * S;
    int lane, w, col, row, mine;   // mine: its first step of a block
    int ch, cg, b, part, n;
    bool live;
    // part `part` (a segment or a block) of a sequence's channel group
    __device__ Place(const RecArgs& a) {
        lane = threadIdx.x & 63;
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        col = lane % LC;
        row = lane / LC;
        mine = (w * R + row) * S;
        const int groups = (a.D + CH - 1) / CH;
        int j = blockIdx.x;
        // (two groups of 32 channels share memory's lines of 128 bytes: on one XCD, of 8 that take workgroups in turn)
        if (CH < kCh && (j | 15) < (int)gridDim.x) j = (j & ~15) | (j & 7) << 1 | (j >> 3 & 1);
        cg = j % groups;
        const int rest = j / groups;
        b = rest % a.B;
        part = rest / a.B;
        ch = cg * CH + col * VEC;
        live = ch < a.D;
        n = a.L;
        if (a.lengths) n = min(max(a.lengths[b], 0), a.L);
    }
    // c softplus(lam) of its channels; whether no channel of the wave goes beyond the series
    __device__ bool decays(const RecArgs& a, float (&kd)[VEC]) const {
        bool near = true;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            kd[v] = live ? rate(a.c, a.lam[ch + v]) : 0.f;
            near &= kd[v] <= kSeries;
        }
        return __all(near);
    }
    // `there` rows of this group's channels from step t0 on (none: nothing is read or written)
    template <typename Q>
    __device__ __amdgpu_buffer_rsrc_t rows(Q* p, long ld, const RecArgs& a, int t0, int there) const {
        const char* base = (const char*)p + (((long)b * a.L + t0) * ld + cg * CH) * sizeof(T);
        return ssm::rsrc(base, there > 0 ? (unsigned)(((long)(there - 1) * ld + min(CH, a.D - cg * CH)) * sizeof(T)) : 0u);
    }
    __device__ unsigned at(long ld, int step) const {   // (dead lanes: past every end)
        return live ? (unsigned)((step * ld + col * VEC) * sizeof(T)) : 0x80000000u;
    }
    template <typename Q>
    __device__ __forceinline__ void load(Raw<T, VEC> (&q)[S], Q* p, long ld, const RecArgs& a, int t0, int there, int first) const {
        const auto r = rows(p, ld, a, t0, there);
        unsigned o = here(at(ld, first));
#pragma unroll
        for (int s = 0; s < S; ++s, o += (unsigned)(ld * sizeof(T))) q[s].load(r, o);
    }
    __device__ __forceinline__ void store(const float (&f)[S][VEC], void* p, long ld, const RecArgs& a, int t0, int there) const {
        const auto r = rows(p, ld, a, t0, there);
        unsigned o = here(at(ld, mine));
#pragma unroll
        for (int s = 0; s < S; ++s, o += (unsigned)(ld * sizeof(T))) put(f[s], r, o, T());
    }
    // zeros for a segment's rows from the sequence's end on
    __device__ void clear(void* p, long ld, const RecArgs& a) const {
        const int s0 = part * a.seg * TB, s1 = min((long)a.L, (long)s0 + (long)a.seg * TB);
        const float none[S][VEC] = {};
        for (int t = max(n, s0); t < s1; t += TB) store(none, p, ld, a, t, min(TB, s1 - t));
    }
};

// The value of a lane (modulo 64).
__device__ __forceinline__ float of_lane(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(lane * 4, __builtin_bit_cast(int, v)));
}

template <int N>
__device__ __forceinline__ bool any_nan(const float (&h)[N]) {
    bool no = false;
#pragma unroll
    for (int v = 0; v < N; ++v) no |= h[v] != h[v];
    return __any(no);
}

// A lane's runs, and their composition over the R rows of a wave: (A, H) becomes the run of all rows up to
// this one, (Ae, He) that of the rows before it. BACK: from this one on, and after it; H the adjoint's.
// SAFE: infinities go through `onto`.
template <int VEC, int S, int R, bool BACK, bool SAFE>
__device__ __forceinline__ void runs(int lane, int row, const float (&d)[S][VEC], const float (&b)[S][VEC], float (&A)[VEC],
                                     float (&H)[VEC], float (&Ae)[VEC], float (&He)[VEC]) {
    static_assert(R <= 2 || (R == 4 && !BACK), "rows of a wave");
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        if (BACK) {   // e <- d (dy + e)
            H[v] = d[S - 1][v] * b[S - 1][v];
            A[v] = d[S - 1][v];
#pragma unroll
            for (int s = S - 2; s >= 0; --s) {
                H[v] = d[s][v] * (b[s][v] + H[v]);
                A[v] *= d[s][v];
            }
        } else {
            H[v] = b[0][v];
            A[v] = d[0][v];
#pragma unroll
            for (int s = 1; s < S; ++s) {
                H[v] = SAFE ? onto(d[s][v], b[s][v], H[v]) : fmaf(d[s][v], H[v], b[s][v]);
                A[v] *= d[s][v];
            }
        }
        Ae[v] = 1.f;
        He[v] = 0.f;
        if constexpr (R == 2) {
            const float A1 = of_lane(A[v], lane + 32), H1 = of_lane(H[v], lane + 32);   // the other row's
            const bool after = row == (BACK ? 0 : 1);
            Ae[v] = after ? A1 : 1.f;
            He[v] = after ? H1 : 0.f;
            H[v] = SAFE ? onto(A[v], H[v], He[v]) : fmaf(A[v], He[v], H[v]);
            A[v] *= Ae[v];
        }
        if constexpr (R == 4) {
#pragma unroll
            for (int k = 1; k < 4; k *= 2) {   // those of the k rows before
                const float A1 = of_lane(A[v], lane - 16 * k), H1 = of_lane(H[v], lane - 16 * k);
                if (row >= k) {
                    H[v] = SAFE ? onto(A[v], H[v], H1) : fmaf(A[v], H1, H[v]);
                    A[v] *= A1;
                }
            }
            const float A1 = of_lane(A[v], lane - 16), H1 = of_lane(H[v], lane - 16);
            Ae[v] = row ? A1 : 1.f;
            He[v] = row ? H1 : 0.f;
        }
    }
}

// ---------------------------------------------------------------- the blocks' (A, H)
// For the segments after them. Without outputs no order binds the lanes: each walks a run of a block on its own, and
// the runs are composed at the end. BACK: of the adjoint, e_{t-1} = a_t (dy_t + e_t), walked from the end.
constexpr int kRunWaves = 8;

// Rows of CH = 128 channels, four a lane, where alignment allows: 1 x 32768 x 1024 bf16 42 us, against 53 with
// rows of 64, one or two a lane, which other rows take.
template <typename T, int VEC, int CH, int TB, bool BACK>
__global__ __launch_bounds__(64 * kRunWaves) void rec_runs(RecArgs a) {
    using P = Place<T, VEC, kRunWaves, CH>;
    constexpr int S = P::S, R = P::R, N = kRunWaves * R, RUN = TB / N;
    static_assert(RUN % S == 0, "whole rows of steps");
    __shared__ float sa[N][CH], sh[N][CH];
    const P p(a);
    const int chl = p.cg * CH + (int)threadIdx.x;
    const bool mine = threadIdx.x < CH && chl < a.D;
    // the entering states go on from here: the caller's may lie where the final ones are written
    float2* const runs = a.runs + (long)p.b * (a.blocks + 1) * a.D;
    if (p.part == 0 && mine) runs[(long)a.blocks * a.D + chl] = make_float2(a.h0 ? a.h0[(long)p.b * a.D + chl] : 0.f, 0.f);
    const int block = p.part + (BACK ? a.seg : 0), t0 = block * TB;   // (none of the last segment; of the first)
    if (t0 >= p.n) return;
    const int there = min(TB, p.n - t0);
    float kd[VEC];
    const bool near = p.decays(a, kd);
    float A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
    const int first = (p.w * R + p.row) * RUN;
    Raw<T, VEC> qx[S], qr[S], qi[S];
    auto fetch = [&](int k) {
        const int at = first + (BACK ? RUN - S - k : k);
        p.load(qr, a.r, a.ldr, a, t0, there, at);
        if (BACK) p.load(qx, a.dy, a.lddy, a, t0, there, at);
        else p.load(qx, a.x, a.ldx, a, t0, there, at), p.load(qi, a.i, a.ldi, a, t0, there, at);
    };
    for (int k = 0; k < RUN; k += S) {
        const int at = first + (BACK ? RUN - S - k : k);
        fetch(k);
        float d[S][VEC], f[S][VEC];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
            qx[s].get(x);
            qr[s].get(r);
            if constexpr (!BACK) qi[s].get(i);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float q;
                decay(kd[v] * open(fall(r[v])), near, d[s][v], q);
                if constexpr (BACK) f[s][v] = x[v];
                else f[s][v] = __builtin_amdgcn_sqrtf(fmaf(q, d[s][v], q)) * (open(fall(i[v])) * x[v]);
            }
        }
        if (at + S > there) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (at + s >= there)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) d[s][v] = 1.f, f[s][v] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < S; ++u)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int s = BACK ? S - 1 - u : u;
                H[v] = BACK ? d[s][v] * (f[s][v] + H[v]) : onto(d[s][v], f[s][v], H[v]);
                A[v] *= d[s][v];
            }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        sa[p.w * R + p.row][p.col * VEC + v] = A[v];
        sh[p.w * R + p.row][p.col * VEC + v] = H[v];
    }
    __syncthreads();
    if (!mine) return;
    float At = 1.f, Ht = 0.f;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int k = BACK ? N - 1 - u : u;
        Ht = onto(sa[k][threadIdx.x], sh[k][threadIdx.x], Ht);
        At *= sa[k][threadIdx.x];
    }
    runs[(long)block * a.D + chl] = make_float2(At, Ht);
}

// By all waves of a workgroup: the state that enters (BACK: leaves) a segment, of channel `lane`. Each wave composes a
// share of the blocks before it (after it); the shares are chained in order.
template <int W, int CH, bool BACK>
__device__ float enter_segment(const RecArgs& a, float2 (&share)[W][CH], int b, int ch, bool has, int from, int to, int w,
                               int lane) {
    const float2* runs = a.runs + (long)b * (a.blocks + 1) * a.D + ch;
    const float h0 = !has ? 0.f : a.runs ? runs[(long)a.blocks * a.D].x : a.h0 ? a.h0[(long)b * a.D + ch] : 0.f;
    if (from >= to) return h0;
    const int each = (to - from + W - 1) / W, k0 = from + w * each, k1 = min(to, k0 + each);
    float A = 1.f, H = 0.f;
#pragma unroll 4
    for (int k = k0; k < k1; ++k) {
        const float2 e = has ? runs[(long)(BACK ? to - 1 - (k - from) : k) * a.D] : make_float2(1.f, 0.f);
        H = onto(e.x, e.y, H);
        A *= e.x;
    }
    share[w][lane] = make_float2(A, H);
    __syncthreads();
    float h = h0;
#pragma unroll
    for (int k = 0; k < W; ++k) h = onto(share[k][lane].x, share[k][lane].y, h);
    return h;
}

// ---------------------------------------------------------------- prompts
template <typename T, int VEC, int W, int CH = kCh>
__global__ __launch_bounds__(64 * W, 4) void rec_kernel(RecArgs a) {
    using P = Place<T, VEC, W, CH>;
    constexpr int S = P::S, R = P::R, TB = P::TB;
    __shared__ float aggA[2][W][CH], aggH[2][W][CH];
    __shared__ float2 share[W][CH];
    const P p(a);
    if (a.pad) p.clear(a.y, a.ldy, a);
    const int last = p.n > 0 ? (p.n - 1) / TB / a.seg : 0;   // the segment of the last token
    if (p.part > last) return;
    const int cl = p.lane % CH, chl = p.cg * CH + cl;   // the channel of what a wave holds by lanes
    const bool has = chl < a.D;
    const int s0 = p.part * a.seg * TB, s1 = min((long)p.n, (long)s0 + (long)a.seg * TB);
    Raw<T, VEC> qx[S], qr[S], qi[S];
    auto fetch = [&](int t0) {
        const int there = min(TB, s1 - t0);   // (none past the end: zeros)
        p.load(qr, a.r, a.ldr, a, t0, there, p.mine);
        p.load(qi, a.i, a.ldi, a, t0, there, p.mine);
        p.load(qx, a.x, a.ldx, a, t0, there, p.mine);
    };
    fetch(s0);
    float kd[VEC];
    const bool near = p.decays(a, kd);
    float st = enter_segment<W, CH, false>(a, share, p.b, chl, has, 0, p.part * a.seg, p.w, cl);
    int buf = 0;
    for (int t0 = s0; t0 < s1; t0 += TB, buf ^= 1) {
        float d[S][VEC], bt[S][VEC];
        by_gates(near, [&](auto close) __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                float x[VEC], r[VEC], i[VEC];
                qx[s].get(x);
                qr[s].get(r);
                qi[s].get(i);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    float u;
                    decay(kd[v] * open(fall(r[v])), close(), d[s][v], u);
                    bt[s][v] = __builtin_amdgcn_sqrtf(fmaf(u, d[s][v], u)) * (open(fall(i[v])) * x[v]);
                }
                if ((s + 1) * VEC % 4 == 0) __builtin_amdgcn_sched_barrier(0);   // (four elements at a time)
            }
        });
        if (t0 + TB > s1) {   // past the end the state stays
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (t0 + p.mine + s >= s1)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) d[s][v] = 1.f, bt[s][v] = 0.f;
        }
        fetch(min(t0 + TB, s1));
        float A[VEC], H[VEC], Ae[VEC], He[VEC];
        runs<VEC, S, R, false, false>(p.lane, p.row, d, bt, A, H, Ae, He);
        if (any_nan(H)) runs<VEC, S, R, false, true>(p.lane, p.row, d, bt, A, H, Ae, He);
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
            next = fmaf(aggA[buf][w][cl], next, aggH[buf][w][cl]);
        }
        if (__any(next != next)) {
            next = st;
            for (int w = 0; w < W; ++w) {
                if (w == p.w) enter = next;
                next = onto(aggA[buf][w][cl], aggH[buf][w][cl], next);
            }
        }
        st = next;
        float h[VEC], g[VEC], y[S][VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            h[v] = g[v] = onto(Ae[v], He[v], CH == 64 && VEC == 1 ? enter : of_lane(enter, p.col * VEC + v));
#pragma unroll
            for (int s = 0; s < S; ++s) y[s][v] = g[v] = fmaf(d[s][v], g[v], bt[s][v]);
        }
        if (any_nan(g)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                g[v] = h[v];
#pragma unroll
                for (int s = 0; s < S; ++s) y[s][v] = g[v] = onto(d[s][v], bt[s][v], g[v]);
            }
        }
        if (a.states && (t0 + p.mine) % kKept == 0 && t0 + p.mine < s1 && p.live) {
            float* o = a.states + ((long)p.b * ((a.L + kKept - 1) / kKept) + (t0 + p.mine) / kKept) * a.D + p.ch;
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = h[v];
        }
        p.store(y, a.y, a.ldy, a, t0, min(TB, s1 - t0));
    }
    if (a.hT && p.part == last && p.w == 0 && has) a.hT[(long)p.b * a.D + chl] = st;
}

// ---------------------------------------------------------------- gradients
// With g_t the gradient of h_t, walked from the last step: g_t = dy_t + a_{t+1} g_{t+1}, and from
// log a = -z, d sqrt(1 - a^2) / d log a = -a^2 / sqrt(1 - a^2):
//   dx = g sqrt(1 - a^2) i,  di = g b (1 - i)   (i: the open gate)
//   q = z dL/dz = g (i x a^2 z / sqrt(1 - a^2) - a z h_{t-1}),  dr = q (1 - sigmoid r)
//   dlam = sum q sigmoid(lam) / softplus(lam),  dh0 = a_1 g_1
// z / sqrt(1 - a^2) goes to 0 with z. The blocks go by from the end; the adjoint's runs e -> A e + G have the same A as
// the states'. The states h_{t-1} are walked again from those that the forward pass kept.
template <typename T, int VEC, int W>
__global__ __launch_bounds__(64 * W, 2) void rec_backward(RecArgs a) {
    using P = Place<T, VEC, W>;
    constexpr int S = P::S, R = P::R, TB = P::TB;
    constexpr int WK = std::min(W, kKept / (R * S));   // waves of a kept state (fewer: sequences of one block)
    static_assert(WK >= 1 && W % WK == 0, "whole kept spans");
    __shared__ float aggA[2][W][kCh], aggH[2][W][kCh], aggG[2][W][kCh];
    __shared__ float2 share[W][kCh];
    const P p(a);
    if (a.pad) {
        p.clear(a.y, a.ldy, a);
        p.clear(a.dr, a.lddr, a);
        p.clear(a.di, a.lddi, a);
    }
    const int chl = p.cg * kCh + p.lane;
    const bool has = chl < a.D;
    const int kept = (a.L + kKept - 1) / kKept;
    const int s0 = p.part * a.seg * TB, s1 = min((long)p.n, (long)s0 + (long)a.seg * TB);
    float sum[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) sum[v] = 0.f;
    if (s1 > s0 || p.part == 0) {
        float kd[VEC];
        const bool near = p.decays(a, kd);
        Raw<T, VEC> qx[S], qr[S], qi[S], qg[S];
        float ks = 0.f;   // the kept state of this wave's span, of channel `lane`
        auto fetch = [&](int t) {
            const int t0 = max(t, s0), there = t < s0 ? 0 : min(TB, s1 - t0);
            p.load(qr, a.r, a.ldr, a, t0, there, p.mine);
            p.load(qg, a.dy, a.lddy, a, t0, there, p.mine);
            p.load(qi, a.i, a.ldi, a, t0, there, p.mine);
            p.load(qx, a.x, a.ldx, a, t0, there, p.mine);
            const int at = t0 + p.w / WK * kKept;
            ks = has && there > 0 && at < s1 ? a.states[((long)p.b * kept + at / kKept) * a.D + chl] : 0.f;
        };
        const int t1 = s1 > s0 ? s0 + (s1 - s0 - 1) / TB * TB : s0 - TB;
        if (t1 >= s0) fetch(t1);
        // the adjoint that leaves a block's first step, of channel `lane`
        float e = enter_segment<W, kCh, true>(a, share, p.b, chl, has, (p.part + 1) * a.seg, p.n > 0 ? (p.n - 1) / TB + 1 : 0, p.w,
                                              p.lane);
        int buf = 0;
        for (int t0 = t1; t0 >= s0; t0 -= TB, buf ^= 1) {
            float d[S][VEC], bt[S][VEC], bi[S][VEC], bj[S][VEC], k1[S][VEC], k2[S][VEC], cr[S][VEC], gy[S][VEC];
            by_gates(near, [&](auto close) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    float x[VEC], r[VEC], i[VEC];
                    qx[s].get(x);
                    qr[s].get(r);
                    qi[s].get(i);
                    qg[s].get(gy[s]);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float er = fall_held(r[v]), ei = fall_held(i[v]);
                        const float gr = open(er), gi = open(ei), z = kd[v] * gr;
                        float q;
                        decay(z, close(), d[s][v], q);
                        const float b2 = fmaf(q, d[s][v], q), inv = __builtin_amdgcn_rsqf(fmaxf(b2, kTiny)), be = b2 * inv;
                        const float u = gi * x[v];
                        bi[s][v] = be * gi;
                        bt[s][v] = be * u;
                        bj[s][v] = bt[s][v] * (ei * gi);
                        k2[s][v] = d[s][v] * z;
                        k1[s][v] = u * d[s][v] * d[s][v] * (z * inv);
                        cr[s][v] = er * gr;
                    }
                    if ((s + 1) * VEC % 4 == 0) __builtin_amdgcn_sched_barrier(0);   // (four elements at a time)
                }
            });
            if (t0 + TB > s1) {
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (t0 + p.mine + s >= s1)
#pragma unroll
                        for (int v = 0; v < VEC; ++v) d[s][v] = 1.f, bt[s][v] = k1[s][v] = k2[s][v] = gy[s][v] = 0.f;
            }
            float hl = ks;
            fetch(t0 - TB);
            float A[VEC], H[VEC], Ae[VEC], He[VEC], Ab[VEC], G[VEC], Ax[VEC], Gx[VEC];
            runs<VEC, S, R, false, false>(p.lane, p.row, d, bt, A, H, Ae, He);
            runs<VEC, S, R, true, false>(p.lane, p.row, d, gy, Ab, G, Ax, Gx);
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
                float h = fmaf(Ae[v], VEC == 1 ? hl : of_lane(hl, p.col * VEC + v), He[v]);
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const float before = h;
                    h = fmaf(d[s][v], h, bt[s][v]);
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
            const int there = min(TB, s1 - t0);
            p.store(bi, a.y, a.ldy, a, t0, there);
            p.store(cr, a.dr, a.lddr, a, t0, there);
            p.store(bj, a.di, a.lddi, a, t0, there);
        }
        if (a.hT && p.part == 0 && p.w == 0 && has) a.hT[(long)p.b * a.D + chl] = e;
    }
    // the workgroup's sums of q, in the order of rows and waves
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        if constexpr (VEC == 2) sum[v] += of_lane(sum[v], p.lane + 32);
        if (p.row == 0) aggA[0][p.w][p.col * VEC + v] = sum[v];
    }
    __syncthreads();
    if (threadIdx.x < kCh && has) {
        float t = 0.f;
        for (int w = 0; w < W; ++w) t += aggA[0][w][threadIdx.x];
        a.sums[((long)p.b * ((a.blocks + a.seg - 1) / a.seg) + p.part) * a.D + chl] = t;
    }
}

// dlam from the segments' sums, in double and in one order.
__global__ __launch_bounds__(1024) void rec_dlam(const float* __restrict__ sums, const float* __restrict__ lam, int n,
                                                 int D, float* __restrict__ dlam) {
    __shared__ double part[16][64];
    const int ch = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + ch;
    double t = 0.;
    if (d < D)
#pragma unroll 4
        for (int k = w; k < n; k += 16) t += (double)sums[(long)k * D + d];
    part[w][ch] = t;
    __syncthreads();
    if (w || d >= D) return;
    for (int k = 1; k < 16; ++k) t += part[k][ch];
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
        decay(rate(a.c, lam[v]) * open(fall((float)r[v])), false, d, q);
        const float bt = __builtin_amdgcn_sqrtf(fmaf(q, d, q)) * (open(fall((float)i[v])) * (float)x[v]);
        h[v] = onto(d, bt, h[v]);
        y[v] = (T)h[v];
    }
    *reinterpret_cast<Fv*>(ph) = h;
    *reinterpret_cast<Tv*>(py) = y;
}

// ---------------------------------------------------------------- plans
constexpr int kWaves = 16, kWavesBack = 8;
constexpr int kNarrow = 32, kWavesNarrow = 8;   // channels and waves of narrow groups

// Blocks and segments of the sequences: as many segments as make the kernels' time least, counted in the time of a
// block on a full chip (one workgroup a CU; us, W = 16 and 8 waves: 7.6, 6.9):
//   - a turn of 256 workgroups takes the blocks of a segment, a last one of fewer at least 0.77 of that (16 blocks of
//     128 workgroups 95 us, of 256 122);
//   - a first pass over the blocks that others follow takes `again` of a block each, spread over the chip, and a launch.
// Of sequences with lengths about 0.6 are taken to be there. us, groups of 64 channels in one segment / by the rule / in twice
// its segments: 1 x 32768 x 1024 633 / 110 / 112, 4 x 2048 x 2048 51 / 51 / 59, 8 x 4096 x 2048 132 / 132 / 173;
// gradients 1090 / 142 / 146, 86 / 70 / 77, 225 / 225 / 278.
// Short sequences leave most of a block of 256 steps empty: up to 16 steps go to single waves, and up to half a block, or four
// blocks where two workgroups a CU are there to share it, to four waves. fp32, us, 16 waves / fewer: 64 x 16 x 1024 46 / 9,
// 256 x 4 x 1024 168 / 12, 64 x 64 x 1024 47 / 16, 64 x 400 x 1024 103 / 78, 32 x 1000 x 1024 113 / 106, but 8 x 200 x 1024
// 12.5 / 13.8 and 64 x 2000 x 1024 416 / 421; gradients, 8 waves / fewer: 41 / 15, 143 / 21, 45 / 27, 161 / 154, 182 / 189.
struct Plan {
    long chains;        // sequences times channel groups
    int blocks, seg;    // blocks of a sequence, and of a segment
    int waves;          // of a workgroup
    int ch;             // channels of a group
    int segments() const { return (blocks + seg - 1) / seg; }
    long groups() const { return chains * segments(); }
};
Plan plan_of(int B, int L, int D, int waves, double again, bool ragged, double* cost = nullptr) {
    const long chain = ssm::cdiv(D, kCh) * B;
    if (L <= 16) return Plan{chain, 1, 1, 1, kCh};
    if (L <= 8 * waves || (L <= 64 * waves && chain * (ragged ? 0.6 : 1.0) >= 512)) {
        const int n = (int)ssm::cdiv(L, 64);
        return Plan{chain, n, n, 4, kCh};
    }
    Plan p{chain, (int)ssm::cdiv(L, 16 * waves), 0, waves, kCh};
    const double chains = p.chains * (ragged ? 0.6 : 1.0);
    double best = 0;
    for (int n = 1; n <= std::min(64, p.blocks); ++n) {
        const int per = (p.blocks + n - 1) / n, segs = (p.blocks + per - 1) / per;
        const double turns = chains * segs / 256, full = (double)(long)turns, rest = turns - full;
        double t = per * (full + (rest > 0 || full == 0 ? std::max(0.77, rest) : 0.0));
        if (segs > 1) t += 0.5 + again * std::max(1.0, chains * (p.blocks - per) / 256);
        if (n == 1 || t < best) best = t, p.seg = per;
    }
    if (cost) *cost = best;
    return p;
}
// Groups of 32 channels put twice the workgroups on sequences that are walked whole, where those are few enough for one a CU:
// a block then takes 0.4 (up to 80 workgroups) to 0.73 (256) of a full chip's. us, wide groups by the rule above / narrow:
// 4 x 2048 x 2048 bf16 50 / 45, fp32 81 / 61, 5 x 1500 x 1536 fp32 with lengths 39 / 27, 2 x 600 x 2048 bf16 24 / 14, but
// 2 x 4096 x 2048 bf16 56 / 71 and 1 x 8192 x 512 fp32 33 / 99. With lengths the segments' share is the less even one: the
// 1.25, and the 0.6 above, are from the ragged batch named here alone.
Plan plan_forward(int B, int L, int D, bool ragged) {
    double best = 0;
    const Plan p = plan_of(B, L, D, kWaves, 0.7, ragged, &best);
    const long n = ssm::cdiv(D, kNarrow) * B;
    if (p.waves != kWaves || n > 256) return p;
    const double there = n * (ragged ? 0.6 : 1.0), t = p.blocks * (0.4 + 0.33 * std::max(0.0, there - 80) / 176);
    return t < best * (ragged ? 1.25 : 1.0) ? Plan{n, p.blocks, p.blocks, kWavesNarrow, kNarrow} : p;
}
Plan plan_backward(int B, int L, int D, bool ragged) { return plan_of(B, L, D, kWavesBack, 0.3, ragged); }

size_t runs_bytes(const Plan& p, int B, int D) {
    return p.segments() > 1 ? ((size_t)B * (p.blocks + 1) * D * sizeof(float2) + 15) / 16 * 16 : 0;
}
size_t sums_bytes(const Plan& p, int B, int D) { return (size_t)B * p.segments() * D * sizeof(float); }
size_t forward_bytes(int B, int L, int D) {
    return std::max(runs_bytes(plan_forward(B, L, D, false), B, D), runs_bytes(plan_forward(B, L, D, true), B, D));
}
size_t backward_bytes(int B, int L, int D) {
    const Plan p = plan_backward(B, L, D, false), q = plan_backward(B, L, D, true);
    return std::max(runs_bytes(p, B, D) + sums_bytes(p, B, D), runs_bytes(q, B, D) + sums_bytes(q, B, D));
}

// VEC channels a lane (4: two in the kernels with outputs).
template <typename T, int VEC, bool BACK>
void launch_runs(const RecArgs& a, int parts, hipStream_t st) {
    constexpr int TB = 16 * (BACK ? kWavesBack : kWaves), CH = VEC == 4 ? 128 : kCh;
    rec_runs<T, VEC, CH, TB, BACK><<<(unsigned)(ssm::cdiv(a.D, CH) * a.B * parts), 64 * kRunWaves, 0, st>>>(a);
}
template <typename T, int VEC>
void launch_forward(const RecArgs& a, const Plan& p, hipStream_t st) {
    if (a.runs) launch_runs<T, VEC, false>(a, (p.segments() - 1) * p.seg, st);
    constexpr int V = std::min(VEC, 2);
    const unsigned n = (unsigned)p.groups();
    if (p.waves == 1) rec_kernel<T, V, 1><<<n, 64, 0, st>>>(a);
    else if (p.waves == 4) rec_kernel<T, V, 4><<<n, 256, 0, st>>>(a);
    else if (p.ch == kNarrow) rec_kernel<T, V, kWavesNarrow, kNarrow><<<n, 64 * kWavesNarrow, 0, st>>>(a);
    else rec_kernel<T, V, kWaves><<<n, 64 * kWaves, 0, st>>>(a);
}
template <typename T, int VEC>
void launch_backward(const RecArgs& a, const Plan& p, float* dlam, hipStream_t st) {
    if (a.runs) launch_runs<T, VEC, true>(a, p.blocks - p.seg, st);
    constexpr int V = std::min(VEC, 2);
    const unsigned n = (unsigned)p.groups();
    if (p.waves == 1) rec_backward<T, V, 1><<<n, 64, 0, st>>>(a);
    else if (p.waves == 4) rec_backward<T, V, 4><<<n, 256, 0, st>>>(a);
    else rec_backward<T, V, kWavesBack><<<n, 64 * kWavesBack, 0, st>>>(a);
    rec_dlam<<<(unsigned)ssm::cdiv(a.D, 64), 1024, 0, st>>>(a.sums, a.lam, a.B * p.segments(), a.D, dlam);
}

// Channels that a lane may load at a time: four or two where D, all strides and the rows' alignment are whole ones.
int vector_of(int dtype, int D, std::initializer_list<std::pair<const void*, long>> ops) {
    const uintptr_t es = dtype == SSM_F32 ? 4 : 2;
    uintptr_t all = (uintptr_t)D;
    for (const auto& o : ops) all |= (uintptr_t)o.second | ((uintptr_t)o.first & (4 * es - 1)) / es | ((uintptr_t)o.first % es ? 1 : 0);
    return all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
}
template <typename T, typename... A>
void forward_of(int vec, A... a) {
    if (vec == 4) launch_forward<T, 4>(a...);
    else if (vec == 2) launch_forward<T, 2>(a...);
    else launch_forward<T, 1>(a...);
}
template <typename T, typename... A>
void backward_of(int vec, A... a) {
    if (vec == 4) launch_backward<T, 4>(a...);
    else if (vec == 2) launch_backward<T, 2>(a...);
    else launch_backward<T, 1>(a...);
}

constexpr long kMaxLd = 1L << 20;   // a block's rows within 2^31 bytes
constexpr long kMaxBlocks = (1L << 22) - 1;   // (launches of 1024 threads in 32 bits)
}  // namespace

extern "C" size_t ssm_gated_recurrence_workspace(int B, int L, int D) {
    return B > 0 && L > 0 && D > 0 ? forward_bytes(B, L, D) : 0;
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
    const Plan p = plan_forward(B, L, D, lengths != nullptr);
    SSM_REQUIRE(p.chains * p.blocks <= kMaxBlocks, "ssm_gated_recurrence: too many sequences, steps or channels");
    const size_t need = ssm_gated_recurrence_workspace(B, L, D);
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
    a.runs = p.segments() > 1 ? static_cast<float2*>(workspace) : nullptr;
    a.B = B; a.L = L; a.D = D; a.blocks = p.blocks; a.seg = p.seg;
    const int vec = vector_of(dtype, D, {{x, ldx}, {r, ldr}, {i, ldi}, {y, ldy}});
    if (dtype == SSM_F32) forward_of<float>(vec, a, p, (hipStream_t)stream);
    else forward_of<__bf16>(vec, a, p, (hipStream_t)stream);
    return ssm::check_launch("ssm_gated_recurrence");
}

extern "C" size_t ssm_gated_recurrence_backward_workspace(int B, int L, int D) {
    if (B <= 0 || L < 0 || D <= 0) return 0;
    return backward_bytes(B, L, D);
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
    const Plan p = plan_backward(B, L, D, lengths != nullptr);
    SSM_REQUIRE(L <= ssm::kMaxSteps && p.chains * p.blocks <= kMaxBlocks,
                "ssm_gated_recurrence_backward: too many sequences, steps or channels");
    const size_t need = ssm_gated_recurrence_backward_workspace(B, L, D);
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
    const size_t runs = runs_bytes(p, B, D);
    a.runs = runs ? static_cast<float2*>(workspace) : nullptr;
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + runs);
    a.B = B; a.L = L; a.D = D; a.blocks = p.blocks; a.seg = p.seg;
    const int vec = vector_of(dtype, D, {{dy, lddy}, {x, ldx}, {r, ldr}, {i, ldi}, {dx, lddx}, {dr, lddr}, {di, lddi}});
    if (dtype == SSM_F32) backward_of<float>(vec, a, p, dlam, (hipStream_t)stream);
    else backward_of<__bf16>(vec, a, p, dlam, (hipStream_t)stream);
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
    // four channels a thread where rows allow it
    const uintptr_t piece = dtype == SSM_F32 ? 15 : 7;
    const bool four = D % 4 == 0 && (ldx | ldr | ldi | ldy) % 4 == 0 && (((uintptr_t)h | (uintptr_t)lam) & 15) == 0 &&
                      (((uintptr_t)x | (uintptr_t)r | (uintptr_t)i | (uintptr_t)y) & piece) == 0;
    const unsigned n = (unsigned)ssm::cdiv((long)B * (four ? D / 4 : D), 256);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SSM_F32) four ? rec_step<float, 4><<<n, 256, 0, st>>>(a) : rec_step<float, 1><<<n, 256, 0, st>>>(a);
    else four ? rec_step<__bf16, 4><<<n, 256, 0, st>>>(a) : rec_step<__bf16, 1><<<n, 256, 0, st>>>(a);
    return ssm::check_launch("ssm_gated_recurrence_step");
}

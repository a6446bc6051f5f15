// Linear attention with a constant decay for each head, chunked for prompts and recurrent for
// single tokens (Katharopoulos et al. 2020; decays as in Sun et al. 2023, section 2):
//   S_t = e^g S_{t-1} + v_t k_t^T  (V x K, fp32);   y_t = scale S_t q_t.
// Query heads h share the keys and values of head h / (H / G).
//
// Chunked form. With C tokens a chunk, S the state before it and i, j its tokens:
//   y_i = scale e^{g (i + 1)} S q_i + sum_{j <= i} scale e^{g (i - j)} (q_i . k_j) v_j
//   S  <- e^{g C} S + sum_j (e^{g (C - 1 - j)} v_j) k_j^T
// One workgroup walks the chunks of a segment of one (sequence, head, part of V) with S in its
// MFMA accumulators. Sequences are cut into segments where (sequence, head, part) alone would
// not fill the chip: a state pass forms each segment's own state, a combine pass the states that
// enter the segments, and the full pass starts from those.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

constexpr unsigned kOut = 0x80000000u;   // a buffer offset past any descriptor

struct LaArgs {
    const void* q; long ldq;
    const void* k; long ldk;
    const void* v; long ldv;
    const float* g;
    float scale;
    const int* lengths;      // (B) or null: L for all
    void* y; long ldy;
    int B, L, H, G, K, V;
    const float* h0;         // (B,H,V,K) or null
    float* hT;               // (B,H,V,K) or null
    float* seg;              // (nseg,B,H,V,K): the segments' own states (the last slot: h0), or,
    int nseg, seglen, vparts, share;   // combined, the states that enter them
    int combined;
};

__device__ __forceinline__ float clamp_g(float g) { return g < -1e30f ? -1e30f : g; }   // (a NaN stays)

// x <- e^{g n} x: as x + (e^{g n} - 1) x from 1/2 on, so that a decay too slow for fp32's e^{g n} is kept,
// and as a product below, where the difference would lose what is left. (Without a branch: the reads
// around it stay ahead of it, and fp32 prompts took 5% longer.)
__device__ __forceinline__ float decayed(float x, float m, float keep) { return fmaf(x, m, keep * x); }

// The same, of a state that may be infinite: it stays so, as it does token by token.
__device__ __forceinline__ float decayed_any(float x, float m, float keep) {
    const float y = decayed(x, m, keep);
    return __builtin_isinf(x) ? x : y;
}

struct Decay {
    float m, keep;   // (of a whole wave)
    __device__ __forceinline__ Decay() : m(0.f), keep(0.f) {}
    __device__ __forceinline__ Decay(float g, int n) {
        const float e = g * (float)n;
        const bool slow = !(e < -0.69f);
        auto whole = [](float x) {
            return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
        };
        m = whole(slow ? expm1f(e) : expf(e));
        keep = whole(slow ? 1.f : 0.f);
    }
    __device__ __forceinline__ float of_any(float x) const { return decayed_any(x, m, keep); }
};

// A value that the compiler forms again in each turn of a loop: the registers that it would hold
// over the loop are wanted for the state and the next chunk's rows (spills read back from memory
// wait behind those rows' loads).
template <typename T>
__device__ __forceinline__ T fresh(T x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ int seq_len(const LaArgs& a, int b) {
    if (!a.lengths) return a.L;
    return max(0, min(a.lengths[b], a.L));
}

// Workgroup order: those that read the same keys and values (the parts of V and the heads of a group) on one
// XCD, the groups, then the sequences and segments, dealt out over the XCDs: a padded batch's long
// sequences are then shared by all of them (8 sequences of up to 1500 tokens, 32 heads: a range of ids an XCD
// took 1.3 times as long). Few groups would leave XCDs idle: then single heads are dealt out.
struct Place {
    int part, h, grp, b, seg;   // seg past the last: none
    __device__ __forceinline__ explicit Place(const LaArgs& a) {
        const int per = a.share * a.vparts, local = blockIdx.x >> 3, units = a.H / a.share;
        const int unit = local / per * 8 + (blockIdx.x & 7), in = local % per;
        part = in % a.vparts;
        h = unit % units * a.share + in / a.vparts;
        grp = h / (a.H / a.G);
        b = unit / units % a.B;
        seg = unit / units / a.B;
    }
};

// The workgroups of a launch over so many segments, and the heads that are dealt out together.
inline unsigned la_groups(LaArgs& a, int segments) {
    const long groups = (long)segments * a.B * a.G;
    a.share = groups % 8 == 0 || groups >= 64 ? a.H / a.G : 1;
    return (unsigned)(8 * ssm::cdiv((long)segments * a.B * (a.H / a.share), 8) * a.share * a.vparts);
}

// ---------------------------------------------------------------- bf16
// Tiles of v_mfma_f32_16x16x32_bf16 (A: row lane % 16, 8 k at 8 (lane / 16); D: column lane % 16,
// rows 4 (lane / 16) + r). Wave w owns VT / 4 columns of V in S^T (rows k, columns v). The
// accumulators of two of its 16 x 16 tiles are, rounded, the A operand of S q^T with the 32 k of
// the block taken in the order (16 t + 4 g + r, 16 (t + 1) + 4 g + r); q is read from LDS in that
// order. The 64 x 64 products q k^T are shared out over the waves by rows i and go through LDS.
//
// 8 sequences of 4096 tokens, 16 heads, K = V = 128, in four segments: the state pass, over three of them,
// takes 60 us (201 MB of rows in, 25 MB of states out: 3.8 TB/s, short of memory speed), the full pass 165, of
// which its loads and stores alone are 120 and the matrix cores' work 51: it is bound by memory and by the
// three barriers a chunk, between which two waves a SIMD cannot keep either busy. Eight waves of 16 columns
// read S q's queries twice as often (1.36 times as long).
//
// Roundings to bf16: the output's alone. What enters a product with 24 bits (S with q, the products q k^T with
// v, and the values of the state update, e^{..} v, with k) enters in three parts of eight bits each. (In two
// parts a call took 196 us in all, now 225, and 2^-17 of a term was left out: all that a sum that cancels holds.)
__device__ __forceinline__ floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// M[row0 .. + 3][col0 + lane % 16] of a row-major LDS tile: inside each 16-lane group lane 4a + b
// receives element b of the 8-byte pieces that lanes a, a + 4, a + 8, a + 12 address.
template <int PITCH>
__device__ __forceinline__ bf16x4 tr_read(const __bf16* base, int row0, int col0, int l16) {
    const __bf16* p = base + (row0 + (l16 >> 2)) * PITCH + col0 + 4 * (l16 & 3);
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)p);
}

__device__ __forceinline__ bf16x8 cat(bf16x4 a, bf16x4 b) {
    return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Pairs of fp32 numbers as three pairs of bf16 whose sums they are: each part has the leading eight bits of
// what the ones before it leave, cut off, not rounded (so that the largest numbers stay finite, and nothing
// is left). ANY: an infinite number's first part is infinite and the others finite, of its sign (NaN else).
struct Parts { unsigned u[3]; };
template <bool ANY = false>
__device__ __forceinline__ Parts split(float a, float b) {
    constexpr float most = 3.402823466e38f;
    auto held = [](float x) { return __builtin_amdgcn_fmed3f(x, -most, most); };
    auto head = [](float x) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u); };
    Parts p;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
        p.u[c] = __builtin_amdgcn_perm(y, x, 0x07060302u);   // (v_perm_b32: their upper halves)
        if (ANY && c == 0) a = held(a), b = held(b);
        a -= head(a);
        b -= head(b);
    }
    return p;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// The larger magnitudes' bits, of two bf16 a dword: 0x7f80 and more is an inf or NaN.
__device__ __forceinline__ u16x2 most_bf16(u16x2 m, unsigned u) {
    return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u & 0x7fff7fffu));
}

constexpr int CB = 64;   // tokens per chunk

template <int KD, int VT, bool STATE>
struct SmemB {
    static constexpr int KP = KD + 8, VP = VT + 8, PP = CB + 8, Y = STATE ? 1 : CB;
    alignas(16) __bf16 q[Y][KP];
    alignas(16) __bf16 k[CB][KP];
    alignas(16) __bf16 v[CB][VP];
    // scale e^{g (i - j)} q_i . k_j, row i, in three parts
    alignas(16) __bf16 p[3][Y][PP];
    float dec[CB + 17];             // place 64 - d: scale e^{g d}, d = i - j (1 behind d = 0)
    alignas(16) float wj[CB];       // e^{g (n - 1 - j)}: the state update's weights
    int odd[2];                     // an inf or NaN in the chunk's v (by the chunk's parity)
};

// 16 bytes (8 elements, columns col .. + 7) from byte offset o on: zeros from column `width` and
// past the descriptor on.
template <bool VEC, bool NT = false>
__device__ __forceinline__ uint4 fetch_b(__amdgpu_buffer_rsrc_t r, unsigned o, int col, int width) {
    if constexpr (VEC) {   // (whole pieces: o is past the descriptor then)
        return NT ? ssm::bload16_nt<uint4>(r, o) : ssm::bload16<uint4>(r, o);
    } else {
        unsigned u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned lo = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(
                r, col + 2 * e < width ? o + 4u * e : kOut, 0, 0);
            const unsigned hi = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(
                r, col + 2 * e + 1 < width ? o + 4u * e + 2u : kOut, 0, 0);
            u[e] = lo | hi << 16;
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// Four elements from byte offset o on, `left` of them inside the row (no more than that are
// touched; an o past the descriptor reads zeros and writes nothing).
template <bool VEC>
__device__ __forceinline__ floatx4 load_f4(__amdgpu_buffer_rsrc_t r, unsigned o, int left) {
    if constexpr (VEC) {
        return ssm::bload16<floatx4>(r, left > 0 ? o : kOut);
    } else {
        floatx4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = ssm::bload4(r, e < left ? o + 4u * e : kOut);
        return x;
    }
}

template <bool VEC>
__device__ __forceinline__ void store_f4(__amdgpu_buffer_rsrc_t r, unsigned o, floatx4 x, int left) {
    if constexpr (VEC) {
        ssm::bstore16(make_float4(x[0], x[1], x[2], x[3]), r, left > 0 ? o : kOut);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) ssm::bstore4(x[e], r, e < left ? o + 4u * e : kOut);
    }
}

// STATE: only the segment's own state (from zero), into its slot.
template <int KD, int VT, bool VEC, bool STATE>
__global__ __launch_bounds__(256, KD == 256 ? 1 : 2) void la_bf16_kernel(LaArgs a) {
    using Smem = SmemB<KD, VT, STATE>;
    constexpr int KT = KD / 16, KB = KD / 32, VW = VT / 64;
    constexpr int KP = Smem::KP, VP = Smem::VP, PP = Smem::PP;
    constexpr int NK = CB * KD / 8 / 256, NV = CB * VT / 8 / 256;
    __shared__ Smem s;

    const Place place(a);
    const int part = place.part, h = place.h, grp = place.grp, b = place.b, seg = place.seg;
    if (seg >= a.nseg - STATE) return;
    const int len = seq_len(a, b);
    const int t_begin = seg * a.seglen, t_end = min(len, t_begin + a.seglen);
    // the segment that ends the sequence writes the final state (segment 0 of an empty one)
    const bool last = seg == (len > 0 ? (len - 1) / a.seglen : 0);
    // (the first segment's state pass also copies h0: hT may alias it, and the last segment may end
    // before another begins)
    const bool copy = STATE && seg == 0 && a.h0;
    if (STATE ? (last || t_begin >= len) && !copy : !last && t_begin >= len) return;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane_g = lane >> 4, lane_i = lane & 15;
    const int v0 = part * VT + 16 * VW * w;     // the wave's first column of V
    const float g = clamp_g(a.g[h]), gl = g * ssm::kLog2e;
    const long state = ((long)b * a.H + h) * a.V * a.K;
    const long slot = (long)a.B * a.H * a.V * a.K;

    floatx4 S[KT][VW];
    const unsigned sbytes = (unsigned)(a.V * a.K) * 4u;
    auto each_state = [&](auto&& f) {
        const int vl = v0 + fresh(lane_i), kl = 4 * fresh(lane_g);
#pragma unroll
        for (int x = 0; x < VW; ++x)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
                f(S[kt][x], (unsigned)((vl + 16 * x) * a.K + kl + 16 * kt) * 4u,
                  vl + 16 * x < a.V ? a.K - kl - 16 * kt : 0);
    };
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int x = 0; x < VW; ++x) S[kt][x] = floatx4{0.f, 0.f, 0.f, 0.f};
    // ---- a chunk's rows in registers, ahead of their staging: piece u of a thread is its column of
    // row 256 u / (pieces per row) further down
    constexpr int RK = 256 / (KD / 8), RV = 256 / (VT / 8);
    uint4 rq[STATE ? 1 : NK], rk[NK], rv[NV];
    const int krow = tid / (KD / 8), kcol = tid % (KD / 8) * 8;
    const int vrow = tid / (VT / 8), vcol = tid % (VT / 8) * 8;
    auto base = [&](const void* p, long ld, int head, int width, int t) {
        return static_cast<const __bf16*>(p) + ((long)b * a.L + t) * ld + (long)head * width;
    };
    auto bytes = [&](long ld, int width, int n) {
        return n > 0 ? (unsigned)(((long)(n - 1) * ld + width) * 2) : 0u;
    };
    const unsigned kdown = (unsigned)a.ldk * (2 * RK), qdown = (unsigned)a.ldq * (2 * RK);
    const unsigned vdown = (unsigned)a.ldv * (2 * RV);
    auto first = [](int row, long ld, int col, int width) {
        return col < width ? ((unsigned)row * (unsigned)ld + (unsigned)col) * 2u : kOut;
    };
    const unsigned koff = first(krow, a.ldk, kcol, a.K), qoff = first(krow, a.ldq, kcol, a.K);
    const unsigned voff = first(vrow, a.ldv, part * VT + vcol, a.V);
    auto fetch = [&](int t) {
        const int n = max(0, min(CB, t_end - t));
        const int tt = min(t, a.L - 1);
        const auto dk = ssm::rsrc(base(a.k, a.ldk, grp, a.K, tt), bytes(a.ldk, a.K, n));
        const auto dv = ssm::rsrc(base(a.v, a.ldv, grp, a.V, tt), bytes(a.ldv, a.V, n));
#pragma unroll
        for (int u = 0; u < NK; ++u) rk[u] = fetch_b<VEC>(dk, koff + u * kdown, kcol, a.K);
#pragma unroll
        for (int u = 0; u < NV; ++u) rv[u] = fetch_b<VEC>(dv, voff + u * vdown, part * VT + vcol, a.V);
        if constexpr (!STATE) {
            // (read once: out of the way of k and v, which the state pass has read before and the other
            // heads of the group read; 4% at 5 sequences of 4096 tokens)
            const auto dq = ssm::rsrc(base(a.q, a.ldq, h, a.K, tt), bytes(a.ldq, a.K, n));
#pragma unroll
            for (int u = 0; u < NK; ++u) rq[u] = fetch_b<VEC, true>(dq, qoff + u * qdown, kcol, a.K);
        }
    };
    if (copy) {
        const auto from = ssm::rsrc(a.h0 + state, sbytes);
        const auto to = ssm::rsrc(a.seg + (a.nseg - 1) * slot + state, sbytes);
        each_state([&](floatx4&, unsigned o, int left) {
            store_f4<VEC>(to, o, load_f4<VEC>(from, o, left), left);
        });
        if (last) return;
    }
    if (tid < 2) s.odd[tid] = 0;
    if (tid < CB + 17) s.dec[tid] = a.scale * ssm::ex2(gl * (float)max(0, 64 - tid));
    if (t_begin < t_end) fetch(t_begin);
    if (!STATE) {
        // h0 (where there are segments, its copy), then the segments' own states, each decayed by a
        // segment's length; or the sum that the combine pass left
        const float* h0 = a.nseg > 1 && a.h0 ? a.seg + (a.nseg - 1) * slot : a.h0;
        if (a.combined) h0 = seg || a.h0 ? a.seg + seg * slot : nullptr;
        if (h0) {
            const auto d = ssm::rsrc(h0 + state, sbytes);
            each_state([&](floatx4& r, unsigned o, int left) { r = load_f4<VEC>(d, o, left); });
        }
        const Decay over(g, a.seglen);
        for (int p = 0; p < seg && !a.combined; ++p) {
            const auto d = ssm::rsrc(a.seg + p * slot + state, sbytes);
            each_state([&](floatx4& r, unsigned o, int left) {
                const floatx4 own = load_f4<VEC>(d, o, left);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = over.of_any(r[e]) + own[e];
            });
        }
    }
    __syncthreads();

    Decay decay;
    int wn = -1;
    int parity = 0;
    for (int t = t_begin; t < t_end; t += CB, parity ^= 1) {
        const int n = min(CB, t_end - t), g4 = fresh(lane_g), l16 = fresh(lane_i);
        if (wn != n) {   // (every wave is past its reads of the weights)
            wn = n;
            decay = Decay(g, n);
            if (tid < CB) s.wj[tid] = ssm::ex2(gl * (float)max(0, n - 1 - tid));
        }
        // ---- staging
        u16x2 most = {0, 0};
#pragma unroll
        for (int u = 0; u < NK; ++u) {
            *reinterpret_cast<uint4*>(&s.k[krow + RK * u][kcol]) = rk[u];
            if constexpr (!STATE) *reinterpret_cast<uint4*>(&s.q[krow + RK * u][kcol]) = rq[u];
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            *reinterpret_cast<uint4*>(&s.v[vrow + RV * u][vcol]) = rv[u];
            if constexpr (!STATE)
                most = most_bf16(most_bf16(most_bf16(most_bf16(most, rv[u].x), rv[u].y), rv[u].z), rv[u].w);
        }
        if (!STATE && max(most.x, most.y) >= 0x7f80) s.odd[parity] = 1;
        __syncthreads();
        if (t + CB < t_end) fetch(t + CB);
        floatx4 Y[STATE ? 1 : VW][4];
        bool any_odd = false;
        float now = decay.m, keep = decay.keep;
        auto each = [&](auto&& f) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int x = 0; x < VW; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float e = S[kt][x][r];
                        f(e);
                        S[kt][x][r] = e;
                    }
        };
        if constexpr (!STATE) {
            any_odd = s.odd[parity] != 0;
            if (tid == 0) s.odd[parity ^ 1] = 0;   // (the next chunk sets it past two barriers)
            // ---- q k^T: wave w forms the rows i of tile w, j up to the diagonal
            auto products = [&](auto wave) {
                constexpr int W = decltype(wave)::value;
                bf16x8 qf[KB];
                floatx4 acc[W + 1];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    qf[kb] = *reinterpret_cast<const bf16x8*>(&s.q[16 * W + l16][32 * kb + 8 * g4]);
#pragma unroll
                for (int jt = 0; jt <= W; ++jt) acc[jt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int jt = 0; jt <= W; ++jt)
                        acc[jt] = mfma(*reinterpret_cast<const bf16x8*>(&s.k[16 * jt + l16][32 * kb + 8 * g4]),
                                       qf[kb], acc[jt]);
                const float* dec = &s.dec[64 - l16 + 4 * g4];
                __bf16* pr = &s.p[0][16 * W + l16][4 * g4];
#pragma unroll
                for (int jt = 0; jt <= (W | 1); ++jt) {
                    Parts p[2] = {};
                    if (jt <= W) {
                        float f[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            f[r] = acc[min(jt, W)][r] * dec[r - 16 * (W - jt)];
                            if (jt == W && l16 < 4 * g4 + r) f[r] = 0.f;
                        }
                        p[0] = split(f[0], f[1]);
                        p[1] = split(f[2], f[3]);
                    }
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        *reinterpret_cast<u32x2*>(pr + c * CB * PP + 16 * jt) = u32x2{p[0].u[c], p[1].u[c]};
                }
            };
            if (w == 0) products(std::integral_constant<int, 0>{});
            else if (w == 1) products(std::integral_constant<int, 1>{});
            else if (w == 2) products(std::integral_constant<int, 2>{});
            else products(std::integral_constant<int, 3>{});
            // ---- S q^T, the next block's q read ahead of each block's products
            bf16x8 qf[2][4];
            auto q_tiles = [&](bf16x8 (&f)[4], int kb) {
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const __bf16* qr = &s.q[16 * it + l16][32 * kb + 4 * g4];
                    f[it] = cat(*reinterpret_cast<const bf16x4*>(qr), *reinterpret_cast<const bf16x4*>(qr + 16));
                }
            };
            auto state_products = [&](auto any) {
                q_tiles(qf[0], 0);
#pragma unroll
                for (int x = 0; x < VW; ++x)
#pragma unroll
                    for (int it = 0; it < 4; ++it) Y[x][it] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    if (kb + 1 < KB) q_tiles(qf[(kb + 1) & 1], kb + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    bf16x8 sf[3][VW];
#pragma unroll
                    for (int x = 0; x < VW; ++x) {
                        ssm::u32x4 u[3];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const floatx4& t = S[2 * kb + (e >> 1)][x];
                            const Parts p = split<decltype(any)::value>(t[2 * (e & 1)], t[2 * (e & 1) + 1]);
#pragma unroll
                            for (int c = 0; c < 3; ++c) u[c][e] = p.u[c];
                        }
#pragma unroll
                        for (int c = 0; c < 3; ++c) sf[c][x] = __builtin_bit_cast(bf16x8, u[c]);
                    }
#pragma unroll
                    for (int c = 2; c >= 0; --c)
#pragma unroll
                        for (int it = 0; it < 4; ++it)
#pragma unroll
                            for (int x = 0; x < VW; ++x) Y[x][it] = mfma(sf[c][x], qf[kb & 1][it], Y[x][it]);
                }
            };
            state_products(std::false_type{});
            // An infinite state makes all outputs of its row NaN there: then once more, with the state taken
            // apart as it is, and decayed here (the decay below is then one half and one half).
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < VW; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum = fmaf(Y[x][0][r], 0.f, sum);
            if (__any(sum != 0.f)) {
                state_products(std::true_type{});
                each([&](float& x) { x = decay.of_any(x); });
                keep = now = 0.5f;
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const float f = s.dec[63 - 16 * it - l16];
#pragma unroll
                for (int x = 0; x < VW; ++x) Y[x][it] *= f;
            }
            __syncthreads();
        }

        auto v_tile = [&](int jb, int x) {
            const int col = 16 * (VW * w + x);
            return cat(tr_read<VP>(&s.v[0][0], 32 * jb + 8 * g4, col, l16),
                       tr_read<VP>(&s.v[0][0], 32 * jb + 8 * g4 + 4, col, l16));
        };
        // ---- P v
        if constexpr (!STATE) {
            if (!any_odd) {
#pragma unroll
                for (int jb = 0; jb < 2; ++jb) {
                    bf16x8 vf[VW], pf[3][4];
#pragma unroll
                    for (int x = 0; x < VW; ++x) vf[x] = v_tile(jb, x);
#pragma unroll
                    for (int c = 0; c < 3; ++c)
#pragma unroll
                        for (int it = 2 * jb; it < 4; ++it)
                            pf[c][it] = *reinterpret_cast<const bf16x8*>(&s.p[c][16 * it + l16][32 * jb + 8 * g4]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 2; c >= 0; --c)
#pragma unroll
                        for (int it = 2 * jb; it < 4; ++it)
#pragma unroll
                            for (int x = 0; x < VW; ++x) Y[x][it] = mfma(vf[x], pf[c][it], Y[x][it]);
                }
            }
        }
        if constexpr (!STATE) {
            if (any_odd) {
                // an inf or NaN in v: term by term, so that a zero weight never meets it
#pragma unroll
                for (int x = 0; x < VW; ++x)
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int i = 16 * it + l16;
                        for (int j = 0; j <= i; ++j) {
                            const float p = (float)s.p[0][i][j] + ((float)s.p[1][i][j] + (float)s.p[2][i][j]);
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                Y[x][it][r] = fmaf(p, (float)s.v[j][16 * (VW * w + x) + 4 * g4 + r], Y[x][it][r]);
                        }
                    }
            }
            const auto dy = ssm::rsrc(static_cast<__bf16*>(a.y) + ((long)b * a.L + t) * a.ldy + (long)h * a.V,
                                      bytes(a.ldy, a.V, n));
#pragma unroll
            for (int x = 0; x < VW; ++x) {
                const int v = v0 + 16 * x + 4 * g4;
                const unsigned o0 = v < a.V ? ((unsigned)l16 * (unsigned)a.ldy + v) * 2u : kOut;
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const unsigned o = o0 + (unsigned)it * ((unsigned)a.ldy * 32u);
                    bf16x4 y;
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = (__bf16)Y[x][it][r];
                    if constexpr (VEC) {
                        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, y), dy, o, 0, 0);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const __bf16 e = y[r];   // (a bit_cast of the element itself reads [0])
                            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, e), dy,
                                                                  v + r < a.V ? o + 2u * r : kOut, 0, 0);
                        }
                    }
                }
            }
        }
        // ---- the state
        each([&](float& x) { x = STATE ? decay.of_any(x) : decayed(x, now, keep); });
        constexpr int KH = KT / 2;
#pragma unroll
        for (int jb = 0; jb < 2; ++jb) {
            bf16x8 kf[KH], parts[VW][3];
            auto k_tiles = [&](int kt0) {
#pragma unroll
                for (int kt = 0; kt < KH; ++kt)
                    kf[kt] = cat(tr_read<KP>(&s.k[0][0], 32 * jb + 8 * g4, 16 * (kt0 + kt), l16),
                                 tr_read<KP>(&s.k[0][0], 32 * jb + 8 * g4 + 4, 16 * (kt0 + kt), l16));
            };
            bf16x8 vf[VW];
#pragma unroll
            for (int x = 0; x < VW; ++x) vf[x] = v_tile(jb, x);
            const floatx4 wa = *reinterpret_cast<const floatx4*>(&s.wj[32 * jb + 8 * g4]);
            const floatx4 wb = *reinterpret_cast<const floatx4*>(&s.wj[32 * jb + 8 * g4 + 4]);
            k_tiles(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < VW; ++x) {
                ssm::u32x4 u[3];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const floatx4& wt = e < 4 ? wa : wb;
                    const Parts p = split((float)vf[x][e] * wt[e & 3], (float)vf[x][e + 1] * wt[(e & 3) + 1]);
#pragma unroll
                    for (int c = 0; c < 3; ++c) u[c][e / 2] = p.u[c];
                }
#pragma unroll
                for (int c = 0; c < 3; ++c) parts[x][c] = __builtin_bit_cast(bf16x8, u[c]);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int c = 2; c >= 0; --c)
#pragma unroll
                    for (int kt = 0; kt < KH; ++kt)
#pragma unroll
                        for (int x = 0; x < VW; ++x)
                            S[KH * half + kt][x] = mfma(kf[kt], parts[x][c], S[KH * half + kt][x]);
                if (half == 0) k_tiles(KH);
            }
            __builtin_amdgcn_sched_barrier(0);
        }

        __syncthreads();
    }

    float* to = STATE ? (last ? nullptr : a.seg + seg * slot) : (last ? a.hT : nullptr);
    if (to) {
        const auto d = ssm::rsrc(to + state, sbytes);
        each_state([&](floatx4& r, unsigned o, int left) { store_f4<VEC>(d, o, r, left); });
    }
}

// ---------------------------------------------------------------- fp32
// The same on v_mfma_f32_16x16x4_f32 (A: row lane % 16, k lane / 16; D as above), every product
// and sum in fp32. Chunks of 32: the quadratic part shrinks with the chunk, and a chunk costs
// nothing else, as S stays in the accumulators. MFMA r of a 16-k block takes k = 4 (lane / 16) + r
// from every lane, so that S and the products q k^T are read as they lie in the accumulators and
// q and k as 16-byte pieces. Bound by the matrix cores: 8 sequences of 4096 tokens, 16 heads, K = V = 128 take
// 530 us, 101 TFLOP/s of the 154 that a large product reaches (5.5 K V + 48 (K + V) operations a token, the
// state pass's among them).
constexpr int CF = 32;

template <int KD, int VT, bool STATE>
struct SmemF {
    static constexpr int KP = KD + 4, VP = VT + 4, PP = CF + 4, Y = STATE ? 1 : CF;
    alignas(16) float q[Y][KP];
    alignas(16) float k[CF][KP];
    alignas(16) float v[CF][VP];
    alignas(16) float p[Y][PP];
    int odd[2];
};

__device__ __forceinline__ floatx4 mfma4(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <int KD, int VT, bool VEC, bool STATE>
__global__ __launch_bounds__(256, KD == 256 ? 1 : 2) void la_f32_kernel(LaArgs a) {
    using Smem = SmemF<KD, VT, STATE>;
    constexpr int KT = KD / 16, VW = VT / 64;
    constexpr int NK = CF * KD / 4 / 256, NV = CF * VT / 4 / 256;
    __shared__ Smem s;

    const Place place(a);
    const int part = place.part, h = place.h, grp = place.grp, b = place.b, seg = place.seg;
    if (seg >= a.nseg - STATE) return;
    const int len = seq_len(a, b);
    const int t_begin = seg * a.seglen, t_end = min(len, t_begin + a.seglen);
    const bool last = seg == (len > 0 ? (len - 1) / a.seglen : 0);
    // (the first segment's state pass also copies h0: hT may alias it, and the last segment may end
    // before another begins)
    const bool copy = STATE && seg == 0 && a.h0;
    if (STATE ? (last || t_begin >= len) && !copy : !last && t_begin >= len) return;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g4 = lane >> 4, l16 = lane & 15;
    const int v0 = part * VT + 16 * VW * w;
    const float g = clamp_g(a.g[h]), gl = g * ssm::kLog2e;
    const long state = ((long)b * a.H + h) * a.V * a.K;
    const long slot = (long)a.B * a.H * a.V * a.K;

    floatx4 S[KT][VW];
    const unsigned sbytes = (unsigned)(a.V * a.K) * 4u;
    auto each_state = [&](auto&& f) {
        const int vl = v0 + fresh(l16), kl = 4 * fresh(g4);
#pragma unroll
        for (int x = 0; x < VW; ++x)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
                f(S[kt][x], (unsigned)((vl + 16 * x) * a.K + kl + 16 * kt) * 4u,
                  vl + 16 * x < a.V ? a.K - kl - 16 * kt : 0);
    };
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int x = 0; x < VW; ++x) S[kt][x] = floatx4{0.f, 0.f, 0.f, 0.f};
    floatx4 rq[STATE ? 1 : NK], rk[NK], rv[NV];
    auto base = [&](const void* p, long ld, int head, int width, int t) {
        return static_cast<const float*>(p) + ((long)b * a.L + t) * ld + (long)head * width;
    };
    auto bytes = [&](long ld, int width, int n) {
        return n > 0 ? (unsigned)(((long)(n - 1) * ld + width) * 4) : 0u;
    };
    auto fetch = [&](int t) {
        const int n = max(0, min(CF, t_end - t));
        const int tt = min(t, a.L - 1), ft = fresh(tid);
        const auto dk = ssm::rsrc(base(a.k, a.ldk, grp, a.K, tt), bytes(a.ldk, a.K, n));
        const auto dv = ssm::rsrc(base(a.v, a.ldv, grp, a.V, tt), bytes(a.ldv, a.V, n));
#pragma unroll
        for (int u = 0; u < NK; ++u) {
            const int e = ft + 256 * u, row = e / (KD / 4), col = e % (KD / 4) * 4;
            rk[u] = load_f4<VEC>(dk, ((unsigned)row * (unsigned)a.ldk + col) * 4u, a.K - col);
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int e = ft + 256 * u, row = e / (VT / 4), col = part * VT + e % (VT / 4) * 4;
            rv[u] = load_f4<VEC>(dv, ((unsigned)row * (unsigned)a.ldv + col) * 4u, a.V - col);
        }
        if constexpr (!STATE) {
            const auto dq = ssm::rsrc(base(a.q, a.ldq, h, a.K, tt), bytes(a.ldq, a.K, n));
#pragma unroll
            for (int u = 0; u < NK; ++u) {
                const int e = ft + 256 * u, row = e / (KD / 4), col = e % (KD / 4) * 4;
                rq[u] = load_f4<VEC>(dq, ((unsigned)row * (unsigned)a.ldq + col) * 4u, a.K - col);
            }
        }
    };
    if (copy) {
        const auto from = ssm::rsrc(a.h0 + state, sbytes);
        const auto to = ssm::rsrc(a.seg + (a.nseg - 1) * slot + state, sbytes);
        each_state([&](floatx4&, unsigned o, int left) {
            store_f4<VEC>(to, o, load_f4<VEC>(from, o, left), left);
        });
        if (last) return;
    }
    if (tid < 2) s.odd[tid] = 0;
    if (t_begin < t_end) fetch(t_begin);
    if (!STATE) {
        // h0 (where there are segments, its copy), then the segments' own states, each decayed by a
        // segment's length; or the sum that the combine pass left
        const float* h0 = a.nseg > 1 && a.h0 ? a.seg + (a.nseg - 1) * slot : a.h0;
        if (a.combined) h0 = seg || a.h0 ? a.seg + seg * slot : nullptr;
        if (h0) {
            const auto d = ssm::rsrc(h0 + state, sbytes);
            each_state([&](floatx4& r, unsigned o, int left) { r = load_f4<VEC>(d, o, left); });
        }
        const Decay over(g, a.seglen);
        for (int p = 0; p < seg && !a.combined; ++p) {
            const auto d = ssm::rsrc(a.seg + p * slot + state, sbytes);
            each_state([&](floatx4& r, unsigned o, int left) {
                const floatx4 own = load_f4<VEC>(d, o, left);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = over.of_any(r[e]) + own[e];
            });
        }
    }
    __syncthreads();

    float wj[2][4];
    Decay decay;
    int wn = -1;
    int parity = 0;
    for (int t = t_begin; t < t_end; t += CF, parity ^= 1) {
        const int n = min(CF, t_end - t);
        const int ft = fresh(tid);
        bool odd = false;
#pragma unroll
        for (int u = 0; u < NK; ++u) {
            const int e = ft + 256 * u, row = e / (KD / 4), col = e % (KD / 4) * 4;
            *reinterpret_cast<floatx4*>(&s.k[row][col]) = rk[u];
            if constexpr (!STATE) *reinterpret_cast<floatx4*>(&s.q[row][col]) = rq[u];
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int e = ft + 256 * u, row = e / (VT / 4), col = e % (VT / 4) * 4;
            *reinterpret_cast<floatx4*>(&s.v[row][col]) = rv[u];
            if constexpr (!STATE) {
#pragma unroll
                for (int c = 0; c < 4; ++c) odd |= !(fabsf(rv[u][c]) < INFINITY);
            }
        }
        if (!STATE && odd) s.odd[parity] = 1;
        __syncthreads();
        if (t + CF < t_end) fetch(t + CF);
        if (wn != n) {
            wn = n;
            decay = Decay(g, n);
#pragma unroll
            for (int jt = 0; jt < 2; ++jt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    wj[jt][r] = ssm::ex2(gl * (float)max(0, n - 1 - (16 * jt + 4 * g4 + r)));
        }

        floatx4 Y[STATE ? 1 : VW][2];
        bool any_odd = false;
        float now = decay.m, keep = decay.keep;
        auto each = [&](auto&& f) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int x = 0; x < VW; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float e = S[kt][x][r];
                        f(e);
                        S[kt][x][r] = e;
                    }
        };
        if constexpr (!STATE) {
            any_odd = s.odd[parity] != 0;
            if (tid == 0) s.odd[parity ^ 1] = 0;
            // ---- q k^T: wave 0 tile (j 0, i 0), wave 1 (0, 1), wave 2 (1, 1); (1, 0) is masked
            if (w < 3) {
                const int jt = w >> 1, it = w > 0;
                floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const floatx4 kf = *reinterpret_cast<const floatx4*>(&s.k[16 * jt + l16][16 * kt + 4 * g4]);
                    const floatx4 qf = *reinterpret_cast<const floatx4*>(&s.q[16 * it + l16][16 * kt + 4 * g4]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc = mfma4(kf[r], qf[r], acc);
                }
                const int i = 16 * it + l16;
                floatx4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int gap = i - (16 * jt + 4 * g4 + r);
                    const float f = a.scale * ssm::ex2(gl * (float)max(gap, 0));
                    o[r] = gap >= 0 ? acc[r] * f : 0.f;
                }
                *reinterpret_cast<floatx4*>(&s.p[i][16 * jt + 4 * g4]) = o;
            }
            // ---- S q^T
#pragma unroll
            for (int x = 0; x < VW; ++x)
#pragma unroll
                for (int it = 0; it < 2; ++it) Y[x][it] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int it = 0; it < 2; ++it) {
                    const floatx4 qf = *reinterpret_cast<const floatx4*>(&s.q[16 * it + l16][16 * kt + 4 * g4]);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int x = 0; x < VW; ++x) Y[x][it] = mfma4(S[kt][x][r], qf[r], Y[x][it]);
                }
            // (as in the bf16 kernel; the products need no change)
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < VW; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum = fmaf(Y[x][0][r], 0.f, sum);
            if (__any(sum != 0.f)) {
                each([&](float& x) { x = decay.of_any(x); });
                keep = now = 0.5f;
            }
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const float f = a.scale * ssm::ex2(fresh(gl) * (float)(16 * it + l16 + 1));
#pragma unroll
                for (int x = 0; x < VW; ++x) Y[x][it] *= f;
            }
            __syncthreads();
        }

        each([&](float& x) { x = STATE ? decay.of_any(x) : decayed(x, now, keep); });
#pragma unroll
        for (int jt = 0; jt < 2; ++jt) {
            float vf[VW][4];
#pragma unroll
            for (int x = 0; x < VW; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    vf[x][r] = s.v[16 * jt + 4 * g4 + r][16 * (VW * w + x) + l16];
            if constexpr (!STATE) {
                if (!any_odd) {
#pragma unroll
                    for (int it = jt; it < 2; ++it) {
                        const floatx4 pf = *reinterpret_cast<const floatx4*>(&s.p[16 * it + l16][16 * jt + 4 * g4]);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int x = 0; x < VW; ++x) Y[x][it] = mfma4(vf[x][r], pf[r], Y[x][it]);
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < VW; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) vf[x][r] *= wj[jt][r];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                float kf[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) kf[r] = s.k[16 * jt + 4 * g4 + r][16 * kt + l16];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int x = 0; x < VW; ++x) S[kt][x] = mfma4(kf[r], vf[x][r], S[kt][x]);
            }
        }

        if constexpr (!STATE) {
            if (any_odd) {
#pragma unroll
                for (int x = 0; x < VW; ++x)
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        const int i = 16 * it + l16;
                        for (int j = 0; j <= i; ++j) {
                            const float p = s.p[i][j];
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                Y[x][it][r] = fmaf(p, s.v[j][16 * (VW * w + x) + 4 * g4 + r], Y[x][it][r]);
                        }
                    }
            }
            const auto dy = ssm::rsrc(static_cast<float*>(a.y) + ((long)b * a.L + t) * a.ldy + (long)h * a.V,
                                      bytes(a.ldy, a.V, n));
#pragma unroll
            for (int it = 0; it < 2; ++it)
#pragma unroll
                for (int x = 0; x < VW; ++x) {
                    const int v = v0 + 16 * x + 4 * g4;
                    store_f4<VEC>(dy, ((unsigned)(16 * it + l16) * (unsigned)a.ldy + v) * 4u, Y[x][it], a.V - v);
                }
        }
        __syncthreads();
    }

    float* to = STATE ? (last ? nullptr : a.seg + seg * slot) : (last ? a.hT : nullptr);
    if (to) {
        const auto d = ssm::rsrc(to + state, sbytes);
        each_state([&](floatx4& r, unsigned o, int left) { store_f4<VEC>(d, o, r, left); });
    }
}

// Entering states of many segments: slot s <- E_s, E_0 = h0 (its copy in the last slot) or 0, E_{s+1} =
// e^{g seglen} E_s + own state of s.
__global__ __launch_bounds__(256) void la_combine_kernel(LaArgs a) {
    const long VK = (long)a.V * a.K, slot = (long)a.B * a.H * VK;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= slot) return;
    const int bh = (int)(i / VK), h = bh % a.H, b = bh / a.H;
    const int len = seq_len(a, b);
    const int used = len > 0 ? (len - 1) / a.seglen + 1 : 1;   // segments that run
    const float x = clamp_g(a.g[h]) * (float)a.seglen;   // (threads of a wave may be of several heads)
    const bool slow = !(x < -0.69f);
    const float m = slow ? expm1f(x) : expf(x), keep = slow ? 1.f : 0.f;
    float* p = a.seg + i;
    float e = a.h0 ? p[(a.nseg - 1) * slot] : 0.f;
    float own = used > 1 ? p[0] : 0.f;   // (own states are read before E takes their slot)
    if (a.h0) p[0] = e;
    constexpr int U = 8;   // loads in flight (16 and 32: 2% of the whole longer)
    for (int sgm = 0; sgm < used - 1; sgm += U) {
        float next[U];
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = sgm + u + 2 < used ? p[(sgm + u + 1) * slot] : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (sgm + u + 1 >= used) break;
            e = decayed_any(e, m, keep) + own;
            p[(sgm + u + 1) * slot] = e;
            own = next[u];
        }
    }
}

// ---------------------------------------------------------------- plan
// Segments: as many as fill the chip once, two workgroups a CU (one more turn for the rest costs as much
// as a whole one: 80 sequences and heads of 4096 tokens take 163 us in 7 segments, 158 in 6), each of
// at least so many tokens that its states' traffic stays small beside its rows'. bf16: 512 where that
// leaves a workgroup for every CU (128 sequences and heads of 1024: 71 us, 73 in segments of 256), else 256.
// fp32 chunks take longer on the matrix cores: 64 (24 of 2000: 83 us, 95 in segments of 256).
//
// Columns of V a workgroup: 128, which share a chunk's q k^T and its rows of q and k (512 sequences and
// heads of 4096 tokens: 624 us, 765 in parts of 64). 64 where V or the registers (K above 128) ask for
// it; where whole sequences fill the chip in parts of 64 and need no state pass (256 sequences and heads
// of 1500 tokens: 144 us, 149 in two segments of 128 columns; of 4096: 385, 398); and where the shortest
// segments would leave CUs idle (8 of 4096: 38 us, 46).
constexpr int kSlots = 512, kCUs = 256;
struct LaPlan { int nseg, seglen, vt, vparts; };
LaPlan la_plan(int dtype, int B, int L, int H, int K, int V) {
    const int C = dtype == SSM_F32 ? CF : CB;
    const long heads = (long)B * H, len = std::max(L, 1), by512 = ssm::cdiv(len, 512);
    const long half = heads * ssm::cdiv(V, 64), full = heads * ssm::cdiv(V, 128);
    const long shortest = ssm::cdiv(len, dtype == SSM_F32 ? 64 : 256);
    LaPlan p;
    p.vt = V <= 64 || K > 128 || (half <= kSlots && 4 * half > 3 * kSlots) || full * shortest < kCUs ? 64 : 128;
    p.vparts = (int)ssm::cdiv(V, p.vt);
    const long wgs = std::max(heads * p.vparts, 1L), fit = std::max(kSlots / wgs, 1L);
    const long most = dtype != SSM_F32 && by512 * wgs >= kCUs ? by512 : shortest;
    const long n = std::min(fit, most);
    p.seglen = (int)(ssm::cdiv(ssm::cdiv(len, n), C) * C);
    p.nseg = (int)std::max(1L, ssm::cdiv(L, p.seglen));
    return p;
}

// A chain of more segments than this is combined once, by a pass of its own (8 sequences of 1500 tokens, 16
// heads, 3 segments: 97 us in a chain, 107 combined; 24 heads of 4096 tokens, 16 segments: 98 and 71).
constexpr int kChain = 4;

template <int KD, int VT, bool VEC>
ssm_status la_launch(int dtype, LaArgs a, hipStream_t st) {
    if (a.nseg > 1) {
        // 64 columns a workgroup, whatever the full pass takes: half the registers, so that more of
        // them share a CU
        LaArgs s = a;
        s.vparts = (int)ssm::cdiv(a.V, 64);
        const unsigned n1 = la_groups(s, a.nseg - 1);
        if (dtype == SSM_F32) la_f32_kernel<KD, 64, VEC, true><<<n1, 256, 0, st>>>(s);
        else la_bf16_kernel<KD, 64, VEC, true><<<n1, 256, 0, st>>>(s);
        if (ssm_status e = ssm::check_launch("ssm_linear_attention (states)")) return e;
        a.combined = a.nseg > kChain;
        if (a.combined) {
            const long m = (long)a.B * a.H * a.V * a.K;
            la_combine_kernel<<<(unsigned)ssm::cdiv(m, 256), 256, 0, st>>>(a);
            if (ssm_status e = ssm::check_launch("ssm_linear_attention (combine)")) return e;
        }
    }
    const unsigned n = la_groups(a, a.nseg);
    if (dtype == SSM_F32) la_f32_kernel<KD, VT, VEC, false><<<n, 256, 0, st>>>(a);
    else la_bf16_kernel<KD, VT, VEC, false><<<n, 256, 0, st>>>(a);
    return ssm::check_launch("ssm_linear_attention");
}

template <bool VEC>
ssm_status la_dispatch(int dtype, const LaArgs& a, int vt, hipStream_t st) {
    if (a.K > 128) return la_launch<256, 64, VEC>(dtype, a, st);
    if (a.K > 64) return vt == 64 ? la_launch<128, 64, VEC>(dtype, a, st)
                                  : la_launch<128, 128, VEC>(dtype, a, st);
    return vt == 64 ? la_launch<64, 64, VEC>(dtype, a, st) : la_launch<64, 128, VEC>(dtype, a, st);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// ---------------------------------------------------------------- one token
// S is read and written once: memory bound (64 sequences of 32 heads, K = V = 128, 270 MB: 51 us, 5.3
// TB/s), past the caches, as the next token's call comes after the layer's other work. 16 lanes hold a row of S (LV x 64 columns in float4
// pieces, or one by one), a wave four rows, a workgroup 16 RV rows of one (sequence, head); the
// loads of all RV rows are in flight before the first is used.
struct LaStepArgs {
    const void* q; long ldq;
    const void* k; long ldk;
    const void* v; long ldv;
    const float* g;
    float scale;
    void* y; long ldy;
    int H, G, K, V, blocks;
    float* h;
};

template <typename T, int KU, int RV, bool VEC>
__global__ __launch_bounds__(256) void la_step_kernel(LaStepArgs a) {
    constexpr int E = 4 * KU;   // columns per lane
    const int l16 = threadIdx.x & 15, row = threadIdx.x >> 4;
    const int blk = blockIdx.x % a.blocks, bh = blockIdx.x / a.blocks;
    const int h = bh % a.H, b = bh / a.H, grp = h / (a.H / a.G);
    const int v0 = blk * 16 * RV + row;
    float* S = a.h + (long)bh * a.V * a.K;
    // column of element e of the lane
    auto col = [&](int e) { return VEC ? 64 * (e >> 2) + 4 * l16 + (e & 3) : 16 * e + l16; };
    float s[RV][E];
#pragma unroll
    for (int r = 0; r < RV; ++r) {
        const int v = v0 + 16 * r;
        const float* p = S + (long)min(v, a.V - 1) * a.K;
        if constexpr (VEC) {
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                const float4 x = col(4 * u) < a.K ? ssm::load_nt4(p + col(4 * u)) : make_float4(0.f, 0.f, 0.f, 0.f);
                s[r][4 * u] = x.x; s[r][4 * u + 1] = x.y; s[r][4 * u + 2] = x.z; s[r][4 * u + 3] = x.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) s[r][e] = col(e) < a.K ? p[col(e)] : 0.f;
        }
    }
    const T* qp = static_cast<const T*>(a.q) + b * a.ldq + (long)h * a.K;
    const T* kp = static_cast<const T*>(a.k) + b * a.ldk + (long)grp * a.K;
    const T* vp = static_cast<const T*>(a.v) + b * a.ldv + (long)grp * a.V;
    float q[E], k[E], vv[RV];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool in = col(e) < a.K;
        q[e] = in ? (float)qp[col(e)] : 0.f;
        k[e] = in ? (float)kp[col(e)] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < RV; ++r) vv[r] = (float)vp[min(v0 + 16 * r, a.V - 1)];
    const Decay decay(clamp_g(a.g[h]), 1);
    float o[RV];
#pragma unroll
    for (int r = 0; r < RV; ++r) {
        float acc = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            s[r][e] = fmaf(vv[r], k[e], decay.of_any(s[r][e]));
            acc = fmaf(s[r][e], q[e], acc);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 16);
        o[r] = acc * a.scale;
    }
    T* yp = static_cast<T*>(a.y) + b * a.ldy + (long)h * a.V;
#pragma unroll
    for (int r = 0; r < RV; ++r) {
        const int v = v0 + 16 * r;
        if (v >= a.V) continue;
        float* p = S + (long)v * a.K;
        if constexpr (VEC) {
#pragma unroll
            for (int u = 0; u < KU; ++u)
                if (col(4 * u) < a.K)
                    ssm::store_nt4(make_float4(s[r][4 * u], s[r][4 * u + 1], s[r][4 * u + 2], s[r][4 * u + 3]),
                                   p + col(4 * u));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (col(e) < a.K) p[col(e)] = s[r][e];
        }
        if (l16 == 0) yp[v] = (T)o[r];
    }
}

template <typename T, int KU, int RV>
void step_launch(const LaStepArgs& a, bool vec, unsigned n, hipStream_t st) {
    if (vec) la_step_kernel<T, KU, RV, true><<<n, 256, 0, st>>>(a);
    else la_step_kernel<T, KU, RV, false><<<n, 256, 0, st>>>(a);
}

template <typename T, int KU>
void step_rows(const LaStepArgs& a, int rv, bool vec, unsigned n, hipStream_t st) {
    if (rv == 4) step_launch<T, KU, 4>(a, vec, n, st);
    else step_launch<T, KU, 1>(a, vec, n, st);
}

template <typename T>
void step_dispatch(const LaStepArgs& a, int rv, bool vec, unsigned n, hipStream_t st) {
    if (a.K <= 64) step_rows<T, 1>(a, rv, vec, n, st);
    else if (a.K <= 128) step_rows<T, 2>(a, rv, vec, n, st);
    else step_rows<T, 4>(a, rv, vec, n, st);
}

}  // namespace

extern "C" size_t ssm_linear_attention_workspace(int dtype, int B, int L, int H, int K, int V) {
    if (B <= 0 || L <= 0 || H <= 0 || K <= 0 || V <= 0) return 0;
    const int nseg = la_plan(dtype, B, L, H, K, V).nseg;
    return nseg > 1 ? sizeof(float) * (size_t)nseg * B * H * V * K : 0;
}

extern "C" ssm_status ssm_linear_attention(int dtype, const void* q, long ldq, const void* k,
                                           long ldk, const void* v, long ldv, const float* g,
                                           float scale, const int* lengths, void* y, long ldy,
                                           int B, int L, int H, int G, int K, int V,
                                           const float* h0, float* hT, void* workspace,
                                           size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_linear_attention: bad dtype");
    SSM_REQUIRE(B >= 0 && L >= 0 && H > 0 && G > 0 && H % G == 0 && K > 0 && V > 0,
                "ssm_linear_attention: bad shape");
    if (K > 256)
        return ssm::fail(SSM_ERR_UNSUPPORTED, "ssm_linear_attention: head dim %d of the keys above 256", K);
    if (B == 0) return SSM_OK;
    SSM_REQUIRE(g && (L == 0 || (q && k && v && y)), "ssm_linear_attention: null input");
    SSM_REQUIRE(L == 0 || (ldq >= (long)H * K && ldk >= (long)G * K && ldv >= (long)G * V &&
                           ldy >= (long)H * V),
                "ssm_linear_attention: row stride below row width");
    const long esz = dtype == SSM_F32 ? 4 : 2, ev = 16 / esz;
    const long lim = (1L << 31) / (CB * esz);   // a chunk's byte offsets are 32-bit
    SSM_REQUIRE(ldq < lim && ldk < lim && ldv < lim && ldy < lim, "ssm_linear_attention: row stride too large");
    LaArgs a{};
    a.q = q; a.ldq = ldq; a.k = k; a.ldk = ldk; a.v = v; a.ldv = ldv; a.g = g; a.scale = scale;
    a.lengths = lengths; a.y = y; a.ldy = ldy; a.B = B; a.L = L; a.H = H; a.G = G; a.K = K; a.V = V;
    a.h0 = h0; a.hT = hT;
    const LaPlan plan = la_plan(dtype, B, L, H, K, V);
    a.nseg = plan.nseg;
    a.seglen = plan.seglen;
    a.vparts = plan.vparts;
    SSM_REQUIRE(L <= ssm::kMaxSteps, "ssm_linear_attention: too long");
    SSM_REQUIRE((long)V * K < (1L << 29), "ssm_linear_attention: state of a head too large");
    SSM_REQUIRE(((double)a.nseg * B + 7) * H * ssm::cdiv(V, 64) <= (double)ssm::kMaxGroups,
                "ssm_linear_attention: too many heads");
    if (a.nseg > 1) {
        const size_t need = ssm_linear_attention_workspace(dtype, B, L, H, K, V);
        SSM_REQUIRE(workspace && workspace_bytes >= need,
                    "ssm_linear_attention: workspace of %zu bytes needed", need);
        SSM_REQUIRE(aligned16(workspace), "ssm_linear_attention: workspace must be 16-byte aligned");
        a.seg = (float*)workspace;
    }
    auto rows = [&](const void* x, long ld, long wide) { return ssm::Rows{x, ld * esz, wide * esz, (long)B * L}; };
    const ssm::Rows rq = rows(q, ldq, (long)H * K), rk = rows(k, ldk, (long)G * K), rv = rows(v, ldv, (long)G * V),
                    ry = rows(y, ldy, (long)H * V), rg = ssm::block(g, 4L * H), rl = ssm::block(lengths, 4L * B),
                    from = ssm::block(h0, 4L * B * H * V * K), to = ssm::block(hT, 4L * B * H * V * K);
    SSM_REQUIRE(!ssm::meets(ry, rq, rk, rv, rg, rl, from), "ssm_linear_attention: y overlaps an input");
    SSM_REQUIRE(!ssm::meets(to, rq, rk, rv, rg, rl, ry) && (h0 == hT || !ssm::meet(to, from)),
                "ssm_linear_attention: hT overlaps y or an input that it is not");
    SSM_REQUIRE(a.nseg == 1 || !ssm::meets(ssm::block(workspace, ssm_linear_attention_workspace(dtype, B, L, H, K, V)),
                                           rq, rk, rv, rg, rl, ry, from, to),
                "ssm_linear_attention: the workspace overlaps another operand");
    const bool vec = K % ev == 0 && V % ev == 0 && (ldq | ldk | ldv | ldy) % ev == 0 &&
                     aligned16(q) && aligned16(k) && aligned16(v) && aligned16(y) &&
                     aligned16(h0) && aligned16(hT);
    return vec ? la_dispatch<true>(dtype, a, plan.vt, (hipStream_t)stream)
               : la_dispatch<false>(dtype, a, plan.vt, (hipStream_t)stream);
}

extern "C" ssm_status ssm_linear_attention_step(int dtype, const void* q, long ldq, const void* k,
                                                long ldk, const void* v, long ldv, const float* g,
                                                float scale, void* y, long ldy, float* h, int B,
                                                int H, int G, int K, int V, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_linear_attention_step: bad dtype");
    SSM_REQUIRE(B >= 0 && H > 0 && G > 0 && H % G == 0 && K > 0 && V > 0,
                "ssm_linear_attention_step: bad shape");
    if (K > 256)
        return ssm::fail(SSM_ERR_UNSUPPORTED, "ssm_linear_attention_step: head dim %d of the keys above 256", K);
    if (B == 0) return SSM_OK;
    SSM_REQUIRE(q && k && v && g && y && h, "ssm_linear_attention_step: null input");
    SSM_REQUIRE(B == 1 || (ldq >= (long)H * K && ldk >= (long)G * K && ldv >= (long)G * V &&
                           ldy >= (long)H * V),
                "ssm_linear_attention_step: row stride below row width");
    LaStepArgs a{q, ldq, k, ldk, v, ldv, g, scale, y, ldy, H, G, K, V, 0, h};
    // four rows a lane group where that still leaves a workgroup for every CU (K = V = 128: 64 sequences of
    // 32 heads 51 us, 68 with one row; one of 12 heads 3.8 us with one, 4.5 with four)
    const int rv = (long)B * H * ssm::cdiv(V, 64) >= 256 ? 4 : 1;
    a.blocks = (int)ssm::cdiv(V, 16 * rv);
    const long n = (long)B * H * a.blocks;
    SSM_REQUIRE(n <= ssm::kMaxGroups, "ssm_linear_attention_step: too many heads");
    const long es = dtype == SSM_F32 ? 4 : 2;
    auto rows = [&](const void* x, long ld, long wide) { return ssm::Rows{x, ld * es, wide * es, B}; };
    const ssm::Rows q_rows = rows(q, ldq, (long)H * K), k_rows = rows(k, ldk, (long)G * K),
                    v_rows = rows(v, ldv, (long)G * V), y_rows = rows(y, ldy, (long)H * V), decays = ssm::block(g, 4L * H);
    SSM_REQUIRE(!ssm::meets(y_rows, q_rows, k_rows, v_rows, decays),
                "ssm_linear_attention_step: y overlaps an input");
    SSM_REQUIRE(!ssm::meets(ssm::block(h, 4L * B * H * V * K), q_rows, k_rows, v_rows, decays, y_rows),
                "ssm_linear_attention_step: the state overlaps y or an input");
    const bool vec = K % 4 == 0 && aligned16(h);
    if (dtype == SSM_F32) step_dispatch<float>(a, rv, vec, (unsigned)n, (hipStream_t)stream);
    else step_dispatch<__bf16>(a, rv, vec, (unsigned)n, (hipStream_t)stream);
    return ssm::check_launch("ssm_linear_attention_step");
}

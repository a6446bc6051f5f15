// Log probabilities of given tokens, entropy and the likeliest tokens of rows of logits, in one pass over them, and
// their gradient. With m = max x, Z = sum e^{x-m}, S = sum e^{x-m} (x - m):
//   log p_j = x_j - m - log Z,   H = -sum p log p = log Z - S / Z
//   dx_j = w (delta_{j,id} - p_j) - v p_j (log p_j + H)   for the gradients w of log p_id and v of H
// A lane keeps its own (m, Z, S) and rescales it where m grows (Milakov & Gimelshein 2018); lanes, waves and
// slices of a row are joined the same way, in one order.
//
// Likeliest tokens: a wave keeps a list of 64 in its lanes, sorted by one key for each logit (larger for larger
// values and, of equal ones, for lower indices). The first 2048 logits give the maximum of each lane, sorted at once;
// from there on a logit enters only past the list's k-th, which few do: about k ln(n / 2048) of a random row.
//
// Memory bound: one read of the logits; the gradient reads and writes each once. 4096 x 50257 bf16 (odd rows at the
// elements' alignment) is read in 93 us (4.4 TB/s), in 121 to 127 behind a gradient's writes, and its gradient takes 151
// (5.4 TB/s), or 134 to 138 behind its forward call, with part of the logits still in the caches; 2047 x 32000 fp32 with five
// alternatives takes 52 us (5.0 TB/s). Lists bound bf16 rows, 45 us for 2047 x 32000 (2.9 TB/s), 117 for 4096 x 50257, and
// few rows: 64 x 128000 fp32 with 20 alternatives 15 us and 5 for the joining, without 7 and 3.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int kMaxTop = 64;
constexpr int kGroups = 4, kWaveRun = 64 * 8 * kGroups, kRun = 4 * kWaveRun;   // logits of a wave's and a workgroup's turn
constexpr float kFloor = -200.f;   // e^kFloor is 0 in fp32: differences are held above it where they multiply a 0
constexpr float kLowest = -3.40282347e38f;
typedef unsigned long long u64;

// Eight elements at p, from element `at` of a row of n on. WHOLE: rows of whole eights, all or none of which is there.
template <bool WHOLE> __device__ __forceinline__ bool inside(int at, int n) { return WHOLE ? at < n : at >= 0 && at <= n - 8; }
template <bool WHOLE> __device__ __forceinline__ void load8(const float* p, int at, int n, float (&f)[8]) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    if (inside<WHOLE>(at, n)) {
        const f4 a = reinterpret_cast<const f4*>(p)[0], b = reinterpret_cast<const f4*>(p)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = a[j], f[4 + j] = b[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = !WHOLE && (unsigned)(at + j) < (unsigned)n ? p[j] : -__builtin_inff();
    }
}
template <bool WHOLE> __device__ __forceinline__ void load8(const __bf16* p, int at, int n, float (&f)[8]) {
    typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(2)));
    if (inside<WHOLE>(at, n)) {
        const u4 a = *reinterpret_cast<const u4*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __builtin_bit_cast(float, j % 2 ? a[j / 2] & 0xffff0000u : a[j / 2] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = !WHOLE && (unsigned)(at + j) < (unsigned)n ? (float)p[j] : -__builtin_inff();
    }
}
template <bool WHOLE> __device__ __forceinline__ void store8(float* p, int at, int n, const float (&f)[8]) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    if (inside<WHOLE>(at, n)) {
        reinterpret_cast<f4*>(p)[0] = f4{f[0], f[1], f[2], f[3]};
        reinterpret_cast<f4*>(p)[1] = f4{f[4], f[5], f[6], f[7]};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!WHOLE && (unsigned)(at + j) < (unsigned)n) p[j] = f[j];
    }
}
template <bool WHOLE> __device__ __forceinline__ void store8(__bf16* p, int at, int n, const float (&f)[8]) {
    typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    if (inside<WHOLE>(at, n)) {
        b8 b;
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = (__bf16)f[j];
        *reinterpret_cast<u4*>(p) = __builtin_bit_cast(u4, b);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!WHOLE && (unsigned)(at + j) < (unsigned)n) p[j] = (__bf16)f[j];
    }
}
// Where a row of bf16 begins in its 16 bytes. The gradient takes rows from there on, with all but their first and last eight
// elements in place (us, eights from the row's first element on / this: 4096 x 32001 bf16 111 / 105, 4096 x 50257 152 / 152, with
// its forward call 262.4 / 261.7, 16000 x 5003 69 / 74; 2048 x 50257 fp32 156 / 163). The sums do not: their order would go by
// where a row lies.
template <bool WHOLE, typename T> __device__ __forceinline__ int lead(const T* row) {
    return WHOLE || sizeof(T) == 4 ? 0 : (int)((uintptr_t)row / sizeof(T) & 7);
}

// ---------------------------------------------------------------- sums
struct Sums {
    float m, z, s;
};
__device__ __forceinline__ float grow(float d) { return ssm::ex2(ssm::kLog2e * d); }   // e^d
__device__ __forceinline__ void raise(Sums& a, float m) {   // the same sums from a maximum m >= a.m
    const float d = fmaxf(a.m - m, kFloor), f = grow(d);
    a.s = f * fmaf(a.z, d, a.s);
    a.z *= f;
    a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    return Sums{m, a.z + b.z, a.s + b.s};
}
__device__ __forceinline__ void take8(Sums& a, const float (&x)[8]) {
    float m = a.m;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, x[j]);
    raise(a, m);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float d = x[j] - m, e = grow(d);
        a.z += e;
        a.s = fmaf(e, fmaxf(d, kFloor), a.s);
    }
}
__device__ __forceinline__ Sums over_wave(Sums a) {
#pragma unroll
    for (int k = 32; k > 0; k /= 2) a = join(a, Sums{__shfl_xor(a.m, k), __shfl_xor(a.z, k), __shfl_xor(a.s, k)});
    return a;
}

// ---------------------------------------------------------------- keys
// Larger for larger values and, of equal ones, for lower indices; never 0; a NaN below all else.
__device__ __forceinline__ u64 key_of(float x, unsigned index) {
    const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);   // (-0 equals 0)
    const unsigned o = x != x ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
    return (u64)o << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(u64 key) {
    const unsigned o = (unsigned)(key >> 32);
    return o == 0u ? __builtin_nanf("") : __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned index_of(u64 key) { return 0xffffffffu - (unsigned)key; }

__device__ __forceinline__ u64 shfl64(u64 v, int lane) {
    return (u64)(unsigned)__shfl((int)(v >> 32), lane) << 32 | (unsigned)__shfl((int)v, lane);
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {   // lane: the same in all lanes
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
// The key of lane ^ J (J a power of two): within a row of 16 lanes by the moves that the vector unit has.
template <int CTRL> __device__ __forceinline__ u64 moved(u64 v) {
    return (u64)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, true) << 32 |
           (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ u64 across(u64 v, int lane, int j) {   // j: a constant after unrolling
    switch (j) {
        case 1: return moved<0xb1>(v);                  // quad_perm 1 0 3 2
        case 2: return moved<0x4e>(v);                  // quad_perm 2 3 0 1
        case 4: return moved<0x1b>(moved<0x141>(v));    // row_half_mirror (^ 7), then quad_perm 3 2 1 0 (^ 3)
        case 8: return moved<0x128>(v);                 // row_ror 8
        default: return shfl64(v, lane ^ j);
    }
}
// The lanes' keys in descending order over the lanes.
__device__ __forceinline__ u64 sorted(u64 v, int lane) {
#pragma unroll
    for (int k = 2; k <= 64; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
            const u64 o = across(v, lane, j);
            const bool high = ((lane & j) == 0) == ((lane & k) == 0);   // this lane takes the larger one
            v = (v > o) == high ? v : o;
        }
    return v;
}
// The 64 largest of two sorted lists, sorted: the larger of each pair of one and the other's mirror, then six levels.
__device__ __forceinline__ u64 merged(u64 a, u64 b, int lane) {
    u64 o = shfl64(b, 63 - lane), v = a > o ? a : o;
#pragma unroll
    for (int j = 32; j > 0; j /= 2) {
        o = across(v, lane, j);
        v = (v > o) == ((lane & j) == 0) ? v : o;
    }
    return v;
}
// A key enters the sorted list, whose last one leaves it.
__device__ __forceinline__ u64 entered(u64 list, u64 key, int lane) {
    const int at = __popcll(__ballot(list > key));
    const u64 below = moved<0x138>(list);   // wave_shr 1
    return lane < at ? list : lane == at ? key : below;
}

struct LogArgs {
    const void* x; long ldx;
    const int* ids;
    float* logp; float* ent; float2* stats;
    int* top; float* toplp;
    Sums* sums; u64* keys;   // the slices' results
    int M, N, k, slices, turns;
};

// By one wave: a row's results from its sums and its sorted list (0: none).
template <typename T>
__device__ __forceinline__ void finish(const LogArgs& a, int row, Sums s, u64 list, int lane) {
    // (nothing left: Z = 0)
    const bool none = s.z == 0.f;
    const float m = fmaxf(s.m, kLowest), logz = none ? -__builtin_inff() : logf(s.z);
    if (lane == 0) {
        if (a.stats) a.stats[row] = make_float2(m, logz);
        const float h = logz - s.s / s.z;
        if (a.ent) a.ent[row] = none || h < 0.f ? 0.f : h;   // (below 0 by rounding)
        if (a.logp) {
            const int id = a.ids[row];
            const bool given = id >= 0 && id < a.N;
            a.logp[row] = !given ? 0.f : none ? -__builtin_inff() : ((float)static_cast<const T*>(a.x)[row * a.ldx + id] - m) - logz;
        }
    }
    if (lane < a.k) {
        a.top[(long)row * a.k + lane] = (int)index_of(list);
        a.toplp[(long)row * a.k + lane] = none ? -__builtin_inff() : (value_of(list) - m) - logz;
    }
}

// (waves a SIMD for its registers, us, five alternatives, 8 waves / 5: bf16 4096 x 50257 117 / 137, 2047 x 32000 45 / 51, but fp32
// 2047 x 32000 58 / 52)
template <typename T, bool TOP, bool WHOLE>
__global__ __launch_bounds__(256, TOP && sizeof(T) == 4 ? 5 : 8) void logprob_kernel(LogArgs a) {
    __shared__ Sums ws[4];
    __shared__ u64 lists[4][TOP ? 64 : 1];
    __shared__ alignas(16) float near[4][TOP ? 512 : 4];
    __shared__ int2 whose[4][TOP ? 64 : 1];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const int begin = slice * a.turns, end = begin + a.turns;
    Sums s{kLowest, 0.f, 0.f};
    u64 list = 0, least = 0;   // least: the k-th of the list
    float bar = 0.f;           // its value
    bool full = false;
    for (int turn = begin; turn < end; ++turn) {
        const int base = turn * kRun + w * kWaveRun;   // (below 2^31: N is at most 2^30)
        if (base >= a.N) break;
        float v[kGroups][8];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) load8<WHOLE>(x + base + (g * 64 + lane) * 8, base + (g * 64 + lane) * 8, a.N, v[g]);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) take8(s, v[g]);
        if constexpr (TOP) {
            int own = -1;
            if (!full) {   // the first turn: the lanes' maxima (any of a lane's logits would do)
                float most = v[0][0];
                int at = 0;
#pragma unroll
                for (int g = 0; g < kGroups; ++g)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool up = v[g][j] > most;
                        most = up ? v[g][j] : most;
                        at = up ? g * 512 + j : at;
                    }
                own = at + base + lane * 8;
                list = sorted(own < a.N ? key_of(most, own) : 0, lane);
                least = lane64(list, a.k - 1);
                bar = least ? value_of(least) : __builtin_nanf("");
            }
            // Lanes with a logit that may enter (of an unfilled list: equal ones too; later, all earlier logits of the wave
            // have lower indices) put their eight side by side, a logit a lane, and those that enter are taken from there.
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                bool some = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) some |= full ? !(v[g][j] <= bar) : !(v[g][j] < bar);
                const u64 lanes = __ballot(some);
                if (!lanes) continue;
                if (some) {
                    const int to = __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0));
                    float4* out = reinterpret_cast<float4*>(near[w] + 8 * to);
                    out[0] = make_float4(v[g][0], v[g][1], v[g][2], v[g][3]);
                    out[1] = make_float4(v[g][4], v[g][5], v[g][6], v[g][7]);
                    whose[w][to] = make_int2(base + (g * 64 + lane) * 8, own);
                }
                __builtin_amdgcn_wave_barrier();
                const int n = 8 * __popcll(lanes);
                for (int k = lane; k - lane < n; k += 64) {
                    u64 key = 0;
                    if (k < n) {
                        const int2 of = whose[w][k / 8];
                        const int at = of.x + k % 8;
                        if (at < a.N && at != of.y) key = key_of(near[w][k], at);   // (of.y: in the list)
                    }
                    u64 left = __ballot(key > least);
                    if (__popcll(left) > 8) {   // (an entry takes about an eighth of a sort and merge)
                        list = merged(list, sorted(key, lane), lane);
                        least = lane64(list, a.k - 1);
                        left = 0;
                    }
                    while (left) {
                        const int l = __builtin_ctzll(left);
                        list = entered(list, lane64(key, l), lane);
                        least = lane64(list, a.k - 1);
                        left &= left - 1;
                        left &= __ballot(key > least);
                    }
                }
                __builtin_amdgcn_wave_barrier();
                bar = least ? value_of(least) : __builtin_nanf("");
            }
            full = least != 0;
        }
    }
    s = over_wave(s);
    if (lane == 0) ws[w] = s;
    if constexpr (TOP) lists[w][lane] = list;
    __syncthreads();
    if (w) return;
    s = join(join(ws[0], ws[1]), join(ws[2], ws[3]));
    if constexpr (TOP)
        for (int o = 1; o < 4; ++o) list = merged(list, lists[o][lane], lane);
    if (a.slices == 1) {
        finish<T>(a, row, s, list, lane);
        return;
    }
    if (lane == 0) a.sums[blockIdx.x] = s;
    if constexpr (TOP)
        if (lane < a.k) a.keys[(long)blockIdx.x * a.k + lane] = list;
}

// The slices of a row together.
template <typename T>
__global__ __launch_bounds__(256) void logprob_join(LogArgs a) {
    __shared__ u64 lists[4][64];
    const int row = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    Sums s{kLowest, 0.f, 0.f};
    if (lane < a.slices) s = a.sums[(long)row * a.slices + lane];
    u64 list = 0;
    if (a.k) {
        const u64* keys = a.keys + (long)row * a.slices * a.k + lane;
        u64 next = lane < a.k && w < a.slices ? keys[(long)w * a.k] : 0;
        for (int c = w; c < a.slices; c += 4) {
            const u64 here = next;
            next = lane < a.k && c + 4 < a.slices ? keys[(long)(c + 4) * a.k] : 0;
            list = merged(list, here, lane);
        }
        lists[w][lane] = list;
        __syncthreads();
        if (w) return;
        for (int o = 1; o < 4; ++o) list = merged(list, lists[o][lane], lane);
    } else if (w) {
        return;
    }
    finish<T>(a, row, over_wave(s), list, lane);
}

struct GradArgs {
    const void* x; long ldx;
    const int* ids;
    const float2* stats;
    const float* ent; const float* dlogp; const float* dent;
    void* dx; long lddx;
    int M, N, pieces;
};

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void logprob_grad(GradArgs a) {
    const int row = blockIdx.x / a.pieces, piece = blockIdx.x - row * a.pieces;
    const float2 st = a.stats[row];
    const int id = a.ids ? a.ids[row] : -1;
    const float w = a.dlogp && id >= 0 && id < a.N ? a.dlogp[row] : 0.f;
    const float v = a.dent ? a.dent[row] : 0.f, h = a.dent ? a.ent[row] : 0.f;
    const bool none = st.y == -__builtin_inff();
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* dx = static_cast<T*>(a.dx) + row * a.lddx;
    const int base = piece * kRun - lead<WHOLE>(dx);
    float f[kGroups][8];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int at = base + (g * 256 + (int)threadIdx.x) * 8;
        load8<WHOLE>(x + at, at, a.N, f[g]);
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int at = base + (g * 256 + (int)threadIdx.x) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float lp = (f[g][j] - st.x) - st.y, p = grow(lp);
            const float d = -p * fmaf(v, fmaxf(lp, kFloor) + h, w);
            f[g][j] = none ? 0.f : at + j == id ? d + w : d;
        }
        store8<WHOLE>(dx + at, at, a.N, f[g]);
    }
}

// Slices of a row: workgroups enough for the chip (four a CU), each of at least one turn (us, 64 x 128000 fp32 with 20
// alternatives, 1 / 4 / 8 / 16 slices: 47 / 25 / 20 / 19; 600 x 50257 fp32, 1 / 3: 22.8 / 25.0).
int slices_of(int M, int N) {
    const long turns = ssm::cdiv(N, kRun);
    return (int)std::max(1L, std::min(std::min(turns, 64L), 1024L / std::max(1, M)));
}

// Rows on 16-byte places.
bool in_place(const void* p, long bytes) { return (((uintptr_t)p | (uintptr_t)bytes) & 15) == 0; }

size_t sums_bytes(int M, int slices) { return ((size_t)M * slices * sizeof(Sums) + 15) / 16 * 16; }

template <typename T, bool WHOLE>
void run_logprobs(const LogArgs& a, hipStream_t st) {
    const unsigned n = (unsigned)((long)a.M * a.slices);
    if (a.k) logprob_kernel<T, true, WHOLE><<<n, 256, 0, st>>>(a);
    else logprob_kernel<T, false, WHOLE><<<n, 256, 0, st>>>(a);
    if (a.slices > 1) logprob_join<T><<<a.M, 256, 0, st>>>(a);
}
template <typename T>
void run_grad(const GradArgs& a, bool whole, hipStream_t st) {
    const unsigned n = (unsigned)((long)a.M * a.pieces);
    if (whole) logprob_grad<T, true><<<n, 256, 0, st>>>(a);
    else logprob_grad<T, false><<<n, 256, 0, st>>>(a);
}

}  // namespace

extern "C" size_t ssm_token_logprobs_workspace(int M, int N, int k) {
    if (M <= 0 || N <= 0 || k < 0 || k > kMaxTop) return 0;
    const int s = slices_of(M, N);
    return s > 1 ? sums_bytes(M, s) + (size_t)M * s * k * sizeof(u64) : 0;
}

extern "C" ssm_status ssm_token_logprobs(int dtype, const void* x, long ldx, const int* ids, int M, int N, int k,
                                         float* logp, float* entropy, float* stats, int* top_ids, float* top_logp,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_token_logprobs: bad dtype");
    SSM_REQUIRE(M >= 0 && N > 0 && N <= ssm::kMaxSteps && k >= 0, "ssm_token_logprobs: bad shape");
    SSM_REQUIRE(k <= N, "ssm_token_logprobs: %d alternatives of %d logits", k, N);
    if (k > kMaxTop) return ssm::fail(SSM_ERR_UNSUPPORTED, "ssm_token_logprobs: %d alternatives, at most %d", k, kMaxTop);
    if (M == 0) return SSM_OK;
    SSM_REQUIRE(x && (!logp || ids) && (k == 0 || (top_ids && top_logp)), "ssm_token_logprobs: null input");
    if (M == 1) ldx = N;
    SSM_REQUIRE(ldx >= N, "ssm_token_logprobs: row stride below row width");
    const int slices = slices_of(M, N);
    SSM_REQUIRE((long)M * slices <= ssm::kMaxGroups, "ssm_token_logprobs: too many rows");
    const size_t need = ssm_token_logprobs_workspace(M, N, k);
    SSM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "ssm_token_logprobs: needs a workspace of %zu bytes", need);
    SSM_REQUIRE(need == 0 || ((uintptr_t)workspace & 15) == 0, "ssm_token_logprobs: workspace must be 16-byte aligned");
    SSM_REQUIRE(((uintptr_t)stats & 7) == 0, "ssm_token_logprobs: stats must be 8-byte aligned");
    const long es = dtype == SSM_F32 ? 4 : 2;
    const ssm::Rows rx{x, ldx * es, N * es, M}, ri = ssm::block(ids, 4L * M), o0 = ssm::block(logp, 4L * M),
                    o1 = ssm::block(entropy, 4L * M), o2 = ssm::block(stats, 8L * M),
                    o3 = ssm::block(k ? top_ids : nullptr, 4L * M * k), o4 = ssm::block(k ? top_logp : nullptr, 4L * M * k),
                    ws = ssm::block(need ? workspace : nullptr, need);
    SSM_REQUIRE(!ssm::meets(o0, rx, ri, o1, o2, o3, o4, ws) && !ssm::meets(o1, rx, ri, o2, o3, o4, ws) &&
                    !ssm::meets(o2, rx, ri, o3, o4, ws) && !ssm::meets(o3, rx, ri, o4, ws) &&
                    !ssm::meets(o4, rx, ri, ws) && !ssm::meets(ws, rx, ri),
                "ssm_token_logprobs: an output or the workspace overlaps another operand");
    LogArgs a{};
    a.x = x; a.ldx = ldx; a.ids = ids; a.logp = logp; a.ent = entropy; a.stats = reinterpret_cast<float2*>(stats);
    a.top = top_ids; a.toplp = top_logp; a.M = M; a.N = N; a.k = k; a.slices = slices;
    a.turns = (int)ssm::cdiv(ssm::cdiv(N, kRun), slices);
    a.sums = static_cast<Sums*>(workspace);
    a.keys = reinterpret_cast<u64*>(static_cast<char*>(workspace) + sums_bytes(M, slices));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SSM_F32) N % 8 ? run_logprobs<float, false>(a, st) : run_logprobs<float, true>(a, st);
    else N % 8 ? run_logprobs<__bf16, false>(a, st) : run_logprobs<__bf16, true>(a, st);
    return ssm::check_launch("ssm_token_logprobs");
}

extern "C" ssm_status ssm_token_logprobs_backward(int dtype, const void* x, long ldx, const int* ids, const float* stats,
                                                  const float* entropy, const float* dlogp, const float* dentropy,
                                                  void* dx, long lddx, int M, int N, void* stream) {
    SSM_REQUIRE(dtype == SSM_F32 || dtype == SSM_BF16, "ssm_token_logprobs_backward: bad dtype");
    SSM_REQUIRE(M >= 0 && N > 0 && N <= ssm::kMaxSteps, "ssm_token_logprobs_backward: bad shape");
    if (M == 0) return SSM_OK;
    SSM_REQUIRE(x && stats && dx && (!dlogp || ids) && (!dentropy || entropy), "ssm_token_logprobs_backward: null input");
    SSM_REQUIRE(((uintptr_t)stats & 7) == 0, "ssm_token_logprobs_backward: stats must be 8-byte aligned");
    if (M == 1) ldx = lddx = N;
    SSM_REQUIRE(ldx >= N && lddx >= N, "ssm_token_logprobs_backward: row stride below row width");
    const long es = dtype == SSM_F32 ? 4 : 2;
    const bool whole = N % 8 == 0 && (dtype == SSM_F32 || in_place(dx, lddx * es));
    const long pieces = ssm::cdiv(whole ? N : N + 7, kRun);
    SSM_REQUIRE(M * pieces <= ssm::kMaxGroups, "ssm_token_logprobs_backward: too many logits");
    const ssm::Rows rx{x, ldx * es, N * es, M}, ox{dx, lddx * es, N * es, M};
    SSM_REQUIRE((dx == x && ldx == lddx) || !ssm::meet(ox, rx), "ssm_token_logprobs_backward: dx overlaps x, which it is not");
    SSM_REQUIRE(!ssm::meets(ox, ssm::block(ids, 4L * M), ssm::block(stats, 8L * M), ssm::block(entropy, 4L * M),
                            ssm::block(dlogp, 4L * M), ssm::block(dentropy, 4L * M)),
                "ssm_token_logprobs_backward: dx overlaps another operand");
    GradArgs a{};
    a.x = x; a.ldx = ldx; a.ids = ids; a.stats = reinterpret_cast<const float2*>(stats); a.ent = entropy;
    a.dlogp = dlogp; a.dent = dentropy; a.dx = dx; a.lddx = lddx; a.M = M; a.N = N; a.pieces = (int)pieces;
    if (dtype == SSM_F32) run_grad<float>(a, whole, (hipStream_t)stream);
    else run_grad<__bf16>(a, whole, (hipStream_t)stream);
    return ssm::check_launch("ssm_token_logprobs_backward");
}

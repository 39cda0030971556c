// Log probabilities of given categories, entropy, log-sum-exp and the likeliest alternatives of rows of logits, and their gradient.
//
//   m = max x, Z = sum e^(x - m), S = sum e^(x - m) (x - m), L = log Z
//   log_prob = (x_t - m) - L      entropy = L - S / Z      lse = m + L      alternatives: value descending, then index ascending
//   dx_j = p_j (A - g_H log p_j) + [j = t] g_lp + [j = top_i] g_top_i,   p_j = e^((x_j - m) - L),
//          A = g_lse - g_lp - sum_i g_top_i - g_H H
//
// m and L are kept apart (not as m + L): with logits around 10^4 their sum has lost the digits that p_j needs.
// A row of nothing but -inf has lse = log_prob = -inf, entropy 0 and gradient 0.  Sums are fp32, the gradient is rounded once.
#include "mmt_common.h"

namespace {

constexpr int kBlock = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -200.f;         // 2^-200 is 0 in fp32: what is below adds nothing, and 0 * -inf has to be 0
constexpr int kMaxParts = 64;            // parts of a row
constexpr int kCandidates = 1024;        // alternatives of one part that are sorted out by counting

struct LogProbsArgs {
    int64_t rows, D, row_stride;
    const void *logits;
    const void *ids;             // int32 / int64 [rows] or NULL
    int ids_bytes, top;
    float *log_prob, *entropy, *lse, *stats;     // stats [rows][4]: m, L, H, 0
    float *top_log_prob;
    int64_t *top_ids;
    // rows in parts: part_elems elements each, `parts` of them; their (m, Z, S, -) and sorted alternatives
    int parts;
    int64_t part_elems;
    float *part_sums;
    unsigned long long *part_top;
    // backward
    const float *g_lp, *g_h, *g_lse, *g_top;
    const float *stats_in;
    const int64_t *top_in;
    void *grad;
    int64_t grad_stride;
};

template <typename T> __device__ __forceinline__ float load1(const T *p) { return *p; }
template <> __device__ __forceinline__ float load1<bf16_t>(const bf16_t *p) { return __uint_as_float((unsigned)*p << 16); }
template <typename T> __device__ __forceinline__ void store1(T *p, float v) { *p = v; }
template <> __device__ __forceinline__ void store1<bf16_t>(bf16_t *p, float v) { *p = (bf16_t)(pack_bf16x2(v, 0.f) & 0xFFFFu); }

// 16 bytes from an address that is aligned to one element only (a row of an odd length begins anywhere)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned w[4]; };
typedef unsigned raw4 __attribute__((ext_vector_type(4), aligned(2)));

// A piece is the 16 bytes of a row that one lane takes at a time.  The last piece of a row that does not end on one begins earlier, so that it ends
// with the row; its elements before e0 belong to the piece in front and read as dead.  dead = -inf.
template <typename T> struct Piece {
    static constexpr int N = 16 / sizeof(T);
    float v[N];
    int s;                               // index of v[0]
    // (I: int where a row is short -- its 64-bit comparisons, one or two an element, are what a short row's time would go into)
    template <typename I>
    __device__ __forceinline__ bool live(int j, I e0, I D) const { return s + j >= e0 && s + j < D; }
    template <typename I>
    __device__ __forceinline__ void load(const T *row, I e0, I D) {
        s = (int)e0;
        if (e0 + N <= D) {
            unpack(*reinterpret_cast<const Raw<T> *>(row + e0));
        } else if (e0 < D && D >= N) {
            s = (int)(D - N);
            unpack(*reinterpret_cast<const Raw<T> *>(row + s));
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = s + j >= e0 ? v[j] : -INFINITY;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = e0 + j < D ? load1(row + e0 + j) : -INFINITY;
        }
    }
    // (no test, so that the loads of several pieces are under way together)  ONCE: passing through the caches without staying, see kOnceBytes
    template <bool ONCE>
    __device__ __forceinline__ void load_whole(const T *row, int64_t e0) {
        s = (int)e0;
        if constexpr (ONCE) {
            const raw4 t = __builtin_nontemporal_load(reinterpret_cast<const raw4 *>(row + e0));
            unpack(Raw<T>{{t.x, t.y, t.z, t.w}});
        } else {
            unpack(*reinterpret_cast<const Raw<T> *>(row + e0));
        }
    }
    __device__ __forceinline__ void unpack(Raw<T> r) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r.w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(r.w[j]); v[2 * j + 1] = bf16_hi(r.w[j]); }
        }
    }
    template <bool ONCE>
    __device__ __forceinline__ void store_whole(T *row, int64_t e0) const {
        Raw<T> r;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[j] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
        }
        if constexpr (ONCE) __builtin_nontemporal_store(raw4{r.w[0], r.w[1], r.w[2], r.w[3]}, reinterpret_cast<raw4 *>(row + e0));
        else *reinterpret_cast<Raw<T> *>(row + e0) = r;
    }
    // v -> the row, where live
    template <typename I>
    __device__ __forceinline__ void store(T *row, I e0, I D) const {
        if (e0 + N <= D) {
            store_whole<false>(row, e0);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (live(j, e0, D)) store1(row + s + j, v[j]);
        }
    }
};

// the category of a row, or -1 where the id names none
__device__ __forceinline__ int64_t given_id(const LogProbsArgs &a, int64_t r) {
    if (!a.ids) return -1;
    const int64_t t = a.ids_bytes == 8 ? static_cast<const int64_t *>(a.ids)[r] : (int64_t)static_cast<const int32_t *>(a.ids)[r];
    return t >= 0 && t < a.D ? t : -1;
}

// unsigned key with the order of the values: NaN above +inf, -0 equal to +0; 0 is below every value's
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return x != x ? 0xFFFFFFFFu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);       // (NaN's key gives a NaN)
}

// reduction over groups of L = 16 or 64 lanes; every lane ends with the result (a wave's is in a scalar register)
template <int L, typename V, typename F>
__device__ __forceinline__ V lanes_reduce(V v, V identity, F f) {
#define MMT_DPP_STEP(ctrl) v = f(v, __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xF, 0xF, true)));
    MMT_DPP_STEP(0xB1)      // quad_perm [1,0,3,2]
    MMT_DPP_STEP(0x4E)      // quad_perm [2,3,0,1]
    MMT_DPP_STEP(0x141)     // row_half_mirror
    MMT_DPP_STEP(0x140)     // row_mirror
#undef MMT_DPP_STEP
    if constexpr (L == 64) {
        const int none = __builtin_bit_cast(int, identity);
        v = f(v, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(none, __builtin_bit_cast(int, v), 0x142, 0xA, 0xF, false)));      // row_bcast:15 into rows 1, 3
        v = f(v, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(none, __builtin_bit_cast(int, v), 0x143, 0xC, 0xF, false)));      // row_bcast:31 into rows 2, 3
        v = __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    }
    return v;
}
__device__ __forceinline__ float fadd(float a, float b) { return a + b; }
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned umin(unsigned a, unsigned b) { return a < b ? a : b; }

// (m, Z, S) of a stretch of a row, S in units of log 2: S = sum e^(x - m) (x - m) / log 2.  m = -inf: nothing (but -inf) so far.
struct Sums {
    float m = -INFINITY, z = 0.f, s = 0.f;
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void add(float x, float b) {
        const float t = (x - b) * kLog2e, e = __builtin_amdgcn_exp2f(t);
        z += e;
        s = fmaf(e, fmaxf(t, kFloor), s);
    }
    __device__ __forceinline__ void raise(float to) {                   // to >= m
        if (m != -INFINITY && to != m) {
            const float t = (m - to) * kLog2e, f = __builtin_amdgcn_exp2f(t);
            s = f * fmaf(z, fmaxf(t, kFloor), s);
            z *= f;
        }
        m = to;
    }
};
// what a row's (m, Z, S) come to; a row of nothing but -inf: Z = 0 (a NaN beside them: Z = NaN)
struct RowResult {
    float m, L, h;
    bool empty;
    __device__ __forceinline__ RowResult(Sums q) {
        m = q.m;
        empty = q.m == -INFINITY && q.z == 0.f;
        L = empty ? 0.f : logf(q.z);
        h = empty ? 0.f : L - q.s / q.z * kLn2;
    }
    __device__ __forceinline__ float log_prob(float x) const { return empty ? -INFINITY : (x - m) - L; }
};
__device__ __forceinline__ void write_row(const LogProbsArgs &a, int64_t r, const RowResult &q, int64_t t, float xt) {
    *reinterpret_cast<float4 *>(a.stats + 4 * r) = make_float4(q.m, q.L, q.h, 0.f);
    a.lse[r] = q.m + q.L;
    a.entropy[r] = q.h;
    if (a.log_prob) a.log_prob[r] = t < 0 ? 0.f : q.log_prob(xt);
}

// ------------------------------------------------------------------------------------------------ rows in the registers of 16 or 64 lanes

// An element as (order key, falling index): greater = earlier alternative, no two are equal.
__device__ __forceinline__ unsigned long long composite(unsigned key, int64_t index) { return ((unsigned long long)key << 32) | (unsigned)~(unsigned)index; }

// A value that at least `want` (<= 64) and, ties apart, at most `most` of a wave's 64 x E values reach, and how many do: a bisection from the top.  It
// begins at the least of `want` or more groups of lanes' greatest values, which is near already; every step is counted by ballots.  (To
// end at exactly `want` instead took the steps that tell neighbours apart: 22 us against 8 at 28 160 rows of 409, 8 alternatives.)
template <int E>
__device__ __forceinline__ unsigned reached_by(const unsigned *key, int want, int most, int &n) {
    unsigned mine = 0u;
#pragma unroll
    for (int i = 0; i < E; ++i) mine = umax(mine, key[i]);
    unsigned hi = mine, low = mine;
#define MMT_GROUP_STEP(groups, other)                                                                                              \
    {                                                                                                                              \
        const unsigned h = other(hi), l = other(low);                                                                              \
        hi = umax(hi, h);                                                                                                          \
        low = want > groups ? umin(low, l) : umax(low, l);                                                                         \
    }
#define MMT_DPP_1(v) (unsigned)__builtin_amdgcn_mov_dpp((int)(v), 0xB1, 0xF, 0xF, true)
#define MMT_DPP_2(v) (unsigned)__builtin_amdgcn_mov_dpp((int)(v), 0x4E, 0xF, 0xF, true)
#define MMT_DPP_4(v) (unsigned)__builtin_amdgcn_mov_dpp((int)(v), 0x141, 0xF, 0xF, true)
#define MMT_DPP_8(v) (unsigned)__builtin_amdgcn_mov_dpp((int)(v), 0x140, 0xF, 0xF, true)
#define MMT_XOR_16(v) (unsigned)__shfl_xor((int)(v), 16)
#define MMT_XOR_32(v) (unsigned)__shfl_xor((int)(v), 32)
    // (lanes that differ in bit 0 first: 32 groups of two, 16 of four, ..; `want` > groups: from here on the least)
    MMT_GROUP_STEP(32, MMT_DPP_1)
    MMT_GROUP_STEP(16, MMT_DPP_2)
    MMT_GROUP_STEP(8, MMT_DPP_4)
    MMT_GROUP_STEP(4, MMT_DPP_8)
    MMT_GROUP_STEP(2, MMT_XOR_16)
    MMT_GROUP_STEP(1, MMT_XOR_32)
#undef MMT_GROUP_STEP
#undef MMT_DPP_1
#undef MMT_DPP_2
#undef MMT_DPP_4
#undef MMT_DPP_8
#undef MMT_XOR_16
#undef MMT_XOR_32
    hi = (unsigned)__builtin_amdgcn_readfirstlane((int)hi);
    unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)low);
    auto count = [&](unsigned at) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) c += __popcll(__ballot(key[i] >= at));
        return c;
    };
    n = count(lo);
    while (n > most && lo < hi) {
        const unsigned mid = hi - (hi - lo) / 2;
        const int c = count(mid);
        if (c >= want) { lo = mid; n = c; }
        else hi = mid - 1;
    }
    return lo;
}

// What lanes of a wave have written to LDS for one another, before they read it (or before they write the next): a wave's LDS operations are done in order,
// so this only keeps the compiler from moving them.
__device__ __forceinline__ void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Alternatives of a row that a wave holds: the elements that reach the bound above side by side in the wave's lanes (two each at most), each counting the
// ones in front of it.  false: more reach it (ties), nothing written.
constexpr int kWaveCandidates = 128;
template <typename T, int E, typename R>
__device__ __forceinline__ bool wave_alternatives(const LogProbsArgs &a, int64_t r, const R &res, const Piece<T> *x, const unsigned *key, int lane, unsigned long long *cand) {
    constexpr int N = Piece<T>::N;
    int n;
    const unsigned lo = reached_by<E>(key, a.top, a.top <= 32 ? 64 : kWaveCandidates, n);
    if (n > kWaveCandidates) return false;
    int base = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const unsigned long long mask = __ballot(key[i] >= lo);
        const int at = base + __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
        if (key[i] >= lo) cand[at] = composite(key[i], x[i / N].s + i % N);
        base += __popcll(mask);
    }
    wave_exchange();
    for (int i = lane; i < n; i += 64) {
        const unsigned long long own = cand[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += cand[j] > own ? 1 : 0;
        if (rank < a.top) {
            a.top_ids[r * a.top + rank] = (unsigned)~(unsigned)own;
            a.top_log_prob[r * a.top + rank] = res.log_prob(key_value((unsigned)(own >> 32)));
        }
    }
    wave_exchange();
    return true;
}

// D <= L * E: L lanes hold a row, E elements each; one read.  For 16 lanes (and ties in the wave's form above) an alternative is the largest key, then the
// lowest index that has it: two reductions each.
template <typename T, int L, int E>
__global__ __launch_bounds__(kBlock) void log_probs_fwd_lanes(LogProbsArgs a) {
    constexpr int N = Piece<T>::N, P = E / N, G = kBlock / L;
    __shared__ unsigned long long cand[L == 64 ? kBlock / 64 * kWaveCandidates : 1];
    const int lane = threadIdx.x % L, D = (int)a.D;
    for (int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / L; r < a.rows; r += (int64_t)gridDim.x * G) {
        const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
        const int64_t t = given_id(a, r);
        Piece<T> x[P];
#pragma unroll
        for (int p = 0; p < P; ++p) x[p].load(row, (p * L + lane) * N, D);
        const float xt = t < 0 ? 0.f : load1(row + t);
        Sums q;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < N; ++j) q.m = fmaxf(q.m, x[p].v[j]);
        q.m = lanes_reduce<L>(q.m, -INFINITY, [](float u, float v) { return fmaxf(u, v); });
        const float b = q.base();
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < N; ++j) q.add(x[p].v[j], b);
        q.z = lanes_reduce<L>(q.z, 0.f, fadd);
        q.s = lanes_reduce<L>(q.s, 0.f, fadd);
        const RowResult res(q);
        if (lane == 0) write_row(a, r, res, t, xt);
        bool done = a.top == 0;
        if (!done) {
            unsigned key[E];
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < N; ++j) key[p * N + j] = x[p].live(j, (p * L + lane) * N, D) ? order_key(x[p].v[j]) : 0u;
            if constexpr (L == 64) done = wave_alternatives<T, E>(a, r, res, x, key, lane, &cand[threadIdx.x / 64 * kWaveCandidates]);
            for (int k = 0; k < a.top && !done; ++k) {
                unsigned best = 0u;
#pragma unroll
                for (int i = 0; i < E; ++i) best = umax(best, key[i]);
                best = lanes_reduce<L>(best, 0u, umax);
                unsigned at = 0xFFFFFFFFu;
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int j = 0; j < N; ++j) at = key[p * N + j] == best ? umin(at, (unsigned)(x[p].s + j)) : at;
                at = lanes_reduce<L>(at, 0xFFFFFFFFu, umin);
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int j = 0; j < N; ++j) key[p * N + j] = (unsigned)(x[p].s + j) == at ? 0u : key[p * N + j];
                if (lane == 0) {
                    a.top_ids[r * a.top + k] = at;
                    a.top_log_prob[r * a.top + k] = res.log_prob(key_value(best));
                }
            }
        }
    }
}

// coefficients of a row's gradient: d = p (A - gh log p), and gt at the given category
struct RowGrad {
    float m, L, A, gh, gt;
    int64_t t;
    bool empty;
    __device__ __forceinline__ RowGrad(const LogProbsArgs &a, int64_t r) {
        const float4 st = *reinterpret_cast<const float4 *>(a.stats_in + 4 * r);
        m = st.x; L = st.y;
        empty = m == -INFINITY && L == L;
        t = given_id(a, r);
        gt = t >= 0 && a.g_lp ? a.g_lp[r] : 0.f;
        gh = a.g_h ? a.g_h[r] : 0.f;
        A = (a.g_lse ? a.g_lse[r] : 0.f) - gt;
        if (a.g_h) A -= gh * st.z;
        if (a.g_top) {
            float g = 0.f;
            for (int k = 0; k < a.top; ++k) g += a.g_top[r * a.top + k];
            A -= g;
        }
        if (empty) { m = L = A = gh = gt = 0.f; t = -1; }                // (x - m = -inf: p = 0)
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float lp = (x - m) - L;
        // (a probability below 2^-126 comes out as 0: its gradient is off by up to 2^-126 |A - gh lp|)
        return __builtin_amdgcn_exp2f(lp * kLog2e) * fmaf(-gh, fmaxf(lp, kFloor), A);
    }
};

template <typename T, int L, int E>
__global__ __launch_bounds__(kBlock) void log_probs_bwd_lanes(LogProbsArgs a) {
    constexpr int N = Piece<T>::N, P = E / N, G = kBlock / L;
    const int lane = threadIdx.x % L, D = (int)a.D;
    for (int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / L; r < a.rows; r += (int64_t)gridDim.x * G) {
        const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
        T *out = static_cast<T *>(a.grad) + r * a.grad_stride;
        Piece<T> x[P];
#pragma unroll
        for (int p = 0; p < P; ++p) x[p].load(row, (p * L + lane) * N, D);
        const RowGrad g(a, r);
        const int t = (int)g.t;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < N; ++j) x[p].v[j] = g(x[p].v[j]) + (x[p].s + j == t ? g.gt : 0.f);
        if (a.g_top && !g.empty)
            for (int k = 0; k < a.top; ++k) {
                const int at = (int)a.top_in[r * a.top + k];
                const float gk = a.g_top[r * a.top + k];
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int j = 0; j < N; ++j) x[p].v[j] += x[p].s + j == at ? gk : 0.f;
            }
#pragma unroll
        for (int p = 0; p < P; ++p) x[p].store(out, (p * L + lane) * N, D);
    }
}

// ------------------------------------------------------------------------------------------------ long rows: a workgroup per part of a row

// the workgroup's (m, Z, S) in every thread; lds: 3 floats per wave
__device__ __forceinline__ Sums block_join(Sums q, float *lds) {
    auto fmx = [](float u, float v) { return fmaxf(u, v); };
    q.raise(lanes_reduce<64>(q.m, -INFINITY, fmx));
    q.z = lanes_reduce<64>(q.z, 0.f, fadd);
    q.s = lanes_reduce<64>(q.s, 0.f, fadd);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { lds[3 * wave] = q.m; lds[3 * wave + 1] = q.z; lds[3 * wave + 2] = q.s; }
    __syncthreads();
    Sums all, one[kBlock / 64];
#pragma unroll
    for (int w = 0; w < kBlock / 64; ++w) {
        one[w].m = lds[3 * w]; one[w].z = lds[3 * w + 1]; one[w].s = lds[3 * w + 2];
        all.m = fmaxf(all.m, one[w].m);
    }
#pragma unroll
    for (int w = 0; w < kBlock / 64; ++w) {
        one[w].raise(all.m);
        all.z += one[w].z;
        all.s += one[w].s;
    }
    __syncthreads();
    return all;
}

// the `top` greatest of cand[0 .. n), in order, handed to put(rank, composite): every one counts those in front of it
template <typename F>
__device__ __forceinline__ void rank_candidates(const unsigned long long *cand, int n, int top, F put) {
    for (int i = threadIdx.x; i < n; i += kBlock) {
        const unsigned long long mine = cand[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += cand[j] > mine ? 1 : 0;
        if (rank < top) put(rank, mine);
    }
}

// Alternatives of a part [begin, end).  Every thread knows its own greatest element's value and the piece that it is in first; the top-th greatest of those
// 256 (key, falling piece) is a bound that at least `top` elements reach, and few more do (a second look at these threads' pieces, now in the
// caches, collects them).  Only a part whose greatest elements crowd in few threads' pieces overflows the list: then one pass for each alternative.
template <typename T, typename F>
__device__ __forceinline__ void part_alternatives(const T *row, int64_t begin, int64_t end, int top, unsigned own_key, unsigned own_piece, bool own_nan,
                                                  unsigned long long *cand, uint8_t *order, int *count, F put) {
    constexpr int N = Piece<T>::N;
    constexpr int W = kBlock / 64;
    unsigned *keys = reinterpret_cast<unsigned *>(cand), *pieces = keys + kBlock;
    keys[threadIdx.x] = own_key;
    pieces[threadIdx.x] = ~own_piece;
    if (threadIdx.x < 2) count[threadIdx.x] = 0;
    __syncthreads();
    unsigned key[W], back[W];                                             // (every wave finds the bound for itself)
    int n;
#pragma unroll
    for (int w = 0; w < W; ++w) key[w] = keys[(threadIdx.x & 63) + 64 * w];
    const unsigned least = reached_by<W>(key, top, 2 * top, n);           // 0: fewer than `top` threads have an element
    unsigned last = 0xFFFFFFFFu;
    if (least && n > 2 * top) {                                           // ties at the bound: the first pieces only
        int above = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            above += __popcll(__ballot(key[w] > least));
            back[w] = key[w] == least ? pieces[(threadIdx.x & 63) + 64 * w] : 0u;
        }
        last = ~reached_by<W>(back, top - above, top, n);
    }
    const float floor = least ? key_value(least) : -INFINITY;
    // The threads with something to look for (their greatest element reaches the bound, or a NaN is among their elements), and their pieces dealt out
    // to all: what is left of the latency of a handful of threads that read on alone (14 us of 57 at 450 rows of 100 003 and one alternative).
    if (own_key >= least || own_nan) order[atomicAdd(&count[0], 1)] = (uint8_t)threadIdx.x;
    __syncthreads();
    const int looking = count[0];
    const int pieces_each = (int)((end - begin + kBlock * N - 1) / (kBlock * N));
    for (int k = threadIdx.x; k < looking * pieces_each; k += kBlock) {
        const unsigned piece = (unsigned)(k / looking) * kBlock + order[k % looking];
        const int64_t e0 = begin + (int64_t)piece * N;
        if (e0 >= end) continue;
        Piece<T> x;
        x.load(row, e0, end);
        bool any = false;
#pragma unroll
        for (int j = 0; j < N; ++j) any = any || !(x.v[j] < floor);
        if (any)
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (x.live(j, e0, end) && !(x.v[j] < floor) && (x.v[j] != floor || piece <= last)) {
                    const int at = atomicAdd(&count[1], 1);
                    if (at < kCandidates) cand[at] = composite(order_key(x.v[j]), x.s + j);
                }
    }
    __syncthreads();
    n = count[1];
    if (n <= kCandidates) {
        rank_candidates(cand, n, top, put);
    } else {
        unsigned long long before = ~0ull;
        for (int k = 0; k < top; ++k) {                                   // the greatest below the one before
            unsigned long long best = 0ull;
            for (int64_t j = begin + threadIdx.x; j < end; j += kBlock) {
                const unsigned long long c = composite(order_key(load1(row + j)), j);
                if (c > best && (c < before || k == 0)) best = c;
            }
            for (int o = 32; o > 0; o >>= 1) { const unsigned long long c = __shfl_xor(best, o); best = c > best ? c : best; }
            __syncthreads();
            if ((threadIdx.x & 63) == 0) cand[threadIdx.x >> 6] = best;
            __syncthreads();
            best = cand[0];
            for (int w = 1; w < kBlock / 64; ++w) best = cand[w] > best ? cand[w] : best;
            before = best;
            if (threadIdx.x == 0) put(k, best);
        }
    }
    __syncthreads();
}

template <typename T, bool TOP, bool ONCE>
__global__ __launch_bounds__(kBlock) void log_probs_fwd_parts(LogProbsArgs a) {
    constexpr int N = Piece<T>::N, U = 4;
    __shared__ float lds[3 * kBlock / 64];
    __shared__ unsigned long long cand[TOP ? kCandidates : 1];
    __shared__ uint8_t order[TOP ? kBlock : 1];
    __shared__ int count[2];
    const int64_t units = a.rows * a.parts;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t r = u / a.parts;
        const int part = (int)(u - r * a.parts);
        const int64_t begin = part * a.part_elems, end = begin + a.part_elems < a.D ? begin + a.part_elems : a.D;
        const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
        const int64_t t = a.parts == 1 ? given_id(a, r) : -1;
        Sums q;
        unsigned piece = 0xFFFFFFFFu, at = threadIdx.x;                   // piece of the first of the greatest elements; current piece
        auto take = [&](const Piece<T> &x) {
            float m = x.v[0];
#pragma unroll
            for (int j = 1; j < N; ++j) m = fmaxf(m, x.v[j]);
            if (TOP) { piece = m > q.m || piece == 0xFFFFFFFFu ? at : piece; at += kBlock; }
            if (m > q.m) q.raise(m);
            const float b = q.base();
#pragma unroll
            for (int j = 0; j < N; ++j) q.add(x.v[j], b);
        };
        int64_t e0 = begin + (int64_t)threadIdx.x * N;
        for (; e0 + (U - 1) * kBlock * N + N <= end; e0 += U * kBlock * N) {
            Piece<T> x[U];
#pragma unroll
            for (int i = 0; i < U; ++i) x[i].template load_whole<ONCE>(row, e0 + i * kBlock * N);
#pragma unroll
            for (int i = 0; i < U; ++i) take(x[i]);
        }
        for (; e0 < end; e0 += kBlock * N) {
            Piece<T> x;
            x.load(row, e0, end);
            take(x);
        }
        const unsigned own_key = piece != 0xFFFFFFFFu ? order_key(q.m) : 0u;
        const bool own_nan = q.z != q.z;
        const Sums all = block_join(q, lds);
        if (a.parts == 1) {
            const RowResult res(all);
            if (threadIdx.x == 0) write_row(a, r, res, t, t < 0 ? 0.f : load1(row + t));
            if constexpr (TOP)
                part_alternatives(row, begin, end, a.top, own_key, piece, own_nan, cand, order, count, [&](int k, unsigned long long c) {
                    a.top_ids[r * a.top + k] = (unsigned)~(unsigned)c;
                    a.top_log_prob[r * a.top + k] = res.log_prob(key_value((unsigned)(c >> 32)));
                });
        } else {
            if (threadIdx.x == 0) { float *o = a.part_sums + 4 * u; o[0] = all.m; o[1] = all.z; o[2] = all.s; }
            if constexpr (TOP) {
                // (a part shorter than `top`, the last of a row, leaves zeros behind: below every element)
                if (end - begin < a.top)
                    for (int k = (int)(end - begin) + threadIdx.x; k < a.top; k += kBlock) a.part_top[u * a.top + k] = 0ull;
                part_alternatives(row, begin, end, a.top, own_key, piece, own_nan, cand, order, count, [&](int k, unsigned long long c) { a.part_top[u * a.top + k] = c; });
            }
        }
    }
}

// the parts of a row together: a workgroup per row
template <typename T, bool TOP>
__global__ __launch_bounds__(kBlock) void log_probs_join(LogProbsArgs a) {
    __shared__ float lds[3 * kBlock / 64];
    __shared__ unsigned long long cand[TOP ? kMaxParts * MMT_LOG_PROBS_MAX_TOP : 1];
    __shared__ unsigned long long bound;
    __shared__ int count;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        // (everything that memory has to give first)
        const unsigned long long *lists = a.part_top + r * a.parts * a.top;
        unsigned long long mine = 0ull;
        if constexpr (TOP) {
            const int heads = kBlock / a.parts < a.top ? kBlock / a.parts : a.top;
            if (threadIdx.x < a.parts * heads) mine = lists[threadIdx.x / heads * a.top + threadIdx.x % heads];
        }
        const int64_t t = given_id(a, r);
        Sums q;
        if (threadIdx.x < a.parts) {
            const float *o = a.part_sums + 4 * (r * a.parts + threadIdx.x);
            q.m = o[0]; q.z = o[1]; q.s = o[2];
        }
        const float xt = t < 0 ? 0.f : load1(static_cast<const T *>(a.logits) + r * a.row_stride + t);
        const RowResult res(block_join(q, lds));
        if (threadIdx.x == 0) write_row(a, r, res, t, xt);
        if constexpr (TOP) {
            // the first entries of all lists, one a thread: at least `top` of them (or all there are), and the top-th greatest bounds the rest
            cand[threadIdx.x] = mine;
            if (threadIdx.x == 0) { bound = 0ull; count = 0; }
            __syncthreads();
            if (mine) {
                int rank = 0;
#pragma unroll 16
                for (int j = 0; j < kBlock; ++j) rank += cand[j] > mine ? 1 : 0;
                if (rank == a.top - 1) bound = mine;
            }
            __syncthreads();
            const unsigned long long least = bound;
            for (int i = threadIdx.x; i < a.parts * a.top; i += kBlock) {
                const unsigned long long c = lists[i];
                if (c && c >= least) cand[atomicAdd(&count, 1)] = c;
            }
            __syncthreads();
            rank_candidates(cand, count, a.top, [&](int k, unsigned long long c) {
                a.top_ids[r * a.top + k] = (unsigned)~(unsigned)c;
                a.top_log_prob[r * a.top + k] = res.log_prob(key_value((unsigned)(c >> 32)));
            });
            __syncthreads();
        }
    }
}

template <typename T, bool ONCE>
__global__ __launch_bounds__(kBlock) void log_probs_bwd_parts(LogProbsArgs a) {
    constexpr int N = Piece<T>::N, U = 2;
    const int64_t units = a.rows * a.parts;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t r = u / a.parts;
        const int64_t begin = (u - r * a.parts) * a.part_elems, end = begin + a.part_elems < a.D ? begin + a.part_elems : a.D;
        const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
        T *out = static_cast<T *>(a.grad) + r * a.grad_stride;
        const RowGrad g(a, r);
        const int t = (int)g.t;
        auto turn = [&](Piece<T> &x) {                                    // logits -> their gradients
            const int given = t - x.s;
#pragma unroll
            for (int j = 0; j < N; ++j) x.v[j] = g(x.v[j]);
            if ((unsigned)given < (unsigned)N)                            // (the one piece of the row that holds the category)
#pragma unroll
                for (int j = 0; j < N; ++j) x.v[j] += j == given ? g.gt : 0.f;
        };
        int64_t e0 = begin + (int64_t)threadIdx.x * N;
        for (; e0 + (U - 1) * kBlock * N + N <= end; e0 += U * kBlock * N) {
            Piece<T> x[U];
#pragma unroll
            for (int i = 0; i < U; ++i) x[i].template load_whole<false>(row, e0 + i * kBlock * N);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                turn(x[i]);
                x[i].template store_whole<ONCE>(out, e0 + i * kBlock * N);
            }
        }
        for (; e0 < end; e0 += kBlock * N) {
            Piece<T> x;
            x.load(row, e0, end);
            turn(x);
            x.store(out, e0, end);
        }
        if (a.g_top && !g.empty) {
            // the alternatives of this part once more, whole, over what another thread has stored: every wave waits for its stores, then all for each other
            __builtin_amdgcn_s_waitcnt(0x0F70);                           // vmcnt(0)
            __syncthreads();
            for (int i = threadIdx.x; i < a.top; i += kBlock) {
                const int64_t at = a.top_in[r * a.top + i];
                if (at < begin || at >= end) continue;
                float d = at == g.t ? g.gt : 0.f;
                for (int k = 0; k < a.top; ++k) d += a.top_in[r * a.top + k] == at ? a.g_top[r * a.top + k] : 0.f;
                store1(out + at, g(load1(row + at)) + d);
            }
        }
    }
}

// Which form takes a row: the registers of 16 lanes up to 256 elements, of a wave up to 2048, else workgroups.  Up to 512 elements without alternatives 16 lanes
// with 32 elements each share a row's closing arithmetic among four rows a wave (28 160 rows of 409: 15.4 us against 17.4 fp32, 12.8 / 16.6 bf16;
// backward, where there is none, 26.3 against 22.2); with alternatives the wave's form counts faster (8: 37.6 / 27.9 us).
constexpr int64_t kLanesMax = 2048;

// How a long row is cut.  2048 workgroups of four waves fill the card (eight a compute unit); fewer rows are cut until there are that many, into parts of at
// least kMinPart elements (below, a part's own reductions and the join cost more than the spread gives).  With alternatives, whose share of a
// part's time does not shrink with it, 1024 (64 rows of 131 072, 20: 19.2 us against 23.0; 1100 of 50 003, 8: 34.2 / 43.3; 700 of 100 003: 48.2 / 44.9).
constexpr int64_t kMinPart = 4096;
int parts_of(int64_t rows, int64_t D, int top) {
    const int64_t want = mmt::ceil_div(top ? 1024 : 2048, rows < 1 ? 1 : rows), most = D / kMinPart;
    const int64_t parts = want < most ? want : most;
    return (int)(parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts);
}
void cut(LogProbsArgs &a, int64_t parts) {
    a.part_elems = mmt::ceil_div(mmt::ceil_div(a.D, parts), 256) * 256;   // (a whole number of pieces)
    a.parts = (int)mmt::ceil_div(a.D, a.part_elems);
}
unsigned grid_of(int64_t units, int64_t most) { return (unsigned)(units < most ? units : most); }

// Logits beyond this are read, and gradients written, without staying in the caches: nothing of them would still be there for the next kernel, and the
// stream itself goes faster (4096 rows of 131 072 bf16: forward 222 -> 183 us; 1021 of 100 003: 62 -> 48, backward 87 -> 76 us).
// Below, the backward finds the logits cached (300 rows of 20 000 fp32: 22 us for both against 25).
constexpr int64_t kOnceBytes = 128 << 20;

template <typename T>
void launch_forward(LogProbsArgs a, hipStream_t st) {
    mmt::TimedSeq seq;
    if (a.D <= kLanesMax) {
        const dim3 g16(grid_of(mmt::ceil_div(a.rows, kBlock / 16), 1 << 16)), g64(grid_of(mmt::ceil_div(a.rows, kBlock / 64), 1 << 16)), b(kBlock);
        if (a.D <= 128) seq.launch(true, log_probs_fwd_lanes<T, 16, 8>, g16, b, 0, st, a);
        else if (a.D <= 256) seq.launch(true, log_probs_fwd_lanes<T, 16, 16>, g16, b, 0, st, a);
        else if (a.D <= 512 && !a.top) seq.launch(true, log_probs_fwd_lanes<T, 16, 32>, g16, b, 0, st, a);
        else if (a.D <= 512) seq.launch(true, log_probs_fwd_lanes<T, 64, 8>, g64, b, 0, st, a);
        else if (a.D <= 1024) seq.launch(true, log_probs_fwd_lanes<T, 64, 16>, g64, b, 0, st, a);
        else seq.launch(true, log_probs_fwd_lanes<T, 64, 32>, g64, b, 0, st, a);
        return;
    }
    const dim3 grid(grid_of(a.rows * a.parts, 1 << 20)), b(kBlock);
    const bool last = a.parts == 1;
    if (a.top) seq.launch(last, log_probs_fwd_parts<T, true, false>, grid, b, 0, st, a);       // (looks at the part twice)
    else if (a.rows * a.D > kOnceBytes / (int64_t)sizeof(T)) seq.launch(last, log_probs_fwd_parts<T, false, true>, grid, b, 0, st, a);
    else seq.launch(last, log_probs_fwd_parts<T, false, false>, grid, b, 0, st, a);
    if (last) return;
    const dim3 rows(grid_of(a.rows, 1 << 20));
    if (a.top) seq.launch(true, log_probs_join<T, true>, rows, b, 0, st, a);
    else seq.launch(true, log_probs_join<T, false>, rows, b, 0, st, a);
}

template <typename T>
void launch_backward(LogProbsArgs a, hipStream_t st) {
    mmt::TimedSeq seq;
    const dim3 b(kBlock);
    if (a.D <= kLanesMax) {
        const dim3 g16(grid_of(mmt::ceil_div(a.rows, kBlock / 16), 1 << 16)), g64(grid_of(mmt::ceil_div(a.rows, kBlock / 64), 1 << 16));
        if (a.D <= 128) seq.launch(true, log_probs_bwd_lanes<T, 16, 8>, g16, b, 0, st, a);
        else if (a.D <= 256) seq.launch(true, log_probs_bwd_lanes<T, 16, 16>, g16, b, 0, st, a);
        else if (a.D <= 512) seq.launch(true, log_probs_bwd_lanes<T, 64, 8>, g64, b, 0, st, a);
        else if (a.D <= 1024) seq.launch(true, log_probs_bwd_lanes<T, 64, 16>, g64, b, 0, st, a);
        else seq.launch(true, log_probs_bwd_lanes<T, 64, 32>, g64, b, 0, st, a);
        return;
    }
    cut(a, mmt::ceil_div(a.D, 16384 / (int64_t)sizeof(T)));
    const dim3 grid(grid_of(a.rows * a.parts, 1 << 20));
    if (a.rows * a.D > kOnceBytes / (int64_t)sizeof(T)) seq.launch(true, log_probs_bwd_parts<T, true>, grid, b, 0, st, a);
    else seq.launch(true, log_probs_bwd_parts<T, false>, grid, b, 0, st, a);
}

int check_rows(const char *who, int64_t rows, int64_t D, int64_t row_stride, int dtype, int ids_bytes, int top) {
    if (rows < 0 || D < 1 || D > 0x7FFFFFFF || row_stride < D || row_stride > (int64_t)1 << 40 || rows > (int64_t)1 << 40)
        return mmt::fail(MMT_ERR_BAD_SHAPE, "%s: bad shape (rows=%lld D=%lld row_stride=%lld)", who, (long long)rows, (long long)D, (long long)row_stride);
    if (dtype != MMT_DTYPE_F32 && dtype != MMT_DTYPE_BF16) return mmt::fail(MMT_ERR_BAD_FLAG, "%s: dtype %d is neither fp32 nor bf16", who, dtype);
    if (ids_bytes != 0 && ids_bytes != 4 && ids_bytes != 8) return mmt::fail(MMT_ERR_BAD_FLAG, "%s: ids of %d bytes", who, ids_bytes);
    if (top < 0 || top > MMT_LOG_PROBS_MAX_TOP || top > D)
        return mmt::fail(MMT_ERR_BAD_SHAPE, "%s: 0 <= top <= min(%d, D) (top=%d D=%lld)", who, MMT_LOG_PROBS_MAX_TOP, top, (long long)D);
    return MMT_OK;
}

}  // namespace

extern "C" int64_t mmt_log_probs_workspace_bytes(int64_t rows, int64_t D, int top, int logits_dtype) {
    if (check_rows("log_probs_workspace_bytes", rows, D, D, logits_dtype, 0, top)) return -1;
    const int64_t parts = rows == 0 || D <= kLanesMax ? 1 : parts_of(rows, D, top);
    return parts == 1 ? 0 : rows * parts * (16 + 8 * top);
}

extern "C" int mmt_log_probs_forward(int64_t rows, int64_t D, const void *logits, int64_t logit_row_stride, int logits_dtype, const void *ids,
                                     int ids_bytes, int top, float *log_prob, float *entropy, float *lse, float *stats, float *top_log_prob,
                                     int64_t *top_ids, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check_rows("log_probs_forward", rows, D, logit_row_stride, logits_dtype, ids_bytes, top)) return rc;
    if (rows == 0) return MMT_OK;
    MMT_REQUIRE_PTR(logits);
    MMT_REQUIRE_PTR(entropy);
    MMT_REQUIRE_PTR(lse);
    MMT_REQUIRE_PTR(stats);
    if ((uintptr_t)stats & 15) return mmt::fail(MMT_ERR_BAD_SHAPE, "log_probs_forward: stats is not 16-byte aligned");
    if (ids_bytes) { MMT_REQUIRE_PTR(ids); MMT_REQUIRE_PTR(log_prob); }
    if (top) { MMT_REQUIRE_PTR(top_log_prob); MMT_REQUIRE_PTR(top_ids); }
    const int64_t need = mmt_log_probs_workspace_bytes(rows, D, top, logits_dtype);
    if (need > 0) {
        MMT_REQUIRE_PTR(workspace);
        if ((uintptr_t)workspace & 15) return mmt::fail(MMT_ERR_WORKSPACE, "log_probs_forward: the workspace is not 16-byte aligned");
        if (workspace_bytes < need) return mmt::fail(MMT_ERR_WORKSPACE, "log_probs_forward: %lld bytes of workspace, %lld needed", (long long)workspace_bytes, (long long)need);
    }
    LogProbsArgs a = {};
    a.rows = rows; a.D = D; a.row_stride = logit_row_stride; a.logits = logits;
    a.ids = ids_bytes ? ids : nullptr; a.ids_bytes = ids_bytes; a.top = top;
    a.log_prob = ids_bytes ? log_prob : nullptr; a.entropy = entropy; a.lse = lse; a.stats = stats; a.top_log_prob = top_log_prob; a.top_ids = top_ids;
    a.parts = 1;
    if (D > kLanesMax) cut(a, parts_of(rows, D, top));
    a.part_sums = static_cast<float *>(workspace);
    a.part_top = reinterpret_cast<unsigned long long *>(static_cast<char *>(workspace) + rows * a.parts * 16);
    if (logits_dtype == MMT_DTYPE_F32) launch_forward<float>(a, (hipStream_t)stream);
    else launch_forward<bf16_t>(a, (hipStream_t)stream);
    return mmt::check_launch("log_probs_forward");
}

extern "C" int mmt_log_probs_backward(int64_t rows, int64_t D, const void *logits, int64_t logit_row_stride, int logits_dtype, const void *ids,
                                      int ids_bytes, int top, const float *stats, const int64_t *top_ids,
                                      const float *grad_log_prob, const float *grad_entropy, const float *grad_lse, const float *grad_top,
                                      void *grad_logits, int64_t grad_row_stride, void *stream) {
    if (int rc = check_rows("log_probs_backward", rows, D, logit_row_stride, logits_dtype, ids_bytes, top)) return rc;
    if (grad_row_stride < D || grad_row_stride > (int64_t)1 << 40)
        return mmt::fail(MMT_ERR_BAD_SHAPE, "log_probs_backward: grad_row_stride=%lld below D=%lld", (long long)grad_row_stride, (long long)D);
    if (rows == 0) return MMT_OK;
    MMT_REQUIRE_PTR(logits);
    MMT_REQUIRE_PTR(stats);
    MMT_REQUIRE_PTR(grad_logits);
    if ((uintptr_t)stats & 15) return mmt::fail(MMT_ERR_BAD_SHAPE, "log_probs_backward: stats is not 16-byte aligned");
    if (grad_logits == logits) return mmt::fail(MMT_ERR_BAD_SHAPE, "log_probs_backward: the gradient cannot overwrite the logits");
    if (ids_bytes) MMT_REQUIRE_PTR(ids);
    if (grad_top) MMT_REQUIRE_PTR(top_ids);
    LogProbsArgs a = {};
    a.rows = rows; a.D = D; a.row_stride = logit_row_stride; a.logits = logits;
    a.ids = ids_bytes ? ids : nullptr; a.ids_bytes = ids_bytes; a.top = top;
    a.g_lp = grad_log_prob; a.g_h = grad_entropy; a.g_lse = grad_lse; a.g_top = top ? grad_top : nullptr;
    a.stats_in = stats; a.top_in = top_ids; a.grad = grad_logits; a.grad_stride = grad_row_stride;
    if (logits_dtype == MMT_DTYPE_F32) launch_backward<float>(a, (hipStream_t)stream);
    else launch_backward<bf16_t>(a, (hipStream_t)stream);
    return mmt::check_launch("log_probs_backward");
}

// Gradient clipping + AdamW over many tensors with the moments in 8 bits (or, per tensor, in 32), and the moments' conversion.
//
// A moment in 8 bits: blocks of 32 elements share a power of two (one byte), the codes are E4M3 (first moment) and E5M2 (second).  The
// power of two makes scaling exact both ways, so a code read, held and written again is the same code, and all rounding is in the codes.
// At beta2 = 0.999 one step changes the second moment by about 0.1 % while neighbouring codes are 12 - 25 % apart: rounding to the
// nearest would never move it.  So the codes are rounded stochastically (the expected value is the fp32 value), by bits that are a hash
// of the element's position and the step's key: no state, the same on every rank.  Only what is stored is rounded: this step's
// parameter update takes the fp32 moments.  A positive second moment is kept at one code step at least: sqrt(v) is a divisor.
//   update: read p 4, g 4, codes 2, scales 2/32; write p 4, codes 2, scales 2/32 = 16.125 bytes an element (fp32 moments: 28)
#include <type_traits>

#include "mmt_common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kTile = 256;              // elements a wave takes at a time: 4 per lane, 8 lanes per block of 32
constexpr int kGrid = 4096;             // most workgroups of the update (2048 / 8192 measured 1 % slower); each adds the norm's partial sums up once
constexpr int kNormGrid = 1024;         // workgroups of the norm launch = partial sums that every workgroup of the update adds up

// From 128 MiB of fp32 on, what is used once passes through the caches without staying: the step's parameters and gradients (84 M elements: 333 -> 297 us),
// an unpacked moment (82 -> 67 us), a moment that is packed (79 -> 76).
constexpr int64_t kOnceElems = 32 << 20;

struct StepRow {
    int64_t grad;
    float decay, step_size, b1, c1, b2, c2, inv_bc2, eps;
};
static_assert(sizeof(StepRow) == 40, "the layout of `steps`");

struct Adam8Args {
    const int32_t *chunk_tensor;
    const int64_t *chunk_off;
    int num_chunks, chunk_elems, num_partials;
    const int64_t *tensors;
    const StepRow *steps;
    unsigned key;
    float max_norm;
    double *partials;
    float *norm_out;
};

__device__ __forceinline__ unsigned mix32(unsigned x) {
    x ^= x >> 16; x *= 0x9E3779B9u;
    x ^= x >> 13; x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// scale byte of a block whose largest magnitude has the bits `top`
template <bool SECOND>
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
    const int e = (int)(top >> 23) + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0) - (SECOND ? 15 : 8);
    return top >= 0x7F800000u ? 255u : (unsigned)(e > 0 ? e : 0);
}
__device__ __forceinline__ float scale_value(unsigned c) {
    return c == 255u ? __uint_as_float(0x7FC00000u) : c == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(c << 23);
}
__device__ __forceinline__ float scale_inverse(unsigned c) { return __uint_as_float((254u - (c == 255u ? 254u : c)) << 23); }

// largest bits among the 8 lanes of a block
__device__ __forceinline__ unsigned max8(unsigned v) {
#define MMT_DPP_MAX(ctrl) { const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, ctrl, 0xF, 0xF, true); v = v > o ? v : o; }
    MMT_DPP_MAX(0xB1)      // quad_perm [1,0,3,2]
    MMT_DPP_MAX(0x4E)      // quad_perm [2,3,0,1]
    MMT_DPP_MAX(0x141)     // row_half_mirror
#undef MMT_DPP_MAX
    return v;
}

template <bool SECOND>
__device__ __forceinline__ void decode4(unsigned codes, float scale, float *out) {
    if constexpr (SECOND) {
        out[0] = __builtin_amdgcn_cvt_f32_bf8((int)codes, 0) * scale; out[1] = __builtin_amdgcn_cvt_f32_bf8((int)codes, 1) * scale;
        out[2] = __builtin_amdgcn_cvt_f32_bf8((int)codes, 2) * scale; out[3] = __builtin_amdgcn_cvt_f32_bf8((int)codes, 3) * scale;
    } else {
        out[0] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 0) * scale; out[1] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 1) * scale;
        out[2] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 2) * scale; out[3] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 3) * scale;
    }
}

// one code; r16: 16 random bits added to the part that is cut off, or (NEAREST) the nearest code, ties to even
template <bool SECOND, bool NEAREST>
__device__ __forceinline__ unsigned encode1(float x, unsigned byte, float inv, unsigned r16) {
    constexpr int MAN = SECOND ? 2 : 3, LOWEST = SECOND ? -14 : -6, CUT = 23 - MAN;
    const unsigned xb = __float_as_uint(x);
    const float u = __uint_as_float(xb & 0x7FFFFFFFu) * inv;                     // exact: a power of two
    const unsigned ub = __float_as_uint(u);
    const unsigned add = NEAREST ? (1u << (CUT - 1)) - 1u + ((ub >> CUT) & 1u) : r16 << (CUT - 16);
    const unsigned normal = ((ub + add) >> CUT) - ((unsigned)(127 + LOWEST - 1) << MAN);
    const float f = u * (float)(1 << (MAN - LOWEST));
    const unsigned below = (unsigned)(NEAREST ? rintf(f) : floorf(f + (float)r16 * 0x1p-16f));
    unsigned code = u >= (LOWEST == -14 ? 0x1p-14f : 0x1p-6f) ? normal : below;
    if (SECOND && x > 0.f && code == 0u) code = 1u;
    code |= (xb >> 24) & 0x80u;
    return byte == 255u ? 0u : code;
}

template <bool SECOND>
__device__ __forceinline__ unsigned encode4_nearest(const float *x, unsigned byte) {
    const float inv = scale_inverse(byte);
    unsigned out = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) out |= encode1<SECOND, true>(x[j], byte, inv, 0u) << (8 * j);
    return out;
}

// The same codes as encode1's, stochastically rounded, in three operations each: scaled by a further 2^-8 (E4M3) / 2^-16 (E5M2), the low bits of the fp32
// exponent ARE the code's, so that the code is a bit field of bits + random.  The lowest codes (multiples of one step, and 0) and blocks near
// the end of fp32's range are put right in a branch that few waves take.
template <bool SECOND>
__device__ __forceinline__ unsigned encode4_stochastic(const float *x, unsigned byte, const unsigned *r16) {
    constexpr int CUT = SECOND ? 21 : 20, DOWN = SECOND ? 16 : 8;
    constexpr float LEAST = SECOND ? 0x1p-30f : 0x1p-14f, STEPS = SECOND ? 0x1p32f : 0x1p17f;      // the lowest normal code, 1 / a step, in scaled units
    const float inv = __uint_as_float((254u - DOWN - (byte > 236u ? 236u : byte)) << 23);
    float u[4];
    unsigned code[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        u[j] = fabsf(x[j]) * inv;
        code[j] = ((__float_as_uint(u[j]) + (r16[j] << (CUT - 16))) >> CUT) & 0x7Fu;
    }
    if (!(fminf(fminf(u[0], u[1]), fminf(u[2], u[3])) >= LEAST) || byte > 236u) {
        if (byte > 236u) {
            const float whole = scale_inverse(byte);
#pragma unroll
            for (int j = 0; j < 4; ++j) code[j] = encode1<SECOND, false>(x[j], byte, whole, r16[j]) & 0x7Fu;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned below = (unsigned)fmaf((float)r16[j], 0x1p-16f, u[j] * STEPS);
                if (SECOND) below = x[j] > 0.f && below == 0u ? 1u : below;
                code[j] = u[j] >= LEAST ? code[j] : below;
            }
        }
    }
    unsigned out = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (!SECOND) code[j] |= (__float_as_uint(x[j]) >> 24) & (byte == 255u ? 0u : 0x80u);
        out |= code[j] << (8 * j);
    }
    return out;
}

__device__ __forceinline__ unsigned top_bits(const float *x) {
    unsigned t = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) { const unsigned b = __float_as_uint(x[j]) & 0x7FFFFFFFu; t = t > b ? t : b; }
    return t;
}

__device__ __forceinline__ double block_sum(double v, double *lds) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.;
#pragma unroll
    for (int w = 0; w < kBlock / 64; ++w) t += lds[w];        // (fixed order: the same bits in every workgroup)
    __syncthreads();
    return t;
}

// the same in all lanes: into scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return __int_as_float(uniform(__float_as_int(v))); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)(((uint64_t)(unsigned)uniform((int)(v >> 32)) << 32) | (unsigned)uniform((int)v));
}

// addresses that come as integers are global ones (a generic pointer's loads count as shared-memory ones too and cannot be waited for one by one)
template <typename T> using Global = __attribute__((address_space(1))) T *;
template <typename T> __device__ __forceinline__ Global<T> global(int64_t at) { return reinterpret_cast<Global<T>>(at); }

// four elements from an address that is aligned to one element only
typedef unsigned four_f32 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned four_bf16 __attribute__((ext_vector_type(2), aligned(2)));

// elements i .. i + 3 of a tensor as fp32; WHOLE: all below `end`, else zeros from there on; ONCE: passing through the caches without staying
template <bool BF16, bool WHOLE, bool ONCE = false>
__device__ __forceinline__ void load4(int64_t base, int64_t i, int64_t end, float *out) {
    using E = typename std::conditional<BF16, bf16_t, float>::type;
    const Global<const E> at = global<const E>(base) + i;
    if (WHOLE || i + 4 <= end) {
        if constexpr (BF16) {
            const Global<const four_bf16> from = reinterpret_cast<Global<const four_bf16>>(at);
            const four_bf16 t = ONCE ? __builtin_nontemporal_load(from) : *from;
            out[0] = bf16_lo(t.x); out[1] = bf16_hi(t.x); out[2] = bf16_lo(t.y); out[3] = bf16_hi(t.y);
        } else {
            const Global<const four_f32> from = reinterpret_cast<Global<const four_f32>>(at);
            const four_f32 t = ONCE ? __builtin_nontemporal_load(from) : *from;
            out[0] = __uint_as_float(t.x); out[1] = __uint_as_float(t.y); out[2] = __uint_as_float(t.z); out[3] = __uint_as_float(t.w);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v = 0.f;
            if (i + j < end) {
                if constexpr (BF16) v = __uint_as_float((unsigned)at[j] << 16);
                else v = at[j];
            }
            out[j] = v;
        }
    }
}

template <bool ONCE = false>
__device__ __forceinline__ void store4(int64_t base, int64_t i, const float *x) {
    const four_f32 t = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    const Global<four_f32> to = global<four_f32>(base + 4 * i);
    if constexpr (ONCE) __builtin_nontemporal_store(t, to);
    else *to = t;
}

template <bool BF16>
__device__ __forceinline__ double sumsq_of(int64_t grad, int64_t off, int64_t end) {
    double s = 0.;
    int64_t i = off + 4 * threadIdx.x;
    constexpr int U = 4;
    for (; i + (U - 1) * 4 * kBlock + 4 <= end; i += U * 4 * kBlock) {
        float g[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) load4<BF16, true>(grad, i + u * 4 * kBlock, end, g[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) s = fma((double)g[u][j], (double)g[u][j], s);        // (the product of two fp32 is exact)
    }
    for (; i < end; i += 4 * kBlock) {
        float g[4];
        load4<BF16, false>(grad, i, end, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) s = fma((double)g[j], (double)g[j], s);
    }
    return s;
}

__global__ __launch_bounds__(kBlock) void adamw8_sumsq(Adam8Args a) {
    __shared__ double lds[kBlock / 64];
    double s = 0.;
    for (int c = blockIdx.x; c < a.num_chunks; c += gridDim.x) {
        const int t = a.chunk_tensor[c];
        const int64_t *row = a.tensors + (int64_t)t * MMT_ADAMW8_COLUMNS;
        const int64_t n = uniform(row[6]), off = uniform(a.chunk_off[c]), grad = uniform(a.steps[t].grad);
        const int64_t end = off + a.chunk_elems < n ? off + a.chunk_elems : n;
        s += uniform(row[8]) == MMT_DTYPE_BF16 ? sumsq_of<true>(grad, off, end) : sumsq_of<false>(grad, off, end);
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = s;
}

// A tensor's row of the table and of this step, the same for all lanes: kept in scalar registers (read through the vector cache, they would be read
// again after every store, which may alias them as far as the compiler knows)
struct Tensor {
    int64_t param, grad, m, v, m_scale, v_scale, shadow, n;
    unsigned position;
    bool bf16;
    float decay, step_size, b1, c1, b2, c2, inv_bc2, eps;
};
__device__ __forceinline__ Tensor tensor_row(const Adam8Args &a, int t) {
    const int64_t *row = a.tensors + (int64_t)t * MMT_ADAMW8_COLUMNS;
    const StepRow h = a.steps[t];
    return Tensor{uniform(row[0]), uniform(h.grad), uniform(row[1]), uniform(row[2]), uniform(row[3]), uniform(row[4]), uniform(row[5]), uniform(row[6]),
                  (unsigned)uniform((int)row[7]), uniform((int)row[8]) == MMT_DTYPE_BF16, uniform(h.decay), uniform(h.step_size), uniform(h.b1),
                  uniform(h.c1), uniform(h.b2), uniform(h.c2), uniform(h.inv_bc2), uniform(h.eps)};
}

// One lane's share of a tile: elements i .. i + 3
template <bool BF16, bool PACKED, bool WHOLE, bool ONCE>
struct Lane4 {
    float p[4], g[4], m[4], v[4];
    unsigned cm, cv, sm, sv;

    __device__ __forceinline__ void load(const Tensor &t, int64_t i, int64_t end) {
        load4<BF16, WHOLE, ONCE>(t.param, i, end, p);
        load4<BF16, WHOLE, ONCE>(t.grad, i, end, g);
        if constexpr (PACKED) {
            cm = *global<const unsigned>(t.m + i);
            cv = *global<const unsigned>(t.v + i);
            sm = global<const uint8_t>(t.m_scale)[i >> 5];
            sv = global<const uint8_t>(t.v_scale)[i >> 5];
        } else {
            load4<false, true>(t.m, i, 0, m);
            load4<false, true>(t.v, i, 0, v);
        }
    }

    // The quotient m / (sqrt(v) + eps) comes from the hardware's approximate square root and reciprocal (1 unit in the last place each): it only moves
    // the parameter by lr times itself, while the moments, whose codes depend on every bit, use exact operations.  The approximate root
    // flushes far below 2^-96: those few (eps = 0 would divide by it) take the exact one.
    __device__ __forceinline__ void step(const Tensor &t, unsigned key, float coef, int64_t i, int64_t end, int lane) {
        if constexpr (PACKED) {
            decode4<false>(cm, scale_value(sm), m);
            decode4<true>(cv, scale_value(sv), v);
        }
        unsigned hash[4];
        if (PACKED || BF16) {
            const unsigned at = t.position + (unsigned)i + key;
#pragma unroll
            for (int j = 0; j < 4; ++j) hash[j] = mix32(at + j);
        }
        float root[4];
        unsigned tiny = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gc = g[j] * coef;
            m[j] = m[j] * t.b1 + gc * t.c1;
            v[j] = v[j] * t.b2 + (gc * t.c2) * gc;
            root[j] = __builtin_amdgcn_sqrtf(v[j]);
            const unsigned b = __float_as_uint(v[j]) - 1u;                // (0 wraps to the top)
            tiny = tiny < b ? tiny : b;
        }
        if (tiny < 0x0F800000u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) root[j] = sqrtf(v[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float denom = fmaf(root[j], t.inv_bc2, t.eps);
            p[j] = fmaf(-(m[j] * t.step_size), __builtin_amdgcn_rcpf(denom), p[j] * t.decay);
            if (!WHOLE && i + j >= end) { m[j] = 0.f; v[j] = 0.f; }
        }
        if constexpr (PACKED) {
            unsigned r1[4], r2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { r1[j] = hash[j] >> 16; r2[j] = hash[j] & 0xFFFFu; }
            const unsigned bm = scale_byte<false>(max8(top_bits(m))), bv = scale_byte<true>(max8(top_bits(v)));
            *global<unsigned>(t.m + i) = encode4_stochastic<false>(m, bm, r1);
            *global<unsigned>(t.v + i) = encode4_stochastic<true>(v, bv, r2);
            if ((lane & 7) == 0) {
                global<uint8_t>(t.m_scale)[i >> 5] = (uint8_t)bm;
                global<uint8_t>(t.v_scale)[i >> 5] = (uint8_t)bv;
            }
        } else {
            store4(t.m, i, m);
            store4(t.v, i, v);
        }
        if (BF16 || t.shadow) {                                           // bf16 parameters: rounded stochastically, like the codes; copies: to nearest
            bf16_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // (bits + 16 random ones: an infinity stays one)
                if (BF16) q[j] = (bf16_t)((__float_as_uint(p[j]) + ((hash[j] * 0x6A09E667u) >> 16)) >> 16);
                else q[j] = (bf16_t)(pack_bf16x2(p[j], 0.f) & 0xFFFFu);
            }
            // A NaN with ones in its low half (from an fp32 gradient through the norm, from an fp32 moment) could be carried past the largest pattern, into 0:
            // it is made the quiet one.  Two comparisons for the four elements.
            if (BF16 && (__builtin_isunordered(p[0], p[1]) || __builtin_isunordered(p[2], p[3]))) {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = p[j] != p[j] ? (bf16_t)0x7FC0 : q[j];
            }
            const Global<bf16_t> to = global<bf16_t>(BF16 ? t.param : t.shadow) + i;
            if (WHOLE || i + 4 <= end) {
                const four_bf16 two = {q[0] | ((unsigned)q[1] << 16), q[2] | ((unsigned)q[3] << 16)};
                if constexpr (ONCE) __builtin_nontemporal_store(two, reinterpret_cast<Global<four_bf16>>(to));
                else *reinterpret_cast<Global<four_bf16>>(to) = two;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < end) to[j] = q[j];
            }
        }
        if constexpr (!BF16) {
            const Global<float> to = global<float>(t.param) + i;
            if (WHOLE || i + 4 <= end) {
                store4<ONCE>(t.param, i, p);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < end) to[j] = p[j];
            }
        }
    }
};

// A wave takes UNROLL tiles at a time: the loads of all of them are under way before the first is computed (fp32: 333 us with two, 344 with one at 84 M elements;
// bf16, bound by its arithmetic: 85 us with two, 77 with one at 31 M).
template <bool BF16, bool PACKED, bool ONCE>
__device__ __forceinline__ void update_chunk(const Tensor &t, unsigned key, float coef, int64_t off, int64_t end) {
    constexpr int UNROLL = BF16 ? 1 : 2, STRIDE = kTile * (kBlock / 64);
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    int64_t i0 = off + wave * kTile;
    for (; i0 + (UNROLL - 1) * STRIDE + kTile <= end; i0 += UNROLL * STRIDE) {
        Lane4<BF16, PACKED, true, ONCE> x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) x[u].load(t, i0 + u * STRIDE + 4 * lane, end);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) x[u].step(t, key, coef, i0 + u * STRIDE + 4 * lane, end, lane);
    }
    for (; i0 < end; i0 += STRIDE) {
        Lane4<BF16, PACKED, false, ONCE> x;
        x.load(t, i0 + 4 * lane, end);
        x.step(t, key, coef, i0 + 4 * lane, end, lane);
    }
}

template <bool ONCE>
__global__ __launch_bounds__(kBlock) void adamw8_update(Adam8Args a) {
    __shared__ double lds[kBlock / 64];
    float coef = 1.f, norm = 0.f;
    if (a.max_norm > 0.f) {
        double s = 0.;
        for (int i = threadIdx.x; i < a.num_partials; i += kBlock) s += a.partials[i];
        const double total = sqrt(block_sum(s, lds));
        const double c = (double)a.max_norm / (total + 1e-6);
        coef = (float)(c < 1. ? c : 1.);
        if (total != total) coef = (float)total;             // a NaN norm poisons the update, like a multiply by a NaN coefficient
        norm = (float)total;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) { a.norm_out[0] = norm; a.norm_out[1] = coef; }
    for (int c = blockIdx.x; c < a.num_chunks; c += gridDim.x) {
        const int t = a.chunk_tensor[c];
        const Tensor row = tensor_row(a, uniform(t));
        const int64_t off = uniform(a.chunk_off[c]), end = off + a.chunk_elems < row.n ? off + a.chunk_elems : row.n;
        if (row.bf16) {
            if (row.m_scale) update_chunk<true, true, ONCE>(row, a.key, coef, off, end);
            else update_chunk<true, false, ONCE>(row, a.key, coef, off, end);
        } else {
            if (row.m_scale) update_chunk<false, true, ONCE>(row, a.key, coef, off, end);
            else update_chunk<false, false, ONCE>(row, a.key, coef, off, end);
        }
    }
}

template <bool SECOND, bool ONCE>
__global__ __launch_bounds__(kBlock) void moment_pack(int64_t n, const float *x, uint8_t *codes, uint8_t *scales) {
    const int64_t blocks4 = (n + 31) / 32 * 8;              // groups of four, whole blocks (eight lanes take part together)
    for (int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x; q < blocks4; q += (int64_t)gridDim.x * kBlock) {
        const int64_t i = 4 * q;
        float v[4];
        load4<false, false, ONCE>((int64_t)x, i, n, v);
        const unsigned byte = scale_byte<SECOND>(max8(top_bits(v)));
        const unsigned c = encode4_nearest<SECOND>(v, byte);
        if (i + 4 <= n) *reinterpret_cast<unsigned *>(codes + i) = c;
        else
            for (int j = 0; j < 4 && i + j < n; ++j) codes[i + j] = (uint8_t)(c >> (8 * j));
        if ((q & 7) == 0) scales[q >> 3] = (uint8_t)byte;
    }
}

template <bool SECOND, bool ONCE>
__global__ __launch_bounds__(kBlock) void moment_unpack(int64_t n, const uint8_t *codes, const uint8_t *scales, float *x) {
    const int64_t groups = (n + 3) / 4;
    for (int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x; q < groups; q += (int64_t)gridDim.x * kBlock) {
        const int64_t i = 4 * q;
        unsigned c = 0;
        if (i + 4 <= n) c = *reinterpret_cast<const unsigned *>(codes + i);
        else
            for (int j = 0; j < 4 && i + j < n; ++j) c |= (unsigned)codes[i + j] << (8 * j);
        float v[4];
        decode4<SECOND>(c, scale_value(scales[q >> 3]), v);
        if (i + 4 <= n) store4<ONCE>((int64_t)x, i, v);
        else
            for (int j = 0; j < 4 && i + j < n; ++j) x[i + j] = v[j];
    }
}

int check_moment(const char *who, int64_t n, const void *codes) {
    if (n < 0 || n > (int64_t)1 << 45) return mmt::fail(MMT_ERR_BAD_SHAPE, "%s: n=%lld", who, (long long)n);
    if ((uintptr_t)codes & 3) return mmt::fail(MMT_ERR_BAD_SHAPE, "%s: the codes are not 4-byte aligned", who);
    return MMT_OK;
}

}  // namespace

extern "C" int mmt_moment_pack(int64_t n, const float *x, int second, void *codes, void *scales, void *stream) {
    if (int rc = check_moment("moment_pack", n, codes)) return rc;
    if (n == 0) return MMT_OK;
    MMT_REQUIRE_PTR(x);
    MMT_REQUIRE_PTR(codes);
    MMT_REQUIRE_PTR(scales);
    const dim3 grid(mmt::stream_grid((n + 31) / 32 * 8, kBlock, 256 * 32));
    uint8_t *c = static_cast<uint8_t *>(codes), *e = static_cast<uint8_t *>(scales);
    mmt::TimedSeq seq;
    auto kernel = n > kOnceElems ? (second ? moment_pack<true, true> : moment_pack<false, true>) : (second ? moment_pack<true, false> : moment_pack<false, false>);
    seq.launch(true, kernel, grid, dim3(kBlock), 0, (hipStream_t)stream, n, x, c, e);
    return mmt::check_launch("moment_pack");
}

extern "C" int mmt_moment_unpack(int64_t n, const void *codes, const void *scales, int second, float *x, void *stream) {
    if (int rc = check_moment("moment_unpack", n, codes)) return rc;
    if (n == 0) return MMT_OK;
    MMT_REQUIRE_PTR(x);
    MMT_REQUIRE_PTR(codes);
    MMT_REQUIRE_PTR(scales);
    const dim3 grid(mmt::stream_grid((n + 3) / 4, kBlock, 256 * 32));
    const uint8_t *c = static_cast<const uint8_t *>(codes), *e = static_cast<const uint8_t *>(scales);
    mmt::TimedSeq seq;
    auto kernel = n > kOnceElems ? (second ? moment_unpack<true, true> : moment_unpack<false, true>) : (second ? moment_unpack<true, false> : moment_unpack<false, false>);
    seq.launch(true, kernel, grid, dim3(kBlock), 0, (hipStream_t)stream, n, c, e, x);
    return mmt::check_launch("moment_unpack");
}

extern "C" int mmt_clip_adamw8_partials(int num_chunks) { return num_chunks < 1 ? 1 : num_chunks < kNormGrid ? num_chunks : kNormGrid; }

extern "C" int mmt_clip_adamw8_step(int num_chunks, int chunk_elems, const int32_t *chunk_tensor, const int64_t *chunk_offset, const int64_t *tensors,
                                    const int64_t *steps, uint32_t key, float max_norm, double *partials, float *norm_out, void *stream) {
    if (num_chunks < 0 || chunk_elems <= 0 || chunk_elems % kTile)
        return mmt::fail(MMT_ERR_BAD_SHAPE, "clip_adamw8_step: chunks of a multiple of %d elements (chunks=%d chunk_elems=%d)", kTile, num_chunks, chunk_elems);
    if (num_chunks == 0) return MMT_OK;
    MMT_REQUIRE_PTR(chunk_tensor);
    MMT_REQUIRE_PTR(chunk_offset);
    MMT_REQUIRE_PTR(tensors);
    MMT_REQUIRE_PTR(steps);
    MMT_REQUIRE_PTR(norm_out);
    if (max_norm > 0.f) MMT_REQUIRE_PTR(partials);
    Adam8Args a = {};
    a.chunk_tensor = chunk_tensor; a.chunk_off = chunk_offset; a.num_chunks = num_chunks; a.chunk_elems = chunk_elems;
    a.tensors = tensors; a.steps = reinterpret_cast<const StepRow *>(steps); a.key = key; a.max_norm = max_norm; a.partials = partials; a.norm_out = norm_out;
    a.num_partials = mmt_clip_adamw8_partials(num_chunks);
    hipStream_t st = (hipStream_t)stream;
    mmt::TimedSeq seq;
    if (max_norm > 0.f) {
        seq.launch(false, adamw8_sumsq, dim3(a.num_partials), dim3(kBlock), 0, st, a);
        if (int rc = mmt::check_launch("clip_adamw8_step(norm)")) return rc;
    }
    // (counted by the chunks: many small tensors count as more than they are)
    const dim3 grid(num_chunks < kGrid ? num_chunks : kGrid);
    if ((int64_t)num_chunks * chunk_elems > kOnceElems) seq.launch(true, adamw8_update<true>, grid, dim3(kBlock), 0, st, a);
    else seq.launch(true, adamw8_update<false>, grid, dim3(kBlock), 0, st, a);
    return mmt::check_launch("clip_adamw8_step(update)");
}

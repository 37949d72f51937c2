// Multi-tensor AdamW step (states in fp32 or in 8 bits) and the global gradient norm (gfx950).
//
// Step t of one element, all in fp32 and rounded after every operation (no contraction, IEEE square root and division):
//   g' = s g;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p  = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// s = grad_scale * clip coefficient, two numbers in device memory.  16-bit parameters have an fp32 master copy that takes
// the update; the parameter is its rounding (the one rounding to fewer bits; without the master copy updates below 2^-9 of
// a bf16 weight would be lost).
//
// 8-bit states.  Blocks of 128 consecutive elements share one exponent byte E per state; an element is an OCP e4m3 code c:
//   m = e4m3(c) 2^(E - 127),   sqrt(v) = e4m3(c') 2^(E' - 127),   E = max(exponent byte of max |x| - 7, 1)
// so that the block's largest value lies in [128, 256): the code above it, 256, is still below the largest one (448).
// sqrt(v) and not v is held: its dynamic range is half of v's.  Rounding to the code is stochastic, with 16 bits per value of
// a hash of (seed, step, tensor, element): to the upper neighbour with the probability that keeps the mean.  Rounding to
// the nearest would freeze the second moment: one step with b2 = 0.999 changes sqrt(v) by about 0.05 %, half a code is
// 3 - 6 %.  A value sqrt(v) > 0 keeps at least the smallest code (2^-9): zero would divide m by eps alone.  Values that are
// not finite do not enter the block's maximum and become the largest code; their parameter is NaN by then, as with 32 bits,
// and their neighbours are not touched.
//
// Bound by memory: 28 bytes per element with fp32 states, 16 with 8-bit states (fp32: p and g in, p out; with 16-bit
// parameters master and g in, master and p out).  120 M bf16 parameters with fp32 states: 618 us, 5.4 TB/s, which is what the best
// copy reaches; 159 M with 8-bit states: 501 us, 5.1 TB/s, the vector units busy 67 % of the time (76 instructions an
// element); 127 tensors of 174 k elements in all: 5.6 us, one launch, bound by its chain of dependent loads.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define OPT_BLOCK 128                // elements that share an exponent byte
#define OPT_ENTRIES 648              // 48-bit entries of the tensors' table in the kernel arguments (3.8 of 4 KiB)
#define OPT_THREADS 256
#define OPT_PER_LANE 8               // consecutive elements of a lane
#define OPT_STRIDE (OPT_THREADS * OPT_PER_LANE)
#define OPT_VEC (1ull << 47)         // flag in a tensor's element count: every pointer allows 16-byte (codes: 8-byte) access

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// The tensors of a launch, in its arguments: a step over small tensors is as long as its launches, so that as many tensors as
// possible share one.  Entry f of tensor k is number f * cap + k: 0 its element count (with OPT_VEC), then its addresses
// (user addresses have 47 bits): parameter, gradient, exp_avg, exp_avg_sq [, master] [, exponent bytes of exp_avg, of
// exp_avg_sq].  129 tensors with fp32 states fit, 92 with 8-bit ones, 324 gradients.
struct OptTable {
    uint32_t lo[OPT_ENTRIES];
    uint32_t hi[OPT_ENTRIES / 2];    // two 16-bit halves
    uint32_t ordinal;                // number of the first tensor (enters the hash)
    int n, cap;                      // tensors, places
    uint32_t span, span_log2;        // elements of a workgroup
};
__device__ __forceinline__ uint64_t opt_entry(const OptTable& t, int field, int k) {
    const int e = field * t.cap + k;
    return ((uint64_t)(t.hi[e >> 1] >> (16 * (e & 1)) & 0xFFFFu) << 32) | t.lo[e];
}

struct AdamwHyper {
    float b1, omb1, b2, omb2, eps, decay, step_size, inv_sqrt_bc2;
    uint32_t key;                    // hash of seed and step
    uint32_t pad;
};

// A published mixing function of 32-bit integers (C. Wellons, 2018; its shifts and multipliers come from a search for low bias).  The
// hash's other constants are published ones too: 2^32 over the golden ratio, and two multipliers of A. Appleby's (2011).
__device__ __host__ inline uint32_t opt_mix(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352dU; x ^= x >> 15; x *= 0x846ca68bU; x ^= x >> 16;
    return x;
}
__device__ __host__ inline uint32_t opt_key(uint64_t seed, uint64_t step) {
    uint32_t k = opt_mix((uint32_t)seed ^ 0x9E3779B9U);
    k = opt_mix(k ^ (uint32_t)(seed >> 32));
    k = opt_mix(k ^ (uint32_t)step);
    return opt_mix(k ^ (uint32_t)(step >> 32));
}
// Hyperparameters of one step in double precision, rounded once (1 - 0.999 in fp32 arithmetic is 1.3e-5 off).
__device__ __host__ inline AdamwHyper opt_hyper(double lr, double b1, double b2, double eps, double wd, long long step, uint64_t seed) {
    AdamwHyper h;
    h.b1 = (float)b1; h.omb1 = (float)(1.0 - b1);
    h.b2 = (float)b2; h.omb2 = (float)(1.0 - b2);
    h.eps = (float)eps; h.decay = (float)(1.0 - lr * wd);
    h.step_size = (float)(lr / (1.0 - pow(b1, (double)step)));
    h.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
    h.key = opt_key(seed, (uint64_t)step);
    h.pad = 0;
    return h;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t opt_scan_step(uint32_t x) {
    return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
// The tensor that this workgroup works on and which of its units: a lane adds the units of a few tensors, a scan over the
// wavefront places them (no table of first workgroups, whose room goes to more tensors).
template <int MOST>
__device__ __forceinline__ int opt_find(const OptTable& t, uint32_t* unit) {
    const int lane = threadIdx.x & 63, per = (t.n + 63) >> 6;
    const auto units = [&](int k) { return (uint32_t)(((opt_entry(t, 0, k) & ~OPT_VEC) + t.span - 1) >> t.span_log2); };
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < (MOST + 63) / 64; ++j) {                    // all loads at once: places without a tensor read the first
        const int k = lane * per + j;
        const bool there = j < per && k < t.n;
        const uint32_t u = units(there ? k : 0);
        mine += there ? u : 0;
    }
    uint32_t up_to = mine;                                          // sum over this lane and those before it
    up_to = opt_scan_step<0x111, 0xf>(up_to);
    up_to = opt_scan_step<0x112, 0xf>(up_to);
    up_to = opt_scan_step<0x114, 0xf>(up_to);
    up_to = opt_scan_step<0x118, 0xf>(up_to);
    up_to = opt_scan_step<0x142, 0xa>(up_to);
    up_to = opt_scan_step<0x143, 0xc>(up_to);
    const uint64_t has = __ballot(blockIdx.x >= up_to - mine && blockIdx.x < up_to);
    const int owner = __builtin_ctzll(has);
    uint32_t rest = blockIdx.x - (uint32_t)__builtin_amdgcn_readlane((int)(up_to - mine), owner);
    int k = __builtin_amdgcn_readfirstlane(owner * per);
    for (uint32_t u; rest >= (u = units(k)); ++k) rest -= u;
    *unit = rest;
    return k;
}

// Eight elements at i: a 16-byte access for each four (16-bit types: eight) where `vec` (the tensor's addresses allow it) and
// all eight exist, single ones otherwise.  FULL: both hold for the whole workgroup, and no branch stands between its loads.
template <bool FULL, typename T>
__device__ __forceinline__ void opt_load(const T* __restrict__ p, uint64_t i, int left, bool vec, float* out) {
    if (FULL || (vec && left >= OPT_PER_LANE)) {
        if constexpr (sizeof(T) == 4) {
            const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p + i), b = *reinterpret_cast<const f32x4_t*>(p + i + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) { out[k] = a[k]; out[4 + k] = b[k]; }
        } else {
            typedef T vec_t __attribute__((ext_vector_type(8)));
            const vec_t a = *reinterpret_cast<const vec_t*>(p + i);
#pragma unroll
            for (int k = 0; k < 8; ++k) out[k] = (float)a[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < OPT_PER_LANE; ++k) out[k] = k < left ? (float)p[i + k] : 0.f;
    }
}
template <bool FULL, typename T>
__device__ __forceinline__ void opt_store(T* __restrict__ p, uint64_t i, int left, bool vec, const float* in) {
    if (FULL || (vec && left >= OPT_PER_LANE)) {
        if constexpr (sizeof(T) == 4) {
            f32x4_t a, b;
#pragma unroll
            for (int k = 0; k < 4; ++k) { a[k] = in[k]; b[k] = in[4 + k]; }
            *reinterpret_cast<f32x4_t*>(p + i) = a;
            *reinterpret_cast<f32x4_t*>(p + i + 4) = b;
        } else {
            typedef T vec_t __attribute__((ext_vector_type(8)));
            vec_t a;
#pragma unroll
            for (int k = 0; k < 8; ++k) a[k] = (T)in[k];
            *reinterpret_cast<vec_t*>(p + i) = a;
        }
    } else {
#pragma unroll
        for (int k = 0; k < OPT_PER_LANE; ++k)
            if (k < left) p[i + k] = (T)in[k];
    }
}
template <bool FULL>
__device__ __forceinline__ void opt_load_codes(const uint8_t* __restrict__ p, uint64_t i, int left, bool vec, uint32_t* out) {
    if (FULL || (vec && left >= OPT_PER_LANE)) {
        const uint2 a = *reinterpret_cast<const uint2*>(p + i);
        out[0] = a.x; out[1] = a.y;
    } else {
        out[0] = out[1] = 0;
#pragma unroll
        for (int k = 0; k < OPT_PER_LANE; ++k)
            if (k < left) out[k >> 2] |= (uint32_t)p[i + k] << (8 * (k & 3));
    }
}
template <bool FULL>
__device__ __forceinline__ void opt_store_codes(uint8_t* __restrict__ p, uint64_t i, int left, bool vec, const uint32_t* in) {
    if (FULL || (vec && left >= OPT_PER_LANE)) {
        *reinterpret_cast<uint2*>(p + i) = make_uint2(in[0], in[1]);
    } else {
#pragma unroll
        for (int k = 0; k < OPT_PER_LANE; ++k)
            if (k < left) p[i + k] = (uint8_t)(in[k >> 2] >> (8 * (k & 3)));
    }
}

template <int N>
__device__ __forceinline__ uint32_t opt_ror(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf, 0xf, false);
}
// Largest value over the 16 lanes that hold a block (one DPP row).
__device__ __forceinline__ uint32_t opt_max16(uint32_t x) {
    x = max(x, opt_ror<8>(x));
    x = max(x, opt_ror<4>(x));
    x = max(x, opt_ror<2>(x));
    return max(x, opt_ror<1>(x));
}
// The exponent byte of a block whose largest finite |x| has the bits `top`.
__device__ __forceinline__ uint32_t opt_exponent(uint32_t top) {
    const int e = (int)(top >> 23) - 7;
    return (uint32_t)max(e, 1);
}
__device__ __forceinline__ float opt_pow2(uint32_t exponent_byte) { return __builtin_bit_cast(float, exponent_byte << 23); }

// e4m3 code of a value that is finite and scaled to its block (>= 0, < 512), rounded up if the 20 bits below the code's last
// one and the 16 random bits (in place, shifted by 4) carry.  Below 2^-6 the steps are 2^-9: adding 2^-6 moves the value
// into the binade that has these steps, which starts at code 0 instead of 8.
__device__ __forceinline__ uint32_t opt_code(float scaled, uint32_t random) {
#pragma clang fp contract(off)
    const bool small = scaled < 0.015625f;
    const float y = small ? scaled + 0.015625f : scaled;
    return (__builtin_bit_cast(uint32_t, y) + random + (small ? 0u - (121u << 23) : 0u - (120u << 23))) >> 20;
}

template <typename P>
struct AdamwTensor {
    P* p;
    const P* g;
    void *m, *v;
    float* master;
    uint8_t *exp_m, *exp_v;
};
// Eight elements of every lane, from i on; `left` of them exist (FULL: all).
template <bool FULL, typename P, bool MASTER, bool EIGHT>
__device__ __forceinline__ void adamw_elements(const AdamwTensor<P>& w, uint64_t i, int left, bool vec, const AdamwHyper& h, float s, uint32_t key) {
#pragma clang fp contract(off)
    float gi[OPT_PER_LANE], pi[OPT_PER_LANE], m[OPT_PER_LANE], r[OPT_PER_LANE];
    opt_load<FULL>(w.g, i, left, vec, gi);
    if constexpr (MASTER) opt_load<FULL>(w.master, i, left, vec, pi);
    else opt_load<FULL>(w.p, i, left, vec, pi);
    if constexpr (EIGHT) {
        uint32_t cm[2], cr[2];
        opt_load_codes<FULL>((const uint8_t*)w.m, i, left, vec, cm);
        opt_load_codes<FULL>((const uint8_t*)w.v, i, left, vec, cr);
        // a power of two times b1 is exact, and the product below rounds as b1 times the moment does
        const float sm = opt_pow2(FULL || left ? w.exp_m[i / OPT_BLOCK] : 0) * h.b1, sr = opt_pow2(FULL || left ? w.exp_v[i / OPT_BLOCK] : 0);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(cm[q], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(cm[q], true);
            const auto c = __builtin_amdgcn_cvt_pk_f32_fp8(cr[q], false), d = __builtin_amdgcn_cvt_pk_f32_fp8(cr[q], true);
            m[4 * q] = a[0] * sm; m[4 * q + 1] = a[1] * sm; m[4 * q + 2] = b[0] * sm; m[4 * q + 3] = b[1] * sm;
            r[4 * q] = c[0] * sr; r[4 * q + 1] = c[1] * sr; r[4 * q + 2] = d[0] * sr; r[4 * q + 3] = d[1] * sr;
        }
    } else {
        opt_load<FULL>((const float*)w.m, i, left, vec, m);
        opt_load<FULL>((const float*)w.v, i, left, vec, r);
    }
    uint32_t top_m = 0, top_r = 0;
#pragma unroll
    for (int e = 0; e < OPT_PER_LANE; ++e) {
        const float ge = gi[e] * s;
        float v = EIGHT ? r[e] * r[e] : r[e];
        m[e] = (EIGHT ? m[e] : h.b1 * m[e]) + h.omb1 * ge;
        v = h.b2 * v + h.omb2 * (ge * ge);
        const float root = __builtin_sqrtf(v);
        const float below = root * h.inv_sqrt_bc2 + h.eps;
        // 8 bits: the vector units are nearly as busy as memory; the reciprocal (1 ulp; `below` is at least eps, and below
        // 1e28, whose reciprocal is normal; an eps under 2^-126 is as none) saves 10 instructions an element
        const float change = EIGHT ? m[e] * __builtin_amdgcn_rcpf(below) : m[e] / below;
        pi[e] = pi[e] * h.decay - h.step_size * change;
        r[e] = EIGHT ? root : v;
    }
    if constexpr (EIGHT) {
#pragma unroll
        for (int e = 0; e < OPT_PER_LANE; e += 2) {
            top_m = max(max(top_m, __builtin_bit_cast(uint32_t, m[e]) << 1), __builtin_bit_cast(uint32_t, m[e + 1]) << 1);
            top_r = max(max(top_r, __builtin_bit_cast(uint32_t, r[e])), __builtin_bit_cast(uint32_t, r[e + 1]));
        }
        top_m >>= 1;
    }
    if constexpr (MASTER) opt_store<FULL>(w.master, i, left, vec, pi);
    opt_store<FULL>(w.p, i, left, vec, pi);
    if constexpr (EIGHT) {
        const bool bad = max(top_m, top_r) >= 0x7F800000u;   // a value that is not finite: the largest of the others
        if (bad) {
            top_m = top_r = 0;
#pragma unroll
            for (int e = 0; e < OPT_PER_LANE; ++e) {
                const uint32_t bm = __builtin_bit_cast(uint32_t, m[e]) & 0x7FFFFFFFu, br = __builtin_bit_cast(uint32_t, r[e]) & 0x7FFFFFFFu;
                top_m = max(top_m, bm < 0x7F800000u ? bm : 0u);
                top_r = max(top_r, br < 0x7F800000u ? br : 0u);
            }
        }
        // elements behind the end are zeros (or not finite, by a scale that is not) and change no maximum
        const uint32_t em = opt_exponent(opt_max16(top_m)), er = opt_exponent(opt_max16(top_r));
        const float um = opt_pow2(254 - em), ur = opt_pow2(254 - er);
        if (bad) {
#pragma unroll
            for (int e = 0; e < OPT_PER_LANE; ++e) {          // 448 times the block's scale: the largest code
                if ((__builtin_bit_cast(uint32_t, m[e]) & 0x7FFFFFFFu) >= 0x7F800000u) m[e] = __builtin_copysignf(448.f * opt_pow2(em), m[e]);
                if ((__builtin_bit_cast(uint32_t, r[e]) & 0x7FFFFFFFu) >= 0x7F800000u) r[e] = 448.f * opt_pow2(er);
            }
        }
        uint32_t cm[2] = {0, 0}, cr[2] = {0, 0};
        const uint32_t lane_key = key ^ (uint32_t)i ^ ((uint32_t)(i >> 32) * 0xC2B2AE35U);      // i is a multiple of 8
#pragma unroll
        for (int e = 0; e < OPT_PER_LANE; ++e) {
            const uint32_t random = opt_mix(lane_key ^ (uint32_t)e), at = 8 * (e & 3);
            const uint32_t a = opt_code(__builtin_fabsf(m[e]) * um, random << 4 & 0xFFFF0u);
            const uint32_t b = max(opt_code(r[e] * ur, random >> 12 & 0xFFFF0u), min(__builtin_bit_cast(uint32_t, r[e]), 1u));
            cm[e >> 2] |= (a | (__builtin_bit_cast(uint32_t, m[e]) >> 24 & 128u)) << at;
            cr[e >> 2] |= b << at;
        }
        opt_store_codes<FULL>((uint8_t*)w.m, i, left, vec, cm);
        opt_store_codes<FULL>((uint8_t*)w.v, i, left, vec, cr);
        if ((threadIdx.x & 15) == 0 && (FULL || left > 0)) {
            w.exp_m[i / OPT_BLOCK] = (uint8_t)em;
            w.exp_v[i / OPT_BLOCK] = (uint8_t)er;
        }
    } else {
        opt_store<FULL>((float*)w.m, i, left, vec, m);
        opt_store<FULL>((float*)w.v, i, left, vec, r);
    }
}

template <typename P, bool MASTER, bool EIGHT>
__global__ __launch_bounds__(OPT_THREADS) void k_adamw(OptTable t, AdamwHyper by_value, const AdamwHyper* __restrict__ in_memory,
                                                       const float* __restrict__ grad_scale, const float* __restrict__ clip) {
    uint32_t unit;
    const int k = opt_find<OPT_ENTRIES / 5>(t, &unit);
    const uint64_t size = opt_entry(t, 0, k), n = size & ~OPT_VEC;
    const bool vec = (size & OPT_VEC) != 0;
    AdamwTensor<P> w = {(P*)opt_entry(t, 1, k), (const P*)opt_entry(t, 2, k), (void*)opt_entry(t, 3, k), (void*)opt_entry(t, 4, k),
                        MASTER ? (float*)opt_entry(t, 5, k) : nullptr, EIGHT ? (uint8_t*)opt_entry(t, MASTER ? 6 : 5, k) : nullptr,
                        EIGHT ? (uint8_t*)opt_entry(t, MASTER ? 7 : 6, k) : nullptr};
    const AdamwHyper h = in_memory ? *in_memory : by_value;
    const float s = (grad_scale ? *grad_scale : 1.f) * (clip ? *clip : 1.f);
    const uint32_t key = EIGHT ? opt_mix(h.key ^ ((t.ordinal + (uint32_t)k) * 0x85EBCA6BU)) : 0;
    uint64_t i = ((uint64_t)unit << t.span_log2) + threadIdx.x * OPT_PER_LANE;
    const uint64_t end = min(n, (uint64_t)(unit + 1) << t.span_log2);
    if (vec && end == (uint64_t)(unit + 1) << t.span_log2) {
        for (; i < end; i += OPT_STRIDE) adamw_elements<true, P, MASTER, EIGHT>(w, i, OPT_PER_LANE, true, h, s, key);
        return;
    }
    // the last workgroup of a tensor, and tensors at odd addresses
    for (uint32_t at = 0; at < t.span; at += OPT_STRIDE, i += OPT_STRIDE) {
        const int left = i < n ? (int)min(n - i, (uint64_t)OPT_PER_LANE) : 0;
        // a wavefront without elements leaves; one with some keeps all its lanes for the blocks' maxima
        if (__ballot(left > 0) == 0) break;
        adamw_elements<false, P, MASTER, EIGHT>(w, i, left, vec, h, s, key);
    }
}

// Step counter and hyperparameters in device memory, for steps that are replayed from a captured graph.
__global__ void k_adamw_advance(long long* __restrict__ step, const float* __restrict__ lr, AdamwHyper* __restrict__ out, double lr_value,
                                double b1, double b2, double eps, double wd, uint64_t seed) {
    const long long now = *step + 1;
    *step = now;
    *out = opt_hyper(lr ? (double)*lr : lr_value, b1, b2, eps, wd, now, seed);
}

// Sum of squares of one unit of elements per workgroup, in double precision: no overflow or underflow of squares of finite
// gradients, and no rounding that shows.  Every partial sum has a place of its own and the second kernel adds them in a fixed
// order, so that equal gradients give equal bits.  Bound by memory: 300 tensors of 41 M fp32 elements in
// all take 33 us with the final kernel, 5.0 TB/s, over gradients in turn; between steps of 41 M parameters 53 + 5 us.
#define OPT_NORM_UNITS 4             // strides of a workgroup, all of them on the way at once
template <typename P>
__global__ __launch_bounds__(OPT_THREADS) void k_grad_norm(OptTable t, double* __restrict__ part) {
    __shared__ double wave_sum[OPT_THREADS / 64];
    uint32_t unit;
    const int k = opt_find<OPT_ENTRIES / 2>(t, &unit);
    const uint64_t size = opt_entry(t, 0, k), n = size & ~OPT_VEC;
    const P* g = (const P*)opt_entry(t, 1, k);
    const uint64_t start = (uint64_t)unit * (OPT_NORM_UNITS * OPT_STRIDE) + threadIdx.x * OPT_PER_LANE;
    double sum = 0.0;
    float x[OPT_NORM_UNITS][OPT_PER_LANE];
    if ((size & OPT_VEC) && (uint64_t)(unit + 1) * (OPT_NORM_UNITS * OPT_STRIDE) <= n) {
#pragma unroll
        for (int u = 0; u < OPT_NORM_UNITS; ++u) opt_load<true>(g, start + u * OPT_STRIDE, OPT_PER_LANE, true, x[u]);
    } else {
#pragma unroll
        for (int u = 0; u < OPT_NORM_UNITS; ++u) {
            const uint64_t i = start + u * OPT_STRIDE;
            opt_load<false>(g, i, i < n ? (int)min(n - i, (uint64_t)OPT_PER_LANE) : 0, (size & OPT_VEC) != 0, x[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < OPT_NORM_UNITS; ++u)
#pragma unroll
        for (int e = 0; e < OPT_PER_LANE; ++e) sum += (double)x[u][e] * (double)x[u][e];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int q = 0; q < OPT_THREADS / 64; ++q) total += wave_sum[q];
        part[blockIdx.x] = total;
    }
}

// out = {norm, min(1, max_norm / (norm + 1e-6))}; a norm that is NaN makes the coefficient NaN, an infinite one makes it 0.
__global__ __launch_bounds__(1024) void k_grad_norm_final(int n, const double* __restrict__ part, const float* __restrict__ grad_scale,
                                                          double max_norm, float* __restrict__ out) {
    __shared__ double wave_sum[16];
    double sum = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 1024) sum += part[i];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int q = 0; q < 16; ++q) total += wave_sum[q];
        const double norm = sqrt(total) * (grad_scale ? fabs((double)*grad_scale) : 1.0);
        const double c = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = c > 1.0 ? 1.f : (float)c;
    }
}

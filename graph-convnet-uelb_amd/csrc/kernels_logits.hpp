// Rules on logits before something is drawn from them, and their gradient (gfx950): penalties for tokens that occurred, a bias,
// a temperature and a mask.
//
// Logits are rows x[o][v][i]: o a request, a position or a (graph, node), v the vocabulary or the next node, i what shares the
// row's history and mask (1 for token logits, the commodities for link scores).  With n the number of times that v stands in
// row o's history behind its prompt, and seen = v stands in it anywhere:
//   x1 = seen ? (x > 0 ? x / rho : x rho) : x
//   y  = (x1 - n alpha_f - (n > 0) alpha_p + bias[v]) / tau,       masked_value where the mask has v off
//   dx = dy / tau * (seen ? (x > 0 ? 1 / rho : rho) : 1),  dbias[r][v] = sum over o = r (mod R) and i of dy / tau;
//   both 0 where v is off, whatever dy and x hold there.
// Everything is fp32 and rounded once to the logits' type.
//
// Bound by memory: one read and one write of the logits (backward: of the gradient; a logit is read where its token is seen).
// A workgroup takes a range of one row's vocabulary and counts the row's history into LDS first (integer atomics: the order
// does not matter), so that there is one launch, no workspace and no second pass over the logits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define LGT_THREADS 256
#define LGT_PER_LANE 8                         // consecutive elements of a lane
#define LGT_STRIDE (LGT_THREADS * LGT_PER_LANE)
#define LGT_SEEN 0x80000000u                   // a count's flag: the token stands in the prompt

struct LogitsArgs {
    const void* x;                 // logits
    void* y;                       // forward: result; backward: gradient of the logits (may be null)
    const void* dy;                // backward: gradient of the result
    long long x_stride, y_stride;  // between rows, in elements (dy has y's)
    int rows, vocab, inner, chunk, chunks;   // vocabulary entries per workgroup, workgroups per row
    const void* history;
    const void *lens, *prompts;
    long long history_len;
    int history_wide, lens_wide;   // 64-bit integers
    int history_rows, mask_rows, bias_rows, rep_rows, pres_rows, freq_rows, temp_rows;   // row o uses entry o mod this
    int mask_type;                 // 0 none, 1 a byte per entry, 2 a bit per entry in 32-bit words, lowest first
    const void* mask;
    const float *bias, *rep, *pres, *freq, *temp;      // rep .. temp: null = the number below
    float rep_value, pres_value, freq_value, temp_value, masked_value;
};

__device__ __forceinline__ float lgt_param(const float* p, int rows, float value, int o) { return p ? p[rows == 1 ? 0 : o % rows] : value; }
__device__ __forceinline__ long long lgt_int(const void* p, int wide, long long i) {
    return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// Counts of the entries [v0, v0 + n) in row o's history, into LDS.
__device__ __forceinline__ void lgt_count(const LogitsArgs& a, int o, int v0, int n, uint32_t* cnt) {
    for (int k = threadIdx.x; k < n; k += LGT_THREADS) cnt[k] = 0;
    __syncthreads();
    const int r = o % a.history_rows;
    long long len = a.lens ? lgt_int(a.lens, a.lens_wide, r) : a.history_len;
    len = len < a.history_len ? len : a.history_len;
    const long long prompt = a.prompts ? lgt_int(a.prompts, a.lens_wide, r) : 0;
    const long long base = (long long)r * a.history_len;
    for (long long l = threadIdx.x; l < len; l += LGT_THREADS) {
        const long long id = lgt_int(a.history, a.history_wide, base + l) - v0;
        if (id >= 0 && id < n) {
            if (l >= prompt) atomicAdd(&cnt[id], 1u);
            else atomicOr(&cnt[id], LGT_SEEN);
        }
    }
    __syncthreads();
}

// Whether the mask leaves entry v of row r.
__device__ __forceinline__ bool lgt_on(const LogitsArgs& a, int r, int v) {
    if (a.mask_type == 0) return true;
    if (a.mask_type == 1) return static_cast<const uint8_t*>(a.mask)[(long long)r * a.vocab + v] != 0;
    const int words = (a.vocab + 31) >> 5;
    return (static_cast<const uint32_t*>(a.mask)[(long long)r * words + (v >> 5)] >> (v & 31)) & 1;
}

template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) LgtVec {      // rows of odd lengths: aligned to elements only
    T v[N];
};

template <typename T, bool BACKWARD>
__global__ __launch_bounds__(LGT_THREADS) void k_logits(LogitsArgs a) {
    extern __shared__ uint32_t cnt[];
    const int o = blockIdx.x / a.chunks, v0 = (blockIdx.x % a.chunks) * a.chunk, n = min(a.chunk, a.vocab - v0);
    if (a.history) lgt_count(a, o, v0, n, cnt);
    const float rho = lgt_param(a.rep, a.rep_rows, a.rep_value, o), inv_rho = 1.f / rho;
    const float inv_tau = 1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o);
    const float pres = lgt_param(a.pres, a.pres_rows, a.pres_value, o), freq = lgt_param(a.freq, a.freq_rows, a.freq_value, o);
    const float* bias = a.bias && !BACKWARD ? a.bias + (long long)(o % a.bias_rows) * a.vocab : nullptr;
    const int mask_row = a.mask_type ? o % a.mask_rows : 0;
    const T* x = static_cast<const T*>(a.x) + (long long)o * a.x_stride;
    const T* dy = BACKWARD ? static_cast<const T*>(a.dy) + (long long)o * a.y_stride : nullptr;
    T* y = static_cast<T*>(a.y) + (long long)o * a.y_stride;
    const int first = v0 * a.inner, end = first + n * a.inner;
    for (int e = first + threadIdx.x * LGT_PER_LANE; e < end; e += LGT_STRIDE) {
        const int left = min(end - e, LGT_PER_LANE);
        float in[LGT_PER_LANE];
        const T* src = BACKWARD ? dy : x;
        if (left == LGT_PER_LANE) {
            const LgtVec<T, LGT_PER_LANE> raw = *reinterpret_cast<const LgtVec<T, LGT_PER_LANE>*>(src + e);
#pragma unroll
            for (int k = 0; k < LGT_PER_LANE; ++k) in[k] = (float)raw.v[k];
        } else {
            for (int k = 0; k < LGT_PER_LANE; ++k) in[k] = k < left ? (float)src[e + k] : 0.f;
        }
        float out[LGT_PER_LANE];
        int v = e / a.inner, i = e - v * a.inner;
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) {
            out[k] = 0.f;
            if (k < left) {
                const uint32_t c = a.history ? cnt[v - v0] : 0;
                const bool on = lgt_on(a, mask_row, v);
                float z = in[k];
                if (BACKWARD) {
                    z *= inv_tau;
                    if (c) z *= (float)x[e + k] > 0.f ? inv_rho : rho;
                    out[k] = on ? z : 0.f;
                } else {
                    const uint32_t times = c & ~LGT_SEEN;
                    if (c) z *= z > 0.f ? inv_rho : rho;
                    if (times) z -= (float)times * freq + pres;
                    if (bias) z += bias[v];
                    out[k] = on ? z * inv_tau : a.masked_value;
                }
                if (++i == a.inner) { i = 0; ++v; }
            }
        }
        if (left == LGT_PER_LANE) {
            LgtVec<T, LGT_PER_LANE> raw;
#pragma unroll
            for (int k = 0; k < LGT_PER_LANE; ++k) raw.v[k] = (T)out[k];
            *reinterpret_cast<LgtVec<T, LGT_PER_LANE>*>(y + e) = raw;
        } else {
            for (int k = 0; k < left; ++k) y[e + k] = (T)out[k];
        }
    }
}

// Gradient of the bias: one wavefront per (r, v) adds the rows o = r, r + R, ... and all i, each lane its own in order.
template <typename T>
__global__ __launch_bounds__(LGT_THREADS) void k_logits_bias_grad(LogitsArgs a, float* __restrict__ dbias) {
    const long long at = (long long)blockIdx.x * (LGT_THREADS / 64) + (threadIdx.x >> 6);
    if (at >= (long long)a.bias_rows * a.vocab) return;
    const int r = (int)(at / a.vocab), v = (int)(at % a.vocab), lane = threadIdx.x & 63;
    const long long many = (long long)(a.rows / a.bias_rows) * a.inner;
    float sum = 0.f;
    for (long long k = lane; k < many; k += 64) {
        const int o = r + (int)(k / a.inner) * a.bias_rows;
        if (!lgt_on(a, a.mask_type ? o % a.mask_rows : 0, v)) continue;
        const T* dy = static_cast<const T*>(a.dy) + (long long)o * a.y_stride + (long long)v * a.inner;
        sum += (float)dy[k % a.inner] * (1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o));
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) dbias[at] = sum;
}

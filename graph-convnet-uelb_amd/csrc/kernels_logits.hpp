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
// A workgroup takes a range of one row's vocabulary and counts the row's history into LDS (integer atomics: the order does not
// matter) while its logits are on the way, so that there is one launch, no workspace and no second pass over the logits.
// The backward pass takes a range of the rows that share a bias row, one after the other, and keeps the bias gradient's sums
// in registers: the gradient is read once for both results.
// Kernel times with everything on: 512 x 131072 bf16, 512 entries of history, bit mask: 56 us (5.0 TB/s of the 5.2 to 5.5 that a copy
// reaches); 64 x 131072 fp32, 2048 entries: 16 us; 2048 x 32000 bf16, 256 entries, shared bias: 64 us forward (9 of them the
// bias' way through L2, 9 the history), 64 + 5 us backward; 800 x 200 x 100 fp32 scores: 29 to 31 us forward, 32 to 35 us backward.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define LGT_THREADS 512                        // four workgroups on a CU: 32 wavefronts
#define LGT_PER_LANE 8                         // consecutive elements of a lane
#define LGT_STRIDE (LGT_THREADS * LGT_PER_LANE)
#define LGT_SEEN 0x80000000u                   // a count's flag: the token stands in the prompt

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

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
    int splits;                    // backward: parts of the rows that share a bias row
    float* dbias;                  // backward: [splits][bias_rows][vocab] or null
    uint32_t blocks;               // workgroups, over both dimensions of the grid (a dimension holds 2^32 threads)
};

__device__ __forceinline__ uint32_t lgt_block() { return blockIdx.y * gridDim.x + blockIdx.x; }

__device__ __forceinline__ float lgt_param(const float* p, int rows, float value, int o) { return p ? p[rows == 1 ? 0 : o % rows] : value; }
__device__ __forceinline__ long long lgt_int(const void* p, int wide, long long i) {
    return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

template <typename T, int N>
struct LgtVecOf {
    typedef T type __attribute__((ext_vector_type(N)));
    typedef type loose __attribute__((aligned(sizeof(T))));      // rows of odd lengths: aligned to elements only
};
template <typename T, int N>
using LgtVec = typename LgtVecOf<T, N>::type;
template <typename T, int N>
__device__ __forceinline__ LgtVec<T, N> lgt_vec(const T* p) { return *reinterpret_cast<const typename LgtVecOf<T, N>::loose*>(p); }

// Counts of the entries [v0, v0 + n) in row o's history, into LDS.  Between two barriers of the workgroup.
__device__ __forceinline__ void lgt_count_one(long long id, long long l, long long prompt, int v0, int n, uint32_t* cnt) {
    const unsigned long long at = (unsigned long long)(id - v0);
    if (at < (unsigned long long)n) {
        if (l >= prompt) atomicAdd(&cnt[at], 1u);
        else atomicOr(&cnt[at], LGT_SEEN);
    }
}
// A lane's first 16 bytes of row r's history, requested before anything else: loads return in order, so that they can be
// counted while the logits are on the way.
__device__ __forceinline__ u32x4_t lgt_first_ids(const LogitsArgs& a, int r) {
    u32x4_t ids = {0, 0, 0, 0};
    const int w = a.history_wide ? 2 : 4;
    if ((long long)(threadIdx.x + 1) * w <= a.history_len)
        ids = lgt_vec<uint32_t, 4>(static_cast<const uint32_t*>(a.history) + ((long long)r * a.history_len + threadIdx.x * w) * (a.history_wide ? 2 : 1));
    return ids;
}
template <bool LONG, typename ID>
__device__ __forceinline__ void lgt_count_ids(const ID* __restrict__ ids, u32x4_t first, long long len, long long prompt, int v0, int n, uint32_t* cnt) {
    constexpr int W = 16 / sizeof(ID), STEP = LGT_THREADS * W, DEEP = 8;
    long long l = (long long)threadIdx.x * W;
    if (l + W <= len) {
        const LgtVec<ID, W> some = __builtin_bit_cast(LgtVec<ID, W>, first);
#pragma unroll
        for (int k = 0; k < W; ++k) lgt_count_one(some[k], l + k, prompt, v0, n, cnt);
        l += STEP;
    }
    if constexpr (LONG) {
        for (; l + (DEEP - 1) * STEP + W <= len; l += DEEP * STEP) {
            LgtVec<ID, W> some[DEEP];
#pragma unroll
            for (int j = 0; j < DEEP; ++j) some[j] = lgt_vec<ID, W>(ids + l + j * STEP);
#pragma unroll
            for (int j = 0; j < DEEP; ++j)
#pragma unroll
                for (int k = 0; k < W; ++k) lgt_count_one(some[j][k], l + j * STEP + k, prompt, v0, n, cnt);
        }
    }
    for (; l + W <= len; l += STEP) {
        const LgtVec<ID, W> some = lgt_vec<ID, W>(ids + l);
#pragma unroll
        for (int k = 0; k < W; ++k) lgt_count_one(some[k], l + k, prompt, v0, n, cnt);
    }
    for (; l < len; ++l) lgt_count_one(ids[l], l, prompt, v0, n, cnt);       // the one lane whose group is cut off
}
template <bool LONG>
__device__ __forceinline__ void lgt_count(const LogitsArgs& a, int o, u32x4_t first, int v0, int n, uint32_t* cnt) {
    for (int k = threadIdx.x * 4; k < n; k += LGT_THREADS * 4) *reinterpret_cast<uint4*>(cnt + k) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int r = o % a.history_rows;
    long long len = a.lens ? lgt_int(a.lens, a.lens_wide, r) : a.history_len;
    len = len < a.history_len ? len : a.history_len;
    const long long prompt = a.prompts ? lgt_int(a.prompts, a.lens_wide, r) : 0, base = (long long)r * a.history_len;
    if (a.history_wide) lgt_count_ids<LONG>(static_cast<const long long*>(a.history) + base, first, len, prompt, v0, n, cnt);
    else lgt_count_ids<LONG>(static_cast<const int*>(a.history) + base, first, len, prompt, v0, n, cnt);
    __syncthreads();
}

// Whether the mask leaves entry v of row r.
__device__ __forceinline__ bool lgt_on(const LogitsArgs& a, int r, int v) {
    if (a.mask_type == 0) return true;
    if (a.mask_type == 1) return static_cast<const uint8_t*>(a.mask)[(long long)r * a.vocab + v] != 0;
    const int words = (a.vocab + 31) >> 5;
    return (static_cast<const uint32_t*>(a.mask)[(long long)r * words + (v >> 5)] >> (v & 31)) & 1;
}
// The same for eight entries from v on, a multiple of 8, of which `left` exist: bit k for v + k.
__device__ __forceinline__ uint32_t lgt_on8(const LogitsArgs& a, int r, int v, int left) {
    if (a.mask_type == 0) return 0xFFu;
    if (left <= 0) return 0;
    if (a.mask_type == 2) return static_cast<const uint8_t*>(a.mask)[(long long)r * (((a.vocab + 31) >> 5) * 4) + (v >> 3)];
    const uint8_t* m = static_cast<const uint8_t*>(a.mask) + (long long)r * a.vocab + v;
    uint32_t on = 0;
    if (left >= LGT_PER_LANE) {
        const LgtVec<uint8_t, LGT_PER_LANE> some = lgt_vec<uint8_t, LGT_PER_LANE>(m);
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) on |= (some[k] != 0 ? 1u : 0u) << k;
    } else {
        for (int k = 0; k < left; ++k) on |= (m[k] != 0 ? 1u : 0u) << k;
    }
    return on;
}

template <typename T>
__device__ __forceinline__ LgtVec<T, LGT_PER_LANE> lgt_load(const T* p, long long e, int left) {
    LgtVec<T, LGT_PER_LANE> raw;
    if (left >= LGT_PER_LANE) {
        raw = lgt_vec<T, LGT_PER_LANE>(p + e);
    } else {
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) raw[k] = k < left ? p[e + k] : (T)0.f;
    }
    return raw;
}
template <typename T>
__device__ __forceinline__ void lgt_store(T* p, long long e, int left, const float* out) {
    if (left >= LGT_PER_LANE) {
        LgtVec<T, LGT_PER_LANE> raw;
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) raw[k] = (T)out[k];
        *reinterpret_cast<typename LgtVecOf<T, LGT_PER_LANE>::loose*>(p + e) = raw;
    } else {
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k)
            if (k < left) p[e + k] = (T)out[k];
    }
}

// ---------------------------------------------------------------------------------------------- token logits (inner = 1)
// LONG: histories of 8192 entries and more are read eight loads at a time (16 rows of 50021 with 32768 entries of int64: 15.5 ->
// 10.6 us, all but 1.5 of it the walk over the history); the code for that costs shorter ones 12 to 15 %.
// Tried and slower: four rows of 4096 with 16-bit counts and their histories counted together (70 us where this takes 58).
template <typename T, int ITER, bool LONG>
__global__ __launch_bounds__(LGT_THREADS) void k_logits(LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t cnt[];
    if (lgt_block() >= a.blocks) return;
    const int o = lgt_block() / a.chunks, v0 = (lgt_block() % a.chunks) * (ITER * LGT_STRIDE), n = min(ITER * LGT_STRIDE, a.vocab - v0);
    const T* x = static_cast<const T*>(a.x) + (long long)o * a.x_stride + v0;
    T* y = static_cast<T*>(a.y) + (long long)o * a.y_stride + v0;
    const int mask_row = a.mask_type ? o % a.mask_rows : 0;
    const float* bias = a.bias ? a.bias + (long long)(o % a.bias_rows) * a.vocab + v0 : nullptr;
    u32x4_t ids = {0, 0, 0, 0};
    if (a.history) ids = lgt_first_ids(a, o % a.history_rows);
    LgtVec<T, LGT_PER_LANE> raw[ITER];
    uint32_t on[ITER];
#pragma unroll
    for (int t = 0; t < ITER; ++t) {
        const int e = t * LGT_STRIDE + threadIdx.x * LGT_PER_LANE;
        raw[t] = lgt_load(x, e, n - e);
        on[t] = lgt_on8(a, mask_row, v0 + e, n - e);
    }
    const float rho = lgt_param(a.rep, a.rep_rows, a.rep_value, o), inv_rho = 1.f / rho;
    const float inv_tau = 1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o);
    const float pres = lgt_param(a.pres, a.pres_rows, a.pres_value, o), freq = lgt_param(a.freq, a.freq_rows, a.freq_value, o);
    if (a.history) lgt_count<LONG>(a, o, ids, v0, n, cnt);
#pragma unroll
    for (int t = 0; t < ITER; ++t) {
        const int e = t * LGT_STRIDE + threadIdx.x * LGT_PER_LANE, left = n - e;
        if (left <= 0) break;
        float z[LGT_PER_LANE];
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) z[k] = (float)raw[t][k];
        if (a.history) {
            uint32_t c[LGT_PER_LANE];
            *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(cnt + e);
            *reinterpret_cast<uint4*>(c + 4) = *reinterpret_cast<const uint4*>(cnt + e + 4);
            if (c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) {
#pragma unroll
                for (int k = 0; k < LGT_PER_LANE; ++k) {
                    const uint32_t times = c[k] & ~LGT_SEEN;
                    if (c[k]) z[k] *= z[k] > 0.f ? inv_rho : rho;
                    if (times) z[k] -= (float)times * freq + pres;
                }
            }
        }
        if (bias) {
            const LgtVec<float, LGT_PER_LANE> b = lgt_load(bias, e, left);
#pragma unroll
            for (int k = 0; k < LGT_PER_LANE; ++k) z[k] += b[k];
        }
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) z[k] = (on[t] >> k) & 1 ? z[k] * inv_tau : a.masked_value;
        lgt_store(y, e, left, z);
    }
}

// Rows r, r + R, ... (R = bias_rows) of one part: the gradient of the logits row by row, that of the bias in registers.  The slope
// needs to know whether a token was seen, not how often: one bit per entry in LDS, so that the bits of LGT_ROWS rows are set in
// one go (all histories together, spread over all lanes), and the rows then stream without a barrier among them.  2048 rows of
// 32000 in bf16: 64 us (50 without a history); row by row, with a barrier each, 86; four rows at a time 99.
#define LGT_ROWS 32
#define LGT_AHEAD 4                              // rows whose loads are on the way together

__device__ __forceinline__ void lgt_see(long long id, int v0, int n, uint32_t* bits) {
    const unsigned long long at = (unsigned long long)(id - v0);
    if (at < (unsigned long long)n) atomicOr(&bits[at >> 5], 1u << (at & 31));
}

template <typename T>
__global__ __launch_bounds__(LGT_THREADS) void k_logits_bwd(LogitsArgs a) {
    constexpr int WORDS = LGT_STRIDE / 32;
    __shared__ uint32_t bits[LGT_ROWS * WORDS];
    __shared__ float slope[LGT_ROWS][2];         // 1 / temperature and repetition penalty of the rows
    __shared__ int length[LGT_ROWS];
    uint32_t at = lgt_block();
    if (at >= a.blocks) return;
    const int v0 = (int)(at % a.chunks) * LGT_STRIDE, n = min(LGT_STRIDE, a.vocab - v0);
    at /= a.chunks;
    const int r = (int)(at % a.bias_rows), part = (int)(at / a.bias_rows), many = a.rows / a.bias_rows;
    const int first = (int)((long long)many * part / a.splits), last = (int)((long long)many * (part + 1) / a.splits);
    const int e = threadIdx.x * LGT_PER_LANE, left = n - e;
    // the histories of a turn as groups of 16 bytes, dealt to the lanes in turn
    const int w = a.history_wide ? 2 : 4, groups = a.history ? (int)((a.history_len + w - 1) / w) : 1;
    const int step_row = LGT_THREADS / groups, step_group = LGT_THREADS % groups;
    float sum[LGT_PER_LANE] = {};
    for (int q = first; q < last; q += LGT_ROWS) {
        const int rows = min(LGT_ROWS, last - q);
        if (q != first) __syncthreads();
        if ((int)threadIdx.x < rows) {
            const int o = r + (q + threadIdx.x) * a.bias_rows;
            slope[threadIdx.x][0] = 1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o);
            slope[threadIdx.x][1] = lgt_param(a.rep, a.rep_rows, a.rep_value, o);
            if (a.history) {
                const long long len = a.lens ? lgt_int(a.lens, a.lens_wide, o % a.history_rows) : a.history_len;
                length[threadIdx.x] = (int)(len < 0 ? 0 : len < a.history_len ? len : a.history_len);
            }
        }
        if (a.history) {
            for (int k = threadIdx.x * 4; k < rows * WORDS; k += LGT_THREADS * 4) *reinterpret_cast<uint4*>(bits + k) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            int j = threadIdx.x / groups, g = threadIdx.x % groups;
            while (j < rows) {
                const int len = length[j], l = g * w;
                const long long base = (long long)((r + (q + j) * a.bias_rows) % a.history_rows) * a.history_len + l;
                if (l + w <= len) {
                    const u32x4_t ids = lgt_vec<uint32_t, 4>(static_cast<const uint32_t*>(a.history) + base * (a.history_wide ? 2 : 1));
                    if (a.history_wide) {
                        lgt_see((long long)(((unsigned long long)ids[1] << 32) | ids[0]), v0, n, bits + j * WORDS);
                        lgt_see((long long)(((unsigned long long)ids[3] << 32) | ids[2]), v0, n, bits + j * WORDS);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) lgt_see((int)ids[k], v0, n, bits + j * WORDS);
                    }
                } else {
                    for (int k = 0; l + k < len; ++k) lgt_see(lgt_int(a.history, a.history_wide, base + k), v0, n, bits + j * WORDS);
                }
                j += step_row;
                g += step_group;
                if (g >= groups) { g -= groups; ++j; }
            }
        }
        __syncthreads();
        if (left <= 0) continue;
        for (int j0 = 0; j0 < rows; j0 += LGT_AHEAD) {
            LgtVec<T, LGT_PER_LANE> raw[LGT_AHEAD], xs[LGT_AHEAD];
            uint32_t on[LGT_AHEAD], seen[LGT_AHEAD] = {};
#pragma unroll
            for (int j = 0; j < LGT_AHEAD; ++j) {
                const int row = min(j0 + j, rows - 1), o = r + (q + row) * a.bias_rows;      // behind the end: the last row again, not used
                raw[j] = lgt_load(static_cast<const T*>(a.dy) + (long long)o * a.y_stride + v0, e, left);
                on[j] = lgt_on8(a, a.mask_type ? o % a.mask_rows : 0, v0 + e, left);
                if (a.history && a.y) {
                    seen[j] = reinterpret_cast<const uint8_t*>(bits + row * WORDS)[threadIdx.x];
                    if (seen[j]) xs[j] = lgt_load(static_cast<const T*>(a.x) + (long long)o * a.x_stride + v0, e, left);
                }
            }
#pragma unroll
            for (int j = 0; j < LGT_AHEAD; ++j) {
                if (j0 + j >= rows) break;
                const float inv_tau = slope[j0 + j][0], rho = slope[j0 + j][1];
                float g[LGT_PER_LANE];
#pragma unroll
                for (int k = 0; k < LGT_PER_LANE; ++k) {
                    g[k] = (on[j] >> k) & 1 ? (float)raw[j][k] * inv_tau : 0.f;
                    sum[k] += g[k];
                }
                if (!a.y) continue;
                if (seen[j] & on[j]) {
                    const float inv_rho = 1.f / rho;
#pragma unroll
                    for (int k = 0; k < LGT_PER_LANE; ++k)
                        if ((seen[j] & on[j]) >> k & 1) g[k] *= (float)xs[j][k] > 0.f ? inv_rho : rho;
                }
                lgt_store(static_cast<T*>(a.y) + (long long)(r + (q + j0 + j) * a.bias_rows) * a.y_stride + v0, e, left, g);
            }
        }
    }
    if (a.dbias && left > 0) lgt_store(a.dbias + ((long long)part * a.bias_rows + r) * a.vocab + v0, e, left, sum);
}

// ---------------------------------------------------------------------------------------------- scores (inner > 1)
// A workgroup's tile: `chunk` vocabulary entries with all their inner elements, which follow each other in memory.  What depends
// on the entry alone stands in LDS: the sum of its additive terms, and two flags in the count's place.
#define LGT_OFF 0x40000000u                    // the mask has the entry off

__device__ __forceinline__ int lgt_entry(int e, float inv_inner) { return (int)((e + 0.5f) * inv_inner); }    // e < 2^22: exact

template <typename T>
__global__ __launch_bounds__(LGT_THREADS) void k_scores(LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t cnt[];
    if (lgt_block() >= a.blocks) return;
    const int o = lgt_block() / a.chunks, v0 = (lgt_block() % a.chunks) * a.chunk, n = min(a.chunk, a.vocab - v0);
    float* add = reinterpret_cast<float*>(cnt + ((a.chunk + 3) & ~3));
    const T* x = static_cast<const T*>(a.x) + (long long)o * a.x_stride + (long long)v0 * a.inner;
    T* y = static_cast<T*>(a.y) + (long long)o * a.y_stride + (long long)v0 * a.inner;
    const int end = n * a.inner;
    u32x4_t ids = {0, 0, 0, 0};
    if (a.history) ids = lgt_first_ids(a, o % a.history_rows);
    LgtVec<T, LGT_PER_LANE> raw = lgt_load(x, threadIdx.x * LGT_PER_LANE, end - (int)threadIdx.x * LGT_PER_LANE);
    const float rho = lgt_param(a.rep, a.rep_rows, a.rep_value, o), inv_rho = 1.f / rho;
    const float inv_tau = 1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o);
    const float pres = lgt_param(a.pres, a.pres_rows, a.pres_value, o), freq = lgt_param(a.freq, a.freq_rows, a.freq_value, o);
    if (a.history) lgt_count<false>(a, o, ids, v0, n, cnt);
    const float* bias = a.bias ? a.bias + (long long)(o % a.bias_rows) * a.vocab + v0 : nullptr;
    const int mask_row = a.mask_type ? o % a.mask_rows : 0;
    for (int v = threadIdx.x; v < n; v += LGT_THREADS) {
        const uint32_t c = a.history ? cnt[v] : 0, times = c & ~LGT_SEEN;
        float z = bias ? bias[v] : 0.f;
        if (times) z -= (float)times * freq + pres;
        add[v] = z;
        cnt[v] = (c ? LGT_SEEN : 0) | (lgt_on(a, mask_row, v0 + v) ? 0 : LGT_OFF);
    }
    __syncthreads();
    const float inv_inner = 1.f / (float)a.inner;
    for (int e = threadIdx.x * LGT_PER_LANE; e < end; e += LGT_STRIDE) {
        if (e >= LGT_STRIDE) raw = lgt_load(x, e, end - e);
        float z[LGT_PER_LANE];
        int v = n == 1 ? 0 : lgt_entry(e, inv_inner), i = e - v * a.inner;
#pragma unroll
        for (int k = 0; k < LGT_PER_LANE; ++k) {
            const uint32_t c = cnt[min(v, n - 1)];
            z[k] = (float)raw[k];
            if (c & LGT_SEEN) z[k] *= z[k] > 0.f ? inv_rho : rho;
            z[k] = c & LGT_OFF ? a.masked_value : (z[k] + add[min(v, n - 1)]) * inv_tau;
            if (++i == a.inner) { i = 0; ++v; }
        }
        lgt_store(y, e, end - e, z);
    }
}

#define LGT_SCORE_ROWS 8                       // rows of a turn
#define LGT_SCORE_ENTRIES (LGT_STRIDE / 2)     // most entries of a tile

// As k_logits_bwd: the histories of a turn's rows first, then their tiles one after the other, the next one on the way.  For the bias
// the tile's gradient goes through LDS (two tiles in turn, one barrier a row): a group of lanes adds an entry's elements, and
// keeps the sum over the rows in a register.
template <typename T>
__global__ __launch_bounds__(LGT_THREADS) void k_scores_bwd(LogitsArgs a) {
    __shared__ uint32_t seen[LGT_SCORE_ROWS * LGT_SCORE_ENTRIES / 32];
    __shared__ float slope[LGT_SCORE_ROWS][2];
    __shared__ int length[LGT_SCORE_ROWS];
    extern __shared__ __align__(16) float tile[];             // with dbias: two of LGT_STRIDE elements; then a flag per (row, entry)
    uint8_t* flag = reinterpret_cast<uint8_t*>(tile + (a.dbias ? 2 * LGT_STRIDE : 0));
    uint32_t at = lgt_block();
    if (at >= a.blocks) return;
    const int v0 = (int)(at % a.chunks) * a.chunk, n = min(a.chunk, a.vocab - v0), end = n * a.inner, words = (n + 31) >> 5;
    at /= a.chunks;
    const int r = (int)(at % a.bias_rows), part = (int)(at / a.bias_rows), many = a.rows / a.bias_rows;
    const int first = (int)((long long)many * part / a.splits), last = (int)((long long)many * (part + 1) / a.splits);
    const float inv_inner = 1.f / (float)a.inner;
    // lanes that add one entry's elements: a power of two, so that they lie in one wavefront
    int group = 1;
    while (group < 64 && group * 2 * n <= LGT_THREADS) group *= 2;
    const int mine = threadIdx.x / group, member = threadIdx.x % group, entries = LGT_THREADS / group;
    const int w = a.history_wide ? 2 : 4, groups = a.history ? (int)((a.history_len + w - 1) / w) : 1;
    const int e0 = threadIdx.x * LGT_PER_LANE;
    const int lane_v = n == 1 ? 0 : lgt_entry(min(e0, end), inv_inner), lane_i = e0 - lane_v * a.inner;
    float sum[LGT_SCORE_ENTRIES / LGT_THREADS] = {};
    for (int q = first; q < last; q += LGT_SCORE_ROWS) {
        const int rows = min(LGT_SCORE_ROWS, last - q);
        const auto row_of = [&](int j) { return r + (q + j) * a.bias_rows; };
        const auto dy_of = [&](int j) { return static_cast<const T*>(a.dy) + (long long)row_of(j) * a.y_stride + (long long)v0 * a.inner; };
        LgtVec<T, LGT_PER_LANE> next = lgt_load(dy_of(0), e0, end - e0);
        if (q != first) __syncthreads();
        if ((int)threadIdx.x < rows) {
            const int o = row_of(threadIdx.x);
            slope[threadIdx.x][0] = 1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o);
            slope[threadIdx.x][1] = lgt_param(a.rep, a.rep_rows, a.rep_value, o);
            if (a.history) {
                const long long len = a.lens ? lgt_int(a.lens, a.lens_wide, o % a.history_rows) : a.history_len;
                length[threadIdx.x] = (int)(len < 0 ? 0 : len < a.history_len ? len : a.history_len);
            }
        }
        if (a.history) {
            for (int k = threadIdx.x; k < rows * words; k += LGT_THREADS) seen[k] = 0;
            __syncthreads();
            const int step_row = LGT_THREADS / groups, step_group = LGT_THREADS % groups;
            int j = threadIdx.x / groups, g = threadIdx.x % groups;
            while (j < rows) {
                const int len = length[j], l = g * w;
                const long long base = (long long)(row_of(j) % a.history_rows) * a.history_len + l;
                for (int k = 0; k < w && l + k < len; ++k) lgt_see(lgt_int(a.history, a.history_wide, base + k), v0, n, seen + j * words);
                j += step_row;
                g += step_group;
                if (g >= groups) { g -= groups; ++j; }
            }
            __syncthreads();
        }
        {
            const int step_row = LGT_THREADS / n, step_v = LGT_THREADS % n;
            int j = threadIdx.x / n, v = threadIdx.x % n;
            while (j < rows) {
                const bool was = a.history && (seen[j * words + (v >> 5)] >> (v & 31) & 1);
                flag[j * n + v] = (was ? 1 : 0) | (lgt_on(a, a.mask_type ? row_of(j) % a.mask_rows : 0, v0 + v) ? 0 : 2);
                j += step_row;
                v += step_v;
                if (v >= n) { v -= n; ++j; }
            }
        }
        __syncthreads();
        for (int j = 0; j < rows; ++j) {
            const float inv_tau = slope[j][0], rho = slope[j][1], inv_rho = 1.f / rho;
            const T* x = static_cast<const T*>(a.x) + (long long)row_of(j) * a.x_stride + (long long)v0 * a.inner;
            T* dx = a.y ? static_cast<T*>(a.y) + (long long)row_of(j) * a.y_stride + (long long)v0 * a.inner : nullptr;
            float* out = tile + (j & 1) * LGT_STRIDE;
            LgtVec<T, LGT_PER_LANE> raw = next;
            if (j + 1 < rows) next = lgt_load(dy_of(j + 1), e0, end - e0);
            for (int e = e0; e < end; e += LGT_STRIDE) {
                const int left = end - e;
                if (e != e0) raw = lgt_load(dy_of(j), e, left);
                float g[LGT_PER_LANE];
                uint32_t was = 0;                                             // bit k: seen, and on
                int v = e == e0 ? lane_v : 0, i = e == e0 ? lane_i : 0;       // more than one stride: one entry
#pragma unroll
                for (int k = 0; k < LGT_PER_LANE; ++k) {
                    const uint32_t c = flag[j * n + min(v, n - 1)];
                    was |= (c == 1 ? 1u : 0u) << k;
                    g[k] = c & 2 ? 0.f : (float)raw[k] * inv_tau;
                    if (++i == a.inner) { i = 0; ++v; }
                }
                if (a.dbias) lgt_store(out, e, left, g);
                if (dx) {
                    if (was) {
                        const LgtVec<T, LGT_PER_LANE> xs = lgt_load(x, e, left);
#pragma unroll
                        for (int k = 0; k < LGT_PER_LANE; ++k)
                            if (was >> k & 1) g[k] *= (float)xs[k] > 0.f ? inv_rho : rho;
                    }
                    lgt_store(dx, e, left, g);
                }
            }
            if (a.dbias) {
                __syncthreads();
                // entries mine, mine + entries, ...: at most 4 passes, as a tile has at most 2048 entries
                for (int p = 0; p < LGT_SCORE_ENTRIES / LGT_THREADS; ++p) {
                    const int v = mine + p * entries;
                    float s = 0.f;
                    if (v < n)
                        for (int i = member; i < a.inner; i += group) s += out[v * a.inner + i];
                    for (int off = group >> 1; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
#pragma unroll
                    for (int z = 0; z < LGT_SCORE_ENTRIES / LGT_THREADS; ++z) sum[z] += z == p ? s : 0.f;
                    if ((p + 1) * entries >= n) break;
                }
            }
        }
    }
    if (a.dbias && member == 0) {
        float* out = a.dbias + ((long long)part * a.bias_rows + r) * a.vocab + v0;
#pragma unroll
        for (int p = 0; p < LGT_SCORE_ENTRIES / LGT_THREADS; ++p) {
            const int v = mine + p * entries;
            if (v < n) out[v] = sum[p];
        }
    }
}

// Gradient of the bias where an entry's inner elements exceed a tile: one wavefront per (r, v) adds the rows r, r + R, ... and
// all i, each lane its own in order.
template <typename T>
__global__ __launch_bounds__(LGT_THREADS) void k_scores_bias_grad(LogitsArgs a, float* __restrict__ dbias) {
    const long long at = (long long)blockIdx.x * (LGT_THREADS / 64) + (threadIdx.x >> 6);
    if (at >= (long long)a.bias_rows * a.vocab) return;
    const int r = (int)(at / a.vocab), v = (int)(at % a.vocab), lane = threadIdx.x & 63;
    float sum = 0.f;
    for (int o = r; o < a.rows; o += a.bias_rows) {
        if (!lgt_on(a, a.mask_type ? o % a.mask_rows : 0, v)) continue;
        const float inv_tau = 1.f / lgt_param(a.temp, a.temp_rows, a.temp_value, o);
        const T* dy = static_cast<const T*>(a.dy) + (long long)o * a.y_stride + (long long)v * a.inner;
        for (int i = lane; i < a.inner; i += 64) sum += (float)dy[i] * inv_tau;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) dbias[at] = sum;
}

// The parts' sums of the bias gradient: 32 columns and 8 groups of parts per workgroup, each group added in order, then the
// groups.
__global__ __launch_bounds__(256) void k_logits_bias_sum(long long n, int splits, const float* __restrict__ part, float* __restrict__ dbias) {
    __shared__ float group_sum[8][32];
    const int column = threadIdx.x & 31, group = threadIdx.x >> 5;
    const long long i = (long long)blockIdx.x * 32 + column;
    const int first = (int)((long long)splits * group / 8), last = (int)((long long)splits * (group + 1) / 8);
    float sum = 0.f;
    if (i < n) {
#pragma unroll 8
        for (int p = first; p < last; ++p) sum += part[p * n + i];
    }
    group_sum[group][column] = sum;
    __syncthreads();
    if (group == 0 && i < n) {
#pragma unroll
        for (int g = 1; g < 8; ++g) sum += group_sum[g][column];
        dbias[i] = sum;
    }
}

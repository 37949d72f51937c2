// C ABI of the logits operators: argument checks and launches.  The entry points are documented in include/gcn_uelb_hip.h.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "../../include/gcn_uelb_hip.h"
#include "host.hpp"
#include "kernels_logits.hpp"

namespace {

int check_rows(const char* what, const void* p, long long n, long long rows) {
    if (p && (n < 1 || n > rows || rows % n)) return fail(-1, "gcn_logits: %lld rows of %s for %lld rows of logits", n, what, rows);
    return 0;
}

// A number whose reciprocal the kernels multiply by: with an infinite one, a logit of 0 would become NaN.
bool divides(float x) { return x > 0.f && std::isfinite(x) && std::isfinite(1.f / x); }

// Vocabulary of a workgroup of k_logits in strides of 4096 entries: two where that leaves 1024 workgroups, so that the history
// is walked half as often (2048 rows of 32000: 65 us with two, 97 with one, 75 with four; 512 of 131072: 56, 82, 62; 1 of 32000:
// 4.5 with two, 4.1 with one).
int token_iterations(long long rows, long long vocab) {
    const auto blocks = [&](long long it) { return rows * ((vocab + it * LGT_STRIDE - 1) / (it * LGT_STRIDE)); };
    if (const char* e = tune_env("GCN_TUNE_LOGITS_IT")) return atoi(e);
    return blocks(2) >= 1024 ? 2 : 1;
}

int fill_args(const gcn_logits_desc* d, LogitsArgs* a) {
    if (!d) return fail(-1, "gcn_logits: null descriptor");
    if (d->type < GCN_F32 || d->type > GCN_F16) return fail(-1, "gcn_logits: unknown type %d", d->type);
    if (d->rows < 0 || d->vocab < 1 || d->inner < 1) return fail(-1, "gcn_logits: %lld x %lld x %lld logits", d->rows, d->vocab, d->inner);
    // 4096 below: the kernels step past the last row or element before they compare
    if (d->rows >= (1ll << 31) - 4096 || d->vocab >= (1ll << 31) || d->inner >= (1ll << 31) || d->vocab * d->inner >= (1ll << 31) - 4096)
        return fail(-2, "gcn_logits: %lld x %lld x %lld logits are too many for 32-bit places in a row", d->rows, d->vocab, d->inner);
    if (d->in_stride < 0 || d->out_stride < d->vocab * d->inner) return fail(-1, "gcn_logits: row strides %lld, %lld", d->in_stride, d->out_stride);
    if (d->history && (d->history_len < 0 || d->history_len >= (1ll << 31) - LGT_THREADS)) return fail(-1, "gcn_logits: history of %lld", d->history_len);
    if (!d->history && (d->history_lens || d->prompt_lens)) return fail(-1, "gcn_logits: lengths without a history");
    if (d->mask_type < 0 || d->mask_type > 2 || (d->mask_type != 0) != (d->mask != nullptr)) return fail(-1, "gcn_logits: mask of type %d", d->mask_type);
    if (!d->repetition_t && !divides(d->repetition)) return fail(-1, "gcn_logits: repetition penalty %g", (double)d->repetition);
    if (!d->temperature_t && !divides(d->temperature)) return fail(-1, "gcn_logits: temperature %g", (double)d->temperature);
    if ((!d->presence_t && !std::isfinite(d->presence)) || (!d->frequency_t && !std::isfinite(d->frequency)))
        return fail(-1, "gcn_logits: presence penalty %g, frequency penalty %g", (double)d->presence, (double)d->frequency);
    const long long rows = std::max(d->rows, 1ll);
    if (d->rows > 0) {
        if (int rc = check_rows("history", d->history, d->history_rows, rows)) return rc;
        if (int rc = check_rows("bias", d->bias, d->bias_rows, rows)) return rc;
        if (int rc = check_rows("mask", d->mask, d->mask_rows, rows)) return rc;
        if (int rc = check_rows("repetition penalties", d->repetition_t, d->repetition_rows, rows)) return rc;
        if (int rc = check_rows("presence penalties", d->presence_t, d->presence_rows, rows)) return rc;
        if (int rc = check_rows("frequency penalties", d->frequency_t, d->frequency_rows, rows)) return rc;
        if (int rc = check_rows("temperatures", d->temperature_t, d->temperature_rows, rows)) return rc;
    }
    *a = LogitsArgs{};
    a->x_stride = d->in_stride; a->y_stride = d->out_stride;
    a->rows = (int)d->rows; a->vocab = (int)d->vocab; a->inner = (int)d->inner;
    if (d->history && d->history_len > 0) {
        a->history = d->history; a->history_len = d->history_len; a->history_wide = d->history_wide;
        a->lens = d->history_lens; a->prompts = d->prompt_lens; a->lens_wide = d->lens_wide;
    }
    a->history_rows = (int)d->history_rows; a->mask_rows = (int)d->mask_rows; a->bias_rows = (int)d->bias_rows;
    a->rep_rows = (int)d->repetition_rows; a->pres_rows = (int)d->presence_rows; a->freq_rows = (int)d->frequency_rows; a->temp_rows = (int)d->temperature_rows;
    a->mask_type = d->mask_type; a->mask = d->mask; a->bias = d->bias;
    a->rep = d->repetition_t; a->pres = d->presence_t; a->freq = d->frequency_t; a->temp = d->temperature_t;
    a->rep_value = d->repetition; a->pres_value = d->presence; a->freq_value = d->frequency; a->temp_value = d->temperature;
    a->masked_value = d->masked_value;
    if (d->inner == 1) {
        a->chunk = LGT_STRIDE * token_iterations(d->rows, d->vocab);
    } else {
        a->chunk = (int)std::max(1ll, std::min(d->vocab, (long long)LGT_STRIDE / d->inner));
    }
    a->chunks = (int)((d->vocab + a->chunk - 1) / a->chunk);
    if (std::max(d->rows, 1ll) * a->chunks > 0x7fffffffll) return fail(-2, "gcn_logits: too many rows");
    return 0;
}

size_t lds_of_fwd(const LogitsArgs& a) {
    if (a.inner == 1) return a.history ? (size_t)a.chunk * sizeof(uint32_t) : 0;
    return (size_t)(((a.chunk + 3) & ~3) + a.chunk) * sizeof(uint32_t);
}

// As many workgroups in two dimensions: one of them holds less than 2^32 threads.
dim3 grid_of(uint32_t blocks) {
    const uint32_t x = std::min(blocks, 1u << 22);
    return dim3(x, (blocks + x - 1) / x);
}

template <typename T>
int launch_fwd(LogitsArgs a, hipStream_t st) {
    a.blocks = (uint32_t)a.rows * a.chunks;
    const dim3 blocks = grid_of(a.blocks);
    const size_t lds = lds_of_fwd(a);
    GCN_PROF_PRE(a.inner == 1 ? "k_logits" : "k_scores");
    const bool wide = a.chunk == 2 * LGT_STRIDE, far = a.history && a.history_len >= 8192;
    if (a.inner > 1) k_scores<T><<<blocks, LGT_THREADS, lds, st>>>(a);
    else if (wide && far) k_logits<T, 2, true><<<blocks, LGT_THREADS, lds, st>>>(a);
    else if (wide) k_logits<T, 2, false><<<blocks, LGT_THREADS, lds, st>>>(a);
    else if (far) k_logits<T, 1, true><<<blocks, LGT_THREADS, lds, st>>>(a);
    else k_logits<T, 1, false><<<blocks, LGT_THREADS, lds, st>>>(a);
    GCN_CHECK_LAUNCH("k_logits");
    return 0;
}

// The backward kernel's own range of a row.
void set_bwd_chunk(LogitsArgs* a) {
    if (a->inner != 1) return;
    a->chunk = LGT_STRIDE;
    a->chunks = (a->vocab + a->chunk - 1) / a->chunk;
}

// Parts of the rows that share a bias row: about 1024 workgroups, but with several rows each where there are enough (a turn's
// histories are counted together; 800 rows of 200 x 100 scores in fp32: 33 us with 4 rows, 41 with 2, 59 with 1), and sums of the
// parts (written and read in fp32) of at most an eighth of the gradient's bytes where that is more than a launch's worth.
int splits_of(const LogitsArgs& a, bool want_bias, int type) {
    const long long many = a.rows / a.bias_rows, per_part = (long long)a.chunks * a.bias_rows;
    const long long splits = std::max(1ll, std::min(many, 1024 / per_part));
    if (!want_bias) return (int)splits;
    const long long data = (long long)a.rows * a.vocab * a.inner * (type == GCN_F32 ? 8 : 4), part = 8ll * a.bias_rows * a.vocab;
    return (int)std::max(1ll, std::min(splits, std::max(data, 32ll << 20) / 8 / part));
}
bool tile_fits(const LogitsArgs& a) { return a.inner <= LGT_STRIDE; }

template <typename T>
int launch_bwd(LogitsArgs a, float* dbias, int splits, float* parts, hipStream_t st) {
    const bool by_tile = dbias && tile_fits(a);
    a.splits = splits;
    a.dbias = by_tile ? (splits > 1 ? parts : dbias) : nullptr;
    if ((long long)a.chunks * a.bias_rows * splits > 0x7fffffffll) return fail(-2, "gcn_logits_process_bwd: too many rows");
    a.blocks = (uint32_t)((long long)a.chunks * a.bias_rows * splits);
    const dim3 blocks = grid_of(a.blocks);
    const size_t lds = (by_tile ? 2 * LGT_STRIDE * sizeof(float) : 0) + (size_t)LGT_SCORE_ROWS * a.chunk;
    if (a.y || by_tile) {
        GCN_PROF_PRE(a.inner == 1 ? "k_logits_bwd" : "k_scores_bwd");
        if (a.inner > 1) k_scores_bwd<T><<<blocks, LGT_THREADS, lds, st>>>(a);
        else k_logits_bwd<T><<<blocks, LGT_THREADS, 0, st>>>(a);
        GCN_CHECK_LAUNCH("k_logits_bwd");
    }
    if (!dbias) return 0;
    const long long n = (long long)a.bias_rows * a.vocab;
    if (!by_tile) {
        const long long blocks = (n + LGT_THREADS / 64 - 1) / (LGT_THREADS / 64);
        GCN_PROF_PRE("k_scores_bias_grad");
        k_scores_bias_grad<T><<<(uint32_t)blocks, LGT_THREADS, 0, st>>>(a, dbias);
        GCN_CHECK_LAUNCH("k_scores_bias_grad");
    } else if (splits > 1) {
        GCN_PROF_PRE("k_logits_bias_sum");
        k_logits_bias_sum<<<(uint32_t)((n + 31) / 32), 256, 0, st>>>(n, splits, parts, dbias);
        GCN_CHECK_LAUNCH("k_logits_bias_sum");
    }
    return 0;
}

}  // namespace

extern "C" {

int gcn_logits_process(const gcn_logits_desc* d, const void* in, void* out, void* stream) {
    LogitsArgs a;
    if (int rc = fill_args(d, &a)) return rc;
    if (a.rows == 0) return 0;
    if (!in || !out) return fail(-1, "gcn_logits_process: null pointer argument");
    a.x = in; a.y = out;
    hipStream_t st = (hipStream_t)stream;
    if (d->type == GCN_F32) return launch_fwd<float>(a, st);
    if (d->type == GCN_BF16) return launch_fwd<__bf16>(a, st);
    return launch_fwd<_Float16>(a, st);
}

size_t gcn_logits_bwd_ws_bytes(const gcn_logits_desc* d) {
    LogitsArgs a;
    if (fill_args(d, &a) || a.rows == 0 || !a.bias) return 0;
    set_bwd_chunk(&a);
    const int splits = splits_of(a, true, d->type);
    return splits > 1 && tile_fits(a) ? (size_t)splits * a.bias_rows * a.vocab * sizeof(float) : 0;
}

int gcn_logits_process_bwd(const gcn_logits_desc* d, const void* in, const void* dout, void* din, float* dbias, void* ws, size_t ws_bytes,
                           void* stream) {
    LogitsArgs a;
    if (int rc = fill_args(d, &a)) return rc;
    if (dbias && !d->bias) return fail(-1, "gcn_logits_process_bwd: gradient of a bias that is not there");
    if (a.rows == 0) return 0;
    if (!in || !dout || (!din && !dbias)) return fail(-1, "gcn_logits_process_bwd: null pointer argument");
    const size_t need = dbias ? gcn_logits_bwd_ws_bytes(d) : 0;
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 3))) return fail(-2, "gcn_logits_process_bwd: workspace too small");
    a.x = in; a.y = din; a.dy = dout;
    set_bwd_chunk(&a);
    if (!dbias) a.bias_rows = 1;
    // a repetition penalty of one changes no slope: the history is not needed
    if (!din || (!a.rep && a.rep_value == 1.f)) a.history = nullptr;
    const int splits = splits_of(a, dbias != nullptr, d->type);
    hipStream_t st = (hipStream_t)stream;
    if (d->type == GCN_F32) return launch_bwd<float>(a, dbias, splits, (float*)ws, st);
    if (d->type == GCN_BF16) return launch_bwd<__bf16>(a, dbias, splits, (float*)ws, st);
    return launch_bwd<_Float16>(a, dbias, splits, (float*)ws, st);
}

}  // extern "C"

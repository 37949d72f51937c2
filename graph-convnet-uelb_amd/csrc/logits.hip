// C ABI of the logits operators: argument checks and launches.  The entry points are documented in include/gcn_uelb_hip.h.
#include <algorithm>

#include "../../include/gcn_uelb_hip.h"
#include "host.hpp"
#include "kernels_logits.hpp"

namespace {

int check_rows(const char* what, const void* p, long long n, long long rows) {
    if (p && (n < 1 || n > rows || rows % n)) return fail(-1, "gcn_logits: %lld rows of %s for %lld rows of logits", n, what, rows);
    return 0;
}

int fill_args(const gcn_logits_desc* d, LogitsArgs* a) {
    if (!d) return fail(-1, "gcn_logits: null descriptor");
    if (d->type < GCN_F32 || d->type > GCN_F16) return fail(-1, "gcn_logits: unknown type %d", d->type);
    if (d->rows < 0 || d->vocab < 1 || d->inner < 1) return fail(-1, "gcn_logits: %lld x %lld x %lld logits", d->rows, d->vocab, d->inner);
    if (d->rows >= (1ll << 31) || d->vocab >= (1ll << 31) || d->inner >= (1ll << 31) || d->vocab * d->inner >= (1ll << 31) - 4096)
        return fail(-2, "gcn_logits: %lld x %lld x %lld logits are too many for 32-bit places in a row", d->rows, d->vocab, d->inner);
    if (d->in_stride < 0 || d->out_stride < d->vocab * d->inner) return fail(-1, "gcn_logits: row strides %lld, %lld", d->in_stride, d->out_stride);
    if (d->history && (d->history_len < 0 || d->history_len >= (1ll << 31) - LGT_THREADS)) return fail(-1, "gcn_logits: history of %lld", d->history_len);
    if (!d->history && (d->history_lens || d->prompt_lens)) return fail(-1, "gcn_logits: lengths without a history");
    if (d->mask_type < 0 || d->mask_type > 2 || (d->mask_type != 0) != (d->mask != nullptr)) return fail(-1, "gcn_logits: mask of type %d", d->mask_type);
    if (!d->repetition_t && !(d->repetition > 0.f)) return fail(-1, "gcn_logits: repetition penalty %g", (double)d->repetition);
    if (!d->temperature_t && !(d->temperature > 0.f)) return fail(-1, "gcn_logits: temperature %g", (double)d->temperature);
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
    // about 1024 workgroups; a range of at least one pass of the workgroup and at most 16384 counts (64 KiB of LDS)
    const long long want = (d->vocab * std::max(d->rows, 1ll) + 1023) / 1024;
    a->chunk = (int)std::min<long long>(16384, std::max<long long>(LGT_STRIDE, (want + LGT_STRIDE - 1) / LGT_STRIDE * LGT_STRIDE));
    a->chunks = (int)((d->vocab + a->chunk - 1) / a->chunk);
    if (d->rows * a->chunks > 0x7fffffffll) return fail(-2, "gcn_logits: too many rows");
    return 0;
}

size_t lds_of(const LogitsArgs& a) { return a.history ? (size_t)std::min(a.chunk, a.vocab) * sizeof(uint32_t) : 0; }

template <typename T, bool BACKWARD>
int launch(const LogitsArgs& a, hipStream_t st) {
    const size_t lds = lds_of(a);
    GCN_PROF_PRE(BACKWARD ? "k_logits_bwd" : "k_logits");
    k_logits<T, BACKWARD><<<(uint32_t)a.rows * a.chunks, LGT_THREADS, lds, st>>>(a);
    GCN_CHECK_LAUNCH("k_logits");
    return 0;
}

template <typename T>
int launch_bias(const LogitsArgs& a, float* dbias, hipStream_t st) {
    const long long waves = (long long)a.bias_rows * a.vocab, blocks = (waves + LGT_THREADS / 64 - 1) / (LGT_THREADS / 64);
    if (blocks > 0x7fffffffll) return fail(-2, "gcn_logits_process_bwd: bias too large");
    GCN_PROF_PRE("k_logits_bias_grad");
    k_logits_bias_grad<T><<<(uint32_t)blocks, LGT_THREADS, 0, st>>>(a, dbias);
    GCN_CHECK_LAUNCH("k_logits_bias_grad");
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
    if (d->type == GCN_F32) return launch<float, false>(a, st);
    if (d->type == GCN_BF16) return launch<__bf16, false>(a, st);
    return launch<_Float16, false>(a, st);
}

int gcn_logits_process_bwd(const gcn_logits_desc* d, const void* in, const void* dout, void* din, float* dbias, void* stream) {
    LogitsArgs a;
    if (int rc = fill_args(d, &a)) return rc;
    if (dbias && !d->bias) return fail(-1, "gcn_logits_process_bwd: gradient of a bias that is not there");
    if (a.rows == 0) return 0;
    if (!in || !dout || (!din && !dbias)) return fail(-1, "gcn_logits_process_bwd: null pointer argument");
    a.x = in; a.y = din; a.dy = dout;
    // a repetition penalty of one changes no slope: the history is not needed
    if (!a.rep && a.rep_value == 1.f) a.history = nullptr;
    hipStream_t st = (hipStream_t)stream;
    if (din) {
        const int rc = d->type == GCN_F32 ? launch<float, true>(a, st) : d->type == GCN_BF16 ? launch<__bf16, true>(a, st) : launch<_Float16, true>(a, st);
        if (rc) return rc;
    }
    if (dbias) {
        const int rc = d->type == GCN_F32 ? launch_bias<float>(a, dbias, st) : d->type == GCN_BF16 ? launch_bias<__bf16>(a, dbias, st) : launch_bias<_Float16>(a, dbias, st);
        if (rc) return rc;
    }
    return 0;
}

}  // extern "C"

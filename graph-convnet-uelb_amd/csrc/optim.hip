// C ABI of the optimizer operators (AdamW step, gradient norm): argument checks, tables and launches.  The entry points are
// documented in include/gcn_uelb_hip.h.
#include <algorithm>
#include <cmath>

#include "../../include/gcn_uelb_hip.h"
#include "host.hpp"
#include "kernels_optim.hpp"

namespace {

constexpr uint64_t kNormSpan = OPT_NORM_UNITS * OPT_STRIDE;       // elements of a workgroup of k_grad_norm

constexpr uint64_t kMostBlocks = 0xffffffffull / OPT_THREADS;       // workgroups of a launch: less than 2^32 threads

int log2_of(uint64_t power) { return __builtin_ctzll(power); }

// Elements of a workgroup of k_adamw: one stride of 2048; two with 8-bit states, where the search for the tensor weighs more,
// once there are workgroups enough.  Per launch, with one / two / four strides: 8-bit states 159 M elements 510 / 501 / 502 us,
// 2.7 M 13.3 / 14.3 / 18.4 us; fp32 states 120 M 620 / 626 / 636 us, 14 M 70 / 74 / 78 us.
uint32_t adamw_span(uint64_t total, bool eight) {
    if (const char* e = tune_env("GCN_TUNE_ADAMW_UNITS")) return (uint32_t)atoi(e) * OPT_STRIDE;
    return eight && total >= (1ull << 25) ? 2 * OPT_STRIDE : OPT_STRIDE;
}

size_t elem_size(int type) { return type == GCN_F32 ? 4 : 2; }

bool aligned_to(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

uint64_t units_of(uint64_t n, uint64_t span) { return (n + span - 1) / span; }

void put(OptTable* t, int field, int k, uint64_t value) {
    const int e = field * t->cap + k;
    t->lo[e] = (uint32_t)value;
    const int shift = 16 * (e & 1);
    t->hi[e >> 1] = (t->hi[e >> 1] & ~(0xFFFFu << shift)) | (uint32_t)(value >> 32 & 0xFFFFu) << shift;
}

// A table has 47 bits for an address.
bool fits(const void* p) { return ((uintptr_t)p >> 47) == 0; }

int check_numel(const char* who, int n, const long long* numel, uint64_t* total) {
    *total = 0;
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0 || numel[k] >= (1ll << 40)) return fail(-1, "%s: tensor %d has %lld elements", who, k, numel[k]);
        *total += (uint64_t)numel[k];
    }
    if (*total >= (1ull << 42)) return fail(-2, "%s: %llu elements in all", who, (unsigned long long)*total);
    return 0;
}

}  // namespace

extern "C" {

size_t gcn_adamw_hyper_bytes(void) { return sizeof(AdamwHyper); }

static int check_adamw(const gcn_adamw_desc* d) {
    if (!d) return fail(-1, "gcn_adamw: null descriptor");
    if (d->n < 0) return fail(-1, "gcn_adamw: n = %d", d->n);
    if (d->param_type < GCN_F32 || d->param_type > GCN_F16) return fail(-1, "gcn_adamw: unknown parameter type %d", d->param_type);
    if (d->state_bits != 32 && d->state_bits != 8) return fail(-1, "gcn_adamw: states of %d bits (32 or 8)", d->state_bits);
    if (!(d->lr >= 0.0) || !(d->eps >= 0.0) || !(d->weight_decay >= 0.0)) return fail(-1, "gcn_adamw: negative lr, eps or weight_decay");
    if (!(d->beta1 >= 0.0 && d->beta1 < 1.0) || !(d->beta2 >= 0.0 && d->beta2 < 1.0)) return fail(-1, "gcn_adamw: betas outside [0, 1)");
    return 0;
}

int gcn_adamw_advance(const gcn_adamw_desc* d, long long* step, const float* lr, void* hyper, void* stream) {
    if (int rc = check_adamw(d)) return rc;
    if (!step || !hyper) return fail(-1, "gcn_adamw_advance: null pointer argument");
    if (!aligned_to(step, 8) || !aligned_to(hyper, 8)) return fail(-1, "gcn_adamw_advance: pointer not aligned to 8 bytes");
    hipStream_t st = (hipStream_t)stream;
    GCN_PROF_PRE("k_adamw_advance");
    k_adamw_advance<<<1, 1, 0, st>>>(step, lr, (AdamwHyper*)hyper, d->lr, d->beta1, d->beta2, d->eps, d->weight_decay, d->seed);
    GCN_CHECK_LAUNCH("k_adamw_advance");
    return 0;
}

int gcn_adamw_step(const gcn_adamw_desc* d, void* const* params, const void* const* grads, float* const* masters, void* const* exp_avg,
                   void* const* exp_avg_sq, unsigned char* const* exp_avg_exp, unsigned char* const* exp_avg_sq_exp, const long long* numel,
                   const float* grad_scale, const float* clip_coef, const void* hyper, void* stream) {
    if (int rc = check_adamw(d)) return rc;
    const bool eight = d->state_bits == 8, half = d->param_type != GCN_F32;
    if (!hyper && d->step < 1) return fail(-1, "gcn_adamw_step: step %lld < 1", d->step);
    if (d->n > 0 && (!params || !grads || !exp_avg || !exp_avg_sq || !numel)) return fail(-1, "gcn_adamw_step: null pointer argument");
    if (d->n > 0 && half != (masters != nullptr)) return fail(-1, "gcn_adamw_step: master copies go with 16-bit parameters, and only with them");
    if (d->n > 0 && eight != (exp_avg_exp != nullptr && exp_avg_sq_exp != nullptr)) return fail(-1, "gcn_adamw_step: exponent bytes go with 8-bit states, and only with them");
    uint64_t total;
    if (int rc = check_numel("gcn_adamw_step", d->n, numel, &total)) return rc;
    const size_t pe = elem_size(d->param_type), se = eight ? 1 : 4;
    for (int k = 0; k < d->n; ++k) {
        if (numel[k] == 0) continue;
        if (!params[k] || !grads[k] || !exp_avg[k] || !exp_avg_sq[k] || (half && !masters[k]) || (eight && (!exp_avg_exp[k] || !exp_avg_sq_exp[k])))
            return fail(-1, "gcn_adamw_step: tensor %d has a null pointer", k);
        if (!aligned_to(params[k], pe) || !aligned_to(grads[k], pe) || !aligned_to(exp_avg[k], se) || !aligned_to(exp_avg_sq[k], se) ||
            (half && !aligned_to(masters[k], 4)))
            return fail(-1, "gcn_adamw_step: tensor %d is not aligned to its elements", k);
        if (!fits(params[k]) || !fits(grads[k]) || !fits(exp_avg[k]) || !fits(exp_avg_sq[k]) || (half && !fits(masters[k])) ||
            (eight && (!fits(exp_avg_exp[k]) || !fits(exp_avg_sq_exp[k]))))
            return fail(-2, "gcn_adamw_step: tensor %d lies beyond the addresses that the kernel's table holds", k);
    }
    hipStream_t st = (hipStream_t)stream;
    const AdamwHyper h = hyper ? AdamwHyper{} : opt_hyper(d->lr, d->beta1, d->beta2, d->eps, d->weight_decay, d->step, d->seed);
    OptTable t = {};
    t.span = adamw_span(total, eight);
    t.span_log2 = log2_of(t.span);
    t.cap = OPT_ENTRIES / (5 + (half ? 1 : 0) + (eight ? 2 : 0));
    for (int k = 0; k < d->n;) {
        t.n = 0;
        t.ordinal = d->first_tensor + (uint32_t)k;
        uint64_t blocks = 0;
        // tensors keep their numbers: an empty one takes a place without workgroups
        for (; k < d->n && t.n < t.cap; ++k, ++t.n) {
            const uint64_t more = units_of((uint64_t)numel[k], t.span);
            if (blocks + more > kMostBlocks) {
                if (t.n == 0) return fail(-2, "gcn_adamw_step: tensor %d is too large for one launch", k);
                break;
            }
            bool vec = aligned_to(params[k], 16) && aligned_to(grads[k], 16) && aligned_to(exp_avg[k], eight ? 8 : 16) && aligned_to(exp_avg_sq[k], eight ? 8 : 16);
            if (half) vec = vec && aligned_to(masters[k], 16);
            put(&t, 0, t.n, (uint64_t)numel[k] | (vec ? OPT_VEC : 0));
            put(&t, 1, t.n, (uint64_t)params[k]);
            put(&t, 2, t.n, (uint64_t)grads[k]);
            put(&t, 3, t.n, (uint64_t)exp_avg[k]);
            put(&t, 4, t.n, (uint64_t)exp_avg_sq[k]);
            int field = 5;
            if (half) put(&t, field++, t.n, (uint64_t)masters[k]);
            if (eight) { put(&t, field++, t.n, (uint64_t)exp_avg_exp[k]); put(&t, field, t.n, (uint64_t)exp_avg_sq_exp[k]); }
            blocks += more;
        }
        if (blocks == 0) continue;
        GCN_PROF_PRE("k_adamw");
#define ADAMW_LAUNCH(P, M, E) k_adamw<P, M, E><<<(uint32_t)blocks, OPT_THREADS, 0, st>>>(t, h, (const AdamwHyper*)hyper, grad_scale, clip_coef)
        if (d->param_type == GCN_F32) { if (eight) ADAMW_LAUNCH(float, false, true); else ADAMW_LAUNCH(float, false, false); }
        else if (d->param_type == GCN_BF16) { if (eight) ADAMW_LAUNCH(__bf16, true, true); else ADAMW_LAUNCH(__bf16, true, false); }
        else { if (eight) ADAMW_LAUNCH(_Float16, true, true); else ADAMW_LAUNCH(_Float16, true, false); }
#undef ADAMW_LAUNCH
        GCN_CHECK_LAUNCH("k_adamw");
    }
    return 0;
}

size_t gcn_grad_norm_ws_bytes(int n, const long long* numel) {
    uint64_t total = 0, blocks = 0;
    if (n < 0 || (n > 0 && !numel) || check_numel("gcn_grad_norm_ws_bytes", n, numel, &total)) return 0;
    for (int k = 0; k < n; ++k) blocks += units_of((uint64_t)numel[k], kNormSpan);
    return std::max<size_t>(blocks, 1) * sizeof(double);
}

int gcn_grad_norm(int n, int type, const void* const* grads, const long long* numel, const float* grad_scale, double max_norm, float* out,
                  void* ws, size_t ws_bytes, void* stream) {
    if (n < 0 || (n > 0 && (!grads || !numel)) || !out) return fail(-1, "gcn_grad_norm: null pointer argument or n = %d", n);
    if (type < GCN_F32 || type > GCN_F16) return fail(-1, "gcn_grad_norm: unknown type %d", type);
    if (!(max_norm >= 0.0)) return fail(-1, "gcn_grad_norm: max_norm %g", max_norm);
    uint64_t total;
    if (int rc = check_numel("gcn_grad_norm", n, numel, &total)) return rc;
    for (int k = 0; k < n; ++k)
        if (numel[k] > 0 && (!grads[k] || !aligned_to(grads[k], elem_size(type)))) return fail(-1, "gcn_grad_norm: tensor %d has a null or misaligned pointer", k);
    for (int k = 0; k < n; ++k)
        if (numel[k] > 0 && !fits(grads[k])) return fail(-2, "gcn_grad_norm: tensor %d lies beyond the addresses that the kernel's table holds", k);
    if (!ws || !aligned_to(ws, 8) || ws_bytes < gcn_grad_norm_ws_bytes(n, numel)) return fail(-2, "gcn_grad_norm: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    double* part = (double*)ws;
    uint64_t done = 0;
    OptTable t = {};
    t.span = (uint32_t)kNormSpan;
    t.span_log2 = log2_of(kNormSpan);
    t.cap = OPT_ENTRIES / 2;
    t.ordinal = 0;
    for (int k = 0; k < n;) {
        t.n = 0;
        uint64_t blocks = 0;
        for (; k < n && t.n < t.cap; ++k, ++t.n) {
            const uint64_t more = units_of((uint64_t)numel[k], kNormSpan);
            if (blocks + more > kMostBlocks) {
                if (t.n == 0) return fail(-2, "gcn_grad_norm: tensor %d is too large for one launch", k);
                break;
            }
            put(&t, 0, t.n, (uint64_t)numel[k] | (aligned_to(grads[k], 16) ? OPT_VEC : 0));
            put(&t, 1, t.n, (uint64_t)grads[k]);
            blocks += more;
        }
        if (blocks == 0) continue;
        GCN_PROF_PRE("k_grad_norm");
        if (type == GCN_F32) k_grad_norm<float><<<(uint32_t)blocks, OPT_THREADS, 0, st>>>(t, part + done);
        else if (type == GCN_BF16) k_grad_norm<__bf16><<<(uint32_t)blocks, OPT_THREADS, 0, st>>>(t, part + done);
        else k_grad_norm<_Float16><<<(uint32_t)blocks, OPT_THREADS, 0, st>>>(t, part + done);
        GCN_CHECK_LAUNCH("k_grad_norm");
        done += blocks;
    }
    if (done > 0x7fffffffull) return fail(-2, "gcn_grad_norm: too many partial sums");
    GCN_PROF_PRE("k_grad_norm_final");
    k_grad_norm_final<<<1, 1024, 0, st>>>((int)done, part, grad_scale, max_norm, out);
    GCN_CHECK_LAUNCH("k_grad_norm_final");
    return 0;
}

}  // extern "C"

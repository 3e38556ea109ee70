// The training step's entry points (include/crukx.h): checks, argument layouts and launches.
#include "step.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <limits>
#include <new>
#include <string>

#include "../../include/crukx.h"
#include "format.h"

static_assert(CRX_BF16 == crx::kBf16 && CRX_F16 == crx::kF16 && CRX_F32 == crx::kF32, "element types");
static_assert(CRX_MEAN_TOKEN == crx::kMeanToken && CRX_MEAN_SEQUENCE == crx::kMeanSequence && CRX_SUM == crx::kSum,
              "reductions");

namespace crx {
namespace {

uint32_t size_of(int32_t dtype) { return dtype == kF32 ? 4 : 2; }

void check_type(int32_t dtype, const char *what) {
    if (dtype != kBf16 && dtype != kF16 && dtype != kF32) throw Invalid(std::string(what) + ": unknown element type");
}

void check_aligned(const void *p, uint32_t bytes, const char *what) {
    if (reinterpret_cast<uintptr_t>(p) % bytes) throw Invalid(std::string(what) + ": data must be aligned to its elements");
}

// Floats (absent ones are at 0), and pairs of them, which are read and written 8 bytes at a time.
template <typename... P>
void check_floats(const P *...p) {
    for (const void *q : {static_cast<const void *>(p)...}) check_aligned(q, 4, "float data");
}
void check_stats(const float *p) { check_aligned(p, 8, "statistics"); }

void launched() {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) throw DeviceError(std::string("kernel launch: ") + hipGetErrorString(e));
}

// body() with its exceptions as status codes
template <typename F>
int32_t guarded_step(char *err, uint64_t errlen, F &&body) {
    auto put = [&](const char *m) {
        if (err && errlen) std::snprintf(err, (size_t)errlen, "%s", m);
    };
    put("");
    try {
        body();
        return CRX_OK;
    } catch (const Invalid &e) {
        put(e.what());
        return CRX_INVALID;
    } catch (const std::bad_alloc &) {
        put("out of memory");
        return CRX_NOMEM;
    } catch (const std::exception &e) {
        put(e.what());
        return CRX_DEVICE;
    } catch (...) {
        put("unknown error");
        return CRX_DEVICE;
    }
}

template <typename T>
At<T> at(const crx_positions &p) {
    return At<T>{static_cast<const T *>(p.p), p.stride_seq, p.stride_token};
}

// The checked logits; false when there is no position to work on.
bool rows_in(const crx_logits *x, RowsIn &o) {
    if (!x) throw Invalid("logits: missing");
    check_type(x->dtype, "logits");
    if (x->id_bytes != 4 && x->id_bytes != 8) throw Invalid("token ids must have 4 or 8 bytes");
    if (!(x->temperature > 0.0) || !std::isfinite(x->temperature)) throw Invalid("temperature must be positive and finite");
    constexpr uint64_t kMost = (1ULL << 31) - 1;
    if (x->seqs > kMost || x->tokens > kMost || (x->tokens && x->seqs > kMost / x->tokens))
        throw Invalid("logits of 2^31 or more positions are not supported");
    if (x->vocab > kMost) throw Invalid("a vocabulary of 2^31 or more ids is not supported");
    if (!x->seqs || !x->tokens) return false;
    if (!x->vocab) throw Invalid("logits: the vocabulary is empty");
    if (!x->x || !x->ids.p) throw Invalid("logits and token ids must not be null");
    check_aligned(x->x, size_of(x->dtype), "logits");
    check_aligned(x->ids.p, (uint32_t)x->id_bytes, "token ids");
    o.x = x->x;
    o.sb = x->stride_seq;
    o.st = x->stride_token;
    o.seqs = (uint32_t)x->seqs;
    o.tokens = (uint32_t)x->tokens;
    o.vocab = (uint32_t)x->vocab;
    o.rows = o.seqs * o.tokens;
    o.row0 = 0;
    o.ids = x->ids.p;
    o.ids_sb = x->ids.stride_seq;
    o.ids_st = x->ids.stride_token;
    o.id_bytes = x->id_bytes;
    o.mask = at<uint8_t>(x->mask);
    // not 0, whatever the temperature: -inf times it has to stay -inf
    const auto inverse = [&](double a) { return std::max((float)(a / x->temperature), std::numeric_limits<float>::denorm_min()); };
    o.c = inverse(1.4426950408889634);
    o.inv_temp = inverse(1.0);
    o.inv_temp_lo = (float)(1.0 / x->temperature - (double)o.inv_temp);
    if (!std::isfinite(o.c)) throw Invalid("temperature is too small for 32-bit arithmetic");
    return true;
}

uint32_t units_of(uint64_t elements) { return (uint32_t)((elements + kUnit - 1) / kUnit); }

// Workgroups of a pass over `units` units, `share` for each
uint32_t blocks_for(uint32_t units, uint32_t share) { return std::min((units + share - 1) / share, 1u << 23); }

// Whether a list's last range can take `more` elements: tensors that follow one another in memory (those of a flat
// buffer) are one range, so a launch holds more of them and none has edges inside.
template <typename L>
bool can_grow(const L &l, uint64_t more, uint32_t most) {
    return l.count && l.first[l.count - 1] + (l.n[l.count - 1] + more) / kUnit < most;
}
template <typename L>
void grow(L &l, uint64_t more) {
    l.n[l.count - 1] += more;
    l.first[l.count] = l.first[l.count - 1] + units_of(l.n[l.count - 1]);
}

// launch(list, type, whether the caches hold the gradients) over the n tensors: those of each type, as
// many in one launch as its arguments hold, at most `most` units
template <typename F>
void over_tensors(int32_t n, void *const *p, const uint64_t *numels, const int32_t *dtypes, uint32_t most, F &&launch) {
    if (n < 0 || (n && (!p || !numels || !dtypes))) throw Invalid("gradients: missing");
    uint64_t bytes = 0;
    for (int32_t i = 0; i < n; ++i) {
        check_type(dtypes[i], "gradients");
        if (numels[i] && !p[i]) throw Invalid("gradients: data must not be null");
        check_aligned(p[i], size_of(dtypes[i]), "gradients");
    }
    for (int32_t i = 0; i < n; ++i) bytes += numels[i] * size_of(dtypes[i]);
    NormList l;
    l.first[0] = 0;
    for (int32_t type : {kBf16, kF16, kF32}) {
        l.count = 0;
        auto flush = [&] {
            if (l.count) launch(l, type, bytes <= kKeepBytes);
            l.count = 0;
        };
        for (int32_t i = 0; i < n; ++i) {
            if (dtypes[i] != type || !numels[i]) continue;
            if (can_grow(l, numels[i], most) && p[i] == static_cast<uint8_t *>(l.p[l.count - 1]) + l.n[l.count - 1] * size_of(type)) {
                grow(l, numels[i]);
                continue;
            }
            uint64_t at = 0;  // a tensor of more units than a launch takes is several entries
            while (at < numels[i]) {
                if (l.count == kNormTensors || l.first[l.count] >= most) flush();
                const uint64_t take = std::min<uint64_t>(numels[i] - at, (uint64_t)kUnit * (most - l.first[l.count]));
                l.p[l.count] = static_cast<uint8_t *>(p[i]) + at * size_of(type);
                l.n[l.count] = take;
                l.first[l.count + 1] = l.first[l.count] + units_of(take);
                ++l.count;
                at += take;
            }
        }
        flush();
    }
}

}  // namespace
}  // namespace crx

using namespace crx;

extern "C" {

uint64_t crx_rows_scratch(uint64_t seqs, uint64_t tokens, uint64_t vocab) {
    const uint64_t rows = seqs * tokens;
    const Parts p = parts_of(rows, vocab);
    return 12 * rows + 4 * (seqs + 2) + (p.n > 1 ? 12 * rows * p.n : 0);
}

int32_t crx_token_logprobs(const crx_logits *x, float *logprobs, float *entropy, float *stats, void *scratch,
                           void *stream, char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        RowsIn in;
        if (!rows_in(x, in)) return;
        if (!logprobs || !scratch) throw Invalid("token_logprobs: no place for the results");
        check_floats(logprobs, entropy, scratch);
        check_stats(stats);
        Parts parts = parts_of(in.rows, in.vocab);
        parts.stat = static_cast<float *>(scratch);
        launch_score(in, parts, ScoreOut{logprobs, entropy, reinterpret_cast<float2 *>(stats)}, x->dtype,
                     static_cast<hipStream_t>(stream));
        launched();
    });
}

int32_t crx_token_logprobs_grad(const crx_logits *x, const float *stats, const float *entropy,
                                const crx_positions *up_logprobs, const crx_positions *up_entropy, void *grad,
                                void *stream, char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        RowsIn in;
        if (!rows_in(x, in)) return;
        GradIn g{};
        g.stats = reinterpret_cast<const float2 *>(stats);
        if (up_logprobs) g.up_logp = at<float>(*up_logprobs);
        if (up_entropy) g.up_entropy = at<float>(*up_entropy);
        g.entropy = entropy;
        g.grad = grad;
        if (!stats || !grad || (g.up_entropy.p && !entropy)) throw Invalid("token_logprobs: no statistics or no place for the gradient");
        check_aligned(grad, size_of(x->dtype), "gradient");
        check_floats(entropy, g.up_logp.p, g.up_entropy.p);
        check_stats(stats);
        launch_rows_grad(in, g, x->dtype, static_cast<hipStream_t>(stream));
        launched();
    });
}

int32_t crx_policy_loss(const crx_logits *x, const crx_policy *p, float *loss, float *kl, float *clipped,
                        float *logprobs, float *stats, float *slope, void *grad, void *scratch, void *stream, char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        const hipStream_t s = static_cast<hipStream_t>(stream);
        RowsIn in;
        const bool any = rows_in(x, in);
        if (!p || !loss || !kl || !clipped) throw Invalid("policy_loss: missing arguments");
        if (p->reduction != kMeanToken && p->reduction != kMeanSequence && p->reduction != kSum)
            throw Invalid("policy_loss: unknown reduction");
        if (!(p->clip_low >= 0.0) || !(p->clip_high >= 0.0)) throw Invalid("policy_loss: the clip range must not be negative");
        check_floats(loss, kl, clipped, logprobs, slope, scratch);
        check_floats(p->old.p, p->advantages.p, p->ref.p);
        check_stats(stats);
        if (p->kl_coef != 0.0 && !p->ref.p && any) throw Invalid("policy_loss: a KL coefficient needs reference log probabilities");
        if (!any) {
            launch_policy_sums(nullptr, 0, 1.0f, loss, kl, clipped, s);
            launched();
            return;
        }
        if (!logprobs || !scratch || !p->old.p || !p->advantages.p) throw Invalid("policy_loss: missing arguments");
        if (grad) check_aligned(grad, size_of(x->dtype), "gradient");
        PolicyIn in_p{};
        in_p.old = at<float>(p->old);
        in_p.adv = at<float>(p->advantages);
        in_p.ref = at<float>(p->ref);
        in_p.low = (float)(1.0 - p->clip_low);
        in_p.high = (float)(1.0 + p->clip_high);
        in_p.kl = (float)p->kl_coef;
        in_p.scale = (float)p->scale;
        in_p.reduction = p->reduction;
        float *const terms = static_cast<float *>(scratch);
        uint32_t *const counts = reinterpret_cast<uint32_t *>(terms + 3 * (uint64_t)in.rows);
        Parts parts = parts_of(in.rows, in.vocab);
        parts.stat = reinterpret_cast<float *>(counts + in.seqs + 2);
        if (in.mask.p && p->reduction != kSum) {
            in_p.counts = counts;
            if (parts.n > 1) parts.counts = counts;  // with the parts' statistics
            else launch_mask_counts(in, counts, s);
        }
        launch_policy(in, parts, in_p, PolicyOut{logprobs, reinterpret_cast<float2 *>(stats), slope, terms, grad}, x->dtype, s);
        launch_policy_sums(terms, in.rows, in_p.scale, loss, kl, clipped, s);
        launched();
    });
}

int32_t crx_policy_loss_grad(const crx_logits *x, const float *stats, const float *slope, const float *upstream,
                             int32_t unless_one, void *grad, void *stream, char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        RowsIn in;
        if (!rows_in(x, in)) return;
        if (!stats || !slope || !upstream || !grad) throw Invalid("policy_loss: no statistics or no place for the gradient");
        check_aligned(grad, size_of(x->dtype), "gradient");
        check_floats(slope, upstream);
        check_stats(stats);
        GradIn g{};
        g.stats = reinterpret_cast<const float2 *>(stats);
        g.slope = slope;
        g.upstream = upstream;
        g.unless_one = unless_one;
        g.grad = grad;
        launch_rows_grad(in, g, x->dtype, static_cast<hipStream_t>(stream));
        launched();
    });
}

// A partial sum of every workgroup; a list of tensors takes one launch per kNormTensors of them, and the
// later launches' workgroups add to the earlier ones' sums.
uint64_t crx_norm_scratch(void) { return 8 * (uint64_t)kNormBlocks; }

int32_t crx_grad_norm(int32_t n, const void *const *grads, const uint64_t *numels, const int32_t *dtypes, float *norm,
                      void *scratch, void *stream, char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        const hipStream_t s = static_cast<hipStream_t>(stream);
        if (!norm || !scratch) throw Invalid("grad_norm: missing arguments");
        check_aligned(scratch, 8, "scratch");
        check_floats(norm);
        double *const partial = static_cast<double *>(scratch);
        uint32_t used = 0;  // partial sums written so far: later launches add to them
        over_tensors(n, const_cast<void *const *>(grads), numels, dtypes, kNormUnits, [&](const NormList &l, int type, bool keep) {
            const uint32_t blocks = std::min(kNormBlocks, blocks_for(l.first[l.count], kNormShare));
            launch_norm_part(l, type, partial, used, keep, blocks, s);
            used = std::max(used, blocks);
        });
        launch_norm_sum(partial, used, norm, s);
        launched();
    });
}

int32_t crx_clip_grads(int32_t n, void *const *grads, const uint64_t *numels, const int32_t *dtypes, const float *norm,
                       double max_norm, void *stream, char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        if (!norm) throw Invalid("clip_grads: missing arguments");
        if (!(max_norm >= 0.0)) throw Invalid("max_norm must not be negative");
        check_floats(norm);
        over_tensors(n, grads, numels, dtypes, kClipUnits, [&](const NormList &l, int type, bool keep) {
            launch_clip(l, type, norm, (float)max_norm, keep, blocks_for(l.first[l.count], kClipShare), static_cast<hipStream_t>(stream));
        });
        launched();
    });
}

int32_t crx_adamw_step(int32_t n, void *const *weights, float *const *masters, float *const *exp_avg,
                       float *const *exp_avg_sq, const void *const *grads, const uint64_t *numels,
                       const int32_t *weight_dtypes, const int32_t *grad_dtypes, const crx_adamw *a, void *stream,
                       char *err, uint64_t errlen) {
    return guarded_step(err, errlen, [&] {
        if (n < 0 || !a || (n && (!weights || !masters || !exp_avg || !exp_avg_sq || !grads || !numels || !weight_dtypes || !grad_dtypes)))
            throw Invalid("adamw: missing arguments");
        if (a->step < 1) throw Invalid("adamw: the first step is 1");
        if (!(a->lr >= 0.0) || !(a->eps >= 0.0) || !(a->weight_decay >= 0.0)) throw Invalid("adamw: lr, eps and weight_decay must not be negative");
        if (!(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0)) throw Invalid("adamw: betas must be in [0, 1)");
        if (a->norm && !(a->max_norm >= 0.0)) throw Invalid("max_norm must not be negative");
        check_floats(a->norm);
        for (int32_t i = 0; i < n; ++i) {
            check_type(weight_dtypes[i], "weights");
            check_type(grad_dtypes[i], "gradients");
            if (numels[i] && (!weights[i] || !masters[i] || !exp_avg[i] || !exp_avg_sq[i] || !grads[i])) throw Invalid("adamw: data must not be null");
            check_aligned(weights[i], size_of(weight_dtypes[i]), "weights");
            check_aligned(grads[i], size_of(grad_dtypes[i]), "gradients");
            check_aligned(masters[i], 4, "masters");
            check_aligned(exp_avg[i], 4, "exp_avg");
            check_aligned(exp_avg_sq[i], 4, "exp_avg_sq");
        }
        AdamArgs k;
        k.beta1 = (float)a->beta1;
        k.beta2 = (float)a->beta2;
        k.one_less_beta1 = (float)(1.0 - a->beta1);
        k.one_less_beta2 = (float)(1.0 - a->beta2);
        k.keep = 1.0 - a->lr * a->weight_decay;
        k.rate = (float)(a->lr / (1.0 - std::pow(a->beta1, (double)a->step)));
        k.root = (float)(1.0 / std::sqrt(1.0 - std::pow(a->beta2, (double)a->step)));
        k.eps = (float)a->eps;
        k.norm = a->norm;
        k.max_norm = (float)a->max_norm;
        AdamList l;
        l.first[0] = 0;
        for (int32_t kinds = 0; kinds < 9; ++kinds) {  // tensors of each pair of types
            const int32_t wtype = kinds / 3, gtype = kinds % 3;
            l.count = 0;
            auto flush = [&] {
                if (l.count)
                    launch_adamw(l, wtype, gtype, k, blocks_for(l.first[l.count], kAdamShare), static_cast<hipStream_t>(stream));
                l.count = 0;
            };
            for (int32_t i = 0; i < n; ++i) {
                if (weight_dtypes[i] != wtype || grad_dtypes[i] != gtype || !numels[i]) continue;
                if (can_grow(l, numels[i], kAdamUnits)) {
                    const uint32_t c = l.count - 1;
                    const uint64_t n = l.n[c];
                    if (weights[i] == static_cast<uint8_t *>(l.w[c]) + n * size_of(wtype) && masters[i] == l.master[c] + n &&
                        exp_avg[i] == l.m[c] + n && exp_avg_sq[i] == l.v[c] + n &&
                        grads[i] == static_cast<const uint8_t *>(l.g[c]) + n * size_of(gtype)) {
                        grow(l, numels[i]);
                        continue;
                    }
                }
                uint64_t at = 0;
                while (at < numels[i]) {
                    if (l.count == kAdamTensors || l.first[l.count] >= kAdamUnits) flush();
                    const uint64_t take = std::min<uint64_t>(numels[i] - at, (uint64_t)kUnit * (kAdamUnits - l.first[l.count]));
                    const uint32_t c = l.count++;
                    l.w[c] = static_cast<uint8_t *>(weights[i]) + at * size_of(wtype);
                    l.master[c] = masters[i] + at;
                    l.m[c] = exp_avg[i] + at;
                    l.v[c] = exp_avg_sq[i] + at;
                    l.g[c] = static_cast<const uint8_t *>(grads[i]) + at * size_of(gtype);
                    l.n[c] = take;
                    l.first[c + 1] = l.first[c] + units_of(take);
                    at += take;
                }
            }
            flush();
        }
        launched();
    });
}

}  // extern "C"

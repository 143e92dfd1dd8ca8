// The calls and the autograd nodes of the losses over token log-probabilities,
// of the log-probabilities themselves, of distillation, sampling and the 8-bit
// checkpoints, as a CPython module over the C ABI.
//
// In Python a loss with its gradient took 125 us of host time for two to five
// launches, the gradient's node alone 60: the engine runs it on a thread of its
// own that has to wait for the interpreter.  Here the engine's thread needs no
// interpreter.
//
// The callers have checked shapes and types.  Only what a kernel can read
// through a pointer is taken, plain tensors on one GPU; for anything else the
// functions return None and the callers' torch operations do it.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <math.h>
#include <stdint.h>

#include <cmath>

#include "../../include/slidefsdp.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int status, const char* what) {
    TORCH_CHECK(status == 0, what, " failed: ", sf_error_string(status), " (status ", status, ")");
}

sf_stream_t stream_of(const Tensor& t) {
    return reinterpret_cast<sf_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// Whether a kernel that reads t's memory gets all of it: no batch of a vmap, no
// wrapper of a transform, no pending negation or conjugation, no forward-mode
// derivative beside it.
bool memory_is_value(const Tensor& t) {
    static const uint64_t allowed = c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView,
                                                         c10::DispatchKey::AutogradCUDA, c10::DispatchKey::AutocastCUDA})
                                        .raw_repr();
    return (t.unsafeGetTensorImpl()->key_set().raw_repr() & ~allowed) == 0 && !t._fw_grad(0).defined();
}

bool plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.is_cuda() && memory_is_value(t);
}

// What the forward saved, as it saved it: hooks may have brought it back otherwise.
bool as_saved(const Tensor& t, at::ScalarType type, c10::Device dev) {
    return t.defined() && t.scalar_type() == type && t.device() == dev && memory_is_value(t) && t.is_contiguous() &&
           t.numel() > 0;
}

// Rows as the kernels read them: elements side by side, any whole number of
// elements that holds a row from one to the next.
bool rows_readable(const Tensor& t) {
    return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}
Tensor rows(const Tensor& t) { return rows_readable(t) ? t : t.contiguous(); }
size_t ld(const Tensor& t) { return size_t(t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1))); }

template <typename T>
T* at_ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// The gradients of a node that is not differentiated again: where that is asked
// for, an error when it comes to it.
variable_list once(const Tensor& upstream, variable_list out) {
    if (!at::GradMode::is_enabled() || !upstream.requires_grad()) return out;
    for (Tensor& t : out) {
        if (!t.defined()) continue;
        auto error = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice a function that can be differentiated once", 1);
        t = (*error)({t.detach().requires_grad_(true)})[0];
    }
    return out;
}

Tensor like(const Tensor& t, at::IntArrayRef shape) { return at::empty(shape, t.options().dtype(at::kFloat)); }

// ---------------------------------------------------------------------------
struct PrefArgs {
    int64_t form;
    double beta, smoothing;
    bool average;
};

struct PrefOut {
    Tensor loss, chosen, rejected, coef;
};

PrefOut pref_forward(const Tensor& logps_, const Tensor& ref_, const Tensor& mask, const PrefArgs& a, bool grad) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor logps = rows(logps_), ref = rows(ref_);
    const int64_t n = logps.size(0), cols = logps.size(1);
    PrefOut o = {like(logps, {}), like(logps, {n / 2}), like(logps, {n / 2}), grad ? like(logps, {n}) : Tensor()};
    const Tensor parts = like(logps, {int64_t(4 * sf_align_parts(n, cols))});
    check(sf_pref_loss(at_ptr<float>(logps), ld(logps), at_ptr<float>(ref), ld(ref), at_ptr<uint8_t>(mask), ld(mask),
                       n / 2, cols, int(a.form), float(a.beta), float(a.smoothing), a.average, parts.data_ptr(),
                       at_ptr<float>(o.loss), at_ptr<float>(o.chosen), at_ptr<float>(o.rejected), at_ptr<float>(o.coef),
                       stream_of(logps)),
          "sf_pref_loss");
    return o;
}

struct Preference : torch::autograd::Function<Preference> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logps, const Tensor& ref, const Tensor& mask,
                                 const PrefArgs& a) {
        PrefOut o = pref_forward(logps, ref, mask, a, true);
        ctx->save_for_backward({o.coef, mask});
        ctx->mark_non_differentiable({o.chosen, o.rejected});
        ctx->set_materialize_grads(false);
        return {o.loss, o.chosen, o.rejected};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& g = grads[0];
        if (!g.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &coef = saved[0], &mask = saved[1];
        Tensor out;
        {
            at::NoGradGuard none;
            const c10::Device dev = g.device();
            if (dev.is_cuda() && memory_is_value(g) && g.scalar_type() == at::kFloat && as_saved(coef, at::kFloat, dev) &&
                mask.scalar_type() == at::kBool && mask.device() == dev && memory_is_value(mask) && rows_readable(mask)) {
                at::AutoDispatchBelowADInplaceOrView below;
                const c10::DeviceGuard guard(dev);
                out = like(coef, mask.sizes());
                check(sf_pref_grad(at_ptr<float>(g), at_ptr<float>(coef), at_ptr<uint8_t>(mask), ld(mask), mask.size(0),
                                   mask.size(1), at_ptr<float>(out), stream_of(coef)),
                      "sf_pref_grad");
            } else {
                const Tensor each = (coef.to(at::kFloat) * g).unsqueeze(-1);
                out = at::where(mask.to(at::kBool), each, at::zeros_like(each));
            }
        }
        variable_list r = once(g, {out});
        return {r[0], Tensor(), Tensor(), Tensor()};
    }
};

// ---------------------------------------------------------------------------
struct PolicyArgs {
    double log_low, log_high, kl_coef;
    bool sequences;
};

struct PolicyOut {
    Tensor loss, kl, clipped, slope, weight;
};

PolicyOut policy_forward(const Tensor& logps_, const Tensor& old_, const Tensor& adv_, const Tensor& mask_,
                         const Tensor& ref_, const PolicyArgs& a, bool grad) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor logps = rows(logps_), old = rows(old_), mask = rows(mask_);
    const bool per_token = adv_.dim() == 2;
    const Tensor adv = per_token ? rows(adv_) : adv_, ref = ref_.defined() ? rows(ref_) : ref_;
    const int64_t n = logps.size(0), cols = logps.size(1);
    PolicyOut o = {like(logps, {}), ref.defined() ? like(logps, {}) : Tensor(), like(logps, {}),
                   grad ? like(logps, {n, cols}) : Tensor(), grad ? like(logps, {n}) : Tensor()};
    const Tensor parts = like(logps, {int64_t(8 * sf_align_parts(n, cols))});
    check(sf_policy_loss(at_ptr<float>(logps), ld(logps), at_ptr<float>(old), ld(old), at_ptr<float>(ref),
                         ref.defined() ? ld(ref) : 0, at_ptr<float>(adv), per_token ? ld(adv) : size_t(adv.stride(0)),
                         per_token, at_ptr<uint8_t>(mask), ld(mask), n, cols, float(a.log_low), float(a.log_high),
                         float(a.kl_coef), a.sequences, parts.data_ptr(), at_ptr<float>(o.loss), at_ptr<float>(o.kl),
                         at_ptr<float>(o.clipped), at_ptr<float>(o.slope), at_ptr<float>(o.weight), stream_of(logps)),
          "sf_policy_loss");
    return o;
}

struct PolicyNode : torch::autograd::Function<PolicyNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logps, const Tensor& old, const Tensor& adv,
                                 const Tensor& mask, const c10::optional<Tensor>& ref, const PolicyArgs& a) {
        PolicyOut o = policy_forward(logps, old, adv, mask, ref.has_value() ? *ref : Tensor(), a, true);
        ctx->save_for_backward({o.slope, o.weight});
        ctx->set_materialize_grads(false);
        if (!o.kl.defined()) {
            ctx->mark_non_differentiable({o.clipped});
            return {o.loss, o.clipped};
        }
        ctx->mark_non_differentiable({o.clipped, o.kl});
        return {o.loss, o.clipped, o.kl};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& g = grads[0];
        if (!g.defined()) return variable_list(6);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &slope = saved[0], &weight = saved[1];
        Tensor out;
        {
            at::NoGradGuard none;
            const c10::Device dev = g.device();
            if (dev.is_cuda() && memory_is_value(g) && g.scalar_type() == at::kFloat &&
                as_saved(slope, at::kFloat, dev) && as_saved(weight, at::kFloat, dev)) {
                at::AutoDispatchBelowADInplaceOrView below;
                const c10::DeviceGuard guard(dev);
                out = like(slope, slope.sizes());
                check(sf_policy_grad(at_ptr<float>(g), at_ptr<float>(weight), at_ptr<float>(slope), slope.size(0),
                                     slope.size(1), at_ptr<float>(out), stream_of(slope)),
                      "sf_policy_grad");
            } else {
                out = slope.to(at::kFloat) * (weight.to(at::kFloat) * g).unsqueeze(-1);
            }
        }
        variable_list all(6);
        all[0] = once(g, {out})[0];
        return all;
    }
};

// ---------------------------------------------------------------------------
// Log-probabilities through logps_tiles_kernel.
struct LogpsArgs {
    int64_t ignore_index;
    double scale;
    int64_t nparts;       // of the hidden gradient's sum over the vocabulary
    int64_t step;         // rows that the backward takes at a time
    bool keep;            // whether the forward keeps the exponentials (then step is all rows)
};

int type_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? SF_DTYPE_BF16 : SF_DTYPE_F16; }
int logits_type(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? SF_DTYPE_F32 : t.scalar_type() == at::kBFloat16 ? SF_DTYPE_BF16 : SF_DTYPE_F16;
}
int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

// As the kernel asks for it: 16-bit operands whose rows start on 16-byte
// boundaries, a sum of whole 64 terms.
bool in_tiles(const Tensor& hidden, const Tensor& weight) {
    if (hidden.scalar_type() != at::kBFloat16 && hidden.scalar_type() != at::kHalf) return false;
    if (hidden.size(1) % 64 != 0) return false;
    for (const Tensor* t : {&hidden, &weight}) {
        const int64_t row = t->stride(0);
        if (t->stride(1) != 1 || row < t->size(1) || row > (int64_t(1) << 22) || row % 8 != 0 ||
            reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0)
            return false;
    }
    return true;
}

// Whether the product looks for rows that it can leave out, prompts above all: a
// launch more, 3 us, where it takes 50 us or more and has more than one tile of
// tokens.  us, every row | those with a label, a fifth, half and nine tenths of
// the rows without: 4092 x 4096 x 128256 3045 | 2555, 1577, 431, 777 x 1024 x
// 50257 102 | 76, 59, 30.
bool skips_rows(int64_t n, int64_t h, int64_t v) { return n > 256 && 2 * n * h * v >= int64_t(1) << 36; }

// The spans' parts of `hidden`'s rows; their results into lse2 and logp.
Tensor tiles(const Tensor& hidden, const Tensor& weight, const int64_t* labels, const LogpsArgs& a, const Tensor& keep,
             float* lse2, float* logp) {
    const int64_t n = hidden.size(0), v = weight.size(0), held = 2 * n * ((v + SF_LOGPS_SPAN - 1) / SF_LOGPS_SPAN);
    const bool skip = skips_rows(n, hidden.size(1), v) && 2 * n * hidden.stride(0) <= int64_t(UINT32_MAX);
    const Tensor parts = like(hidden, {held + n + (skip ? n + 1 : 0)});
    float* p = at_ptr<float>(parts);
    int32_t* order = skip ? reinterpret_cast<int32_t*>(p + held + n) : nullptr;
    check(sf_logps_tiles(weight.data_ptr(), weight.stride(0), v, hidden.data_ptr(), hidden.stride(0), n, hidden.size(1),
                         labels, a.ignore_index, float(a.scale), type_of(hidden), p, p + held, order,
                         keep.defined() ? keep.data_ptr() : nullptr, keep.defined() ? keep.stride(0) : 0, lse2, logp,
                         stream_of(hidden)),
          "sf_logps_tiles");
    return parts;
}

struct LogpsOut {
    Tensor logp, lse2, keep, parts;
};

LogpsOut logps_forward(const Tensor& hidden, const Tensor& weight, const Tensor& labels, const LogpsArgs& a) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = hidden.size(0);
    LogpsOut o = {like(hidden, {n}), like(hidden, {n}), Tensor(), Tensor()};
    if (a.keep) o.keep = at::empty({up(n, 64), up(weight.size(0), SF_LOGPS_SPAN)}, hidden.options());
    o.parts = tiles(hidden, weight, at_ptr<int64_t>(labels), a, o.keep, at_ptr<float>(o.lse2), at_ptr<float>(o.logp));
    return o;
}

int64_t tiles_of(int64_t rows, int64_t cols) { return ((rows + 255) / 256) * ((cols + 255) / 256); }

// Whether the hidden gradient's product in `nparts` parts is
// sf_logps_hidden_product: over 64 tiles of 256 x 256, whose parts fill rounds of
// the chip.  With fewer tiles a library's smaller ones win: 300 x 4096 x 32000 (32)
// 99 | 118 us, 200 x 1024 x 32000 (4) 34 | 48.
bool own_hidden_product(int64_t n, int64_t h, int64_t row) {
    return tiles_of(n, h) > 64 && row <= int64_t(1) << 22;
}

// out = row weight * (d @ weight), rounded once.
void hidden_product(const Tensor& keep, int64_t n, const Tensor& weight, int64_t nparts, const float* row_weight,
                    const float* norm, const Tensor& out) {
    const int64_t v = weight.size(0), h = weight.size(1), row = keep.stride(0);
    const bool own = own_hidden_product(n, h, row);
    const int64_t part = own || nparts == 1 ? v : v / nparts / 8 * 8, done = own ? v : nparts * part;
    Tensor parts = like(keep, {nparts, n, h});
    if (own) {
        check(sf_logps_hidden_product(keep.data_ptr(), row, n, weight.data_ptr(), weight.stride(0), v, h, int(nparts),
                                      at_ptr<float>(parts), type_of(keep), stream_of(keep)),
              "sf_logps_hidden_product");
    } else if (nparts == 1) {
        Tensor whole = parts.select(0, 0);
        at::mm_out(whole, keep.as_strided({n, v}, {row, 1}), weight, at::kFloat);
    } else {
        at::bmm_out(parts, keep.as_strided({nparts, n, part}, {part, row, 1}),
                    weight.as_strided({nparts, part, h}, {part * h, h, 1}), at::kFloat);
    }
    const char *d = static_cast<const char*>(keep.data_ptr()), *w = static_cast<const char*>(weight.data_ptr());
    check(sf_logps_sum(at_ptr<float>(parts), int(nparts), n, h, out.data_ptr(), type_of(keep), d + 2 * done, row,
                       w + 2 * done * h, v - done, row_weight, norm, stream_of(keep)),
          "sf_logps_sum");
}

// Whether the weight gradient of a call in one piece is formed by
// sf_logps_weight_grad: up to 256 tokens always.  Beyond, a library's product wins
// with few tiles, 2000 x 512 x 4096 (32) 22 | 41 us, 834 x 896 x 6640 (104) 25 | 24,
// 400 x 1024 x 16000 (252) 25 | 19, and in bf16 by 2 to 4 % with the largest
// products: 4000 x 3584 x 152064 3318 | 3399, 8190 x 5120 x 152064 9340 | 9706, but
// 6500 x 2048 x 128256 2700 | 2584, 8190 x 2560 x 50257 1732 | 1597.  Of fp16 it is
// into fp32 and has to be scaled: 4000 x 3584 x 152064 4297 | 3541.
bool own_weight_grad(int64_t n, int64_t h, int64_t v, int64_t row, bool fp16) {
    if (row > int64_t(1) << 22 || n > int64_t(1) << 21) return false;   // what its offsets hold
    return n <= 256 || (tiles_of(h, v) >= 96 && (fp16 || double(n) * h * v <= 2e12));
}

// Whether the hidden gradient of a call in one piece is formed by
// sf_logps_hidden_grad instead of a library's product and a scaling: where the
// host's time for those, 18 to 22 us more, is longer.  Whole calls with this
// gradient, us, product | kernel: 126 x 512 x 4096 60 | 43, 64 x 1024 x 8192 63 |
// 49, 250 x 4096 x 4096 95 | 74; not with more to do, 1000 x 2048 x 4096 94 | 95,
// 2000 x 4096 x 1000 97 | 122, nor with more words for a workgroup, 128 x 2048 x
// 16384 86 | 85, 32 x 2048 x 32000 61 | 142.
bool own_hidden_grad(int64_t n, int64_t h, int64_t v) { return v <= 8192 && n * h * v <= int64_t(1) << 32; }

// Both gradients (undefined where not needed) from D, `step` rows at a time, all
// of them where it was kept.  fill(first row, rows, rows padded, their hidden rows,
// keep, row weights, norm or null) makes D of so many rows in keep's first, and with
// the first rows the weights of all.  divided: bf16's D may be over norm too.
template <typename Fill>
std::pair<Tensor, Tensor> products(const Tensor& hidden, const Tensor& weight, Tensor keep, int64_t step, int64_t nparts,
                                   bool need_hidden, bool need_weight, bool divided, const Fill& fill) {
    const int64_t n = hidden.size(0), h = hidden.size(1), v = weight.size(0), row = up(v, SF_LOGPS_SPAN);
    const bool fp16 = hidden.scalar_type() == at::kHalf;
    const bool one = step == n;
    const sf_stream_t st = stream_of(hidden);
    const int type = type_of(hidden);
    const Tensor scalars = like(hidden, {n + 3});
    float* const by = at_ptr<float>(scalars);
    const bool own = one && own_weight_grad(n, h, v, row, fp16);
    // What D is divided by leaves before the results are rounded: in the own products, or of few
    // tiles with a pass over them.
    float* const norm = fp16 || (divided && one && (own || tiles_of(h, v) < 96)) ? by + n : nullptr;
    Tensor gh, gw;
    if (need_hidden) gh = at::empty({n, h}, hidden.options());
    if (need_weight) gw = at::empty({v, h}, own || (one && norm == nullptr) ? weight.options() : weight.options().dtype(at::kFloat));
    if (!keep.defined()) keep = at::empty({up(step, 64), row}, hidden.options());
    for (int64_t s = 0; s < n; s += step) {
        const int64_t m = std::min(n - s, step), pad = up(m, 64);
        const Tensor hc = one ? hidden : hidden.narrow(0, s, m);
        fill(s, m, pad, hc, keep, by, norm);
        if (need_hidden && one && own_hidden_grad(n, h, v))
            check(sf_logps_hidden_grad(keep.data_ptr(), row, n, weight.data_ptr(), weight.stride(0), v, h,
                                       by, norm, type, gh.data_ptr(), st),
                  "sf_logps_hidden_grad");
        else if (need_hidden)
            hidden_product(keep, m, weight, nparts, by + s, norm,
                           one ? gh : gh.narrow(0, s, m));
        if (!need_weight) continue;
        if (fp16 && !own) {
            // into fp32, of rows as they lie: 4096 x 4096 x 128256 4.2 ms, of transposed ones 28.8
            const Tensor weighted = at::empty({m, h}, hidden.options());
            check(sf_logps_weighted(hc.data_ptr(), hc.stride(0), m, h, by + s, type, weighted.data_ptr(), st),
                  "sf_logps_weighted");
            const Tensor dt = keep.as_strided({v, m}, {1, row});
            if (s == 0) at::mm_out(gw, dt, weighted, at::kFloat);
            else at::addmm_out(gw, gw, dt, weighted, at::kFloat);
            continue;
        }
        // transposed: of bf16 the product with an operand laid out along the sum is
        // faster, 3.3 ms there instead of 4.0
        const Tensor ht = at::empty({h, pad}, hidden.options());
        check(sf_logps_hidden(hc.data_ptr(), hc.stride(0), m, h, by + s, type, ht.data_ptr(), pad, st),
              "sf_logps_hidden");
        if (own) {
            check(sf_logps_weight_grad(keep.data_ptr(), row, pad, v, ht.data_ptr(), h, norm,
                                       type, gw.data_ptr(), st),
                  "sf_logps_weight_grad");
            break;
        }
        const Tensor dt = keep.as_strided({v, pad}, {1, row}), hp = ht.t();
        if (one && norm == nullptr) at::mm_out(gw, dt, hp);
        else if (s == 0) at::mm_out(gw, dt, hp, at::kFloat);
        else at::addmm_out(gw, gw, dt, hp, at::kFloat);
    }
    if (need_weight && gw.scalar_type() != weight.scalar_type()) {
        // its factor leaves before the rounding
        if (norm != nullptr) {
            const Tensor out = at::empty({v, h}, weight.options());
            check(sf_ce_scale(norm, norm + 1, nullptr, nullptr, 0, at_ptr<float>(gw),
                              out.data_ptr(), size_t(v * h), type, st),
                  "sf_ce_scale");
            gw = out;
        } else {
            gw = gw.to(weight.scalar_type());
        }
    }
    return {gh, gw};
}

std::pair<Tensor, Tensor> logps_backward(const Tensor& grad, const Tensor& hidden, const Tensor& weight,
                                         const Tensor& labels, const Tensor& logp, const Tensor& lse2, const Tensor& keep,
                                         Tensor parts, const LogpsArgs& a, bool need_hidden, bool need_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = hidden.size(0), v = weight.size(0), row = up(v, SF_LOGPS_SPAN);
    const bool kept = keep.defined();
    const int64_t step = kept ? n : std::min(n, a.step);
    const int type = type_of(hidden);
    const int64_t* y = at_ptr<int64_t>(labels);
    Tensor again;   // results of the product made again
    if (!kept) again = like(hidden, {2, step});
    return products(hidden, weight, keep, step, a.nparts, need_hidden, need_weight, false,
                    [&](int64_t s, int64_t m, int64_t pad, const Tensor& hc, const Tensor& d, float* by, float* norm) {
        if (!kept) parts = tiles(hc, weight, y + s, a, d, at_ptr<float>(again), at_ptr<float>(again) + step);
        check(sf_logps_keep_grad(d.data_ptr(), row, m, pad, v, parts.data_ptr(), y + s, a.ignore_index,
                                 at_ptr<float>(lse2) + s, at_ptr<float>(logp) + s, type, at_ptr<float>(grad) + s,
                                 s == 0 ? n : 0, float(a.scale), by, norm, type == SF_DTYPE_F16, stream_of(hidden)),
              "sf_logps_keep_grad");
    });
}

struct LinearLogps : torch::autograd::Function<LinearLogps> {
    static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& labels,
                          const LogpsArgs& a) {
        LogpsOut o = logps_forward(hidden, weight, labels, a);
        ctx->save_for_backward({hidden, weight, labels, o.logp, o.lse2});
        ctx->set_materialize_grads(false);
        // not among the saved tensors: the backward overwrites it, and gives it up
        if (a.keep) {
            ctx->saved_data["keep"] = o.keep;
            ctx->saved_data["parts"] = o.parts;
        }
        ctx->saved_data["ignore_index"] = a.ignore_index;
        ctx->saved_data["scale"] = a.scale;
        ctx->saved_data["nparts"] = a.nparts;
        ctx->saved_data["step"] = a.step;
        return o.logp;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& g = grads[0];
        if (!g.defined()) return variable_list(4);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &hidden = saved[0], &weight = saved[1], &labels = saved[2], &logp = saved[3], &lse2 = saved[4];
        auto& data = ctx->saved_data;
        const LogpsArgs a = {data["ignore_index"].toInt(), data["scale"].toDouble(), data["nparts"].toInt(),
                             data["step"].toInt(), false};
        const bool need_hidden = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1);
        Tensor gh, gw;
        {
            at::NoGradGuard none;
            const c10::Device dev = g.device();
            if (dev.is_cuda() && memory_is_value(g) && hidden.device() == dev && weight.device() == dev &&
                memory_is_value(hidden) && memory_is_value(weight) && weight.scalar_type() == hidden.scalar_type() &&
                in_tiles(hidden, weight) && as_saved(labels, at::kLong, dev) && as_saved(logp, at::kFloat, dev) &&
                as_saved(lse2, at::kFloat, dev) && (a.nparts == 1 || weight.is_contiguous())) {
                const c10::DeviceGuard guard(dev);
                Tensor keep, parts;
                if (auto it = data.find("keep"); it != data.end()) {
                    keep = it->second.toTensor();
                    parts = data["parts"].toTensor();
                    // a second backward of a retained graph makes it again
                    data.erase("keep");
                    data.erase("parts");
                }
                std::tie(gh, gw) = logps_backward(g.to(at::kFloat).contiguous(), hidden, weight, labels, logp, lse2, keep,
                                                  parts, a, need_hidden, need_weight);
            } else {
                const Tensor w = weight.to(at::kFloat), lse = lse2.to(at::kFloat) * std::log(2.0);
                const Tensor valid = labels != a.ignore_index, inside = labels.ge(0).logical_and(labels < w.size(0));
                const Tensor index = at::where(valid.logical_and(inside), labels, at::zeros_like(labels));
                const Tensor counts = valid.logical_and(g != 0).unsqueeze(-1);
                const Tensor h = at::where(counts, hidden.to(at::kFloat), at::zeros({}, w.options()));
                const Tensor p = at::exp(at::matmul(h, w.t()) * a.scale - lse.unsqueeze(1));
                Tensor dz = (at::one_hot(index, w.size(0)) - p) * (g.to(at::kFloat) * a.scale).unsqueeze(-1);
                dz = at::where(counts, dz, at::zeros_like(dz));
                dz = at::where(counts.logical_and(inside.logical_not().unsqueeze(-1)), at::full_like(dz, NAN), dz);
                if (need_hidden) gh = at::matmul(dz, w).to(hidden.scalar_type());
                if (need_weight) gw = at::matmul(dz.transpose(-1, -2), h).to(weight.scalar_type());
            }
        }
        variable_list r = once(g, {gh, gw});
        return {r[0], r[1], Tensor(), Tensor()};
    }
};

// ---------------------------------------------------------------------------
// Distillation.  16-bit operands as logps_tiles_kernel takes them go through it; of
// others a library's product leaves fp32 logits, and the gradients' products are
// fp32, in pieces of 1 GiB.
struct DistillArgs {
    int64_t form;
    bool rest;
    double scale;
    int64_t nparts, step;   // as LogpsArgs
    bool keep, masked;
};

struct DistillOut {
    Tensor loss, keep, parts;
    // [n, k] or as include/slidefsdp.h says, for the backward
    Tensor words, starts, status, slopes, stats;
    Tensor order;         // where keep's rows are close: of which tokens they are
};

// Rows of logits of one piece.
int64_t piece_rows(int64_t n, int64_t v) { return std::min(n, std::max(int64_t(1), (int64_t(1) << 28) / v)); }

void product32(const Tensor& out, const Tensor& hidden, const Tensor& weight) {
    Tensor to = out;
    if (hidden.scalar_type() == at::kFloat) at::mm_out(to, hidden, weight.t());
    else at::mm_out(to, hidden, weight.t(), at::kFloat);
}

bool skips_masked(int64_t n, const Tensor& hidden, int64_t v) {
    return skips_rows(n, hidden.size(1), v) && 2 * n * hidden.stride(0) <= int64_t(UINT32_MAX);
}

// Whether a masked call keeps the rows of D close, so that both gradients' products leave out
// what has no loss, as the forward's does: where the weight gradient's product is the
// framework's own, of 96 tiles or more.  How many rows there are is known on the device alone.
// Loss and both gradients in us, all rows | close, nothing masked, a fifth, half: 4092 x 4096 x
// 128256 10450 | 10516, 8968, 5499; 8190 x 5120 x 152064 30584 | 30915, 26577, 15796; 4096 x
// 1024 x 32000 923 | 924, 817, 620; 512 x 4096 x 32000 542 | 549, 532, 502.
bool keeps_close(int64_t n, const Tensor& hidden, int64_t v) {
    return skips_masked(n, hidden, v) && tiles_of(hidden.size(1), v) >= 96 && n < int64_t(1) << 22 &&
           v <= (int64_t(1) << 22) - SF_LOGPS_SPAN;
}

Tensor distill_tiles(const Tensor& hidden, const Tensor& weight, const Tensor& words, const Tensor& starts,
                     const Tensor& status, int64_t first, double scale, const Tensor& keep, const Tensor& picked,
                     bool masked, const Tensor& close) {
    const int64_t n = hidden.size(0), v = weight.size(0), k = words.size(1);
    const int64_t held = 2 * n * ((v + SF_LOGPS_SPAN - 1) / SF_LOGPS_SPAN);
    const bool skip = masked && skips_masked(n, hidden, v), own = skip && !close.defined();
    const Tensor parts = like(hidden, {held + (own ? n + 1 : 0)});
    int32_t* order = close.defined() ? at_ptr<int32_t>(close)
                     : own           ? reinterpret_cast<int32_t*>(at_ptr<float>(parts) + held)
                                     : nullptr;
    check(sf_distill_tiles(weight.data_ptr(), weight.stride(0), v, hidden.data_ptr(), hidden.stride(0), n, hidden.size(1),
                           at_ptr<int32_t>(words) + first * k, at_ptr<uint8_t>(starts) + first * starts.size(1),
                           at_ptr<uint8_t>(status) + first, int(k), float(scale), type_of(hidden), parts.data_ptr(),
                           at_ptr<float>(picked), order, keep.defined() ? keep.data_ptr() : nullptr,
                           keep.defined() ? keep.stride(0) : 0, close.defined(), stream_of(hidden)),
          "sf_distill_tiles");
    return parts;
}

DistillOut distill_forward(const Tensor& hidden_, const Tensor& weight_, const Tensor& ids_, const Tensor& logps_,
                           const Tensor& mask, const DistillArgs& a, bool grad) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor ids = rows(ids_), logps = rows(logps_), hidden = rows(hidden_), weight = rows(weight_);
    const int64_t n = hidden.size(0), v = weight.size(0), k = ids.size(1);
    const bool whole = !in_tiles(hidden_, weight_);
    const int64_t spans = whole ? 1 : (v + SF_LOGPS_SPAN - 1) / SF_LOGPS_SPAN;
    const sf_stream_t st = stream_of(hidden);
    const auto bytes = hidden.options().dtype(at::kByte);
    DistillOut o;
    o.loss = like(hidden, {n});
    o.words = at::empty({n, k}, hidden.options().dtype(at::kInt));
    o.starts = at::empty({n, spans + 1}, bytes);
    o.status = at::empty({n}, bytes);
    const Tensor lists = like(hidden, {2, n, k});   // the teacher's, the products
    float *teacher = at_ptr<float>(lists), *picked = teacher + n * k;
    if (grad) o.slopes = like(hidden, {n, k}), o.stats = like(hidden, {4, n});
    check(sf_distill_lists(at_ptr<int64_t>(ids), ld(ids), at_ptr<float>(logps), ld(logps), at_ptr<uint8_t>(mask), n, int(k), v,
                           whole, at_ptr<int32_t>(o.words), teacher, at_ptr<uint8_t>(o.starts), at_ptr<uint8_t>(o.status), st),
          "sf_distill_lists");
    if (whole) {
        const int64_t step = piece_rows(n, v);
        const Tensor buf = like(hidden, {step, v});
        o.parts = like(hidden, {n, 2});
        for (int64_t s = 0; s < n; s += step) {
            const int64_t m = std::min(step, n - s);
            product32(buf.narrow(0, 0, m), hidden.narrow(0, s, m), weight);
            check(sf_distill_rows(at_ptr<float>(buf), v, m, v, at_ptr<int32_t>(o.words) + s * k,
                                  at_ptr<uint8_t>(o.starts) + s * 2, int(k), float(a.scale), at_ptr<float>(o.parts) + 2 * s,
                                  picked + s * k, st),
                  "sf_distill_rows");
        }
    } else {
        if (a.keep && grad) o.keep = at::empty({up(n, 64), up(v, SF_LOGPS_SPAN)}, hidden.options());
        if (o.keep.defined() && mask.defined() && keeps_close(n, hidden, v)) o.order = at::empty({n + 1}, o.words.options());
        o.parts = distill_tiles(hidden, weight, o.words, o.starts, o.status, 0, a.scale, o.keep, lists.select(0, 1),
                                mask.defined(), o.order);
    }
    check(sf_distill_loss(o.parts.data_ptr(), n, whole, picked, teacher, at_ptr<uint8_t>(o.starts), at_ptr<uint8_t>(o.status),
                          n, int(k), v, a.scale, int(a.form), a.rest, hidden.data_ptr(), ld(hidden), weight.data_ptr(),
                          ld(weight), hidden.size(1), logits_type(hidden), at_ptr<int32_t>(o.words), at_ptr<float>(o.loss), at_ptr<float>(o.slopes),
                          at_ptr<float>(o.stats), n, st),
          "sf_distill_loss");
    return o;
}

// Both gradients by fp32 products of whole logits, in pieces.
std::pair<Tensor, Tensor> distill_backward_whole(const Tensor& grad, const Tensor& hidden, const Tensor& weight,
                                                 const DistillOut& o, const DistillArgs& a, bool need_hidden,
                                                 bool need_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = hidden.size(0), v = weight.size(0), k = o.words.size(1), step = piece_rows(n, v);
    const Tensor none = at::zeros({}, grad.options());
    const Tensor by = at::where(o.status.eq(0).logical_or(grad.eq(0)), none, grad * a.scale * o.stats.select(0, 0)).unsqueeze(1);
    const Tensor buf = like(hidden, {step, v});
    const Tensor w32 = need_hidden ? weight.to(at::kFloat) : Tensor();
    Tensor gh, gw;
    if (need_hidden) gh = like(hidden, hidden.sizes());
    if (need_weight) gw = at::zeros(weight.sizes(), grad.options());
    for (int64_t s = 0; s < n; s += step) {
        const int64_t m = std::min(step, n - s);
        const Tensor d = buf.narrow(0, 0, m), f = by.narrow(0, s, m);
        product32(d, hidden.narrow(0, s, m), weight);
        check(sf_distill_grad(at_ptr<float>(buf), v, m, v, at_ptr<int32_t>(o.words) + s * k, at_ptr<uint8_t>(o.starts) + s * 2,
                              at_ptr<uint8_t>(o.status) + s, int(k), float(a.scale), at_ptr<float>(o.slopes) + s * k,
                              at_ptr<float>(o.stats) + s, n, at_ptr<float>(grad) + s, stream_of(hidden)),
              "sf_distill_grad");
        if (need_hidden) {
            Tensor to = gh.narrow(0, s, m);
            at::mm_out(to, d, w32);
            to.mul_(f).masked_fill_(f == 0, 0);
        }
        if (need_weight) {
            const Tensor h = hidden.narrow(0, s, m).to(at::kFloat).masked_fill(f == 0, 0) * f;
            at::addmm_out(gw, gw, d.t(), h);
        }
    }
    if (need_hidden) gh = gh.to(hidden.scalar_type());
    if (need_weight) gw = gw.to(weight.scalar_type());
    return {gh, gw};
}

// Both gradients from rows of D that are close.
std::pair<Tensor, Tensor> distill_backward_close(const Tensor& grad, const Tensor& hidden, const Tensor& weight,
                                                 const DistillOut& o, const DistillArgs& a, bool need_hidden,
                                                 bool need_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = hidden.size(0), h = hidden.size(1), v = weight.size(0), k = o.words.size(1);
    const int64_t row = o.keep.stride(0), pad = up(n, 64);
    const int type = type_of(hidden);
    const sf_stream_t st = stream_of(hidden);
    const int32_t *order = at_ptr<int32_t>(o.order), *live = order + n;
    const Tensor scalars = like(hidden, {n + 3});
    float *by = at_ptr<float>(scalars), *norm = by + n;
    const bool own = own_hidden_product(n, h, row);
    check(sf_distill_weight(at_ptr<float>(grad), at_ptr<float>(o.stats), at_ptr<uint8_t>(o.status), n, float(a.scale), type, by,
                            norm, st),
          "sf_distill_weight");
    check(sf_distill_keep_grad(o.keep.data_ptr(), row, n, pad, v, o.parts.data_ptr(), at_ptr<int32_t>(o.words),
                               at_ptr<uint8_t>(o.starts), at_ptr<uint8_t>(o.status), int(k), at_ptr<float>(o.slopes),
                               at_ptr<float>(o.stats), n, type, at_ptr<float>(grad), float(a.scale), norm, order,
                               need_hidden && !own ? n : 0, st),
          "sf_distill_keep_grad");
    Tensor gh, gw;
    if (need_hidden) {
        gh = at::empty({n, h}, hidden.options());
        // of the framework's own product as many as 1 GiB holds, of which the device takes what suits the rows
        const int64_t most = std::min<int64_t>({16, (v + 1999) / 2000, (int64_t(1) << 28) / (n * h)});
        const int64_t nparts = own ? std::max<int64_t>(most, 1) : a.nparts;
        Tensor parts = like(hidden, {nparts, n, h});
        const Tensor place = at::empty({n}, o.order.options());
        const int64_t part = own || nparts == 1 ? v : v / nparts / 8 * 8, done = own ? v : nparts * part;
        if (own) {
            check(sf_distill_hidden_product(o.keep.data_ptr(), row, n, live, weight.data_ptr(), weight.stride(0), v, h,
                                            int(nparts), at_ptr<float>(parts), type, st),
                  "sf_distill_hidden_product");
        } else if (nparts == 1) {
            Tensor whole = parts.select(0, 0);
            at::mm_out(whole, o.keep.as_strided({n, v}, {row, 1}), weight, at::kFloat);
        } else {
            at::bmm_out(parts, o.keep.as_strided({nparts, n, part}, {part, row, 1}),
                        weight.as_strided({nparts, part, h}, {part * h, h, 1}), at::kFloat);
        }
        check(sf_distill_sum(at_ptr<float>(parts), int(nparts), own, n, h, order, at_ptr<uint8_t>(o.status), at_ptr<int32_t>(place),
                             by, norm, o.keep.data_ptr(), row, weight.data_ptr(), weight.stride(0), done, v, type,
                             gh.data_ptr(), st),
              "sf_distill_sum");
    }
    if (need_weight) {
        gw = at::empty({v, h}, weight.options());
        const Tensor ht = at::empty({h, pad}, hidden.options());
        check(sf_distill_hidden(hidden.data_ptr(), hidden.stride(0), n, h, order, by, ht.data_ptr(), pad, st),
              "sf_distill_hidden");
        check(sf_distill_weight_grad(o.keep.data_ptr(), row, pad, live, v, ht.data_ptr(), h, norm + 2, type, gw.data_ptr(), st),
              "sf_distill_weight_grad");
    }
    return {gh, gw};
}

std::pair<Tensor, Tensor> distill_backward(const Tensor& grad, const Tensor& hidden, const Tensor& weight,
                                           const DistillOut& o, const DistillArgs& a, bool need_hidden, bool need_weight) {
    if (!in_tiles(hidden, weight)) return distill_backward_whole(grad, hidden, weight, o, a, need_hidden, need_weight);
    if (o.keep.defined() && o.order.defined())
        return distill_backward_close(grad, hidden, weight, o, a, need_hidden, need_weight);
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = hidden.size(0), v = weight.size(0), k = o.words.size(1), row = up(v, SF_LOGPS_SPAN);
    const bool kept = o.keep.defined();
    const int64_t step = kept ? n : std::min(n, a.step);
    const int type = type_of(hidden);
    Tensor parts = o.parts, again;   // products of the words, made again
    if (!kept) again = like(hidden, {step, k});
    return products(hidden, weight, o.keep, step, a.nparts, need_hidden, need_weight, true,
                    [&](int64_t s, int64_t m, int64_t pad, const Tensor& hc, const Tensor& d, float* by, float* norm) {
        if (!kept) parts = distill_tiles(hc, weight, o.words, o.starts, o.status, s, a.scale, d, again, a.masked, Tensor());
        if (s == 0)
            check(sf_distill_weight(at_ptr<float>(grad), at_ptr<float>(o.stats), at_ptr<uint8_t>(o.status), n, float(a.scale),
                                    type, by, norm, stream_of(hidden)),
                  "sf_distill_weight");
        check(sf_distill_keep_grad(d.data_ptr(), row, m, pad, v, parts.data_ptr(), at_ptr<int32_t>(o.words) + s * k,
                                   at_ptr<uint8_t>(o.starts) + s * o.starts.size(1), at_ptr<uint8_t>(o.status) + s, int(k),
                                   at_ptr<float>(o.slopes) + s * k, at_ptr<float>(o.stats) + s, n, type,
                                   at_ptr<float>(grad) + s, float(a.scale), norm, nullptr, 0, stream_of(hidden)),
              "sf_distill_keep_grad");
    });
}

// The gradients by torch operations, where what was saved came back as something else.
std::pair<Tensor, Tensor> distill_backward_torch(const Tensor& grad_, const Tensor& hidden, const Tensor& weight,
                                                 const DistillOut& o, const DistillArgs& a, bool need_hidden,
                                                 bool need_weight) {
    const Tensor grad = grad_.to(at::kFloat), w = weight.to(at::kFloat), stats = o.stats.to(at::kFloat);
    const Tensor taught = o.status.eq(1), bad = o.status.eq(2), counts = grad.ne(0).logical_and(o.status.ne(0));
    const Tensor h = at::where(counts.unsqueeze(1), hidden.to(at::kFloat), at::zeros({}, w.options()));
    const int64_t v = w.size(0), k = o.words.size(1);
    // a token's words: those before its last count; the others' slots go to a column behind
    const Tensor n = o.starts.select(1, o.starts.size(1) - 1).to(at::kLong).unsqueeze(1);
    const Tensor there = at::arange(k, n.options()).unsqueeze(0) < n;
    const Tensor at = at::where(there, o.words.to(at::kLong), at::full_like(n, v));
    const Tensor z = (at::matmul(h, w.t()) - stats.select(0, 1).unsqueeze(1)) * (a.scale / std::log(2.0));
    Tensor d = at::exp2(z - stats.select(0, 2).unsqueeze(1)) * stats.select(0, 3).unsqueeze(1);
    d = at::cat({d, at::zeros({d.size(0), 1}, d.options())}, 1);
    d = d.scatter(1, at, at::where(there, o.slopes.to(at::kFloat), at::zeros({}, d.options()))).narrow(1, 0, v);
    d = d * (grad * a.scale * stats.select(0, 0)).unsqueeze(1);
    d = at::where(counts.logical_and(taught).unsqueeze(1), d, at::zeros_like(d));
    d = at::where(counts.logical_and(bad).unsqueeze(1), at::full_like(d, NAN), d);
    Tensor gh, gw;
    if (need_hidden) gh = at::matmul(d, w).to(hidden.scalar_type());
    if (need_weight) gw = at::matmul(d.t(), h).to(weight.scalar_type());
    return {gh, gw};
}

struct LinearDistill : torch::autograd::Function<LinearDistill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& ids,
                          const Tensor& logps, const c10::optional<Tensor>& mask, const DistillArgs& a) {
        DistillOut o = distill_forward(hidden, weight, ids, logps, mask.has_value() ? *mask : Tensor(), a, true);
        ctx->save_for_backward({hidden, weight, o.words, o.starts, o.status, o.slopes, o.stats});
        ctx->set_materialize_grads(false);
        // not among the saved tensors: the backward overwrites it, and gives it up
        if (o.keep.defined()) {
            ctx->saved_data["keep"] = o.keep;
            ctx->saved_data["parts"] = o.parts;
            if (o.order.defined()) ctx->saved_data["order"] = o.order;
        }
        ctx->saved_data["scale"] = a.scale;
        ctx->saved_data["nparts"] = a.nparts;
        ctx->saved_data["step"] = a.step;
        ctx->saved_data["masked"] = a.masked;
        return o.loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& g = grads[0];
        if (!g.defined()) return variable_list(6);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &hidden = saved[0], &weight = saved[1];
        DistillOut o;
        o.words = saved[2], o.starts = saved[3], o.status = saved[4], o.slopes = saved[5], o.stats = saved[6];
        auto& data = ctx->saved_data;
        const DistillArgs a = {0, true, data["scale"].toDouble(), data["nparts"].toInt(), data["step"].toInt(), false,
                               data["masked"].toBool()};
        const bool need_hidden = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1);
        Tensor gh, gw;
        {
            at::NoGradGuard none;
            const c10::Device dev = g.device();
            const bool tiles = hidden.device() == dev && weight.device() == dev && in_tiles(hidden, weight);
            const int64_t spans = tiles ? (weight.size(0) + SF_LOGPS_SPAN - 1) / SF_LOGPS_SPAN : 1;
            if (dev.is_cuda() && memory_is_value(g) && hidden.device() == dev && weight.device() == dev &&
                memory_is_value(hidden) && memory_is_value(weight) && weight.scalar_type() == hidden.scalar_type() &&
                as_saved(o.words, at::kInt, dev) && as_saved(o.starts, at::kByte, dev) && o.starts.size(1) == spans + 1 &&
                as_saved(o.status, at::kByte, dev) && as_saved(o.slopes, at::kFloat, dev) &&
                as_saved(o.stats, at::kFloat, dev) && (!tiles || a.nparts == 1 || weight.is_contiguous())) {
                const c10::DeviceGuard guard(dev);
                if (auto it = data.find("keep"); it != data.end()) {
                    o.keep = it->second.toTensor();
                    o.parts = data["parts"].toTensor();
                    if (auto at = data.find("order"); at != data.end()) o.order = at->second.toTensor();
                    // a second backward of a retained graph makes it again
                    data.erase("keep");
                    data.erase("parts");
                    data.erase("order");
                }
                std::tie(gh, gw) = distill_backward(g.to(at::kFloat).contiguous(), hidden, weight, o, a, need_hidden,
                                                    need_weight);
            } else {
                std::tie(gh, gw) = distill_backward_torch(g, hidden, weight, o, a, need_hidden, need_weight);
            }
        }
        variable_list r = once(g, {gh, gw});
        return {r[0], r[1], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ---------------------------------------------------------------------------
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

// pref_loss(logps, ref, mask, form, beta, smoothing, average): (loss, chosen, rejected), or None
PyObject* pref_loss(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *l, *r, *m;
    int form, average;
    double beta, smoothing;
    if (!PyArg_ParseTuple(args, "OOOiddp", &l, &r, &m, &form, &beta, &smoothing, &average)) return nullptr;
    if (!plain(l) || !plain(r) || !plain(m)) Py_RETURN_NONE;
    const Tensor &logps = THPVariable_Unpack(l), &ref = THPVariable_Unpack(r);
    const c10::DeviceGuard guard(logps.device());
    const Tensor mask = rows(THPVariable_Unpack(m));
    const PrefArgs a = {form, beta, smoothing, average != 0};
    if (at::GradMode::is_enabled() && logps.requires_grad()) {
        const variable_list o = Preference::apply(logps, ref, mask, a);
        return Py_BuildValue("NNN", wrap(o[0]), wrap(o[1]), wrap(o[2]));
    }
    const PrefOut o = pref_forward(logps, ref, mask, a, false);
    return Py_BuildValue("NNN", wrap(o.loss), wrap(o.chosen), wrap(o.rejected));
    END_HANDLE_TH_ERRORS
}

// policy_loss(logps, old, advantages, mask, ref or None, log_low, log_high, kl_coef, sequences):
// (loss, kl or None, clipped), or None
PyObject* policy_loss(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *l, *o_, *ad, *m, *r;
    double low, high, kl;
    int sequences;
    if (!PyArg_ParseTuple(args, "OOOOOdddp", &l, &o_, &ad, &m, &r, &low, &high, &kl, &sequences)) return nullptr;
    if (!plain(l) || !plain(o_) || !plain(ad) || !plain(m) || (r != Py_None && !plain(r))) Py_RETURN_NONE;
    const Tensor& logps = THPVariable_Unpack(l);
    const Tensor &old = THPVariable_Unpack(o_), &adv = THPVariable_Unpack(ad), &mask = THPVariable_Unpack(m);
    const Tensor ref = r == Py_None ? Tensor() : THPVariable_Unpack(r);
    const c10::DeviceGuard guard(logps.device());
    const PolicyArgs a = {low, high, kl, sequences != 0};
    Tensor loss, kl_mean, clipped;
    if (at::GradMode::is_enabled() && logps.requires_grad()) {
        const c10::optional<Tensor> given = ref.defined() ? c10::optional<Tensor>(ref) : c10::nullopt;
        const variable_list o = PolicyNode::apply(logps, old, adv, mask, given, a);
        loss = o[0], clipped = o[1];
        if (o.size() > 2) kl_mean = o[2];
    } else {
        const PolicyOut o = policy_forward(logps, old, adv, mask, ref, a, false);
        loss = o.loss, clipped = o.clipped, kl_mean = o.kl;
    }
    PyObject* k = kl_mean.defined() ? wrap(kl_mean) : Py_NewRef(Py_None);
    return Py_BuildValue("NNN", wrap(loss), k, wrap(clipped));
    END_HANDLE_TH_ERRORS
}

// linear_logps(hidden, weight, labels, ignore_index, scale, nparts, step, keep): log-probabilities, or None
PyObject* linear_logps(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *h, *w, *y;
    long long ignore, nparts, step;
    double scale;
    int keep;
    if (!PyArg_ParseTuple(args, "OOOLdLLp", &h, &w, &y, &ignore, &scale, &nparts, &step, &keep)) return nullptr;
    if (!plain(h) || !plain(w) || !plain(y)) Py_RETURN_NONE;
    const Tensor &hidden = THPVariable_Unpack(h), &weight = THPVariable_Unpack(w), &labels = THPVariable_Unpack(y);
    if (hidden.numel() == 0 || !in_tiles(hidden, weight)) Py_RETURN_NONE;
    const c10::DeviceGuard guard(hidden.device());
    const bool grad = at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad());
    const LogpsArgs a = {ignore, scale, nparts, step, keep != 0 && grad};
    return wrap(grad ? LinearLogps::apply(hidden, weight, labels, a) : logps_forward(hidden, weight, labels, a).logp);
    END_HANDLE_TH_ERRORS
}

// linear_distill(hidden, weight, ids, logps, mask or None, form, rest, scale, nparts, step, keep): each token's
// loss, or None
PyObject* linear_distill(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *h, *w, *i, *l, *m;
    int form, rest, keep;
    double scale;
    long long nparts, step;
    if (!PyArg_ParseTuple(args, "OOOOOipdLLp", &h, &w, &i, &l, &m, &form, &rest, &scale, &nparts, &step, &keep)) return nullptr;
    if (!plain(h) || !plain(w) || !plain(i) || !plain(l) || (m != Py_None && !plain(m))) Py_RETURN_NONE;
    const Tensor &hidden = THPVariable_Unpack(h), &weight = THPVariable_Unpack(w);
    const Tensor &ids = THPVariable_Unpack(i), &logps = THPVariable_Unpack(l);
    if (hidden.numel() == 0) Py_RETURN_NONE;
    const c10::DeviceGuard guard(hidden.device());
    const Tensor mask = m == Py_None ? Tensor() : THPVariable_Unpack(m).contiguous();
    const bool grad = at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad());
    const DistillArgs a = {form, rest != 0, scale, nparts, step, keep != 0, mask.defined()};
    if (!grad) return wrap(distill_forward(hidden, weight, ids, logps, mask, a, false).loss);
    const c10::optional<Tensor> given = mask.defined() ? c10::optional<Tensor>(mask) : c10::nullopt;
    return wrap(LinearDistill::apply(hidden, weight, ids, logps, given, a));
    END_HANDLE_TH_ERRORS
}

// act8_pack(x, dtype, format, bytes): packed, or None
PyObject* act8_pack(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject* o;
    int dtype, format;
    long long bytes;
    if (!PyArg_ParseTuple(args, "OiiL", &o, &dtype, &format, &bytes)) return nullptr;
    if (!plain(o)) Py_RETURN_NONE;
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor& given = THPVariable_Unpack(o);
    const c10::DeviceGuard guard(given.device());
    const Tensor x = given.contiguous(), out = at::empty({bytes}, x.options().dtype(at::kByte));
    check(sf_act8_pack(x.data_ptr(), dtype, size_t(x.numel()), out.data_ptr(), format, stream_of(x)), "sf_act8_pack");
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// act8_unpack(packed, shape, dtype, format): the elements, or None.  shape: a
// tuple of sizes that packed holds.
PyObject* act8_unpack(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *p, *shape;
    int dtype, format;
    if (!PyArg_ParseTuple(args, "OO!ii", &p, &PyTuple_Type, &shape, &dtype, &format)) return nullptr;
    if (!plain(p)) Py_RETURN_NONE;
    c10::SmallVector<int64_t, 6> sizes;
    uint64_t n = 1;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) {
        const int64_t k = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
        if (k == -1 && PyErr_Occurred()) return nullptr;
        if (k <= 0 || n > (uint64_t(1) << 48) / uint64_t(k)) Py_RETURN_NONE;
        n *= uint64_t(k);
        sizes.push_back(k);
    }
    const Tensor& packed = THPVariable_Unpack(p);
    if (packed.scalar_type() != at::kByte || !packed.is_contiguous() ||
        reinterpret_cast<uintptr_t>(packed.data_ptr()) % 16 != 0 ||
        uint64_t(packed.numel()) != (n + SF_ACT8_BLOCK - 1) / SF_ACT8_BLOCK * SF_ACT8_BLOCK_BYTES)
        Py_RETURN_NONE;
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(packed.device());
    const auto type = dtype == SF_DTYPE_F32 ? at::kFloat : dtype == SF_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
    const Tensor out = at::empty(sizes, packed.options().dtype(type));
    check(sf_act8_unpack(packed.data_ptr(), format, size_t(n), out.data_ptr(), dtype, stream_of(packed)),
          "sf_act8_unpack");
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// Rows of logits [.., vocab] as the kernels read them.
Tensor as_rows(const Tensor& t) { return rows(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }
Tensor rows_work(const Tensor& logits) {
    const size_t bytes = sf_rows_work(logits.size(0), logits.size(1), logits_type(logits));
    return at::empty({int64_t(bytes)}, logits.options().dtype(at::kByte));
}

// top_logps(logits, k, temperature): (logps, ids), or None
PyObject* top_logps(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject* o;
    int k;
    double temperature;
    if (!PyArg_ParseTuple(args, "Oid", &o, &k, &temperature)) return nullptr;
    if (!plain(o)) Py_RETURN_NONE;
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor& given = THPVariable_Unpack(o);
    if (given.size(-1) > (int64_t(1) << 30) || given.numel() / given.size(-1) >= (int64_t(1) << 31)) Py_RETURN_NONE;
    const c10::DeviceGuard guard(given.device());
    const Tensor x = as_rows(given), work = rows_work(x);
    c10::SmallVector<int64_t, 6> shape(given.sizes().begin(), given.sizes().end());
    shape.back() = k;
    const Tensor logps = like(x, shape), ids = at::empty(shape, x.options().dtype(at::kLong));
    check(sf_top_logps(x.data_ptr(), logits_type(x), ld(x), x.size(0), x.size(1), k, temperature, work.data_ptr(),
                       at_ptr<float>(logps), at_ptr<int64_t>(ids), stream_of(x)),
          "sf_top_logps");
    return Py_BuildValue("NN", wrap(logps), wrap(ids));
    END_HANDLE_TH_ERRORS
}

// sample_tokens(logits, uniforms, temperature, temperatures or None, top_k, top_ks or None, top_p, top_ps or None,
// min_p, min_ps or None): (ids, logps), or None
PyObject* sample_tokens(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *l, *u, *own[4];
    double t, p, m;
    long long k;
    if (!PyArg_ParseTuple(args, "OOdOLOdOdO", &l, &u, &t, &own[0], &k, &own[1], &p, &own[2], &m, &own[3])) return nullptr;
    if (!plain(l) || !plain(u)) Py_RETURN_NONE;
    for (PyObject* o : own)
        if (o != Py_None && !plain(o)) Py_RETURN_NONE;
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor& given = THPVariable_Unpack(l);
    if (given.size(-1) > (int64_t(1) << 30) || given.numel() / given.size(-1) >= (int64_t(1) << 31)) Py_RETURN_NONE;
    const c10::DeviceGuard guard(given.device());
    const Tensor x = as_rows(given), uniforms = THPVariable_Unpack(u).contiguous(), work = rows_work(x);
    Tensor each[4];
    for (int i = 0; i < 4; ++i)
        if (own[i] != Py_None) each[i] = THPVariable_Unpack(own[i]).contiguous();
    const Tensor ids = at::empty(uniforms.sizes(), x.options().dtype(at::kLong)), logps = like(x, uniforms.sizes());
    check(sf_sample_tokens(x.data_ptr(), logits_type(x), ld(x), x.size(0), x.size(1), at_ptr<float>(uniforms), t,
                           at_ptr<float>(each[0]), k, at_ptr<int64_t>(each[1]), p, at_ptr<float>(each[2]), m,
                           at_ptr<float>(each[3]), work.data_ptr(), at_ptr<int64_t>(ids), at_ptr<float>(logps),
                           stream_of(x)),
          "sf_sample_tokens");
    return Py_BuildValue("NN", wrap(ids), wrap(logps));
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"pref_loss", pref_loss, METH_VARARGS, "(loss, chosen, rejected), or None."},
    {"policy_loss", policy_loss, METH_VARARGS, "(loss, kl, clipped), or None."},
    {"linear_logps", linear_logps, METH_VARARGS, "Log-probabilities, or None."},
    {"linear_distill", linear_distill, METH_VARARGS, "Each token's loss, or None."},
    {"act8_pack", act8_pack, METH_VARARGS, "Packed elements, or None."},
    {"act8_unpack", act8_unpack, METH_VARARGS, "Restored elements, or None."},
    {"top_logps", top_logps, METH_VARARGS, "(logps, ids), or None."},
    {"sample_tokens", sample_tokens, METH_VARARGS, "(ids, logps), or None."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sf_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sf_ops(void) {
    PyObject* m = PyModule_Create(&module);
    // the tensors' layout and the nodes are this torch's alone
    if (m != nullptr && PyModule_AddStringConstant(m, "TORCH_VERSION", SF_TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}

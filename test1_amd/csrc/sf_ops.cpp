// The calls and the autograd nodes of the losses over token log-probabilities,
// of the log-probabilities themselves and of the 8-bit checkpoints, as a
// CPython module over the C ABI.
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
                    const Tensor& norm, const Tensor& out) {
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
                       w + 2 * done * h, v - done, row_weight, at_ptr<float>(norm), stream_of(keep)),
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

// Both gradients (undefined where not needed).  What was kept turns into the
// gradient of the logits in place; without it, it is made again, `step` rows at
// a time.
std::pair<Tensor, Tensor> logps_backward(const Tensor& grad, const Tensor& hidden, const Tensor& weight,
                                         const Tensor& labels, const Tensor& logp, const Tensor& lse2, Tensor keep,
                                         Tensor parts, const LogpsArgs& a, bool need_hidden, bool need_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = hidden.size(0), h = hidden.size(1), v = weight.size(0), row = up(v, SF_LOGPS_SPAN);
    const bool kept = keep.defined(), fp16 = hidden.scalar_type() == at::kHalf;
    const int64_t step = kept ? n : std::min(n, a.step);
    const bool one = step == n;
    const sf_stream_t st = stream_of(hidden);
    const int type = type_of(hidden);
    const int64_t* y = at_ptr<int64_t>(labels);
    const float *lp = at_ptr<float>(logp), *l2 = at_ptr<float>(lse2);
    const Tensor by = like(hidden, {n}), norm = like(hidden, {2});
    const bool own = one && own_weight_grad(n, h, v, row, fp16);
    Tensor gh, gw, again;
    if (need_hidden) gh = at::empty({n, h}, hidden.options());
    if (need_weight) gw = at::empty({v, h}, own || (one && !fp16) ? weight.options() : weight.options().dtype(at::kFloat));
    if (!kept) {
        keep = at::empty({up(step, 64), row}, hidden.options());
        again = like(hidden, {2, step});
    }
    for (int64_t s = 0; s < n; s += step) {
        const int64_t m = std::min(n - s, step), pad = up(m, 64);
        const Tensor hc = one ? hidden : hidden.narrow(0, s, m);
        if (!kept) {
            float* results = at_ptr<float>(again);
            parts = tiles(hc, weight, y + s, a, keep, results, results + step);
        }
        check(sf_logps_keep_grad(keep.data_ptr(), row, m, pad, v, parts.data_ptr(), y + s, a.ignore_index, l2 + s, lp + s,
                                 type, at_ptr<float>(grad) + s, s == 0 ? n : 0, float(a.scale), at_ptr<float>(by),
                                 at_ptr<float>(norm), fp16, st),
              "sf_logps_keep_grad");
        if (need_hidden && one && own_hidden_grad(n, h, v))
            check(sf_logps_hidden_grad(keep.data_ptr(), row, n, weight.data_ptr(), weight.stride(0), v, h,
                                       at_ptr<float>(by), fp16 ? at_ptr<float>(norm) : nullptr, type, gh.data_ptr(), st),
                  "sf_logps_hidden_grad");
        else if (need_hidden)
            hidden_product(keep, m, weight, a.nparts, at_ptr<float>(by) + s, fp16 ? norm : Tensor(),
                           one ? gh : gh.narrow(0, s, m));
        if (!need_weight) continue;
        if (fp16 && !own) {
            // into fp32, of rows as they lie: 4096 x 4096 x 128256 4.2 ms, of transposed ones 28.8
            const Tensor weighted = at::empty({m, h}, hidden.options());
            check(sf_logps_weighted(hc.data_ptr(), hc.stride(0), m, h, at_ptr<float>(by) + s, type, weighted.data_ptr(), st),
                  "sf_logps_weighted");
            const Tensor dt = keep.as_strided({v, m}, {1, row});
            if (s == 0) at::mm_out(gw, dt, weighted, at::kFloat);
            else at::addmm_out(gw, gw, dt, weighted, at::kFloat);
            continue;
        }
        // transposed: of bf16 the product with an operand laid out along the sum is
        // faster, 3.3 ms there instead of 4.0
        const Tensor ht = at::empty({h, pad}, hidden.options());
        check(sf_logps_hidden(hc.data_ptr(), hc.stride(0), m, h, at_ptr<float>(by) + s, type, ht.data_ptr(), pad, st),
              "sf_logps_hidden");
        if (own) {
            check(sf_logps_weight_grad(keep.data_ptr(), row, pad, v, ht.data_ptr(), h, fp16 ? at_ptr<float>(norm) : nullptr,
                                       type, gw.data_ptr(), st),
                  "sf_logps_weight_grad");
            break;
        }
        const Tensor dt = keep.as_strided({v, pad}, {1, row}), hp = ht.t();
        if (one) at::mm_out(gw, dt, hp);
        else if (s == 0) at::mm_out(gw, dt, hp, at::kFloat);
        else at::addmm_out(gw, gw, dt, hp, at::kFloat);
    }
    if (need_weight && gw.scalar_type() != weight.scalar_type()) {
        // fp16's factor leaves before the rounding
        if (fp16) {
            const Tensor out = at::empty({v, h}, weight.options());
            check(sf_ce_scale(at_ptr<float>(norm), at_ptr<float>(norm) + 1, nullptr, nullptr, 0, at_ptr<float>(gw),
                              out.data_ptr(), size_t(v * h), type, st),
                  "sf_ce_scale");
            gw = out;
        } else {
            gw = gw.to(weight.scalar_type());
        }
    }
    return {gh, gw};
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

PyMethodDef methods[] = {
    {"pref_loss", pref_loss, METH_VARARGS, "(loss, chosen, rejected), or None."},
    {"policy_loss", policy_loss, METH_VARARGS, "(loss, kl, clipped), or None."},
    {"linear_logps", linear_logps, METH_VARARGS, "Log-probabilities, or None."},
    {"act8_pack", act8_pack, METH_VARARGS, "Packed elements, or None."},
    {"act8_unpack", act8_unpack, METH_VARARGS, "Restored elements, or None."},
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

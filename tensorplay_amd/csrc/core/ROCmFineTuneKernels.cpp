// ROCm backend of the fine-tuning operators (FineTune.h): shape, dtype and device
// checks, then one call of the C-ABI launch layer (include/tpr_rocm.h) each.
#include "FineTune.h"

#include <cstring>
#include <string>

#include "Allocator.h"
#include "Dispatcher.h"
#include "Exception.h"
#include "tpr_rocm.h"

namespace tensorplay {
namespace rocm {
namespace {

void check(int rc, const char* op) {
    if (rc == TPR_OK) return;
    const std::string msg = std::string(op) + ": " + tpr_last_error();
    if (rc == TPR_ERR_UNSUPPORTED_DTYPE || rc == TPR_ERR_NOT_IMPLEMENTED) TP_THROW(NotImplementedError, msg);
    if (rc == TPR_ERR_INVALID_ARG) TP_THROW(ValueError, msg);
    TP_THROW(RuntimeError, msg);
}

bool is_elem(DType t) { return t == DType::Float32 || t == DType::Float16 || t == DType::BFloat16; }

const Tensor* opt(const OptTensor& t) { return t && t->defined() ? &*t : nullptr; }

void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

// An argument beside `self`: on its device, of this dtype and number of elements; dense.
Tensor arg(const Tensor& t, const Tensor& self, DType dtype, int64_t numel, const char* op, const char* name) {
    if (t.device() != self.device())
        TP_THROW(RuntimeError, std::string(op) + ": " + name + " is on another device than the input");
    if (t.dtype() != dtype)
        TP_THROW(NotImplementedError, std::string(op) + ": " + name + " must be " + toString(dtype));
    if (t.numel() != numel)
        TP_THROW(RuntimeError, std::string(op) + ": " + name + " has " + std::to_string(t.numel()) + " elements, " +
                                   std::to_string(numel) + " expected");
    return t.contiguous();
}

OptTensor opt_arg(const OptTensor& t, const Tensor& self, DType dtype, int64_t numel, const char* op, const char* name) {
    if (!opt(t)) return std::nullopt;
    return arg(*t, self, dtype, numel, op, name);
}

struct Workspace {
    std::shared_ptr<void> mem;
    size_t bytes;
    Workspace(size_t n, const Device& d) : bytes(n) {
        if (n) mem = allocate(n, d);
    }
};

// Logits as rows at one stride (made dense where their leading dims have several), and
// their targets.
struct Logits {
    Tensor x, target;
    tpr_logits_desc d;
    int64_t rows() const { return d.rows; }
};

Logits logits(const Tensor& self, const Tensor& target, double temperature, int64_t ignore_index, const char* op) {
    if (!is_elem(self.dtype()))
        TP_THROW(NotImplementedError, std::string(op) + " not implemented for dtype " + toString(self.dtype()) +
                                          " on ROCm (float32 / float16 / bfloat16)");
    if (self.dim() == 0) TP_THROW(RuntimeError, std::string(op) + ": logits need at least one dim");
    const int64_t nd = self.dim(), vocab = self.shape()[nd - 1];
    if (std::vector<int64_t>(self.shape().begin(), self.shape().end() - 1) != target.shape())
        TP_THROW(RuntimeError, std::string(op) + ": target must have the logits' shape without the last dim");
    Logits l;
    std::memset(&l.d, 0, sizeof l.d);
    l.d.rows = target.numel();
    l.target = arg(target, self, DType::Int64, l.d.rows, op, "target");
    // one stride for the leading dims?
    int64_t size = 1, stride = vocab;
    bool ok = vocab <= 1 || self.strides()[nd - 1] == 1, first = true;
    for (int64_t i = nd - 2; i >= 0 && ok; --i) {
        if (self.shape()[i] == 1) continue;
        if (first) stride = self.strides()[i];
        else ok = self.strides()[i] == stride * size;
        first = false;
        size *= self.shape()[i];
    }
    if (ok && stride < 0) ok = false;
    l.x = ok ? self : self.contiguous();
    l.d.dtype = (int32_t)self.dtype();
    l.d.vocab = vocab;
    l.d.row_stride = ok ? stride : vocab;
    l.d.ignore_index = ignore_index;
    l.d.temperature = temperature;
    return l;
}

std::vector<int64_t> with_pair(std::vector<int64_t> s) {
    s.push_back(2);
    return s;
}

// coef * scale * d logp / d logits; scale a one-element tensor or null
Tensor logits_grad(const Tensor& coef, const Tensor* scale, const Tensor& self, const Tensor& target, const Tensor& lse,
                   double temperature, int64_t ignore_index, const char* op, const char* coef_name) {
    const Logits l = logits(self, target, temperature, ignore_index, op);
    const Tensor c = arg(coef, self, DType::Float32, l.rows(), op, coef_name);
    const Tensor s = arg(lse, self, DType::Float32, 2 * l.rows(), op, "lse");
    Tensor g;
    if (scale) g = arg(*scale, self, DType::Float32, 1, op, "grad");
    Tensor out = Tensor::empty(self.shape(), self.dtype(), self.device());
    DeviceGuard guard(self.device());
    check(tpr_token_logprob_backward(&l.d, static_cast<const float*>(c.data_ptr()),
                                     scale ? static_cast<const float*>(g.data_ptr()) : nullptr, l.x.data_ptr(),
                                     static_cast<const int64_t*>(l.target.data_ptr()),
                                     static_cast<const float*>(s.data_ptr()), out.data_ptr(),
                                     currentStream(self.device().index)),
          op);
    return out;
}

struct PolicyOut {
    Tensor loss, logp, lse, coef, grad;
};

PolicyOut policy(const Tensor& self, const Tensor& target, const Tensor& old_logp, const Tensor& advantage,
                 const OptTensor& ref_logp, const OptTensor& weight, double clip_low, double clip_high, double kl_coef,
                 double temperature, int64_t ignore_index, bool with_grad, const char* op) {
    const Logits l = logits(self, target, temperature, ignore_index, op);
    const int64_t n = l.rows();
    const Tensor old = arg(old_logp, self, DType::Float32, n, op, "old_logp");
    const Tensor adv = arg(advantage, self, DType::Float32, n, op, "advantage");
    const OptTensor ref = opt_arg(ref_logp, self, DType::Float32, n, op, "ref_logp");
    const OptTensor w = opt_arg(weight, self, DType::Float32, n, op, "weight");
    PolicyOut o;
    const Device dev = self.device();
    o.loss = Tensor::empty({}, DType::Float32, dev);
    o.logp = Tensor::empty(target.shape(), DType::Float32, dev);
    if (with_grad) {
        o.grad = Tensor::empty(self.shape(), self.dtype(), dev);
    } else {
        o.lse = Tensor::empty(with_pair(target.shape()), DType::Float32, dev);
        o.coef = Tensor::empty(target.shape(), DType::Float32, dev);
    }
    const tpr_policy_desc p{clip_low, clip_high, kl_coef};
    const Workspace ws(tpr_policy_loss_workspace_bytes(&l.d), dev);
    DeviceGuard guard(dev);
    auto f = [](const Tensor* t) { return static_cast<float*>(ptr(t)); };
    check(tpr_policy_loss(&l.d, &p, l.x.data_ptr(), static_cast<const int64_t*>(l.target.data_ptr()), f(&old), f(&adv),
                          f(opt(ref)), f(opt(w)), f(&o.loss), f(&o.logp), with_grad ? nullptr : f(&o.lse),
                          with_grad ? nullptr : f(&o.coef), with_grad ? o.grad.data_ptr() : nullptr, ws.mem.get(),
                          ws.bytes, currentStream(dev.index)),
          op);
    return o;
}

Tensor run_dropout(const Tensor& self, double p, int64_t seed, int64_t offset, const char* op) {
    if (!is_elem(self.dtype()))
        TP_THROW(NotImplementedError, std::string(op) + " not implemented for dtype " + toString(self.dtype()) +
                                          " on ROCm (float32 / float16 / bfloat16)");
    const Tensor x = self.contiguous();
    const int64_t cols = self.dim() ? self.shape()[self.dim() - 1] : 1;
    Tensor out = Tensor::empty(self.shape(), self.dtype(), self.device());
    DeviceGuard guard(self.device());
    check(tpr_dropout(x.data_ptr(), (int32_t)self.dtype(), cols ? self.numel() / cols : 0, cols, p, seed, offset,
                      out.data_ptr(), currentStream(self.device().index)),
          op);
    return out;
}

// Rows of a tensor, also where they have no columns
int64_t leading(const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.shape()[i];
    return n;
}

// What both passes of the end of a block share: descriptor and checked weights.
struct Block {
    tpr_gated_norm_desc d;
    Tensor pre;
    OptTensor post, gate;
};

Block block(const Tensor& self, DType residual, const Tensor& pre_weight, double eps, const OptTensor& post_weight,
            const OptTensor& gate, double scale, double p, int64_t seed, int64_t offset, const char* op) {
    if (!is_elem(self.dtype()))
        TP_THROW(NotImplementedError, std::string(op) + " not implemented for dtype " + toString(self.dtype()) +
                                          " on ROCm (float32 / float16 / bfloat16)");
    if (self.dim() == 0) TP_THROW(RuntimeError, std::string(op) + ": the input needs at least one dim");
    if (residual != self.dtype() && residual != DType::Float32)
        TP_THROW(NotImplementedError, std::string(op) + ": the residual must be of the input's dtype or float32");
    Block b;
    std::memset(&b.d, 0, sizeof b.d);
    b.d.cols = self.shape()[self.dim() - 1];
    b.d.rows = leading(self);
    b.d.dtype = (int32_t)self.dtype();
    b.d.residual_dtype = (int32_t)residual;
    b.d.eps = eps;
    b.d.residual_scale = scale;
    b.d.p = p;
    b.d.seed = seed;
    b.d.offset = offset;
    b.pre = arg(pre_weight, self, self.dtype(), b.d.cols, op, "pre_weight");
    b.post = opt_arg(post_weight, self, self.dtype(), b.d.cols, op, "post_weight");
    if (const Tensor* g = opt(gate)) {
        if (g->dim() == 0 || g->shape()[g->dim() - 1] != b.d.cols)
            TP_THROW(RuntimeError, std::string(op) + ": gate's last dim must be the input's");
        b.d.gates = leading(*g);
        if (b.d.rows > 0 && b.d.gates == 0)   // the descriptor's "no gate"
            TP_THROW(ValueError, std::string(op) + ": gates must divide the rows, and there are none");
        b.gate = arg(*g, self, self.dtype(), b.d.gates * b.d.cols, op, "gate");
    }
    return b;
}

}  // namespace

std::tuple<Tensor, Tensor> token_logprob_kernel(const Tensor& self, const Tensor& target, double temperature,
                                                int64_t ignore_index) {
    const char* op = "token_logprob";
    const Logits l = logits(self, target, temperature, ignore_index, op);
    const Device dev = self.device();
    Tensor logp = Tensor::empty(target.shape(), DType::Float32, dev);
    Tensor lse = Tensor::empty(with_pair(target.shape()), DType::Float32, dev);
    const Workspace ws(tpr_token_logprob_workspace_bytes(&l.d), dev);
    DeviceGuard guard(dev);
    check(tpr_token_logprob(&l.d, l.x.data_ptr(), static_cast<const int64_t*>(l.target.data_ptr()),
                            static_cast<float*>(logp.data_ptr()), static_cast<float*>(lse.data_ptr()), ws.mem.get(),
                            ws.bytes, currentStream(dev.index)),
          op);
    return {logp, lse};
}

Tensor token_logprob_backward_kernel(const Tensor& grad, const Tensor& self, const Tensor& target, const Tensor& lse,
                                     double temperature, int64_t ignore_index) {
    return logits_grad(grad, nullptr, self, target, lse, temperature, ignore_index, "token_logprob_backward", "grad");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss_kernel(const Tensor& self, const Tensor& target,
                                                              const Tensor& old_logp, const Tensor& advantage,
                                                              OptTensor ref_logp, OptTensor weight, double clip_low,
                                                              double clip_high, double kl_coef, double temperature,
                                                              int64_t ignore_index) {
    const PolicyOut o = policy(self, target, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef,
                               temperature, ignore_index, false, "policy_loss");
    return {o.loss, o.logp, o.lse, o.coef};
}

std::tuple<Tensor, Tensor, Tensor> policy_loss_and_grad_kernel(const Tensor& self, const Tensor& target,
                                                               const Tensor& old_logp, const Tensor& advantage,
                                                               OptTensor ref_logp, OptTensor weight, double clip_low,
                                                               double clip_high, double kl_coef, double temperature,
                                                               int64_t ignore_index) {
    const PolicyOut o = policy(self, target, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef,
                               temperature, ignore_index, true, "policy_loss_and_grad");
    return {o.loss, o.logp, o.grad};
}

Tensor policy_loss_backward_kernel(const Tensor& grad, const Tensor& coef, const Tensor& self, const Tensor& target,
                                   const Tensor& lse, double temperature, int64_t ignore_index) {
    return logits_grad(coef, &grad, self, target, lse, temperature, ignore_index, "policy_loss_backward", "coef");
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> preference_loss_kernel(const Tensor& self, const Tensor& target,
                                                                          const Tensor& offsets, const Tensor& ref_logp,
                                                                          double beta, double label_smoothing,
                                                                          int64_t ignore_index) {
    const char* op = "preference_loss";
    if (self.dim() != 2) TP_THROW(RuntimeError, "preference_loss: logits must be 2-D [tokens, vocab]");
    const Logits l = logits(self, target, 1.0, ignore_index, op);
    if (offsets.dim() != 1 || offsets.numel() < 3 || offsets.numel() % 2 == 0)
        TP_THROW(RuntimeError, "preference_loss: offsets must be [2 pairs + 1] of one pair or more");
    const int64_t seqs = offsets.numel() - 1;
    const Tensor off = arg(offsets, self, DType::Int64, seqs + 1, op, "offsets");
    const Tensor ref = arg(ref_logp, self, DType::Float32, seqs, op, "ref_logp");
    const Device dev = self.device();
    Tensor loss = Tensor::empty({}, DType::Float32, dev);
    Tensor reward = Tensor::empty({seqs}, DType::Float32, dev);
    Tensor logp = Tensor::empty(target.shape(), DType::Float32, dev);
    Tensor lse = Tensor::empty(with_pair(target.shape()), DType::Float32, dev);
    Tensor coef = Tensor::empty(target.shape(), DType::Float32, dev);
    const Workspace ws(tpr_preference_loss_workspace_bytes(&l.d, seqs / 2), dev);
    DeviceGuard guard(dev);
    auto f = [](const Tensor& t) { return static_cast<float*>(t.data_ptr()); };
    check(tpr_preference_loss(&l.d, seqs / 2, beta, label_smoothing, l.x.data_ptr(),
                              static_cast<const int64_t*>(l.target.data_ptr()),
                              static_cast<const int64_t*>(off.data_ptr()), f(ref), f(loss), f(reward), f(logp), f(lse),
                              f(coef), ws.mem.get(), ws.bytes, currentStream(dev.index)),
          op);
    return {loss, reward, logp, lse, coef};
}

Tensor preference_loss_backward_kernel(const Tensor& grad, const Tensor& coef, const Tensor& self, const Tensor& target,
                                       const Tensor& lse, int64_t ignore_index) {
    return logits_grad(coef, &grad, self, target, lse, 1.0, ignore_index, "preference_loss_backward", "coef");
}

Tensor dropout_kernel(const Tensor& self, double p, int64_t seed, int64_t offset) {
    return run_dropout(self, p, seed, offset, "dropout");
}
Tensor dropout_backward_kernel(const Tensor& grad, double p, int64_t seed, int64_t offset) {
    return run_dropout(grad, p, seed, offset, "dropout_backward");
}

std::tuple<Tensor, Tensor, OptTensor, Tensor> gated_residual_norm_kernel(const Tensor& self, const Tensor& residual,
                                                                         const Tensor& pre_weight, double eps,
                                                                         OptTensor post_weight, OptTensor gate,
                                                                         double residual_scale, double p, int64_t seed,
                                                                         int64_t offset) {
    const char* op = "gated_residual_norm";
    const Block b = block(self, residual.dtype(), pre_weight, eps, post_weight, gate, residual_scale, p, seed, offset, op);
    if (residual.shape() != self.shape()) TP_THROW(RuntimeError, "gated_residual_norm: residual must have the input's shape");
    const Tensor x = self.contiguous();
    const Tensor h = arg(residual, self, residual.dtype(), self.numel(), op, "residual");
    const Device dev = self.device();
    Tensor out = Tensor::empty(self.shape(), residual.dtype(), dev);
    Tensor y = Tensor::empty(self.shape(), self.dtype(), dev);
    const std::vector<int64_t> rows(self.shape().begin(), self.shape().end() - 1);
    Tensor rpre = Tensor::empty(rows, DType::Float32, dev);
    OptTensor rpost;
    if (opt(b.post)) rpost = Tensor::empty(rows, DType::Float32, dev);
    DeviceGuard guard(dev);
    check(tpr_gated_norm(&b.d, x.data_ptr(), h.data_ptr(), b.pre.data_ptr(), ptr(opt(b.post)), ptr(opt(b.gate)),
                         out.data_ptr(), y.data_ptr(), static_cast<float*>(ptr(opt(rpost))),
                         static_cast<float*>(rpre.data_ptr()), currentStream(dev.index)),
          op);
    return {out, y, rpost, rpre};
}

std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> gated_residual_norm_backward_kernel(
    const Tensor& grad_y, OptTensor grad_residual, const Tensor& self, const Tensor& out, OptTensor rstd_post,
    const Tensor& rstd_pre, const Tensor& pre_weight, OptTensor post_weight, OptTensor gate, double residual_scale,
    double p, int64_t seed, int64_t offset) {
    const char* op = "gated_residual_norm_backward";
    const Block b = block(self, out.dtype(), pre_weight, 0.0, post_weight, gate, residual_scale, p, seed, offset, op);
    if (out.shape() != self.shape() || grad_y.shape() != self.shape() ||
        (opt(grad_residual) && grad_residual->shape() != self.shape()))
        TP_THROW(RuntimeError, "gated_residual_norm_backward: out and the gradients must have the input's shape");
    if (opt(post_weight) && !opt(rstd_post))
        TP_THROW(RuntimeError, "gated_residual_norm_backward: post_weight needs rstd_post");
    const int64_t n = self.numel();
    const Tensor x = self.contiguous();
    const Tensor gy = arg(grad_y, self, self.dtype(), n, op, "grad_y");
    const OptTensor go = opt_arg(grad_residual, self, out.dtype(), n, op, "grad_residual");
    const Tensor o = arg(out, self, out.dtype(), n, op, "out");
    const OptTensor rpost = opt_arg(opt(post_weight) ? rstd_post : std::nullopt, self, DType::Float32, b.d.rows, op,
                                    "rstd_post");
    const Tensor rpre = arg(rstd_pre, self, DType::Float32, b.d.rows, op, "rstd_pre");
    const Device dev = self.device();
    Tensor gx = Tensor::empty(self.shape(), self.dtype(), dev);
    Tensor gh = Tensor::empty(self.shape(), out.dtype(), dev);
    Tensor gpre = Tensor::empty(b.pre.shape(), self.dtype(), dev);
    OptTensor gpost, ggate;
    if (opt(b.post)) gpost = Tensor::empty(b.post->shape(), self.dtype(), dev);
    if (opt(b.gate)) ggate = Tensor::empty(b.gate->shape(), self.dtype(), dev);
    const Workspace ws(tpr_gated_norm_backward_workspace_bytes(&b.d), dev);
    DeviceGuard guard(dev);
    check(tpr_gated_norm_backward(&b.d, gy.data_ptr(), ptr(opt(go)), x.data_ptr(), o.data_ptr(),
                                  static_cast<const float*>(ptr(opt(rpost))), static_cast<const float*>(rpre.data_ptr()),
                                  b.pre.data_ptr(), ptr(opt(b.post)), ptr(opt(b.gate)), gx.data_ptr(), gh.data_ptr(),
                                  gpre.data_ptr(), ptr(opt(gpost)), ptr(opt(ggate)), ws.mem.get(), ws.bytes,
                                  currentStream(dev.index)),
          op);
    return {gx, gh, gpre, gpost, ggate};
}

}  // namespace rocm

// ---- dispatch: each function calls the kernel registered under its name ----------
#define TP_FINETUNE_OPS(X)                                                                                       \
    X(token_logprob) X(token_logprob_backward) X(policy_loss) X(policy_loss_and_grad) X(policy_loss_backward)    \
    X(preference_loss) X(preference_loss_backward) X(dropout) X(dropout_backward) X(gated_residual_norm)         \
    X(gated_residual_norm_backward)

TENSORPLAY_LIBRARY_IMPL(ROCm, FineTuneKernels) {
#define TP_FINETUNE_IMPL(name) m.impl<decltype(rocm::name##_kernel)>("finetune::" #name, rocm::name##_kernel);
    TP_FINETUNE_OPS(TP_FINETUNE_IMPL)
#undef TP_FINETUNE_IMPL
}

namespace {
// The stub's argument types are those of the public function, and the kernel's own.
template <typename Sig>
struct Stub;
template <typename R, typename... A>
struct Stub<R(A...)> {
    template <typename... B>
    static R call(const char* name, const Tensor& on, B&&... a) {
        return DispatchStub<R, A...>::call(name, computeDispatchKey(on.device()), std::forward<B>(a)...);
    }
};
#define TP_FINETUNE_CHECK(name) \
    static_assert(std::is_same<decltype(tensorplay::name), decltype(rocm::name##_kernel)>::value, #name);
TP_FINETUNE_OPS(TP_FINETUNE_CHECK)
#undef TP_FINETUNE_CHECK
}  // namespace

std::tuple<Tensor, Tensor> token_logprob(const Tensor& self, const Tensor& target, double temperature,
                                         int64_t ignore_index) {
    return Stub<decltype(token_logprob)>::call("finetune::token_logprob", self, self, target, temperature, ignore_index);
}
Tensor token_logprob_backward(const Tensor& grad, const Tensor& self, const Tensor& target, const Tensor& lse,
                              double temperature, int64_t ignore_index) {
    return Stub<decltype(token_logprob_backward)>::call("finetune::token_logprob_backward", self, grad, self, target,
                                                        lse, temperature, ignore_index);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss(const Tensor& self, const Tensor& target, const Tensor& old_logp,
                                                       const Tensor& advantage, OptTensor ref_logp, OptTensor weight,
                                                       double clip_low, double clip_high, double kl_coef,
                                                       double temperature, int64_t ignore_index) {
    return Stub<decltype(policy_loss)>::call("finetune::policy_loss", self, self, target, old_logp, advantage,
                                             std::move(ref_logp), std::move(weight), clip_low, clip_high, kl_coef,
                                             temperature, ignore_index);
}
std::tuple<Tensor, Tensor, Tensor> policy_loss_and_grad(const Tensor& self, const Tensor& target,
                                                        const Tensor& old_logp, const Tensor& advantage,
                                                        OptTensor ref_logp, OptTensor weight, double clip_low,
                                                        double clip_high, double kl_coef, double temperature,
                                                        int64_t ignore_index) {
    return Stub<decltype(policy_loss_and_grad)>::call("finetune::policy_loss_and_grad", self, self, target, old_logp,
                                                      advantage, std::move(ref_logp), std::move(weight), clip_low,
                                                      clip_high, kl_coef, temperature, ignore_index);
}
Tensor policy_loss_backward(const Tensor& grad, const Tensor& coef, const Tensor& self, const Tensor& target,
                            const Tensor& lse, double temperature, int64_t ignore_index) {
    return Stub<decltype(policy_loss_backward)>::call("finetune::policy_loss_backward", self, grad, coef, self, target,
                                                      lse, temperature, ignore_index);
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> preference_loss(const Tensor& self, const Tensor& target,
                                                                   const Tensor& offsets, const Tensor& ref_logp,
                                                                   double beta, double label_smoothing,
                                                                   int64_t ignore_index) {
    return Stub<decltype(preference_loss)>::call("finetune::preference_loss", self, self, target, offsets, ref_logp,
                                                 beta, label_smoothing, ignore_index);
}
Tensor preference_loss_backward(const Tensor& grad, const Tensor& coef, const Tensor& self, const Tensor& target,
                                const Tensor& lse, int64_t ignore_index) {
    return Stub<decltype(preference_loss_backward)>::call("finetune::preference_loss_backward", self, grad, coef, self,
                                                          target, lse, ignore_index);
}
Tensor dropout(const Tensor& self, double p, int64_t seed, int64_t offset) {
    return Stub<decltype(dropout)>::call("finetune::dropout", self, self, p, seed, offset);
}
Tensor dropout_backward(const Tensor& grad, double p, int64_t seed, int64_t offset) {
    return Stub<decltype(dropout_backward)>::call("finetune::dropout_backward", grad, grad, p, seed, offset);
}
std::tuple<Tensor, Tensor, OptTensor, Tensor> gated_residual_norm(const Tensor& self, const Tensor& residual,
                                                                  const Tensor& pre_weight, double eps,
                                                                  OptTensor post_weight, OptTensor gate,
                                                                  double residual_scale, double p, int64_t seed,
                                                                  int64_t offset) {
    return Stub<decltype(gated_residual_norm)>::call("finetune::gated_residual_norm", self, self, residual, pre_weight,
                                                     eps, std::move(post_weight), std::move(gate), residual_scale, p,
                                                     seed, offset);
}
std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> gated_residual_norm_backward(
    const Tensor& grad_y, OptTensor grad_residual, const Tensor& self, const Tensor& out, OptTensor rstd_post,
    const Tensor& rstd_pre, const Tensor& pre_weight, OptTensor post_weight, OptTensor gate, double residual_scale,
    double p, int64_t seed, int64_t offset) {
    return Stub<decltype(gated_residual_norm_backward)>::call(
        "finetune::gated_residual_norm_backward", self, grad_y, std::move(grad_residual), self, out,
        std::move(rstd_post), rstd_pre, pre_weight, std::move(post_weight), std::move(gate), residual_scale, p, seed,
        offset);
}

}  // namespace tensorplay

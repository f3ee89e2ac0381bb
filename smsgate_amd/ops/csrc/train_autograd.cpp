// smsgate_amd — autograd of the training operators (models/train_ops.py), without Python.
//
// A small step's call is host time: autograd runs a GPU backward on a thread of its own, and a
// Python Function there waits for the interpreter lock and then takes its steps in Python.
// Here both directions are one C++ call each: sizes, workspaces from torch's allocator, one
// entry of the kernel library on the current stream of the tensors' device.  No state is kept
// between calls.  Arguments are checked by models/train_ops.py before they come here.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "train_ops.hpp"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// Launches on the tensors' device (current or not), on its current stream.
template <typename F, typename... A>
void run(const Tensor& at, const char* name, F fn, A... args) {
  const c10::DeviceGuard guard(at.device());
  const hipStream_t st = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(at.device().index()).stream();
  const int rc = fn(args..., st);
  TORCH_CHECK(rc == 0, name, " failed (rc=", rc, ")");
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool off16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0; }

// `t` contiguous and on a 16-byte border (a copy where it is not)
Tensor aligned(const Tensor& t) {
  const Tensor c = t.contiguous();
  return off16(c) ? c.clone(at::MemoryFormat::Contiguous) : c;
}

// `t` [B, heads, T, D] itself when its rows can be read 16 bytes at a time, else a copy
Tensor rows16(const Tensor& t) {
  const auto s = t.strides();
  return s[3] == 1 && (s[0] | s[1] | s[2]) % 8 == 0 && !off16(t) ? t : aligned(t);
}

Tensor words(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// The gradients of a backward that can be run but not differentiated: under create_graph they
// carry a function that raises.  linear: they depend on the incoming gradient alone.
variable_list once(const variable_list& grads, variable_list out, bool linear) {
  if (!at::GradMode::is_enabled() || (linear && !grads[0].requires_grad())) return out;
  variable_list some;
  for (Tensor& t : out)
    if (t.defined()) some.push_back(t.requires_grad_());
  const auto err = std::make_shared<torch::autograd::DelayedError>(
      "the training operators' gradients cannot be differentiated again", (int64_t)some.size());
  some = (*err)(std::move(some));
  size_t i = 0;
  for (Tensor& t : out)
    if (t.defined()) t = some[i++];
  return out;
}

struct Embed : torch::autograd::Function<Embed> {
  static int vec16(const Tensor& a, const Tensor& b, int64_t H) {
    return !off16(a) && !off16(b) && H * a.element_size() % 16 == 0;
  }
  static int code(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& table_, const Tensor& ids_, const Maybe& add_,
                        double scale) {
    const Tensor table = table_.contiguous(), ids = ids_.contiguous();
    const Tensor add = add_ ? add_->contiguous() : Tensor();
    const int64_t V = table.size(0), H = table.size(1), n = ids.numel();
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(H);
    const Tensor x = at::empty(shape, table.options());
    if (n)
      run(table, "embed_fwd", sg_embed_fwd, ptr(ids), ptr(add), (int)(ids.scalar_type() == at::kLong), ptr(table),
          ptr(x), (int)n, (int)V, (int)H, (float)scale, code(table), vec16(table, x, H));
    ctx->save_for_backward({ids, add});
    ctx->saved_data["V"] = V;
    ctx->saved_data["scale"] = scale;
    return x;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    Tensor dt;
    {
      const at::NoGradGuard no;
      const Tensor &ids = saved[0], &add = saved[1], dx = grads[0].contiguous();
      const int64_t V = ctx->saved_data["V"].toInt(), H = dx.size(-1), n = ids.numel();
      dt = at::empty({V, H}, dx.options());
      if (n) {
        const int units = sg_embed_grad_ws((int)(add.defined() ? 2 * n : n), (int)V, (int)H);  // of 256 bytes
        const Tensor ws = units ? words(dx, 64L * units) : Tensor();
        run(dx, "embed_grad", sg_embed_grad, ptr(ids), ptr(add), (int)(ids.scalar_type() == at::kLong), ptr(dx),
            ptr(dt), (int)n, (int)V, (int)H, (float)ctx->saved_data["scale"].toDouble(), code(dx), vec16(dx, dt, H),
            ptr(ws), units);
      } else {
        dt.zero_();
      }
    }
    return once(grads, {dt, Tensor(), Tensor(), Tensor()}, true);
  }
};

struct Attention : torch::autograd::Function<Attention> {
  struct Sizes {
    int B, nh, T, D, nkv, fp16;
    long strides[9];
    int64_t stats;  // 32-bit words of the rows' statistics
    Sizes(const Tensor& q, const Tensor& k, const Tensor& v)
        : B(q.size(0)), nh(q.size(1)), T(q.size(2)), D(q.size(3)), nkv(k.size(1)),
          fp16(q.scalar_type() == at::kHalf) {
      int i = 0;
      for (const Tensor* t : {&q, &k, &v})
        for (int d = 0; d < 3; ++d) strides[i++] = t->stride(d);
      stats = (int64_t)B * nh * sg_attn_rows(T);
    }
  };

  // grad: whether a gradient may be asked for
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Maybe& lens_,
                        double scale, bool causal, bool grad) {
    const Tensor q = rows16(q_), k = rows16(k_), v = rows16(v_);
    const Tensor lens = lens_ ? lens_->contiguous() : Tensor();
    const Sizes s(q, k, v);
    const Tensor out = at::empty({s.B, s.T, (int64_t)s.nh * s.D}, q.options());
    // the rows' statistics, and behind them what rounding took from out, for the backward's D
    const Tensor keep = words(q, s.stats + (grad ? out.numel() / 2 : 0));
    float* lse = keep.data_ptr<float>();
    run(q, "attn_fwd", sg_attn_fwd, ptr(q), ptr(k), ptr(v), ptr(lens), ptr(out), grad ? (void*)(lse + s.stats) : nullptr,
        lse, (const void*)s.strides, s.B, s.T, s.nh, s.nkv, s.D, (int)causal, s.fp16, (float)scale);
    ctx->save_for_backward({q, k, v, lens, out, keep});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    Tensor dq, dk, dv;
    {
      const at::NoGradGuard no;
      const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[4], &keep = saved[5];
      const Tensor dout = aligned(grads[0]);
      const Sizes s(q, k, v);
      dq = at::empty(q.sizes(), q.options());
      dk = at::empty(k.sizes(), k.options());
      dv = at::empty(v.sizes(), v.options());
      const bool split = sg_attn_split(s.B, s.T, s.nh, s.nkv);
      const Tensor ws = words(q, s.stats + (s.fp16 ? sg_attn_maxima(s.B) : 0) + (split ? 2L * s.B * s.nh * s.T * s.D : 0));
      float* lse = keep.data_ptr<float>();
      run(q, "attn_bwd", sg_attn_bwd, ptr(q), ptr(k), ptr(v), ptr(saved[3]), ptr(out), (const void*)(lse + s.stats),
          (const void*)lse, ptr(dout), ptr(dq), ptr(dk), ptr(dv), ptr(ws), (const void*)s.strides, s.B, s.T, s.nh, s.nkv,
          s.D, (int)ctx->saved_data["causal"].toBool(), s.fp16, (float)ctx->saved_data["scale"].toDouble());
    }
    return once(grads, {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()}, false);
  }
};

struct Loss : torch::autograd::Function<Loss> {
  struct Plan {
    int64_t hc, ec, state, fwd, bwd;  // elements of hc, ec and state (16 bits), 32-bit words of the workspaces
    Plan(int N, int V, int H) {
      int p[6];
      const int rc = sg_loss_plan(N, V, H, p);
      TORCH_CHECK(rc == 0, "loss_plan failed (rc=", rc, ")");
      hc = (int64_t)p[0] * p[1];
      ec = (int64_t)p[2] * p[1];
      state = p[3] * 128L;
      fwd = p[4] * 64L;
      bwd = p[5] * 64L;
    }
  };

  static Tensor forward(AutogradContext* ctx, const Tensor& h_, const Tensor& table_, const Tensor& labels_, int64_t mode,
                        int64_t ignore) {
    const Tensor h = aligned(h_), table = aligned(table_), labels = labels_.contiguous();
    const int V = table.size(0), H = table.size(1), N = labels.numel(), fp16 = h.scalar_type() == at::kHalf;
    const Plan p(N, V, H);
    // the labelled rows and the table as the products read them, and the rows' places and
    // statistics: kept for the backward
    const Tensor keep = at::empty({p.hc + p.ec + p.state}, h.options()), ws = words(h, p.fwd);
    const Tensor loss = mode == 2 ? at::empty(labels.sizes(), ws.options()) : at::empty({}, ws.options());
    uint16_t* hc = static_cast<uint16_t*>(keep.data_ptr());
    run(h, "loss_fwd", sg_loss_fwd, ptr(h), ptr(table), ptr(labels), (int)(labels.scalar_type() == at::kLong),
        (int)ignore, hc, hc + p.hc, hc + p.hc + p.ec, ptr(ws), ptr(loss), N, V, H, (int)mode, fp16);
    ctx->save_for_backward({keep});
    ctx->saved_data["shape"] = h_.sizes().vec();
    ctx->saved_data["V"] = (int64_t)V;
    ctx->saved_data["mode"] = mode;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    Tensor dh, dt;
    {
      const at::NoGradGuard no;
      const Tensor &keep = saved[0], g = grads[0].contiguous();
      const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
      const int64_t H = shape.back(), V = ctx->saved_data["V"].toInt();
      int64_t N = 1;
      for (size_t i = 0; i + 1 < shape.size(); ++i) N *= shape[i];
      const Plan p(N, V, H);
      if (ctx->needs_input_grad(0)) dh = at::empty(shape, keep.options());
      if (ctx->needs_input_grad(1)) dt = at::empty({V, H}, keep.options());
      const Tensor ws = words(keep, p.bwd);
      uint16_t* hc = static_cast<uint16_t*>(keep.data_ptr());
      run(keep, "loss_bwd", sg_loss_bwd, (const void*)hc, (const void*)(hc + p.hc), (void*)(hc + p.hc + p.ec), ptr(g),
          ptr(ws), ptr(dh), ptr(dt), (int)N, (int)V, (int)H, (int)ctx->saved_data["mode"].toInt(),
          (int)(keep.scalar_type() == at::kHalf));
    }
    return once(grads, {dh, dt, Tensor(), Tensor(), Tensor()}, false);
  }
};

// Capturing a call whose leaf takes part in a living eager graph is refused: the leaf's
// accumulation node belongs to that graph's stream, autograd would wait for it in the captured
// backward, and the process would end.
void no_eager_graph(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return;
  const auto st = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA((*inputs.begin())->device().index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing(st.stream(), &status) == hipSuccess, "hipStreamIsCapturing failed");
  if (status == hipStreamCaptureStatusNone) return;
  for (const Tensor* t : inputs) {
    if (!t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto of = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!of || *of == st.unwrap(),
                "a captured call shares a leaf with a living eager graph: drop that graph's results first");
  }
}

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& lens, double scale, bool causal) {
  no_eager_graph({&q, &k, &v});
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  return Attention::apply(q, k, v, lens, scale, causal, grad);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("embed", [](const Tensor& table, const Tensor& ids, const Maybe& add, double scale) {
    no_eager_graph({&table});
    return Embed::apply(table, ids, add, scale);
  }, free);
  m.def("attention", &attention, free);
  m.def("loss", [](const Tensor& h, const Tensor& table, const Tensor& labels, int64_t mode, int64_t ignore) {
    no_eager_graph({&h, &table});
    return Loss::apply(h, table, labels, mode, ignore);
  }, free);
  m.def("rows16", &rows16);
}

// Autograd nodes of the embedding lookup and of the relation GRU.  A node written in Python runs its backward on the
// engine's thread, which waits for the interpreter's lock that the calling thread holds.  3,080 tokens of 512 x 200 with
// their gradient, pass after pass: 84 us with a node in Python, 50 with this one (19 of them the kernels); torch's indexing
// with its backward takes 76 to 79, a product by 2 with its backward, which is the engine's own cost, 41.  The GRU's three
// calls of a training sample: 0.22 ms in Python, 0.1 here.
//
// Host code only: the kernels are libregcn_hip.so's, whose entries `bind` is given by the library that Python loaded.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "../../include/regcn_hip.h"

#include <algorithm>
#include <cstdint>

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Entries {
  decltype(&regcn_embedding) lookup;
  decltype(&regcn_embedding_grad_workspace_bytes) grad_bytes;
  decltype(&regcn_embedding_grad) grad;
  decltype(&regcn_kreduce_workspace_floats) kreduce_floats;
  decltype(&regcn_kreduce_gemm_f32) kreduce;
  decltype(&regcn_last_error_string) error;
} entry;

int type_of(const Tensor& t) {
  return t.scalar_type() == torch::kFloat ? REGCN_F32 : t.scalar_type() == torch::kBFloat16 ? REGCN_BF16 : REGCN_F16;
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// scale * table[idx], as autograd._embedding_rows.
Tensor rows(const Tensor& table, const Tensor& idx, double scale) {
  auto shape = idx.sizes().vec();
  shape.push_back(table.size(1));
  const c10::DeviceGuard guard(table.device());
  Tensor out = at::empty(shape, table.options().requires_grad(false));
  if (out.numel()) {
    const int rc = entry.lookup(table.data_ptr(), table.stride(0), idx.data_ptr(), idx.scalar_type() == torch::kLong, idx.numel(),
                                table.size(0), (int32_t)table.size(1), type_of(table), (float)scale, out.data_ptr(), stream_of(table));
    TORCH_CHECK(rc == 0, "regcn_embedding failed (rc=", rc, "): ", entry.error());
  }
  return out;
}

// The sums of g's rows by index, as autograd._embedding_sums.
Tensor sums(const Tensor& grad, const Tensor& idx, int64_t V, double scale, int64_t pad) {
  const c10::DeviceGuard guard(grad.device());
  const Tensor g = grad.contiguous();
  const int64_t n = idx.numel(), d = g.size(-1);
  Tensor out = at::empty({V, d}, g.options().requires_grad(false));
  if (out.numel()) {
    const int64_t bytes = entry.grad_bytes(n, V, (int32_t)d);
    const Tensor ws = at::empty({bytes}, g.options().dtype(torch::kByte).requires_grad(false));
    const int rc = entry.grad(g.data_ptr(), idx.data_ptr(), idx.scalar_type() == torch::kLong, n, V, (int32_t)d, pad, type_of(g),
                              (float)scale, out.data_ptr(), ws.data_ptr(), (size_t)bytes, stream_of(g));
    TORCH_CHECK(rc == 0, "regcn_embedding_grad failed (rc=", rc, "): ", entry.error());
  }
  return out;
}

struct Lookup : Function<Lookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& idx, double scale, int64_t pad) {
    ctx->save_for_backward({idx});
    ctx->saved_data["V"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    return rows(table, idx, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g);
};

// The gradient as a function of g: linear, its own gradient a lookup without the rows of the tokens that it leaves out.
struct Sums : Function<Sums> {
  static Tensor forward(AutogradContext* ctx, const Tensor& g, const Tensor& idx, int64_t V, double scale, int64_t pad) {
    ctx->save_for_backward({idx});
    ctx->saved_data["V"] = V;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    return sums(g, idx, V, scale, pad);
  }
  static variable_list backward(AutogradContext* ctx, variable_list gg) {
    const Tensor idx = ctx->get_saved_variables()[0];
    const int64_t V = ctx->saved_data["V"].toInt(), pad = ctx->saved_data["pad"].toInt();
    const Tensor left = idx.lt(0).logical_or(idx.ge(V)).logical_or(idx.eq(pad)).unsqueeze(-1);
    const Tensor out = Lookup::apply(gg[0].contiguous(), idx, ctx->saved_data["scale"].toDouble(), -1);
    return {out.masked_fill(left, 0.0), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

variable_list Lookup::backward(AutogradContext* ctx, variable_list g) {
  const Tensor idx = ctx->get_saved_variables()[0];
  const int64_t V = ctx->saved_data["V"].toInt(), pad = ctx->saved_data["pad"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  // create_graph: the gradient is differentiable in g
  return {torch::GradMode::is_enabled() ? Sums::apply(g[0], idx, V, scale, pad) : sums(g[0], idx, V, scale, pad), Tensor(), Tensor(),
          Tensor()};
}

// A GRU cell's gates and new state from its two products, by torch's fused kernels.  Theirs for the backward would sum the
// biases' gradients on several workgroups, which does not replay in a HIP graph: both are one product with a row of ones here,
// as autograd.colsum.
struct GruGates : Function<GruGates> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gi, const Tensor& gh, const Tensor& h, const Tensor& b_ih, const Tensor& b_hh) {
    auto [out, ws] = at::_thnn_fused_gru_cell(gi, gh, h, b_ih, b_hh);
    ctx->save_for_backward({ws});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gy) {
    const c10::DeviceGuard guard(gy[0].device());
    auto [di, dh, dx, none_i, none_h] = at::_thnn_fused_gru_cell_backward(gy[0].contiguous(), ctx->get_saved_variables()[0], false);
    Tensor db;
    if (ctx->needs_input_grad(3) || ctx->needs_input_grad(4)) {
      const Tensor both = at::cat({di, dh}, 1), ones = at::ones({both.size(0), 1}, both.options());
      const int64_t K = both.size(0), N = both.size(1);
      db = at::empty({2, N / 2}, both.options());
      const Tensor ws = at::empty({std::max<int64_t>(1, (int64_t)entry.kreduce_floats(K, 1, (int32_t)N))}, both.options());
      const int rc = entry.kreduce(ones.data_ptr<float>(), 1, both.data_ptr<float>(), 1, K, 1, (int32_t)N, nullptr, 0, db.data_ptr<float>(),
                                   ws.data_ptr<float>(), stream_of(both));
      TORCH_CHECK(rc == 0, "regcn_kreduce_gemm_f32 failed (rc=", rc, "): ", entry.error());
    }
    return {di, dh, dx, db.defined() ? db[0] : Tensor(), db.defined() ? db[1] : Tensor()};
  }
};

void bind(uintptr_t lookup, uintptr_t grad_bytes, uintptr_t grad, uintptr_t kreduce_floats, uintptr_t kreduce, uintptr_t error) {
  entry.lookup = reinterpret_cast<decltype(entry.lookup)>(lookup);
  entry.grad_bytes = reinterpret_cast<decltype(entry.grad_bytes)>(grad_bytes);
  entry.grad = reinterpret_cast<decltype(entry.grad)>(grad);
  entry.kreduce_floats = reinterpret_cast<decltype(entry.kreduce_floats)>(kreduce_floats);
  entry.kreduce = reinterpret_cast<decltype(entry.kreduce)>(kreduce);
  entry.error = reinterpret_cast<decltype(entry.error)>(error);
}

}  // namespace

PYBIND11_MODULE(_node, m) {
  m.def("bind", &bind, "Addresses of regcn_embedding, regcn_embedding_grad_workspace_bytes, regcn_embedding_grad, "
                       "regcn_kreduce_workspace_floats, regcn_kreduce_gemm_f32, regcn_last_error_string");
  m.def("gru_gates",
        [](const Tensor& gi, const Tensor& gh, const Tensor& h, const Tensor& b_ih, const Tensor& b_hh) {
          return GruGates::apply(gi, gh, h, b_ih, b_hh);
        },
        "A GRU cell's new state from its two products (fp32, on a HIP device)");
  m.def("lookup", [](const Tensor& table, const Tensor& idx, double scale, int64_t pad) { return Lookup::apply(table, idx, scale, pad); },
        "scale * table[idx] with its gradient; arguments as autograd.embedding has checked them");
}

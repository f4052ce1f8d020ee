// The embedding lookup's autograd nodes.  A node written in Python runs its backward on the engine's thread, which waits
// for the interpreter's lock that the calling thread holds.  3,080 tokens of 512 x 200 with their gradient, pass after
// pass: 84 us with a node in Python, 50 with this one (19 of them the kernels); torch's indexing with its backward takes 76 to
// 79, a product by 2 with its backward, which is the engine's own cost, 41.
//
// Host code only: the kernels are libregcn_hip.so's, whose entries `bind` is given by the library that Python loaded.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <cstdint>

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Entries {
  int (*lookup)(const void*, int64_t, const void*, int32_t, int64_t, int64_t, int32_t, int32_t, float, void*, void*);
  int64_t (*grad_bytes)(int64_t, int64_t, int32_t);
  int (*grad)(const void*, const void*, int32_t, int64_t, int64_t, int32_t, int64_t, int32_t, float, void*, void*, size_t, void*);
  const char* (*error)();
} entry;

int type_of(const Tensor& t) {  // REGCN_F32, REGCN_BF16, REGCN_F16
  return t.scalar_type() == torch::kFloat ? 0 : t.scalar_type() == torch::kBFloat16 ? 1 : 2;
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

void bind(uintptr_t lookup, uintptr_t grad_bytes, uintptr_t grad, uintptr_t error) {
  entry.lookup = reinterpret_cast<decltype(entry.lookup)>(lookup);
  entry.grad_bytes = reinterpret_cast<decltype(entry.grad_bytes)>(grad_bytes);
  entry.grad = reinterpret_cast<decltype(entry.grad)>(grad);
  entry.error = reinterpret_cast<decltype(entry.error)>(error);
}

}  // namespace

PYBIND11_MODULE(_node, m) {
  m.def("bind", &bind, "Addresses of regcn_embedding, regcn_embedding_grad_workspace_bytes, regcn_embedding_grad, "
                       "regcn_last_error_string");
  m.def("lookup", [](const Tensor& table, const Tensor& idx, double scale, int64_t pad) { return Lookup::apply(table, idx, scale, pad); },
        "scale * table[idx] with its gradient; arguments as autograd.embedding has checked them");
}

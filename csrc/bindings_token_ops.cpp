// PyTorch bindings of the operators at the ends of a training step (token
// log probabilities, scaled embedding) and of the 8-bit activations.  They
// allocate their results themselves: one call from Python per pass.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>
#include <tuple>

#include "kernels_api.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return msb::kF32;
    case at::kHalf: return msb::kF16;
    case at::kBFloat16: return msb::kBF16;
    default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
  }
  return -1;
}

cudaStream_t stream_of(const at::Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void check_contig(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_matrix(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  // (an axis of one element may have any stride)
  TORCH_CHECK(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1) &&
                  (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
              name, " must be a row-major matrix (unit column stride)");
  TORCH_CHECK(t.size(1) > 0 && t.size(1) < std::numeric_limits<int>::max() - 1024, name,
              " is too wide");
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// ------------------------------------------------------- 8-bit activations
constexpr int64_t kBlk = 32;

std::tuple<at::Tensor, at::Tensor> packed_like(const at::Tensor& t, int64_t rows, int64_t width) {
  const int64_t nb = (width + kBlk - 1) / kBlk;
  return {at::empty({rows, nb * kBlk}, t.options().dtype(at::kChar)),
          at::empty({rows, nb}, t.options().dtype(at::kByte))};
}

void check_packed(const at::Tensor& codes, const at::Tensor& scales, int64_t rows, int64_t width) {
  check_contig(codes, "codes");
  check_contig(scales, "scales");
  const int64_t nb = (width + kBlk - 1) / kBlk;
  TORCH_CHECK(codes.scalar_type() == at::kChar && codes.dim() == 2 && codes.size(0) == rows &&
                  codes.size(1) == nb * kBlk, "codes: int8 [rows, 32 * blocks]");
  TORCH_CHECK(scales.scalar_type() == at::kByte && scales.dim() == 2 && scales.size(0) == rows &&
                  scales.size(1) == nb, "scales: uint8 [rows, blocks]");
  TORCH_CHECK(scales.device() == codes.device(), "codes and scales on different devices");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(codes.data_ptr()) & 15) == 0,
              "codes must be 16-byte aligned");
}

unsigned char* bytes(const at::Tensor& t) { return t.data_ptr<uint8_t>(); }
signed char* codes_of(const at::Tensor& t) {
  return reinterpret_cast<signed char*>(t.data_ptr<int8_t>());
}

std::tuple<at::Tensor, at::Tensor> pack8(const at::Tensor& x) {
  check_matrix(x, "x");
  c10::cuda::CUDAGuard g(x.device());
  auto out = packed_like(x, x.size(0), x.size(1));
  msb::pack8(x.data_ptr(), row_stride(x), codes_of(std::get<0>(out)), bytes(std::get<1>(out)),
             x.size(0), (int)x.size(1), dtype_code(x), stream_of(x));
  return out;
}

// a new tensor of `shape`; dtype: an msb::DType code
at::Tensor unpack8(const at::Tensor& codes, const at::Tensor& scales, at::IntArrayRef shape,
                   int64_t code) {
  TORCH_CHECK(code == msb::kF32 || code == msb::kF16 || code == msb::kBF16, "dtype code");
  const at::ScalarType dtype =
      code == msb::kF32 ? at::kFloat : code == msb::kF16 ? at::kHalf : at::kBFloat16;
  TORCH_CHECK(codes.dim() == 2 && !shape.empty() && shape.back() > 0,
              "codes: int8 [rows, 32 * blocks] of a shape");
  const int64_t rows = codes.size(0), width = shape.back();
  check_packed(codes, scales, rows, width);
  c10::cuda::CUDAGuard g(codes.device());
  at::Tensor x = at::empty(shape, codes.options().dtype(dtype));
  TORCH_CHECK(x.numel() == rows * width && width < (1LL << 31) - 1024, "shape of another tensor");
  msb::unpack8(codes_of(codes), bytes(scales), x.data_ptr(), rows, (int)width, (int)code,
               stream_of(codes));
  return x;
}

// without `save`, codes and scales come back empty
std::tuple<at::Tensor, at::Tensor, at::Tensor> swiglu8_fwd(const at::Tensor& gu, bool save) {
  check_contig(gu, "gu");
  const int64_t F = gu.size(-1) / 2;
  TORCH_CHECK(gu.size(-1) == 2 * F && F > 0 && F < (1LL << 30), "gu: [..., 2 F]");
  const int64_t rows = gu.numel() / (2 * F);
  c10::cuda::CUDAGuard g(gu.device());
  auto shape = gu.sizes().vec();
  shape.back() = F;
  at::Tensor h = at::empty(shape, gu.options());
  auto packed = packed_like(gu, save ? 2 * rows : 0, F);
  msb::swiglu8_fwd(gu.data_ptr(), h.data_ptr(), save ? codes_of(std::get<0>(packed)) : nullptr,
                   bytes(std::get<1>(packed)), rows, (int)F, dtype_code(gu), stream_of(gu));
  return {h, std::get<0>(packed), std::get<1>(packed)};
}

at::Tensor swiglu8_bwd(const at::Tensor& dh, const at::Tensor& codes, const at::Tensor& scales) {
  check_contig(dh, "dh");
  const int64_t F = dh.size(-1), rows = F > 0 ? dh.numel() / F : 0;
  TORCH_CHECK(F > 0 && F < (1LL << 30), "dh: [..., F]");
  check_packed(codes, scales, 2 * rows, F);
  TORCH_CHECK(codes.device() == dh.device(), "dh and codes on different devices");
  c10::cuda::CUDAGuard g(dh.device());
  auto shape = dh.sizes().vec();
  shape.back() = 2 * F;
  at::Tensor dgu = at::empty(shape, dh.options());
  msb::swiglu8_bwd(dh.data_ptr(), codes_of(codes), bytes(scales), dgu.data_ptr(), rows, (int)F,
                   dtype_code(dh), stream_of(dh));
  return dgu;
}

// ------------------------------------------------ token log probabilities
using OptT = c10::optional<at::Tensor>;

bool given(const OptT& t) { return t.has_value() && t->defined(); }

const long long* tokens_of(const at::Tensor& t, int64_t n, const at::Tensor& like) {
  check_contig(t, "tokens");
  TORCH_CHECK(t.scalar_type() == at::kLong && t.numel() == n, "tokens: int64, one a row");
  TORCH_CHECK(t.device() == like.device(), "tokens on another device");
  return reinterpret_cast<const long long*>(t.data_ptr<int64_t>());
}

// (logprobs, entropy or none, top logprobs [..., k], top tokens [..., k], stats [M, 3]), in the
// tokens' shape
std::tuple<at::Tensor, OptT, OptT, OptT, at::Tensor> logprob_fwd(
    const at::Tensor& logits, const at::Tensor& tokens, double temperature, bool entropy,
    int64_t k, int64_t ignore_index) {
  check_matrix(logits, "logits");
  const int64_t M = logits.size(0), V = logits.size(1);
  const long long* tok = tokens_of(tokens, M, logits);
  TORCH_CHECK(k >= 0 && k <= 32 && k <= V, "top_k must be in [0, 32] and at most V");
  TORCH_CHECK(M < (1LL << 31), "too many rows");
  c10::cuda::CUDAGuard g(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor lp = at::empty(tokens.sizes(), f32), stats = at::empty({M, 3}, f32);
  OptT ent, tlp, ttok;
  if (entropy) ent = at::empty(tokens.sizes(), f32);
  if (k > 0) {
    auto shape = tokens.sizes().vec();
    shape.push_back(k);
    tlp = at::empty(shape, f32);
    ttok = at::empty(shape, logits.options().dtype(at::kLong));
  }
  msb::logprob_fwd(logits.data_ptr(), row_stride(logits), tok, M, (int)V, (float)temperature,
                   ignore_index, (int)k, lp.data_ptr<float>(),
                   entropy ? ent->data_ptr<float>() : nullptr,
                   k > 0 ? tlp->data_ptr<float>() : nullptr,
                   k > 0 ? reinterpret_cast<long long*>(ttok->data_ptr<int64_t>()) : nullptr,
                   stats.data_ptr<float>(), dtype_code(logits), stream_of(logits));
  return {lp, ent, tlp, ttok, stats};
}

// an upstream gradient as the contiguous fp32 [n] that the kernel reads
at::Tensor grad_f32(const OptT& g, int64_t n, const at::Tensor& like) {
  if (!given(g)) return at::Tensor();
  TORCH_CHECK(g->numel() == n && g->device() == like.device(), "gradient: one value a result");
  return g->to(at::kFloat).contiguous();
}

const float* fptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// dlogits [M, V]; its rows are padded to 64 values where the logits' rows are padded
at::Tensor logprob_bwd(const at::Tensor& logits, const at::Tensor& tokens, const OptT& top_tokens,
                       const at::Tensor& stats, const OptT& g_logp, const OptT& g_ent,
                       const OptT& g_top, double temperature, int64_t ignore_index) {
  check_matrix(logits, "logits");
  const int64_t M = logits.size(0), V = logits.size(1);
  const long long* tok = tokens_of(tokens, M, logits);
  check_contig(stats, "stats");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.numel() == M * 3, "stats: fp32 [M, 3]");
  int64_t k = 0;
  const long long* tt = nullptr;
  c10::cuda::CUDAGuard g(logits.device());
  if (given(top_tokens) && given(g_top)) {
    TORCH_CHECK(top_tokens->dim() >= 1 && top_tokens->size(-1) <= 32, "top tokens: [..., k]");
    k = top_tokens->size(-1);
    tt = tokens_of(*top_tokens, M * k, logits);
  }
  const at::Tensor gl = grad_f32(g_logp, M, logits), ge = grad_f32(g_ent, M, logits),
                   gt = k > 0 ? grad_f32(g_top, M * k, logits) : at::Tensor();
  const int64_t ld = row_stride(logits) > V ? (V + 63) / 64 * 64 : V;
  at::Tensor dx = at::empty({M, ld}, logits.options());
  msb::logprob_bwd(logits.data_ptr(), row_stride(logits), tok, M, (int)V, (float)temperature,
                   ignore_index, (int)k, tt, stats.data_ptr<float>(), fptr(gl), fptr(ge), fptr(gt),
                   dx.data_ptr(), ld, dtype_code(logits), stream_of(logits));
  return ld == V ? dx : dx.narrow(1, 0, V);
}

// ------------------------------------------------------- scaled embedding
// (out, list): with `sort`, the tokens' list for the backward, else none
std::tuple<at::Tensor, OptT> scaled_embedding_fwd(const at::Tensor& idx, const at::Tensor& weight,
                                                  double scale, int64_t padding, bool sort) {
  check_contig(weight, "weight");
  check_matrix(weight, "weight");
  const int64_t n = idx.numel(), V = weight.size(0), C = weight.size(1);
  const long long* tok = tokens_of(idx, n, weight);
  TORCH_CHECK(V > 0 && V < (1LL << 31) && n < (1LL << 31) && C < (1LL << 30) &&
                  n * ((C + 255) / 256) < (1LL << 34), "too large");
  c10::cuda::CUDAGuard g(weight.device());
  auto shape = idx.sizes().vec();
  shape.push_back(C);
  at::Tensor out = at::empty(shape, weight.options());
  OptT list;
  if (sort) list = at::empty({4 * n}, weight.options().dtype(at::kInt));
  msb::scaled_embedding_fwd(tok, weight.data_ptr(), out.data_ptr(), n, (int)C, V, (float)scale,
                            padding, sort ? (unsigned*)list->data_ptr<int>() : nullptr,
                            dtype_code(weight), stream_of(weight));
  return {out, list};
}

// the gradient added into `sink` [V, C], or, without one, as a new tensor
at::Tensor scaled_embedding_bwd(const at::Tensor& dout, const at::Tensor& list, int64_t V,
                                double scale, const OptT& sink) {
  check_contig(dout, "dout");
  check_contig(list, "list");
  const int64_t C = dout.size(-1), n = list.numel() / 4;
  TORCH_CHECK(list.scalar_type() == at::kInt && dout.dim() >= 1 && C > 0 &&
                  dout.numel() == n * C && list.device() == dout.device(),
              "dout: [tokens, C], with the list of its lookup");
  c10::cuda::CUDAGuard g(dout.device());
  at::Tensor grad;
  if (given(sink)) {
    check_contig(*sink, "sink");
    TORCH_CHECK(sink->dim() == 2 && sink->size(0) == V && sink->size(1) == C &&
                    sink->scalar_type() == dout.scalar_type() && sink->device() == dout.device(),
                "sink: a [V, C] gradient of dout's type");
    grad = *sink;
  } else {
    grad = at::empty({V, C}, dout.options());
  }
  at::Tensor ws = at::empty({msb::scaled_embedding_ws(n, (int)C)}, dout.options().dtype(at::kInt));
  msb::scaled_embedding_bwd(dout.data_ptr(), (const unsigned*)list.data_ptr<int>(),
                            grad.data_ptr(), given(sink), (unsigned*)ws.data_ptr<int>(), n, (int)C,
                            V, (float)scale, dtype_code(dout), stream_of(dout));
  return grad;
}

}  // namespace

// ------------------------------------------------------------- autograd
// The operators' autograd functions.  In C++ they cost the host a third of what
// they do in Python, which is what small calls are bound by.
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// Whether `t` needs a node in the graph.  Forward-mode tangents have no kernels:
// without a node they would be lost, so they are refused here.
bool wants_grad(const at::Tensor& t, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), op,
                              ": forward-mode derivatives are not implemented on CUDA");
  return at::GradMode::is_enabled() && t.requires_grad();
}

// The gradients come from kernels and have no graph of their own: under
// create_graph they would count as constants.
void first_derivative_only(const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), op,
                              ": second derivatives (create_graph=True) are not implemented on CUDA");
}

OptT some(const at::Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

// `t` as rows of its last axis with unit column stride; copied where no view is
at::Tensor as_rows(const at::Tensor& t) {
  at::Tensor m = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  const bool rows = (m.stride(1) == 1 || m.size(1) == 1) &&
                    (m.size(0) <= 1 || m.stride(0) >= m.size(1));
  return rows ? m : m.contiguous();
}

struct TokenLogprobs : public Function<TokenLogprobs> {
  // logprobs, then the entropy and the top log probabilities and tokens asked for
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits,
                               const at::Tensor& tokens, double temperature, bool entropy,
                               int64_t k, int64_t ignore_index) {
    const at::Tensor rows = as_rows(logits), tok = tokens.contiguous();
    auto [lp, ent, tlp, ttok, stats] = logprob_fwd(rows, tok, temperature, entropy, k, ignore_index);
    variable_list out = {lp};
    if (entropy) out.push_back(*ent);
    if (k > 0) {
      out.push_back(*tlp);
      out.push_back(*ttok);
    }
    if (ctx != nullptr) {
      ctx->set_materialize_grads(false);
      if (k > 0) ctx->mark_non_differentiable({out.back()});
      ctx->save_for_backward({rows, tok, k > 0 ? *ttok : at::Tensor(), stats});
      if (logits.dim() != 2) ctx->saved_data["shape"] = logits.sizes().vec();
      ctx->saved_data["temperature"] = temperature;
      ctx->saved_data["entropy"] = entropy;
      ctx->saved_data["ignore_index"] = ignore_index;
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_derivative_only("token_logprobs");
    const bool entropy = ctx->saved_data["entropy"].toBool();
    const at::Tensor none, &gl = g[0], &ge = entropy ? g[1] : none;
    const size_t top = entropy ? 2 : 1;
    const at::Tensor& gt = g.size() > top ? g[top] : none;
    at::Tensor dx;
    if (gl.defined() || ge.defined() || gt.defined()) {
      const auto saved = ctx->get_saved_variables();
      dx = logprob_bwd(saved[0], saved[1], some(saved[2]), saved[3], some(gl), some(ge), some(gt),
                       ctx->saved_data["temperature"].toDouble(),
                       ctx->saved_data["ignore_index"].toInt());
      const auto shape = ctx->saved_data.find("shape");
      if (shape != ctx->saved_data.end()) dx = dx.view(shape->second.toIntVector());
    }
    return {dx, none, none, none, none, none};
  }
};

variable_list token_logprobs(const at::Tensor& logits, const at::Tensor& tokens,
                             double temperature, bool entropy, int64_t k, int64_t ignore_index) {
  if (wants_grad(logits, "token_logprobs"))
    return TokenLogprobs::apply(logits, tokens, temperature, entropy, k, ignore_index);
  return TokenLogprobs::forward(nullptr, logits, tokens, temperature, entropy, k, ignore_index);
}

struct ScaledEmbedding : public Function<ScaledEmbedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& idx, const at::Tensor& weight,
                            double scale, int64_t padding, bool sink) {
    auto [out, list] = scaled_embedding_fwd(idx.contiguous(), weight.contiguous(), scale, padding,
                                            ctx != nullptr);
    if (ctx != nullptr) {
      // the weight itself for its gradient, not for its values
      ctx->save_for_backward({*list});
      if (sink) ctx->saved_data["weight"] = weight;
      ctx->saved_data["rows"] = weight.size(0);
      ctx->saved_data["scale"] = scale;
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_derivative_only("scaled_embedding");
    const at::Tensor none;
    const at::Tensor dout = g[0].contiguous();
    OptT sink;
    if (ctx->saved_data.count("weight") != 0) {
      const at::Tensor weight = ctx->saved_data["weight"].toTensor();
      const at::Tensor& grad = weight.grad();
      if (grad.defined() && grad.scalar_type() == weight.scalar_type() &&
          grad.sizes() == weight.sizes() && grad.is_contiguous())
        sink = grad;
    }
    const at::Tensor dw =
        scaled_embedding_bwd(dout, ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                             ctx->saved_data["scale"].toDouble(), sink);
    return {none, given(sink) ? none : dw, none, none, none};
  }
};

// `sink`: weight is a parameter, whose gradient is added to in place where it has one
at::Tensor scaled_embedding(const at::Tensor& idx, const at::Tensor& weight, double scale,
                            int64_t padding, bool sink) {
  if (wants_grad(weight, "scaled_embedding"))
    return ScaledEmbedding::apply(idx, weight, scale, padding, sink);
  return ScaledEmbedding::forward(nullptr, idx, weight, scale, padding, sink);
}

struct SwiGLU8 : public Function<SwiGLU8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& gu) {
    auto [h, codes, scales] = swiglu8_fwd(gu.contiguous(), ctx != nullptr);
    if (ctx != nullptr) ctx->save_for_backward({codes, scales});
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_derivative_only("swiglu with save_bits=8");
    const auto saved = ctx->get_saved_variables();
    return {swiglu8_bwd(g[0].contiguous(), saved[0], saved[1])};
  }
};

at::Tensor swiglu8(const at::Tensor& gu) {
  return wants_grad(gu, "swiglu with save_bits=8") ? SwiGLU8::apply(gu) : SwiGLU8::forward(nullptr, gu);
}

std::tuple<at::Tensor, at::Tensor> pack_rows(const at::Tensor& x) {
  return pack8(as_rows(x.requires_grad() ? x.detach() : x));
}

}  // namespace

void register_token_ops(pybind11::module_& mod) {
  mod.def("token_logprobs", &token_logprobs);
  mod.def("scaled_embedding", &scaled_embedding);
  mod.def("swiglu8", &swiglu8);
  mod.def("pack_rows", &pack_rows);
  // without a graph (the backward passes trust what their forward left, and are
  // reached through it alone)
  mod.def("logprob_fwd", &logprob_fwd);
  mod.def("scaled_embedding_fwd", &scaled_embedding_fwd);
  mod.def("unpack8", &unpack8);
}

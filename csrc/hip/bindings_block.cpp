// torch glue of the dense-block operators (block_norm.hip, block_fp8.hip):
// shape checks, allocation and the autograd nodes.  Every entry runs on its
// tensors' device and that device's current stream; nothing outlives the call
// but the tensors it returns or saves.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <torch/extension.h>

#include "block_ops.h"

namespace py = pybind11;
using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace pbx {
namespace {

using OptTensor = c10::optional<Tensor>;  // an autograd node takes no undefined tensor

#define BK_CHECK(cond, ...) TORCH_CHECK(cond, "pbx block: ", __VA_ARGS__)

// a launch that the runtime refused is reported by the call that made it
void launched() { C10_HIP_KERNEL_LAUNCH_CHECK(); }

hipStream_t stream_of(const Tensor& t) { return at::hip::getCurrentHIPStream(t.device().index()).stream(); }

BlockType block_type(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return kF32;
    case torch::kBFloat16: return kBF16;
    case torch::kFloat16: return kF16;
    default: BK_CHECK(false, name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
  }
  return kF32;
}

void first_order_only() {
  BK_CHECK(!at::GradMode::is_enabled(), "the backward pass of this operator cannot be differentiated again");
}

// [M, D] rows with unit column stride: the tensor itself when it has them (any
// row stride of at least D), else a contiguous copy
Tensor rows_of(const Tensor& t, int64_t M, int64_t D) {
  if (t.dim() == 2 && (D == 1 || t.stride(1) == 1) && (M <= 1 || t.stride(0) >= D)) return t;
  return t.contiguous().view({M, D});
}
int64_t ld_of(const Tensor& t, int64_t M, int64_t D) { return M <= 1 ? D : t.stride(0); }

// ------------------------------------------------------------------ dropout mask
struct MaskOpts {
  int64_t thr;  // round(p 2^16)
  double up;    // scale of a kept value
  int64_t seed, offset;
};

MaskArgs mask_args(const MaskOpts& o, const Tensor& seed, const Tensor& like) {
  MaskArgs m;
  BK_CHECK(o.thr >= 0 && o.thr <= 65536, "dropout threshold out of range");
  m.thr = (uint32_t)o.thr;
  m.up = (float)o.up;
  m.seed_v = o.seed;
  m.offset_v = o.offset;
  if (seed.defined() && o.thr) {
    BK_CHECK(seed.scalar_type() == torch::kInt64 && seed.numel() == 2 && seed.is_contiguous() &&
                 seed.device() == like.device(),
             "a seed tensor is a contiguous int64 [2] = (seed, offset) on the input's device");
    m.seed = seed.data_ptr<int64_t>();
  }
  return m;
}

class DropoutFn : public torch::autograd::Function<DropoutFn> {
 public:
  static Tensor run(const Tensor& x, MaskArgs m) {
    auto xc = x.contiguous();
    auto y = torch::empty(x.sizes(), xc.options());
    launch_dropout(xc.data_ptr(), y.data_ptr(), x.numel(), block_type(x, "x"), m, stream_of(x));
    launched();
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& seed_t, MaskOpts o, bool grad) {
    c10::DeviceGuard guard(x.device());
    const Tensor seed = seed_t.value_or(Tensor());
    MaskArgs m = mask_args(o, seed, x);
    Tensor used;
    if (m.seed && grad) {  // the caller's tensor may have moved on by the time of the backward
      used = torch::empty({2}, seed.options());
      m.seed_out = used.data_ptr<int64_t>();
    }
    auto y = run(x, m);
    ctx->save_for_backward({used});
    ctx->saved_data["thr"] = o.thr;
    ctx->saved_data["up"] = o.up;
    ctx->saved_data["seed"] = o.seed;
    ctx->saved_data["offset"] = o.offset;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order_only();
    c10::DeviceGuard guard(g[0].device());
    const Tensor used = ctx->get_saved_variables()[0];
    const MaskArgs m = mask_args({ctx->saved_data["thr"].toInt(), ctx->saved_data["up"].toDouble(),
                                  ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt()},
                                 used, g[0]);
    return {run(g[0], m), Tensor(), Tensor(), Tensor()};
  }
};

// Whether an autograd node will be recorded for these inputs.  While the
// stream captures, an input that an eager graph on the default stream made, or
// a leaf whose accumulator such a graph keeps alive, is refused: the backward
// would hand its gradient over to that stream, which may not take part in a
// capture, and end the process.
bool wants_grad(std::initializer_list<OptTensor> ts, const Tensor& like) {
  if (!at::GradMode::is_enabled()) return false;
  bool any = false;
  for (const OptTensor& t : ts) any |= t.has_value() && t->requires_grad();
  if (!any) return false;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  C10_HIP_CHECK(hipStreamIsCapturing(stream_of(like), &status));
  if (status == hipStreamCaptureStatusNone) return true;
  for (const OptTensor& t : ts) {
    if (!t.has_value() || !t->requires_grad()) continue;
    const auto node = t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn();
    const auto s = node ? node->stream() : c10::nullopt;
    BK_CHECK(!s.has_value() || s->id() != 0,
             "the stream captures a graph while an eager autograd graph of the same leaf is alive; drop its outputs first");
  }
  return true;
}

Tensor block_dropout(const Tensor& x, const OptTensor& seed, int64_t thr, double up, int64_t seed_v,
                     int64_t offset_v) {
  BK_CHECK(x.is_cuda(), "x must be a GPU tensor");
  block_type(x, "x");
  return DropoutFn::apply(x, seed, MaskOpts{thr, up, seed_v, offset_v}, wants_grad({x}, x));
}

// ------------------------------------------------------------------ gated residual norm
struct ResidualOpts {
  int64_t post, pre, gate_kind;
  bool sigmoid;
  double x_scale, y_scale, eps;
  MaskOpts mask;
};

class ResidualFn : public torch::autograd::Function<ResidualFn> {
 public:
  // inputs: x, y, gate, post_w, post_b, pre_w, pre_b, seed
  static ResidualArgs args(const ResidualOpts& o, const Tensor& y, int64_t M, int64_t D) {
    ResidualArgs a;
    a.M = M;
    a.D = (int)D;
    a.post = (int)o.post;
    a.pre = (int)o.pre;
    a.gate_kind = (int)o.gate_kind;
    a.sigmoid = o.sigmoid;
    a.x_scale = (float)o.x_scale;
    a.y_scale = (float)o.y_scale;
    a.eps = (float)o.eps;
    a.t = block_type(y, "y");
    return a;
  }
  static const float* vec(const Tensor& t, bool wanted, int64_t D, const Tensor& like, const char* name) {
    if (!wanted) return nullptr;
    BK_CHECK(t.defined() && t.scalar_type() == torch::kFloat32 && t.dim() == 1 && t.size(0) == D &&
                 t.is_contiguous() && t.device() == like.device(),
             name, " must be a contiguous float32 [", D, "] on the input's device");
    return t.data_ptr<float>();
  }
  static void params(ResidualArgs& a, const Tensor& like, const Tensor& gate, const Tensor& post_w,
                     const Tensor& post_b, const Tensor& pre_w, const Tensor& pre_b) {
    a.post_w = vec(post_w, a.post != kNormNone, a.D, like, "post_weight");
    a.post_b = vec(post_b, a.post == kNormLayer, a.D, like, "post_bias");
    a.pre_w = vec(pre_w, a.pre != kNormNone, a.D, like, "pre_weight");
    a.pre_b = vec(pre_b, a.pre == kNormLayer, a.D, like, "pre_bias");
    if (a.gate_kind == kGateChannel) a.gate = vec(gate, true, a.D, like, "gate");
    if (a.gate_kind == kGateRow) {
      BK_CHECK(gate.defined() && gate.scalar_type() == torch::kFloat32 && gate.numel() == a.M && gate.is_contiguous() &&
                   gate.device() == like.device(),
               "a row gate must be a contiguous float32 with one value for each row, on the input's device");
      a.gate = gate.data_ptr();
    }
    if (a.gate_kind == kGateFull) {
      BK_CHECK(gate.defined() && gate.scalar_type() == like.scalar_type() && gate.dim() == 2 && gate.size(0) == a.M &&
                   gate.size(1) == a.D && (a.D == 1 || gate.stride(1) == 1) && gate.device() == like.device(),
               "a full gate must have y's shape, type and device");
      a.gate = gate.data_ptr();
      a.ldg = ld_of(gate, a.M, a.D);
    }
  }

  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const OptTensor& gate_t,
                               const OptTensor& post_wt, const OptTensor& post_bt, const OptTensor& pre_wt,
                               const OptTensor& pre_bt, const OptTensor& seed_t, ResidualOpts o, bool any) {
    c10::DeviceGuard guard(x.device());
    auto v = [](const OptTensor& t) { return t.value_or(Tensor()); };
    const Tensor gate = v(gate_t), post_w = v(post_wt), post_b = v(post_bt), pre_w = v(pre_wt), pre_b = v(pre_bt),
                 seed = v(seed_t);
    const int64_t D = x.size(-1), M = D ? x.numel() / D : 0;
    BK_CHECK(M < (int64_t(1) << 31), "too many rows");
    ResidualArgs a = args(o, y, M, D);
    a.stream_t = block_type(x, "x");
    BK_CHECK(a.stream_t == a.t || a.stream_t == kF32, "x must have y's type or float32");
    BK_CHECK(y.sizes() == x.sizes() && y.device() == x.device(), "x and y must have one shape and device");
    BK_CHECK(D <= kResidualMaxD, "at most ", kResidualMaxD, " columns, not ", D);
    const Tensor xr = rows_of(x, M, D), yr = rows_of(y, M, D);
    Tensor gr = gate;
    if (o.gate_kind == kGateRow) gr = gate.contiguous();
    if (o.gate_kind == kGateFull) gr = rows_of(gate, M, D);
    auto c = [](const Tensor& t) { return t.defined() ? t.contiguous() : t; };
    if (o.gate_kind == kGateChannel) gr = c(gate);
    const Tensor pw = c(post_w), pb = c(post_b), qw = c(pre_w), qb = c(pre_b);
    params(a, yr, gr, pw, pb, qw, qb);
    a.mask = mask_args(o.mask, seed, x);
    Tensor r = torch::empty(x.sizes(), x.options().memory_format(c10::MemoryFormat::Contiguous));
    Tensor h = o.pre ? torch::empty(y.sizes(), y.options().memory_format(c10::MemoryFormat::Contiguous)) : Tensor();
    Tensor stats, used;
    if (any) {
      stats = torch::empty({M, 4}, x.options().dtype(torch::kFloat32));
      a.stats = stats.data_ptr<float>();
      if (a.mask.seed) {
        used = torch::empty({2}, seed.options());
        a.mask.seed_out = used.data_ptr<int64_t>();
      }
    }
    a.x = xr.data_ptr();
    a.ldx = ld_of(xr, M, D);
    a.y = yr.data_ptr();
    a.ldy = ld_of(yr, M, D);
    a.r = r.data_ptr();
    a.h = o.pre ? h.data_ptr() : nullptr;
    launch_residual_fwd(a, stream_of(x));
    launched();
    if (any) {
      // the copies that were made, or views of the inputs: either way what the kernel read
      ctx->save_for_backward({xr, yr, gr, pw, pb, qw, qb, used});
      ctx->saved_data["stats"] = stats;
      for (auto& kv : std::initializer_list<std::pair<const char*, int64_t>>{
               {"post", o.post}, {"pre", o.pre}, {"gk", o.gate_kind}, {"sig", (int64_t)o.sigmoid},
               {"thr", o.mask.thr}, {"seed", o.mask.seed}, {"off", o.mask.offset}})
        ctx->saved_data[kv.first] = kv.second;
      ctx->saved_data["xs"] = o.x_scale;
      ctx->saved_data["ys"] = o.y_scale;
      ctx->saved_data["up"] = o.mask.up;
      ctx->saved_data["shape"] = x.sizes().vec();
      ctx->saved_data["gs"] = gate.defined() ? c10::IValue(gate.sizes().vec()) : c10::IValue(std::vector<int64_t>{});
    }
    ctx->set_materialize_grads(false);
    if (o.pre) return {r, h};
    return {r};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order_only();
    const auto sv = ctx->get_saved_variables();
    auto& sd = ctx->saved_data;
    const Tensor &x = sv[0], &y = sv[1], &gate = sv[2], &post_w = sv[3], &post_b = sv[4], &pre_w = sv[5],
                 &pre_b = sv[6], &used = sv[7];
    c10::DeviceGuard guard(x.device());
    ResidualOpts o{sd["post"].toInt(), sd["pre"].toInt(), sd["gk"].toInt(), sd["sig"].toInt() != 0, sd["xs"].toDouble(),
                   sd["ys"].toDouble(), 0.0, {sd["thr"].toInt(), sd["up"].toDouble(), sd["seed"].toInt(), sd["off"].toInt()}};
    const auto shape = sd["shape"].toIntVector();
    const int64_t M = x.size(0), D = x.size(1);
    ResidualArgs a = args(o, y, M, D);
    a.stream_t = block_type(x, "x");
    params(a, y, gate, post_w, post_b, pre_w, pre_b);
    a.mask = mask_args(o.mask, used, x);
    const Tensor stats = sd["stats"].toTensor();
    a.stats = stats.data_ptr<float>();
    a.x = x.data_ptr();
    a.ldx = ld_of(x, M, D);
    a.y = y.data_ptr();
    a.ldy = ld_of(y, M, D);
    Tensor dr, dh;
    if (g[0].defined()) {
      dr = rows_of(g[0], M, D);
      a.dr = dr.data_ptr();
      a.lddr = ld_of(dr, M, D);
    }
    if (o.pre && g[1].defined()) {
      dh = rows_of(g[1], M, D);
      a.dh = dh.data_ptr();
      a.lddh = ld_of(dh, M, D);
    }
    // edges: the tensor arguments that forward() got, in order, without the absent ones
    const bool have[7] = {true, true, gate.defined(), post_w.defined(), post_b.defined(), pre_w.defined(), pre_b.defined()};
    auto want = [&](int i) {
      if (!have[i]) return false;
      int edge = 0;
      for (int j = 0; j < i; ++j) edge += have[j];
      return ctx->needs_input_grad(edge);
    };
    auto like_x = x.options(), like_y = y.options(), f32 = x.options().dtype(torch::kFloat32);
    variable_list out(10);
    if (want(0)) a.dx = (out[0] = torch::empty(shape, like_x)).data_ptr();
    if (want(1)) a.dy = (out[1] = torch::empty(shape, like_y)).data_ptr();
    if (want(2)) {
      out[2] = torch::empty(sd["gs"].toIntVector(), o.gate_kind == kGateFull ? like_y : f32);
      a.dgate = out[2].data_ptr();
    }
    float** vecs[4] = {&a.dpost_w, &a.dpost_b, &a.dpre_w, &a.dpre_b};
    for (int i = 0; i < 4; ++i)
      if (want(3 + i)) *vecs[i] = (out[3 + i] = torch::empty({D}, f32)).data_ptr<float>();
    if (M == 0) {  // no row: the sums over rows are zero
      for (auto& t : out)
        if (t.defined()) t.zero_();
      return out;
    }
    Tensor slab;
    if (const int nvec = residual_nvec(a)) {
      slab = torch::empty({(int64_t)residual_slab_rows(M, (int)D), nvec, D}, f32);
      a.slab = slab.data_ptr<float>();
    }
    launch_residual_bwd(a, stream_of(x));
    launched();
    return out;
  }
};

std::vector<Tensor> block_residual(const Tensor& x, const Tensor& y, const OptTensor& gate,
                                   const OptTensor& post_w, const OptTensor& post_b,
                                   const OptTensor& pre_w, const OptTensor& pre_b,
                                   const OptTensor& seed, int64_t post, int64_t pre, int64_t gate_kind,
                                   bool sigmoid, double x_scale, double y_scale, double eps, int64_t thr,
                                   double up, int64_t seed_v, int64_t offset_v) {
  BK_CHECK(x.is_cuda() && y.is_cuda(), "x and y must be GPU tensors");
  BK_CHECK(x.dim() >= 1, "x must have at least one dimension");
  BK_CHECK(post >= 0 && post <= 2 && pre >= 0 && pre <= 2 && gate_kind >= 0 && gate_kind <= 3, "unknown kind");
  return ResidualFn::apply(
      x, y, gate, post_w, post_b, pre_w, pre_b, seed,
      ResidualOpts{post, pre, gate_kind, sigmoid, x_scale, y_scale, eps, {thr, up, seed_v, offset_v}},
      wants_grad({x, y, gate, post_w, post_b, pre_w, pre_b}, x));
}

// ------------------------------------------------------------------ 8-bit fc
constexpr int64_t kFp8MaxDim = 65535 * 128;  // keeps tiles, rows and columns in 32 bits

void fp8_dims(int64_t a, int64_t b) {
  BK_CHECK(a <= kFp8MaxDim && b <= kFp8MaxDim, "fp8: at most ", kFp8MaxDim, " rows or columns");
}

// codes and exponent bytes of a [rows, K] matrix, in a part of an allocation
struct Fp8Buf {
  uint8_t* codes = nullptr;
  int64_t rows = 0, K = 0;
  uint8_t* scales() const { return codes + rows * fp8_kp(K); }
  static int64_t bytes(int64_t rows, int64_t K) { return (rows * (fp8_kp(K) + fp8_sp(K)) + 255) / 256 * 256; }
};
// parts of one allocation, each at a multiple of 256 bytes
class Parts {
 public:
  int64_t add(int64_t bytes) {
    const int64_t at = size_;
    size_ += (bytes + 255) / 256 * 256;
    return at;
  }
  void allocate(const Tensor& like) { mem = torch::empty({size_}, like.options().dtype(torch::kUInt8)); }
  uint8_t* at(int64_t offset) const { return mem.data_ptr<uint8_t>() + offset; }
  Fp8Buf blocks(int64_t offset, int64_t rows, int64_t K) const { return {at(offset), rows, K}; }
  Tensor mem;

 private:
  int64_t size_ = 0;
};

Fp8QuantArgs quant_args(const Tensor& x, int64_t M, int64_t K, bool tile) {
  Fp8QuantArgs q;
  q.x = x.data_ptr();
  q.t = block_type(x, "x");
  q.M = M;
  q.K = K;
  q.ld = ld_of(x, M, K);
  q.tile = tile;
  return q;
}

Fp8GemmArgs gemm_args(const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, int64_t M, int64_t N,
                      int64_t K, const float* bias, const Tensor& c) {
  Fp8GemmArgs g;
  g.a = a;
  g.sa = sa;
  g.b = b;
  g.sb = sb;
  g.M = (int)M;
  g.N = (int)N;
  g.K = K;
  g.bias = bias;
  g.c = c.data_ptr();
  g.ct = block_type(c, "the result");
  return g;
}
Fp8GemmArgs gemm_args(const Fp8Buf& a, const Fp8Buf& b, const float* bias, const Tensor& c) {
  return gemm_args(a.codes, a.scales(), b.codes, b.scales(), a.rows, b.rows, a.K, bias, c);
}
void fp8_product(Fp8GemmArgs g, const Tensor& c) {
  g.ksplit = fp8_gemm_ksplit(g.M, g.N, g.K);
  Tensor slab;
  if (g.ksplit > 1) {
    slab = torch::empty({(int64_t)g.ksplit, g.M, g.N}, c.options().dtype(torch::kFloat32));
    g.slab = slab.data_ptr<float>();
  }
  launch_fp8_gemm(g, stream_of(c));
  launched();
}

const float* bias_of(const Tensor& b, int64_t N, const Tensor& like) {
  if (!b.defined()) return nullptr;
  BK_CHECK(b.scalar_type() == torch::kFloat32 && b.numel() == N && b.is_contiguous() && b.device() == like.device(),
           "a bias is a contiguous float32 [", N, "] on the input's device");
  return b.data_ptr<float>();
}

// x [M, K] -> (codes, scales) in blocks along K, or of x^T in blocks along M
std::vector<Tensor> block_fp8_quantize(const Tensor& x, bool tile, bool transposed) {
  BK_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) > 0, "x must be a GPU matrix");
  c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1);
  fp8_dims(M, K);
  const Tensor xr = rows_of(x.detach(), M, K);
  auto q = quant_args(xr, M, K, tile);
  const int64_t rows = transposed ? K : M, cols = transposed ? M : K;
  auto codes = torch::empty({rows, fp8_kp(cols)}, x.options().dtype(torch::kFloat8_e4m3fn));
  auto scales = torch::empty({rows, fp8_sp(cols)}, x.options().dtype(torch::kUInt8));
  uint8_t* c = reinterpret_cast<uint8_t*>(codes.data_ptr());
  (transposed ? q.col_codes : q.row_codes) = c;
  (transposed ? q.col_scales : q.row_scales) = scales.data_ptr<uint8_t>();
  launch_fp8_quant(q, stream_of(x));
  launched();
  return {codes, scales};
}

void check_blocks(const Tensor& codes, const Tensor& scales, int64_t K, const char* name) {
  BK_CHECK(codes.is_cuda() && codes.scalar_type() == torch::kFloat8_e4m3fn && codes.dim() == 2 && codes.is_contiguous() &&
               codes.size(1) == fp8_kp(K) && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
           name, " codes must be a contiguous float8_e4m3fn [rows, ", fp8_kp(K), "] at a 16-byte address");
  BK_CHECK(scales.device() == codes.device() && scales.scalar_type() == torch::kUInt8 && scales.dim() == 2 &&
               scales.is_contiguous() && scales.size(0) == codes.size(0) && scales.size(1) == fp8_sp(K) &&
               reinterpret_cast<uintptr_t>(scales.data_ptr()) % 4 == 0,
           name, " scales must be a contiguous uint8 [rows, ", fp8_sp(K), "] beside the codes");
  fp8_dims(codes.size(0), K);
}
const uint8_t* bytes(const Tensor& t) { return reinterpret_cast<const uint8_t*>(t.data_ptr()); }

Tensor block_fp8_matmul(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, int64_t K,
                        const OptTensor& bias, at::ScalarType out) {
  check_blocks(a, sa, K, "a");
  check_blocks(b, sb, K, "b");
  BK_CHECK(a.device() == b.device(), "a and b must be on one device");
  c10::DeviceGuard guard(a.device());
  const Tensor bc = bias.has_value() ? bias->detach().contiguous() : Tensor();
  auto c = torch::empty({a.size(0), b.size(0)}, a.options().dtype(out));
  fp8_product(gemm_args(bytes(a), bytes(sa), bytes(b), bytes(sb), a.size(0), b.size(0), K, bias_of(bc, b.size(0), a), c), c);
  return c;
}

// y = q(x) q(W) + b with a packed weight (codes of W^T)
Tensor block_fp8_fc_packed(const Tensor& x, const Tensor& codes, const Tensor& scales, const OptTensor& b) {
  BK_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) > 0, "x must be a GPU matrix");
  check_blocks(codes, scales, x.size(1), "weight");
  BK_CHECK(codes.device() == x.device(), "x and the weight must be on one device");
  c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), O = codes.size(0);
  fp8_dims(M, O);
  const Tensor xr = rows_of(x.detach(), M, K), bc = b.has_value() ? b->detach().contiguous() : Tensor();
  auto q = quant_args(xr, M, K, false);
  Parts tmp;
  tmp.add(Fp8Buf::bytes(M, K));
  tmp.allocate(x);
  const Fp8Buf xq = tmp.blocks(0, M, K);
  q.row_codes = xq.codes;
  q.row_scales = xq.scales();
  launch_fp8_quant(q, stream_of(x));
  launched();
  auto y = torch::empty({M, O}, x.options().memory_format(c10::MemoryFormat::Contiguous));
  fp8_product(gemm_args(xq.codes, xq.scales(), bytes(codes), bytes(scales), M, O, K, bias_of(bc, O, x), y), y);
  return y;
}

// Training: x and dy are held in blocks along K / O for the forward and dx
// and, from the same read, in blocks along the batch for dW; W in 128 x 128
// blocks, whose codes serve the forward and dx alike.  What the backward keeps
// is 8 bits a value: x^T's codes and W's.
class Fp8FcFn : public torch::autograd::Function<Fp8FcFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& W, const OptTensor& b, bool grad) {
    c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), K = x.size(1), O = W.size(1);
    const Tensor xr = rows_of(x, M, K), Wr = rows_of(W, K, O), bc = b.has_value() ? b->contiguous() : Tensor();
    const bool need_dx = grad && x.requires_grad(), need_dw = grad && W.requires_grad();
    auto s = stream_of(x);
    // the forward's own: codes of W^T and x; the backward's: codes of W (for dx) and x^T (for dW)
    Parts tmp, kept;
    const int64_t at_wt = tmp.add(Fp8Buf::bytes(O, K)), at_xq = tmp.add(Fp8Buf::bytes(M, K));
    tmp.allocate(x);
    const Fp8Buf wt = tmp.blocks(at_wt, O, K), xq = tmp.blocks(at_xq, M, K);
    const int64_t at_wq = need_dx ? kept.add(Fp8Buf::bytes(K, O)) : 0, at_xt = need_dw ? kept.add(Fp8Buf::bytes(K, M)) : 0;
    if (need_dx || need_dw) kept.allocate(x);
    auto qw = quant_args(Wr, K, O, true);
    qw.col_codes = wt.codes;
    qw.col_scales = wt.scales();
    if (need_dx) {
      const Fp8Buf wq = kept.blocks(at_wq, K, O);
      qw.row_codes = wq.codes;
      qw.row_scales = wq.scales();
    }
    auto qx = quant_args(xr, M, K, false);
    qx.row_codes = xq.codes;
    qx.row_scales = xq.scales();
    if (need_dw) {
      const Fp8Buf xt = kept.blocks(at_xt, K, M);
      qx.col_codes = xt.codes;
      qx.col_scales = xt.scales();
    }
    launch_fp8_quant_two(qx, qw, s);
    launched();
    auto y = torch::empty({M, O}, x.options().memory_format(c10::MemoryFormat::Contiguous));
    fp8_product(gemm_args(xq, wt, bias_of(bc, O, x), y), y);
    ctx->save_for_backward({kept.mem});
    ctx->saved_data["wq"] = at_wq;
    ctx->saved_data["xt"] = at_xt;
    ctx->saved_data["M"] = M;
    ctx->saved_data["K"] = K;
    ctx->saved_data["O"] = O;
    ctx->saved_data["wt"] = (int64_t)W.scalar_type();
    ctx->saved_data["bs"] = b.has_value() ? c10::IValue(b->sizes().vec()) : c10::IValue();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order_only();
    c10::DeviceGuard guard(g[0].device());
    auto& sd = ctx->saved_data;
    const int64_t M = sd["M"].toInt(), K = sd["K"].toInt(), O = sd["O"].toInt();
    const auto sv = ctx->get_saved_variables();
    const bool has_b = !sd["bs"].isNone();
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1),
               want_b = has_b && ctx->needs_input_grad(2);
    const Tensor dy = rows_of(g[0], M, O);
    Tensor dx, dW, db;
    auto q = quant_args(dy, M, O, false);
    Parts tmp;
    const int64_t at_dq = want_x ? tmp.add(Fp8Buf::bytes(M, O)) : 0, at_dt = want_w ? tmp.add(Fp8Buf::bytes(O, M)) : 0,
                  at_slab = want_b ? tmp.add((M + 127) / 128 * O * 4) : 0;
    if (want_x) dx = torch::empty({M, K}, dy.options());
    if (want_w) dW = torch::empty({K, O}, dy.options().dtype((at::ScalarType)sd["wt"].toInt()));
    if (want_b) db = torch::empty(sd["bs"].toIntVector(), dy.options().dtype(torch::kFloat32));
    if (M == 0) {  // no row: the sums over rows are zero
      if (want_w) dW.zero_();
      if (want_b) db.zero_();
      return {dx, dW, db, Tensor()};
    }
    if (!(want_x || want_w || want_b)) return {dx, dW, db, Tensor()};
    uint8_t* kept = sv[0].defined() ? sv[0].data_ptr<uint8_t>() : nullptr;
    // the products' arguments but for the temporaries' addresses, which the slices decide on
    Fp8GemmArgs gx, gw;
    bool two = false;
    int64_t at_gx = 0, at_gw = 0;
    const Fp8Buf wq{kept + sd["wq"].toInt(), K, O}, xt{kept + sd["xt"].toInt(), K, M};
    if (want_x) gx = gemm_args(Fp8Buf{nullptr, M, O}, wq, nullptr, dx);
    if (want_w) gw = gemm_args(xt, Fp8Buf{nullptr, O, M}, nullptr, dW);
    if (want_x && want_w && fp8_gemm_two_split(gx, gw)) {
      two = true;
      if (gx.ksplit > 1) at_gx = tmp.add((int64_t)gx.ksplit * M * K * 4);
      if (gw.ksplit > 1) at_gw = tmp.add((int64_t)gw.ksplit * K * O * 4);
    }
    tmp.allocate(dy);
    const Fp8Buf dq = tmp.blocks(at_dq, M, O), dt = tmp.blocks(at_dt, O, M);
    if (want_x) {
      gx.a = q.row_codes = dq.codes;
      q.row_scales = dq.scales();
      gx.sa = dq.scales();
    }
    if (want_w) {
      q.col_codes = dt.codes;
      q.col_scales = dt.scales();
      gw.b = dt.codes;
      gw.sb = dt.scales();
    }
    if (want_b) {
      q.slab = reinterpret_cast<float*>(tmp.at(at_slab));
      if (!two) q.colsum = db.data_ptr<float>();
    }
    launch_fp8_quant(q, stream_of(dy));
    launched();
    if (two) {
      gx.slab = reinterpret_cast<float*>(tmp.at(at_gx));
      gw.slab = reinterpret_cast<float*>(tmp.at(at_gw));
      launch_fp8_gemm_two(gx, gw, q.slab, (M + 127) / 128, O, want_b ? db.data_ptr<float>() : nullptr, stream_of(dy));
      launched();
    } else {
      if (want_x) fp8_product(gx, dx);
      if (want_w) fp8_product(gw, dW);
    }
    return {dx, dW, db, Tensor()};
  }
};

Tensor block_fp8_fc(const Tensor& x, const Tensor& W, const OptTensor& b) {
  BK_CHECK(x.is_cuda() && x.dim() == 2 && W.dim() == 2 && x.size(1) == W.size(0) && x.size(1) > 0 && W.size(1) > 0 &&
               x.device() == W.device(),
           "x [N, K] and W [K, O] must be GPU matrices on one device");
  block_type(x, "x");
  block_type(W, "W");
  fp8_dims(x.size(0), x.size(1));
  fp8_dims(W.size(1), 1);
  return Fp8FcFn::apply(x, W, b, wants_grad({x, W, b}, x));
}

}  // namespace

void bind_block(py::module_& m) {
  m.def("block_dropout", &block_dropout);
  m.def("block_residual", &block_residual);
  m.def("block_fp8_quantize", &block_fp8_quantize);
  m.def("block_fp8_matmul", [](const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, int64_t K,
                               const OptTensor& bias, py::object dtype) {
    return block_fp8_matmul(a, sa, b, sb, K, bias, torch::python::detail::py_object_to_dtype(dtype));
  });
  m.def("block_fp8_fc_packed", &block_fp8_fc_packed);
  m.def("block_fp8_fc", &block_fp8_fc);
}

}  // namespace pbx

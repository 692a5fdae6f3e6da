// ATen face of the feed-forward operators: linear, gated_linear, dropout, residual_norm.
//
// Each has an explicit forward / backward pair (what the model's units call) and a differentiable form whose autograd node is
// C++, so that a training call costs no Python in its backward pass.  All checks are on the host, wrong arguments raise
// ValueError.  Launches go to PyTorch's current stream of the inputs' device; workspaces come from the caching allocator for
// the one call, so streams and captured graphs never share one.
#include "torch_hip.h"
#include "ddl_kernels.h"
#include "ffn_common.h"
#include "ffn_misc.h"
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <string>

namespace {

using at::Tensor;
using OptT = std::optional<Tensor>;
using ddl::cur_stream;
namespace ffn = ddl::ffn;
#define BAD_UNLESS(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

int type_of(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat: return ffn::F32;
    case at::kBFloat16: return ffn::BF16;
    case at::kHalf: return ffn::F16;
    default: break;
  }
  BAD_UNLESS(false, op, ": float32, bfloat16 or float16 expected, got ", t.scalar_type());
  return 0;
}
// The tensor whose memory holds its values: PyTorch marks lazily negated views (the imaginary part of a conjugate) and zeros without
// memory, which its own operators resolve in its dispatcher and a kernel that reads memory would not see.
Tensor in_memory(const Tensor& t) {
  if (!t.defined() || !(t.is_neg() || t._is_zerotensor())) return t;
  return t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg();
}
bool has(const OptT& t) { return t.has_value() && t->defined(); }
Tensor get(const OptT& t) { return has(t) ? *t : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
long up(long n, long to) { return (n + to - 1) / to * to; }

// The operators have a backward pass and no forward-mode derivative.  Their kernels see values only, so a tangent would be lost without a
// word: a call on a dual tensor is refused.
void no_tangent(const Tensor& t, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), op,
                              ": no forward-mode derivative (an argument is a dual tensor of torch.autograd.forward_ad)");
}
void no_tangents(std::initializer_list<const Tensor*> ts, const char* op) {
  for (const Tensor* t : ts) no_tangent(*t, op);
}

// torch.jit.trace and make_fx record what goes through PyTorch's dispatcher; these calls do not.  A recorded program would hold this
// call's result as a constant, so a call is refused while either records.
void not_recorded(const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                              op, ": cannot be recorded by torch.jit.trace or make_fx");
}

// `t` may stand beside `x` in a call: same device and type
void check_like(const Tensor& t, const Tensor& x, const char* op, const char* name) {
  BAD_UNLESS(t.device() == x.device(), op, ": ", name, " is on ", t.device(), ", the input on ", x.device());
  BAD_UNLESS(t.scalar_type() == x.scalar_type(), op, ": ", name, " is ", t.scalar_type(), ", the input ", x.scalar_type());
}
int rows_fit(int64_t n, const char* op) {
  BAD_UNLESS(n <= (1 << 30), op, ": at most 2^30 rows, got ", n);
  return (int)n;
}
int width_fits(int64_t n, const char* op) {                          // a launch has fewer than 2^32 threads, up to 32 a column
  BAD_UNLESS(n <= (1 << 26), op, ": rows of at most 2^26 columns, got ", n);
  return (int)n;
}
// [.., C] as [rows, C] whose columns are contiguous
Tensor rows_of(const Tensor& t) {
  const int64_t c = t.size(-1);
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  Tensor v = t.dim() == 2 ? t : t.reshape({rows, c});
  return c > 1 && v.numel() > 0 && v.stride(1) != 1 ? v.contiguous() : v;
}
long row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : up(t.size(1), 16); }
bool rows_aligned(const Tensor& t) {
  return aligned(t.data_ptr()) && (t.size(0) <= 1 || t.stride(0) * t.element_size() % 16 == 0);
}

// An operand of a product: 16-byte aligned rows of whole 16-byte chunks.  A tensor that is not laid out so (odd widths, a column
// slice, a transposed view) is packed into a copy whose rows are padded with zeros to 128 bytes, one pass over it.  Training
// keeps the copy instead of the tensor, so the backward pass finds it packed: [rows, padded] with the width known from elsewhere.
// An operand owns the tensor it is packed from: the packing launch comes after all operands are set up, and memory given back before
// it could become one of the others' copies.
struct Operand {
  Tensor keep, source;
  const void* p = nullptr;
  long ld = 0;
};
long line(int64_t n, const Tensor& like) { return up(n, 128 / like.element_size()); }
bool is_operand(const Tensor& t) {
  const int64_t epc = 16 / t.element_size();
  return t.numel() == 0 || ((t.size(1) <= 1 || t.stride(1) == 1) && t.size(1) % epc == 0 && rows_aligned(t));
}
// t: 2-D [rows, width] of any strides, or packed already.  What has to be packed joins `todo`, for one launch.
Operand operand(const Tensor& t, int64_t width, ffn::PackArgs& todo) {
  Operand o;
  o.source = t;
  if (t.size(1) != width) {
    o.keep = t;
    o.p = t.data_ptr();
    o.ld = t.size(1);
    return o;
  }
  if (is_operand(t)) {
    o.keep = t;
    o.p = t.numel() ? t.data_ptr() : nullptr;
    o.ld = row_stride(t);
    return o;
  }
  o.ld = line(t.size(1), t);
  o.keep = at::empty({t.size(0), o.ld}, t.options());
  ffn::PackItem& it = todo.item[todo.count++];
  it.src = t.data_ptr();
  it.dst = o.keep.data_ptr();
  it.s_row = t.stride(0);
  it.s_col = t.stride(1);
  it.ld = o.ld;
  it.rows = t.size(0);
  it.cols = (int)t.size(1);
  o.p = o.keep.data_ptr();
  return o;
}
Operand own_operand(const Tensor& padded) {                          // a padded buffer of ours
  Operand o;
  o.keep = padded;
  o.p = padded.data_ptr();
  o.ld = padded.size(1);
  return o;
}

void set_out(ffn::Epilogue& e, int i, const Tensor& out) {
  e.out[i] = out.data_ptr();
  e.ldo = out.size(1);
  e.out_vec = (i == 0 || e.out_vec) && aligned(out.data_ptr()) && out.size(1) * out.element_size() % 16 == 0;
}
void run_gemm(int dtype, ffn::GemmArgs& g, const Tensor& like) {
  const ffn::GemmPlan plan = ffn::gemm_plan(dtype, g);
  BAD_UNLESS(plan.bm > 0, "a product of ", g.M, " x ", g.N, " results is more than one launch holds");
  Tensor ws;
  if (plan.partial_floats > 0) {
    ws = at::empty({plan.partial_floats}, like.options().dtype(at::kFloat));
    g.partial = ws.data_ptr<float>();
  }
  ffn::launch_gemm(dtype, g, plan, cur_stream());
}

// ---- linear and gated_linear ------------------------------------------------------------------------------------------
int check_act(int64_t act, const char* op) {
  BAD_UNLESS(act >= 0 && act < ffn::N_ACT, op, ": unknown activation ", act);
  return (int)act;
}
void check_product(const Tensor& x, const Tensor& w, const OptT& b, const char* op, const char* wname, const char* bname) {
  BAD_UNLESS(x.is_cuda(), op, ": GPU tensor expected");
  type_of(x, op);
  BAD_UNLESS(x.dim() >= 1 && w.dim() == 2, op, ": x [.., K] and ", wname, " [N, K] expected, got ", x.sizes(), " and ", w.sizes());
  BAD_UNLESS(x.size(-1) == w.size(1), op, ": x ", x.sizes(), " and ", wname, " ", w.sizes(), " differ in their last size");
  check_like(w, x, op, wname);
  if (has(b)) {
    BAD_UNLESS(b->dim() == 1 && b->size(0) == w.size(0), op, ": ", bname, " [", w.size(0), "] expected, got ", b->sizes());
    check_like(*b, x, op, bname);
  }
}
std::vector<int64_t> out_sizes(const Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}

// The three products of [M, K] x [N, K]^T as the kernels see them
ffn::GemmArgs forward_shape(int M, int K, int N, bool dual) {
  ffn::GemmArgs g;
  g.N = N; g.M = M; g.K = K;
  g.dual = dual;
  return g;
}
ffn::GemmArgs dx_shape(int M, int K, int N, int weights) {           // dx[m][k] = sum over weights, n of dz[m][n] w[n][k]
  ffn::GemmArgs g;
  g.N = K; g.M = M; g.K = N;
  g.nseg = weights;
  g.p_kc = false;
  return g;
}
ffn::GemmArgs dw_shape(int M, int K, int N, int weights) {           // dw[n][k] = sum over m of dz[m][n] x[m][k]
  ffn::GemmArgs g;
  g.N = K; g.M = N; g.K = M;
  g.nout = weights;
  g.p_kc = g.q_kc = false;
  return g;
}
// -> rows and columns of the tile, splits: what the cost rule gives a product of more than FEW_ROWS rows (host only)
std::tuple<int, int, int> product_plan(const std::string& what, const std::string& type, int64_t M, int64_t K, int64_t N, bool dual) {
  BAD_UNLESS(what == "forward" || what == "dx" || what == "dw", "product_plan: forward, dx or dw expected, got ", what);
  BAD_UNLESS(type == "fp32" || type == "bf16" || type == "fp16", "product_plan: fp32, bf16 or fp16 expected, got ", type);
  const int m = rows_fit(M, "product_plan"), k = width_fits(K, "product_plan"), n = width_fits(N, "product_plan"), weights = dual ? 2 : 1;
  const ffn::GemmArgs g = what == "forward" ? forward_shape(m, k, n, dual) : what == "dx" ? dx_shape(m, k, n, weights)
                                                                                         : dw_shape(m, k, n, weights);
  const ffn::GemmPlan plan = ffn::gemm_plan(type == "fp32" ? ffn::F32 : type == "bf16" ? ffn::BF16 : ffn::F16, g);
  return {plan.bm, plan.bn, plan.splits};
}

// What a product keeps for its backward pass: the fp32 sums z (one or two planes [M, ldz]; none without an activation), and x and the
// weights as they were packed (otherwise as given).
struct Kept { Tensor z, x, w[2]; };

// One or two weights -> out [M, N].
Tensor product_forward(const Tensor& x_in, const Tensor& w0_in, const Tensor& w1_in, const Tensor& b0_in, const Tensor& b1_in,
                       const Tensor& res_in, int act, bool keep_sums, Kept* kept, const char* op) {
  const Tensor x = in_memory(x_in), w0 = in_memory(w0_in), w1 = in_memory(w1_in), b0 = in_memory(b0_in), b1 = in_memory(b1_in),
               res = in_memory(res_in);
  const int dtype = type_of(x, op);
  const Tensor x2 = rows_of(x);
  const int M = rows_fit(x2.size(0), op), K = width_fits(x2.size(1), op), N = width_fits(w0.size(0), op);
  const bool dual = w1.defined();
  Tensor out = at::empty({M, N}, x.options()), z;
  if (keep_sums) z = at::empty({dual ? 2 : 1, M, up(N, 16)}, x.options().dtype(at::kFloat));
  if (kept != nullptr) *kept = {z, x, {w0, w1}};
  if (M == 0 || N == 0) return out;
  ffn::Epilogue e;
  set_out(e, 0, out);
  e.act = act;
  Tensor bias0 = b0.defined() ? b0.contiguous() : b0, bias1 = b1.defined() ? b1.contiguous() : b1, r2;
  e.bias[0] = ptr(bias0);
  e.bias[1] = ptr(bias1);
  e.bias_vec = aligned(e.bias[0]) && aligned(e.bias[1]);
  if (res.defined()) {
    r2 = rows_of(res);
    e.residual = r2.data_ptr();
    e.ldr = row_stride(r2);
    e.res_vec = rows_aligned(r2);
  }
  if (keep_sums) {
    e.ldz = z.size(2);
    e.z[0] = z.data_ptr<float>();
    if (dual) e.z[1] = e.z[0] + (long)M * e.ldz;
  }
  if (M <= ffn::FEW_ROWS) {
    const Tensor wa = rows_of(w0), wb = dual ? rows_of(w1) : w1;
    ffn::FewRowsArgs f;
    f.N = N; f.M = M; f.K = K;
    f.dual = dual;
    f.vec = is_operand(wa) && is_operand(x2) && (!dual || is_operand(wb));
    f.ep = e;
    if (K > 0) {
      f.w[0] = wa.data_ptr();
      f.ldw[0] = row_stride(wa);
      if (dual) {
        f.w[1] = wb.data_ptr();
        f.ldw[1] = row_stride(wb);
      }
      f.x = x2.data_ptr();
      f.ldx = row_stride(x2);
    }
    ffn::launch_few_rows(dtype, f, cur_stream());
    return out;
  }
  ffn::PackArgs todo;
  const Operand xo = operand(x2, K, todo), wo = operand(w0, K, todo), vo = dual ? operand(w1, K, todo) : Operand();
  ffn::launch_pack(dtype, todo, cur_stream());
  if (kept != nullptr) {
    if (xo.keep.size(1) != K) kept->x = xo.keep;
    if (wo.keep.size(1) != K) kept->w[0] = wo.keep;
    if (dual && vo.keep.size(1) != K) kept->w[1] = vo.keep;
  }
  ffn::GemmArgs g = forward_shape(M, K, N, dual);
  g.p[0] = wo.p; g.ldp[0] = wo.ld;
  g.p[1] = vo.p; g.ldp[1] = vo.ld;
  g.q[0] = xo.p; g.ldq[0] = xo.ld;
  g.ep = e;
  run_gemm(dtype, g, x);
  return out;
}

// Gradients of a product with one or two weights [N, K] from dy [.., N] and what the forward pass kept.
struct ProductGrads { Tensor dx, dw[2], db[2]; };
ProductGrads product_backward(const Tensor& dy, const Kept& kept, int64_t width, int act, bool need_dx, bool need_dw, bool need_db,
                              const char* op) {
  not_recorded(op);
  const Tensor x = in_memory(kept.x), w0 = in_memory(kept.w[0]), w1 = in_memory(kept.w[1]), &z = kept.z;
  const int dtype = type_of(x, op);
  const Tensor x2 = rows_of(x), dy2 = rows_of(in_memory(dy));
  const int M = rows_fit(dy2.size(0), op), K = width_fits(width, op), N = width_fits(dy2.size(1), op);
  const bool dual = w1.defined();
  const int D = dual ? 2 : 1;
  ProductGrads r;
  if (need_dx) r.dx = at::empty({M, K}, x.options());
  for (int d = 0; d < D; ++d) {
    if (need_dw) r.dw[d] = at::empty({N, K}, x.options());
    if (need_db) r.db[d] = at::empty({N}, x.options());
  }
  if (M == 0 || N == 0) {                                            // sums over nothing
    if (need_dx) r.dx.zero_();
    for (int d = 0; d < D; ++d) {
      if (need_dw) r.dw[d].zero_();
      if (need_db) r.db[d].zero_();
    }
    return r;
  }
  // dz in padded rows; without an activation dz is dy itself.  The 16-bit products read dz rounded to their type: with the outputs' own
  // rounding that makes a gradient's error sqrt(2) times one rounding, where many of them average.  Few rows may not average (one
  // row, 64 columns: 1.57 times the rounding alone, four columns: 3), and their products have time to spare.  So up to FEW_ROWS rows
  // dz comes in two parts, the rounded one in rows 0 .. M-1 and what it lacks in rows M .. 2M-1: d_x sums both rows' outputs in
  // fp32 before it rounds, d_w adds the parts before it multiplies.  Above that the other way, two parts for every product, was not taken:
  // the matrix cores are what bounds the large ones, and both gradients would multiply twice as much.
  // fp16: dz, which is no result, may lie outside the type's range where the gradients lie inside.  It is held times a power of two
  // (act_bwd_rescale_kernel), and the products' fp32 sums are scaled back.
  const bool make_dz = z.defined() && (need_dx || need_dw);
  const bool few = M <= ffn::FEW_ROWS, two = make_dz && dtype != ffn::F32 && few;
  const int R = two ? 2 * M : M;
  Tensor dz, range;
  const float* scale = nullptr;                                      // what dz is held in (fp16)
  Operand dzo[2], wo[2], xo;
  ffn::PackArgs todo;
  if (make_dz) {
    dz = at::empty({D, R, line(N, x)}, x.options());
    for (int d = 0; d < D; ++d) dzo[d] = own_operand(dz[d]);
  } else if (need_dx || (need_dw && !few)) {
    dzo[0] = operand(dy2, N, todo);
  }
  if (K > 0 && need_dx) {
    wo[0] = operand(w0, K, todo);
    if (dual) wo[1] = operand(w1, K, todo);
  }
  if (K > 0 && need_dw && !few) xo = operand(x2, K, todo);
  ffn::launch_pack(dtype, todo, cur_stream());
  if (make_dz || need_db) {
    ffn::ActBwdArgs b;
    b.dy = dy2.data_ptr();
    b.ldy = row_stride(dy2);
    b.dy_vec = rows_aligned(dy2);
    b.act = act;
    b.dual = dual;
    b.M = M; b.N = N;
    b.two = two;
    b.ldd = line(N, x);
    b.ldz = up(N, 16);
    Tensor part;
    if (z.defined())
      for (int d = 0; d < D; ++d) {
        b.z[d] = z.data_ptr<float>() + (long)d * M * b.ldz;
        if (make_dz) b.dz[d] = const_cast<void*>(dzo[d].p);
      }
    b.chunks = ffn::act_bwd_chunks(dtype, M, N);
    if (make_dz && dtype == ffn::F16) {
      const int64_t tiles = ffn::act_bwd_tiles(dtype, b);
      range = at::empty({tiles + 1}, x.options().dtype(at::kFloat));
      b.range = range.data_ptr<float>();
      scale = b.scale = b.range + tiles;
    }
    void* outs[2] = {need_db ? r.db[0].data_ptr() : nullptr, need_db && dual ? r.db[1].data_ptr() : nullptr};
    if (need_db && b.chunks == 1) {
      b.db[0] = outs[0];
      b.db[1] = outs[1];
    } else if (need_db) {
      part = at::empty({b.chunks, D, N}, x.options().dtype(at::kFloat));
      b.part = part.data_ptr<float>();
    }
    ffn::launch_act_bwd(dtype, b, cur_stream());
    if (b.part != nullptr) {
      ffn::launch_colsum(dtype, b.part, b.chunks, D, N, outs, cur_stream());
    }
  }
  if (K == 0) return r;
  if (need_dx) {
    ffn::GemmArgs g = dx_shape(R, K, N, D);
    g.halves = two;
    for (int d = 0; d < D; ++d) {
      g.p[d] = wo[d].p; g.ldp[d] = wo[d].ld;
      g.q[d] = dzo[d].p; g.ldq[d] = dzo[d].ld;
    }
    set_out(g.ep, 0, r.dx);
    g.ep.scale = scale;
    run_gemm(dtype, g, x);
  }
  if (need_dw && few) {
    ffn::OuterArgs o;
    o.M = M; o.N = N; o.K = K;
    o.nout = D;
    o.x = x2.data_ptr();
    o.ldx = row_stride(x2);
    o.x_vec = rows_aligned(x2);
    o.two = two;
    o.scale = scale;
    o.ldd = make_dz ? dzo[0].ld : row_stride(dy2);
    o.out_vec = (int64_t)K * x.element_size() % 16 == 0;
    for (int d = 0; d < D; ++d) {
      o.dz[d] = make_dz ? dzo[d].p : dy2.data_ptr();
      o.out[d] = r.dw[d].data_ptr();
    }
    ffn::launch_outer(dtype, o, cur_stream());
  } else if (need_dw) {
    ffn::GemmArgs g = dw_shape(M, K, N, D);
    g.p[0] = xo.p; g.ldp[0] = xo.ld;
    for (int d = 0; d < D; ++d) {
      g.q[d] = dzo[d].p; g.ldq[d] = dzo[d].ld;
      set_out(g.ep, d, r.dw[d]);
    }
    g.ep.scale = scale;
    run_gemm(dtype, g, x);
  }
  return r;
}

void no_second_derivative(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": no second derivative (backward was called with create_graph)");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// what linear checks; then the pieces that the model's units call: forward -> (y, z), backward -> (dx, dw, db)
void check_linear(const Tensor& x, const Tensor& w, const OptT& b, const OptT& res, int64_t act) {
  const Tensor bias = get(b), residual = get(res);
  not_recorded("linear");
  no_tangents({&x, &w, &bias, &residual}, "linear");
  check_product(x, w, b, "linear", "weight", "bias");
  check_act(act, "linear");
  if (has(res)) {
    check_like(*res, x, "linear", "residual");
    BAD_UNLESS(res->sizes().vec() == out_sizes(x, w.size(0)), "linear: residual ", res->sizes(), " where the result is ",
               out_sizes(x, w.size(0)));
  }
}
std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const OptT& b, const OptT& res, int64_t act, bool keep) {
  check_linear(x, w, b, res, act);
  ddl::DeviceGuard guard(x.device());
  Kept kept;
  Tensor y = product_forward(x, w, Tensor(), get(b), Tensor(), get(res), (int)act, keep && act != ffn::ACT_NONE, &kept, "linear");
  return {y.view(out_sizes(x, w.size(0))), kept.z};
}
void check_dy(const Tensor& dy, const Tensor& x, int64_t n, const char* op) {
  no_tangent(dy, op);
  check_like(dy, x, op, "the output's gradient");
  BAD_UNLESS(dy.sizes().vec() == out_sizes(x, n), op, ": gradient ", dy.sizes(), " where the result is ", out_sizes(x, n));
}
// the sums that the forward pass keeps: fp32 [planes, rows of x, n rounded up to 16]
void check_kept(const Tensor& z, int64_t planes, const Tensor& x, int64_t n, const char* op) {
  int64_t rows = 1;                                                  // not numel / K: K may be zero
  for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
  BAD_UNLESS(z.defined() && z.is_contiguous() && z.scalar_type() == at::kFloat && z.dim() == 3 && z.size(0) == planes &&
                 z.size(1) == rows && z.size(2) == up(n, 16) && z.device() == x.device(),
             op, ": the backward pass needs the sums kept by the forward pass of the same call");
}
std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const OptT& z, int64_t act,
                                                   bool need_dx, bool need_dw, bool need_db) {
  check_linear(x, w, OptT(), OptT(), act);
  check_dy(dy, x, w.size(0), "linear");
  BAD_UNLESS(act == ffn::ACT_NONE || has(z), "linear: the backward pass of an activation needs the sums kept by the forward pass");
  ddl::DeviceGuard guard(x.device());
  const Tensor zz = act == ffn::ACT_NONE ? Tensor() : get(z);
  if (zz.defined()) check_kept(zz, 1, x, w.size(0), "linear");
  auto r = product_backward(dy, {zz, x, {w, Tensor()}}, x.size(-1), (int)act, need_dx, need_dw, need_db, "linear");
  return {need_dx ? r.dx.view(x.sizes()) : r.dx, r.dw[0], r.db[0]};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
// Which inputs of a node want a gradient.  The node numbers its edges over the tensors that were given, so the absent optional
// ones are remembered as gaps: bit i of `given` is tensor argument i.
struct Needs {
  AutogradContext* ctx;
  int64_t given;
  static void remember(AutogradContext* ctx, std::initializer_list<bool> given) {
    int64_t m = 0, i = 0;
    for (bool g : given) m |= (int64_t)g << i++;
    ctx->saved_data["given"] = m;
  }
  explicit Needs(AutogradContext* c) : ctx(c), given(c->saved_data["given"].toInt()) {}
  bool operator()(int i) const {
    return (given >> i & 1) && ctx->needs_input_grad((size_t)__builtin_popcountll(given & ((1ll << i) - 1)));
  }
};
// PyTorch hands a gradient to the next node on the stream where that node was made.  A leaf's accumulation node is made by the leaf's first
// use and lives as long as a result of it (or a hook): an eager result that is alive puts it on the default stream, and to wait for that
// stream ends a capture, and the process with it.  So a backward pass that is being captured refuses such a gradient, before anything
// is launched for it.
void no_capture_onto_default_stream(const char* op) {
  const auto here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA();
  if (here.unwrap().id() == 0) return;                               // the default stream itself: nothing is captured on it
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  DDL_HIP_CHECK(hipStreamIsCapturing(here.stream(), &status));
  const auto node = torch::autograd::get_current_node();
  if (status == hipStreamCaptureStatusNone || !node) return;
  for (uint32_t i = 0; i < node->num_outputs(); ++i) {
    const auto& next = node->next_edge(i).function;
    if (!next || !node->task_should_compute_output(i)) continue;
    const auto stream = next->stream();
    TORCH_CHECK(!stream.has_value() || stream->id() != 0, op, ": this backward pass is being captured, and a gradient goes to ",
                next->name(), " on the default stream, which would break the capture.  An eager result of the same tensor is alive, or a "
                "hook holds its node: free it before the capture, or use the tensor on the capturing stream first");
  }
}
struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& b, const OptT& res, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    Needs::remember(ctx, {true, true, has(b), has(res)});
    ddl::DeviceGuard guard(x.device());
    Kept kept;
    Tensor y = product_forward(x, w, Tensor(), get(b), Tensor(), get(res), (int)act, act != ffn::ACT_NONE, &kept, "linear");
    ctx->save_for_backward({kept.x, kept.w[0], kept.z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["width"] = x.size(-1);
    ctx->set_materialize_grads(false);
    return y.view(out_sizes(x, w.size(0)));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("linear");
    if (!grads[0].defined()) return variable_list(5);
    no_tangent(grads[0], "linear");
    no_capture_onto_default_stream("linear");
    const auto saved = ctx->get_saved_variables();
    const Needs need(ctx);
    ddl::DeviceGuard guard(grads[0].device());
    const int64_t width = ctx->saved_data["width"].toInt();
    auto r = product_backward(grads[0], {saved[2], saved[0], {saved[1], Tensor()}}, width, (int)ctx->saved_data["act"].toInt(), need(0),
                              need(1), need(2), "linear");
    return {need(0) ? r.dx.view(out_sizes(grads[0], width)) : r.dx, r.dw[0], r.db[0], need(3) ? grads[0] : Tensor(), Tensor()};
  }
};
Tensor linear(const Tensor& x, const Tensor& w, const OptT& b, const OptT& res, int64_t act) {
  const Tensor bb = get(b), rr = get(res);
  if (wants_grad({&x, &w, &bb, &rr})) {
    check_linear(x, w, b, res, act);
    return LinearFn::apply(x, w, b, res, act);
  }
  return std::get<0>(linear_forward(x, w, b, res, act, false));
}

void check_gated(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptT& bg, const OptT& bu, int64_t act) {
  const Tensor b0 = get(bg), b1 = get(bu);
  not_recorded("gated_linear");
  no_tangents({&x, &wg, &wu, &b0, &b1}, "gated_linear");
  check_product(x, wg, bg, "gated_linear", "w_gate", "b_gate");
  check_product(x, wu, bu, "gated_linear", "w_up", "b_up");
  BAD_UNLESS(wg.sizes() == wu.sizes(), "gated_linear: w_gate ", wg.sizes(), " and w_up ", wu.sizes(), " differ");
  BAD_UNLESS(has(bg) == has(bu), "gated_linear: both biases or none");
  check_act(act, "gated_linear");
}
std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptT& bg, const OptT& bu,
                                         int64_t act, bool keep) {
  check_gated(x, wg, wu, bg, bu, act);
  ddl::DeviceGuard guard(x.device());
  Kept kept;
  Tensor h = product_forward(x, wg, wu, get(bg), get(bu), Tensor(), (int)act, keep, &kept, "gated_linear");
  return {h.view(out_sizes(x, wg.size(0))), kept.z};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_backward(const Tensor& dy, const Tensor& x, const Tensor& wg,
                                                                  const Tensor& wu, const Tensor& z, int64_t act, bool need_dx,
                                                                  bool need_dw, bool need_db) {
  check_gated(x, wg, wu, OptT(), OptT(), act);
  check_dy(dy, x, wg.size(0), "gated_linear");
  check_kept(z, 2, x, wg.size(0), "gated_linear");
  ddl::DeviceGuard guard(x.device());
  auto r = product_backward(dy, {z, x, {wg, wu}}, x.size(-1), (int)act, need_dx, need_dw, need_db, "gated_linear");
  return {need_dx ? r.dx.view(x.sizes()) : r.dx, r.dw[0], r.dw[1], r.db[0], r.db[1]};
}
struct GatedFn : torch::autograd::Function<GatedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const OptT& bg, const OptT& bu,
                        int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    Needs::remember(ctx, {true, true, true, has(bg), has(bu)});
    ddl::DeviceGuard guard(x.device());
    Kept kept;
    Tensor h = product_forward(x, wg, wu, get(bg), get(bu), Tensor(), (int)act, true, &kept, "gated_linear");
    ctx->save_for_backward({kept.x, kept.w[0], kept.w[1], kept.z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["width"] = x.size(-1);
    ctx->set_materialize_grads(false);
    return h.view(out_sizes(x, wg.size(0)));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("gated_linear");
    if (!grads[0].defined()) return variable_list(6);
    no_tangent(grads[0], "gated_linear");
    no_capture_onto_default_stream("gated_linear");
    const auto s = ctx->get_saved_variables();
    const Needs need(ctx);
    ddl::DeviceGuard guard(grads[0].device());
    const int64_t width = ctx->saved_data["width"].toInt();
    auto r = product_backward(grads[0], {s[3], s[0], {s[1], s[2]}}, width, (int)ctx->saved_data["act"].toInt(), need(0),
                              need(1) || need(2), need(3) || need(4), "gated_linear");
    auto only = [&](int i, const Tensor& t) { return need(i) ? t : Tensor(); };
    return {need(0) ? r.dx.view(out_sizes(grads[0], width)) : r.dx, only(1, r.dw[0]), only(2, r.dw[1]), only(3, r.db[0]),
            only(4, r.db[1]), Tensor()};
  }
};
Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptT& bg, const OptT& bu, int64_t act) {
  const Tensor b0 = get(bg), b1 = get(bu);
  if (wants_grad({&x, &wg, &wu, &b0, &b1})) {
    check_gated(x, wg, wu, bg, bu, act);
    return GatedFn::apply(x, wg, wu, bg, bu, act);
  }
  return std::get<0>(gated_forward(x, wg, wu, bg, bu, act, false));
}

// ---- dropout ------------------------------------------------------------------------------------------------------------
void check_dropout(const Tensor& x, double p, const Tensor& key, const OptT& res) {
  not_recorded("dropout");
  no_tangent(x, "dropout");
  no_tangent(get(res), "dropout");
  BAD_UNLESS(x.is_cuda(), "dropout: GPU tensor expected");
  type_of(x, "dropout");
  BAD_UNLESS(p >= 0. && p <= 1., "dropout: p must lie in [0, 1], got ", p);
  BAD_UNLESS(key.scalar_type() == at::kLong && key.numel() == 2 && key.device() == x.device(),
             "dropout: key must be two int64 values (seed, call) on the input's device");
  if (has(res)) {
    check_like(*res, x, "dropout", "residual");
    BAD_UNLESS(res->sizes() == x.sizes(), "dropout: residual ", res->sizes(), " where x is ", x.sizes());
  }
}
Tensor dropout_apply(const Tensor& x, double p, const Tensor& key, const OptT& res) {
  check_dropout(x, p, key, res);
  ddl::DeviceGuard guard(x.device());
  const Tensor xc = in_memory(x).contiguous(), rc = has(res) ? in_memory(*res).contiguous() : Tensor(),
               kc = in_memory(key).contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  ffn::DropoutArgs a;
  a.x = xc.data_ptr();
  a.residual = rc.defined() ? rc.data_ptr() : nullptr;
  a.y = y.data_ptr();
  a.n = x.numel();
  a.key = kc.data_ptr<int64_t>();
  a.p = p;
  ffn::launch_dropout(type_of(x, "dropout"), a, cur_stream());
  return y;
}
struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& key, const OptT& res, double p) {
    at::AutoDispatchBelowADInplaceOrView below;
    Needs::remember(ctx, {true, true, has(res)});
    ctx->save_for_backward({key});
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);
    return dropout_apply(x, p, key, res);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("dropout");
    if (!grads[0].defined()) return variable_list(4);
    no_tangent(grads[0], "dropout");
    no_capture_onto_default_stream("dropout");
    const Needs need(ctx);
    Tensor dx;
    if (need(0))
      dx = dropout_apply(grads[0], ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0], OptT());
    return {dx, Tensor(), need(2) ? grads[0] : Tensor(), Tensor()};
  }
};
Tensor dropout(const Tensor& x, double p, const Tensor& key, const OptT& res) {
  const Tensor rr = get(res);
  if (wants_grad({&x, &rr})) {
    check_dropout(x, p, key, res);
    return DropoutFn::apply(x, key, res, p);
  }
  return dropout_apply(x, p, key, res);
}
Tensor rng_keys(Tensor state, int64_t n) {
  not_recorded("rng_keys");
  DDL_CHECK_DEV(state); DDL_CHECK_CONTIG(state);
  BAD_UNLESS(state.scalar_type() == at::kLong && state.numel() == 2, "rng_keys: state must be two int64 values");
  BAD_UNLESS(n >= 1 && n <= (1 << 20), "rng_keys: 1 .. 2^20 keys, got ", n);
  ddl::DeviceGuard guard(state.device());
  Tensor keys = at::empty({n, 2}, state.options());
  ffn::launch_rng_keys(state.data_ptr<int64_t>(), keys.data_ptr<int64_t>(), (int)n, cur_stream());
  return keys;
}

// ---- residual_norm --------------------------------------------------------------------------------------------------------
struct NormIn {
  Tensor x, y, gate, post_w, post_b, pre_w, pre_b;
  bool layer = false;
  double eps = 0., scale = 1.;
};
// Beside a single row [C] both kinds of gate have its shape: one of x's type is taken element by element, another is a channel gate.
bool full_gate(const NormIn& in) {
  return in.gate.defined() && (in.gate.dim() != 1 || (in.x.dim() == 1 && in.gate.scalar_type() == in.x.scalar_type()));
}
// The checks alone: nothing is copied or launched.
void check_norm(const NormIn& in) {
  const char* op = "residual_norm";
  not_recorded(op);
  no_tangents({&in.x, &in.y, &in.gate, &in.post_w, &in.post_b, &in.pre_w, &in.pre_b}, op);
  BAD_UNLESS(in.x.is_cuda(), op, ": GPU tensor expected");
  type_of(in.x, op);
  BAD_UNLESS(in.x.dim() >= 1 && in.x.size(-1) >= 1, op, ": x [.., C] with C >= 1 expected, got ", in.x.sizes());
  const int64_t C = in.x.size(-1);
  BAD_UNLESS(C <= ffn::NORM_MAX_C, op, ": rows of at most ", ffn::NORM_MAX_C, " columns, got ", C);
  rows_fit(in.x.numel() / C, op);
  BAD_UNLESS(in.eps >= 0., op, ": eps must not be negative");
  BAD_UNLESS(in.layer || !(in.post_b.defined() || in.pre_b.defined()), op, ": an RMS norm has no bias");
  BAD_UNLESS(in.post_w.defined() || !in.post_b.defined(), op, ": post_bias without post_weight");
  BAD_UNLESS(in.pre_w.defined() || !in.pre_b.defined(), op, ": pre_bias without pre_weight");
  BAD_UNLESS(in.y.defined() || !(in.gate.defined() || in.post_w.defined()), op, ": gate or post_weight without a branch");
  BAD_UNLESS(in.y.defined() || in.pre_w.defined(), op, ": neither a branch nor pre_weight: nothing to do");
  if (in.y.defined()) {
    check_like(in.y, in.x, op, "the branch");
    BAD_UNLESS(in.y.sizes() == in.x.sizes(), op, ": branch ", in.y.sizes(), " where x is ", in.x.sizes());
  }
  at::ScalarType pt = in.x.scalar_type();
  bool first = true;
  auto param = [&](const Tensor& t, const char* name) {
    if (!t.defined()) return;
    BAD_UNLESS(t.dim() == 1 && t.size(0) == C, op, ": ", name, " [", C, "] expected, got ", t.sizes());
    BAD_UNLESS(t.device() == in.x.device(), op, ": ", name, " is on another device");
    BAD_UNLESS(t.scalar_type() == in.x.scalar_type() || t.scalar_type() == at::kFloat, op, ": ", name, " must be float32 or ",
               in.x.scalar_type());
    BAD_UNLESS(first || t.scalar_type() == pt, op, ": weights, biases and a channel gate share one type");
    pt = t.scalar_type();
    first = false;
  };
  param(in.post_w, "post_weight");
  param(in.post_b, "post_bias");
  param(in.pre_w, "pre_weight");
  param(in.pre_b, "pre_bias");
  if (full_gate(in)) {
    check_like(in.gate, in.x, op, "a gate of x's shape");
    BAD_UNLESS(in.gate.sizes() == in.x.sizes(), op, ": gate [", C, "] or of x's shape ", in.x.sizes(), " expected, got ",
               in.gate.sizes());
  } else {
    param(in.gate, "gate");
  }
}
// The inputs as the kernels read them: rows behind each other.  The backward pass keeps these, so a strided input is copied once.
NormIn contiguous(const NormIn& in) {
  NormIn c = in;
  for (Tensor* t : {&c.x, &c.y, &c.gate, &c.post_w, &c.post_b, &c.pre_w, &c.pre_b})
    if (t->defined()) *t = in_memory(*t).contiguous();
  return c;
}
// of checked, contiguous inputs
ffn::NormArgs norm_args(const NormIn& in) {
  ffn::NormArgs a;
  a.C = (int)in.x.size(-1);
  a.M = (int)(in.x.numel() / a.C);
  a.layer = in.layer;
  a.eps = (float)in.eps;
  a.scale = (float)in.scale;
  a.post = in.post_w.defined();
  a.pre = in.pre_w.defined();
  a.gate_kind = !in.gate.defined() ? ffn::GATE_NONE : full_gate(in) ? ffn::GATE_FULL : ffn::GATE_CHANNEL;
  at::ScalarType pt = in.x.scalar_type();
  for (const Tensor* t : {&in.post_w, &in.pre_w, &in.gate})          // all vectors have one type
    if (t->defined() && !(t == &in.gate && full_gate(in))) pt = t->scalar_type();
  a.param_f32 = pt == at::kFloat;
  a.x = ptr(in.x); a.y = ptr(in.y); a.gate = ptr(in.gate);
  a.post_w = ptr(in.post_w); a.post_b = ptr(in.post_b);
  a.pre_w = ptr(in.pre_w); a.pre_b = ptr(in.pre_b);
  a.vec = a.C * in.x.element_size() % 16 == 0;
  for (const void* p : {a.x, a.y, a.gate, a.post_w, a.post_b, a.pre_w, a.pre_b}) a.vec = a.vec && aligned(p);
  return a;
}
// -> r (undefined without a branch), h (undefined without a pre norm), statistics [4, M] if `keep`
// (checked, contiguous inputs)
std::tuple<Tensor, Tensor, Tensor> norm_forward(const NormIn& in, bool keep) {
  ddl::DeviceGuard guard(in.x.device());
  ffn::NormArgs a = norm_args(in);
  Tensor r, h, st;
  if (in.y.defined()) r = at::empty(in.x.sizes(), in.x.options());
  if (a.pre) h = at::empty(in.x.sizes(), in.x.options());
  if (keep) st = at::empty({4, a.M}, in.x.options().dtype(at::kFloat));
  a.r = r.defined() ? r.data_ptr() : nullptr;
  a.h = h.defined() ? h.data_ptr() : nullptr;
  a.stats = keep ? st.data_ptr<float>() : nullptr;
  if (a.M > 0) ffn::launch_norm_fwd(type_of(in.x, "residual_norm"), a, cur_stream());
  return {r, h, st};
}
struct NormGrads { Tensor dx, dy, v[5]; };                           // v: gate, post_w, post_b, pre_w, pre_b
NormGrads norm_backward(const NormIn& in, const Tensor& st, const Tensor& dr, const Tensor& dh, bool need_dx, bool need_dy,
                        bool need_gate, bool need_post_w, bool need_post_b, bool need_pre_w, bool need_pre_b) {
  ddl::DeviceGuard guard(in.x.device());
  ffn::NormArgs a = norm_args(in);
  const int dtype = type_of(in.x, "residual_norm");
  NormGrads g;
  BAD_UNLESS(st.defined() && st.is_contiguous() && st.scalar_type() == at::kFloat && st.numel() == 4 * (int64_t)a.M &&
                 st.device() == in.x.device(), "residual_norm: the backward pass needs the statistics kept by the forward pass");
  a.stats = st.data_ptr<float>();
  Tensor drc, dhc;
  auto grad = [&](const Tensor& t, Tensor& c) -> const void* {
    if (!t.defined()) return nullptr;
    no_tangent(t, "residual_norm");
    check_like(t, in.x, "residual_norm", "an output's gradient");
    BAD_UNLESS(t.sizes() == in.x.sizes(), "residual_norm: gradient ", t.sizes(), " where x is ", in.x.sizes());
    c = in_memory(t).contiguous();
    a.vec = a.vec && aligned(c.data_ptr());
    return c.data_ptr();
  };
  a.dr = grad(dr, drc);
  a.dh = a.pre ? grad(dh, dhc) : nullptr;
  if (need_dx) { g.dx = at::empty(in.x.sizes(), in.x.options()); a.dx = g.dx.data_ptr(); }
  if (need_dy) { g.dy = at::empty(in.x.sizes(), in.x.options()); a.dy = g.dy.data_ptr(); }
  const bool full = a.gate_kind == ffn::GATE_FULL;
  if (need_gate && full) { g.v[0] = at::empty(in.x.sizes(), in.x.options()); a.dgate = g.v[0].data_ptr(); }
  const bool need[5] = {need_gate && !full, need_post_w, need_post_b, need_pre_w, need_pre_b};
  const Tensor* like[5] = {&in.gate, &in.post_w, &in.post_b, &in.pre_w, &in.pre_b};
  void* outs[5] = {};
  bool any = false;
  for (int i = 0; i < 5; ++i)
    if (need[i]) {
      g.v[i] = at::empty({a.C}, like[i]->options());
      outs[i] = g.v[i].data_ptr();
      any = true;
    }
  if (a.M == 0) {
    for (auto& t : g.v) if (t.defined()) t.zero_();
    return g;
  }
  Tensor part;
  a.groups = ffn::norm_bwd_groups(a.M, a.C);
  if (any) {
    part = at::empty({a.groups, 5, a.C}, in.x.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  Tensor means;
  if (any && a.dh != nullptr && ffn::norm_bwd_wants_means(a.C)) {
    means = at::empty({2, a.M}, in.x.options().dtype(at::kFloat));
    a.means = means.data_ptr<float>();
  }
  ffn::launch_norm_bwd(dtype, a, cur_stream());
  if (any) ffn::launch_colsum(a.param_f32 ? (int)ffn::F32 : dtype, a.part, a.groups, 5, a.C, outs, cur_stream());
  return g;
}
NormIn norm_in(const Tensor& x, const OptT& y, const OptT& gate, const OptT& post_w, const OptT& post_b, const OptT& pre_w,
               const OptT& pre_b, bool layer, double eps, double scale) {
  NormIn in;
  in.x = x;
  in.y = get(y); in.gate = get(gate);
  in.post_w = get(post_w); in.post_b = get(post_b);
  in.pre_w = get(pre_w); in.pre_b = get(pre_b);
  in.layer = layer;
  in.eps = eps; in.scale = scale;
  return in;
}
struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptT& y, const OptT& gate, const OptT& post_w,
                               const OptT& post_b, const OptT& pre_w, const OptT& pre_b, bool layer, double eps, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    Needs::remember(ctx, {true, has(y), has(gate), has(post_w), has(post_b), has(pre_w), has(pre_b)});
    const NormIn in = contiguous(norm_in(x, y, gate, post_w, post_b, pre_w, pre_b, layer, eps, scale));
    auto [r, h, st] = norm_forward(in, true);
    ctx->save_for_backward({in.x, in.y, in.gate, in.post_w, in.post_b, in.pre_w, in.pre_b, st});
    ctx->saved_data["layer"] = layer;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    variable_list out;
    if (r.defined()) out.push_back(r);
    if (h.defined()) out.push_back(h);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("residual_norm");
    not_recorded("residual_norm");
    const auto v = ctx->get_saved_variables();
    const NormIn in = norm_in(v[0], v[1], v[2], v[3], v[4], v[5], v[6], ctx->saved_data["layer"].toBool(),
                              ctx->saved_data["eps"].toDouble(), ctx->saved_data["scale"].toDouble());
    Tensor dr, dh;
    if (in.y.defined()) {
      dr = grads[0];
      if (in.pre_w.defined()) dh = grads[1];
    } else {
      dh = grads[0];
    }
    variable_list out(10);
    if (!dr.defined() && !dh.defined()) return out;
    no_capture_onto_default_stream("residual_norm");
    const Needs need(ctx);
    NormGrads g = norm_backward(in, v[7], dr, dh, need(0), need(1), need(2), need(3), need(4), need(5), need(6));
    out[0] = g.dx;
    out[1] = g.dy;
    for (int i = 0; i < 5; ++i) out[2 + i] = g.v[i];
    return out;
  }
};
// -> (r, h); r is x itself without a branch, h is None without a pre norm
std::tuple<Tensor, OptT> residual_norm(const Tensor& x, const OptT& y, const OptT& gate, const OptT& post_w, const OptT& post_b,
                                       const OptT& pre_w, const OptT& pre_b, bool layer, double eps, double scale) {
  const NormIn in = norm_in(x, y, gate, post_w, post_b, pre_w, pre_b, layer, eps, scale);
  check_norm(in);
  ddl::DeviceGuard guard(x.device());
  Tensor r, h;
  if (wants_grad({&in.x, &in.y, &in.gate, &in.post_w, &in.post_b, &in.pre_w, &in.pre_b})) {
    auto out = NormFn::apply(x, y, gate, post_w, post_b, pre_w, pre_b, layer, eps, scale);
    size_t i = 0;
    if (in.y.defined()) r = out[i++];
    if (in.pre_w.defined()) h = out[i];
  } else {
    std::tie(r, h, std::ignore) = norm_forward(contiguous(in), false);
  }
  return {r.defined() ? r : x, h.defined() ? OptT(h) : OptT()};
}

}  // namespace

void register_ffn_ops(pybind11::module_& m) {
  m.def("linear", &linear);
  m.def("linear_forward", &linear_forward, "-> (y, kept sums)");
  m.def("linear_backward", &linear_backward, "-> (dx, dweight, dbias)");
  m.def("product_plan", &product_plan, "(forward | dx | dw, type, M, K, N, dual) -> (tile rows, tile columns, splits)");
  m.def("gated_linear", &gated_linear);
  m.def("gated_forward", &gated_forward, "-> (h, kept sums)");
  m.def("gated_backward", &gated_backward, "-> (dx, dw_gate, dw_up, db_gate, db_up)");
  m.def("dropout", &dropout);
  m.def("rng_keys", &rng_keys, "state (seed, calls) -> n keys (seed, call); calls += n");
  m.def("residual_norm", &residual_norm);
  m.def("norm_forward", [](const Tensor& x, const OptT& y, const OptT& gate, const OptT& post_w, const OptT& post_b, const OptT& pre_w,
                           const OptT& pre_b, bool layer, double eps, double scale, bool keep) {
    const NormIn in = norm_in(x, y, gate, post_w, post_b, pre_w, pre_b, layer, eps, scale);
    check_norm(in);
    ddl::DeviceGuard guard(x.device());
    return norm_forward(contiguous(in), keep);
  }, "-> (r, h, statistics)", py::arg("x"), py::arg("branch"), py::arg("gate"), py::arg("post_weight"), py::arg("post_bias"),
        py::arg("pre_weight"), py::arg("pre_bias"), py::arg("layer"), py::arg("eps"), py::arg("scale"), py::arg("keep") = true);
  m.def("norm_backward", [](const Tensor& x, const OptT& y, const OptT& gate, const OptT& post_w, const OptT& post_b, const OptT& pre_w,
                            const OptT& pre_b, bool layer, double eps, double scale, const Tensor& stats, const OptT& dr, const OptT& dh) {
    const NormIn in = norm_in(x, y, gate, post_w, post_b, pre_w, pre_b, layer, eps, scale);
    check_norm(in);
    ddl::DeviceGuard guard(x.device());
    NormGrads g = norm_backward(contiguous(in), stats, get(dr), get(dh), true, has(y), has(gate), has(post_w), has(post_b), has(pre_w), has(pre_b));
    return std::make_tuple(g.dx, g.dy, g.v[0], g.v[1], g.v[2], g.v[3], g.v[4]);
  }, "-> (dx, dbranch, dgate, dpost_w, dpost_b, dpre_w, dpre_b)");
}

// Operators of other layer forms: norms and rotation of query and key heads.
#include "host.h"

namespace hyc_host {

static int elem_type(at::ScalarType t) { return t == at::kBFloat16 ? HYC_BF16 : t == at::kHalf ? HYC_F16 : t == at::kFloat ? HYC_F32 : -1; }
static int elem_type(const Tensor& t, const char* what) {
  const int e = elem_type(t.scalar_type());
  TORCH_CHECK_VALUE(e >= 0, what, " must be bf16, fp16 or fp32, got ", t.scalar_type());
  return e;
}
static bool on16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// ---- norms and rotation of query and key heads
// [batch, seq, heads, d] with adjacent channels and 16-byte rows, as it is or as a copy; the strides of its first three dimensions
static Tensor head_view(const Tensor& t_in, int64_t (&stride)[3]) {
  Tensor t = t_in;
  const int64_t e = 16 / t.element_size();
  auto fits = [&]() {
    if (t.stride(3) != 1 || !on16(t)) return false;
    for (int i = 0; i < 3; ++i) {
      stride[i] = t.size(i) > 1 ? t.stride(i) : 0;
      if (stride[i] % e != 0) return false;
    }
    return true;
  };
  if (t.numel() > 0 && !fits()) {
    t = t.contiguous();
    if (!fits()) { t = t.clone(); fits(); }      // (contiguous, but begins off a 16-byte boundary)
  }
  return t;
}
// a table of `rows` angles as [rows, >= half], with a row stride that the library takes (expanded and overlapping rows are copied)
static Tensor angle_table(const Tensor& t_in, int64_t half, const char* what) {
  TORCH_CHECK_VALUE(t_in.dim() >= 2 && t_in.numel() == t_in.size(-2) * t_in.size(-1) && t_in.size(-1) >= half, what,
                    " must be a [positions, >= rotary_dim / 2] table, got shape ", t_in.sizes());
  Tensor t = t_in.dim() == 2 ? t_in : t_in.reshape({t_in.size(-2), t_in.size(-1)});
  if (elem_type(t.scalar_type()) < 0) t = t.to(at::kFloat);
  if (t.numel() > 0 && (t.stride(1) != 1 || !on16(t) || (t.size(0) > 1 && (t.stride(0) < half || t.stride(0) % (16 / t.element_size()) != 0))))
    t = t.narrow(1, 0, half).clone(at::MemoryFormat::Contiguous);
  return t;
}

namespace {
struct QkNorm {
  hyc_qk_norm a = {};
  Tensor hold[8];

  void inputs(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& cos_in, const Tensor& sin_in, double eps,
              const OptTensor& pos, const std::optional<int64_t>& rotary_dim) {
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
                      "q and k must be [batch, seq_len, heads, head_dim] with the same batch, length and head size, got ", q.sizes(), " and ", k.sizes());
    TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type(), "q and k must have one type, got ", q.scalar_type(), " and ", k.scalar_type());
    const int64_t d = q.size(3), rot = rotary_dim.value_or(d);
    TORCH_CHECK_VALUE(d >= 16 && d % 16 == 0 && d <= 512, "head_dim must be a multiple of 16 up to 512, got ", d);
    TORCH_CHECK_VALUE(rot >= 16 && rot % 16 == 0 && rot <= d, "rotary_dim must be a multiple of 16 from 16 to head_dim, got ", rot);
    TORCH_CHECK_VALUE(q.size(2) >= 1 && k.size(2) >= 1, "q and k need a head each");
    TORCH_CHECK_VALUE(q.size(2) <= 65536 && k.size(2) <= 65536 && q.size(0) * q.size(1) <= 0x7fffffffll, "more than 65536 heads or 2^31 - 1 tokens");
    TORCH_CHECK_VALUE(qw.numel() == d && kw.numel() == d && qw.scalar_type() == kw.scalar_type(),
                      "q_weight and k_weight must have head_dim = ", d, " entries and one type");
    a.batch = q.size(0); a.seq = q.size(1); a.head_dim = (int)d; a.rotary_dim = (int)rot; a.eps = (float)eps;
    a.heads[0] = (int)q.size(2); a.heads[1] = (int)k.size(2);
    a.type = elem_type(q, "q and k"); a.w_type = elem_type(qw, "q_weight and k_weight");
    hold[0] = head_view(q, a.x_stride[0]); hold[1] = head_view(k, a.x_stride[1]);
    const Tensor* w[2] = {&qw, &kw};
    for (int i = 0; i < 2; ++i) {
      Tensor& c = hold[2 + i];
      c = w[i]->contiguous();
      if (!on16(c)) c = c.clone();
      a.x[i] = data(hold[i]); a.weight[i] = data(c);
    }
    Tensor cos = angle_table(cos_in, rot / 2, "cos"), sin = angle_table(sin_in, rot / 2, "sin");
    TORCH_CHECK_VALUE(cos.size(0) == sin.size(0), "cos and sin must have the same number of positions");
    if (sin.scalar_type() != cos.scalar_type()) { cos = cos.to(at::kFloat); sin = sin.to(at::kFloat); }
    a.cos_t = data(cos); a.sin_t = data(sin); a.ld_cos = cos.stride(0); a.ld_sin = sin.stride(0);
    a.table_rows = cos.size(0); a.table_type = elem_type(cos.scalar_type());
    hold[4] = cos; hold[5] = sin;
    if (cos.size(0) <= 1) a.ld_cos = a.ld_sin = (rot / 2 + 7) / 8 * 8;
    if (given(pos)) {
      TORCH_CHECK_VALUE(pos->dim() == 2 && (pos->size(0) == a.batch || pos->size(0) == 1) && pos->size(1) == a.seq &&
                            (pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt),
                        "position_ids must be int32 or int64 [batch or 1, seq_len], got ", pos->scalar_type(), " ", pos->sizes());
      a.position_ids = data(*pos);
      a.pos_is_int64 = pos->scalar_type() == at::kLong;
      a.pos_stride[0] = pos->size(0) == 1 ? 0 : pos->stride(0);
      a.pos_stride[1] = pos->stride(1);
    } else {
      TORCH_CHECK_VALUE(cos.size(0) >= a.seq, "the rotary tables have ", cos.size(0), " positions, the sequence ", a.seq);
    }
  }
};
}  // namespace

static std::tuple<Tensor, Tensor> qk_norm_rope_forward(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                                                       const Tensor& sin, double eps, const OptTensor& pos, const std::optional<int64_t>& rotary_dim) {
  require_cuda({&q, &k, &qw, &kw, &cos, &sin, opt(pos)});
  OnDevice on(q);
  QkNorm n;
  n.inputs(q, k, qw, kw, cos, sin, eps, pos, rotary_dim);
  const Tensor oq = empty(q.sizes(), q, q.scalar_type()), ok = empty(k.sizes(), k, k.scalar_type());
  n.a.out[0] = data(oq); n.a.out[1] = data(ok);
  check(hyc_qk_norm_rope_fwd(&n.a, on.stream), "hyc_qk_norm_rope_fwd");
  return {oq, ok};
}

static std::tuple<Tensor, Tensor, OptTensor, OptTensor> qk_norm_rope_backward(const Tensor& dq, const Tensor& dk, const Tensor& q, const Tensor& k,
                                                                              const Tensor& qw, const Tensor& kw, const Tensor& cos, const Tensor& sin,
                                                                              double eps, const OptTensor& pos, const std::optional<int64_t>& rotary_dim,
                                                                              bool needs_weight_grad) {
  require_cuda({&q, &k, &dq, &dk, &qw, &kw, &cos, &sin, opt(pos)});
  OnDevice on(q);
  QkNorm n;
  n.inputs(q, k, qw, kw, cos, sin, eps, pos, rotary_dim);
  TORCH_CHECK_VALUE(dq.sizes() == q.sizes() && dk.sizes() == k.sizes(), "the gradients must have the shapes ", q.sizes(), " and ", k.sizes(), ", got ",
                    dq.sizes(), " and ", dk.sizes());
  TORCH_CHECK_VALUE(dq.scalar_type() == q.scalar_type() && dk.scalar_type() == q.scalar_type(), "the gradients must have the type of q and k, ", q.scalar_type());
  n.hold[6] = head_view(dq, n.a.dy_stride[0]); n.hold[7] = head_view(dk, n.a.dy_stride[1]);
  n.a.dy[0] = data(n.hold[6]); n.a.dy[1] = data(n.hold[7]);
  const Tensor oq = empty(q.sizes(), q, q.scalar_type()), ok = empty(k.sizes(), k, k.scalar_type());
  n.a.out[0] = data(oq); n.a.out[1] = data(ok);
  OptTensor wq, wk;
  Tensor ws;
  size_t bytes = 0;
  if (needs_weight_grad) {
    wq = empty(qw.sizes(), qw, qw.scalar_type()); wk = empty(kw.sizes(), kw, kw.scalar_type());
    bytes = hyc_qk_norm_rope_workspace_bytes(n.a.head_dim);
    ws = empty({(int64_t)bytes}, q, at::kByte);
  }
  check(hyc_qk_norm_rope_bwd(&n.a, data(wq), data(wk), data(ws), bytes, on.stream), "hyc_qk_norm_rope_bwd");
  return {oq, ok, wq, wk};
}

// ---- softmax with a learned bias per bucket of relative positions
static hyc_relative_bias relative_bias_args(const Tensor& x, double scale, const Tensor& edges, bool both, bool causal, int64_t q_offset) {
  TORCH_CHECK_VALUE(x.dim() == 4, "expected a [batch, heads, n, S] map, got shape ", x.sizes());
  TORCH_CHECK_VALUE(x.size(3) >= 1, "the last dimension is empty (shape ", x.sizes(), ")");
  TORCH_CHECK_VALUE(x.size(3) <= HYC_RELATIVE_BIAS_MAX_COLS, "rows of more than ", (int)HYC_RELATIVE_BIAS_MAX_COLS, " columns");
  TORCH_CHECK_VALUE(x.size(1) >= 1, "the map has no heads");
  TORCH_CHECK_VALUE(x.size(0) * x.size(1) * x.size(2) <= 0x7fffffffll, "more than 2^31 - 1 rows");
  TORCH_CHECK_VALUE(std::abs(q_offset) < (1ll << 29), "q_offset is out of range: ", q_offset);
  TORCH_CHECK_VALUE(!edges.is_cuda() && edges.scalar_type() == at::kInt && edges.dim() == 1 && edges.is_contiguous() && edges.numel() >= 1,
                    "the buckets' edges must be an int32 vector on the host");
  hyc_relative_bias a = {};
  a.batch = x.size(0); a.heads = (int)x.size(1); a.n = x.size(2); a.cols = x.size(3); a.q_offset = q_offset;
  a.host_edges = (const int32_t*)edges.data_ptr(); a.side = (int)edges.numel(); a.both = both; a.causal = causal;
  a.type = elem_type(x, "the map"); a.scale = (float)scale;
  return a;
}

static Tensor softmax_relative_bias_forward(const Tensor& scores, double scale, const Tensor& table, const Tensor& edges, bool both, const OptTensor& mask,
                                            bool causal, int64_t q_offset, bool inplace) {
  require_cuda({&scores, &table, opt(mask)});
  OnDevice on(scores);
  hyc_relative_bias a = relative_bias_args(scores, scale, edges, both, causal, q_offset);
  TORCH_CHECK_VALUE(!inplace || scores.is_contiguous(), "inplace needs contiguous scores");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == (both ? 2 : 1) * a.side && table.size(1) == a.heads, "the table must be [", (both ? 2 : 1) * a.side,
                    " buckets, ", a.heads, " heads], got ", table.sizes());
  const Tensor x = scores.contiguous(), t = table.contiguous();
  const Tensor out = inplace ? x : empty(x.sizes(), x, x.scalar_type());
  Tensor mk;
  if (given(mask)) {
    mk = *mask;
    TORCH_CHECK_VALUE(mk.dim() == 4 && mk.size(3) == a.cols && (mk.size(2) == 1 || mk.size(2) == a.n) && (mk.size(1) == 1 || mk.size(1) == a.heads) &&
                          (mk.size(0) == 1 || mk.size(0) == a.batch),
                      "attention_mask must be [b or 1, h or 1, n or 1, S], got ", mk.sizes());
    a.mask_type = elem_type(mk, "attention_mask");
    if (mk.stride(3) != 1) mk = mk.contiguous();
    a.mask = data(mk);
    a.mask_b = mk.size(0) == 1 ? 0 : mk.stride(0); a.mask_h = mk.size(1) == 1 ? 0 : mk.stride(1); a.mask_row = mk.size(2) == 1 ? 0 : mk.stride(2);
  }
  a.x = data(x); a.out = data(out); a.table = data(t); a.table_type = elem_type(t, "the table");
  check(hyc_softmax_relative_bias_fwd(&a, on.stream), "hyc_softmax_relative_bias_fwd");
  return inplace ? scores : out;
}

static std::tuple<Tensor, Tensor> softmax_relative_bias_backward(const Tensor& map, const Tensor& grad, double scale, const Tensor& edges, bool both,
                                                                 bool causal, int64_t q_offset) {
  require_cuda({&map, &grad});
  OnDevice on(map);
  hyc_relative_bias a = relative_bias_args(map, scale, edges, both, causal, q_offset);
  TORCH_CHECK_VALUE(grad.sizes() == map.sizes() && grad.scalar_type() == map.scalar_type(), "the gradient must have the map's shape and type, ",
                    map.scalar_type(), " ", map.sizes(), ", got ", grad.scalar_type(), " ", grad.sizes());
  const Tensor x = map.contiguous(), g = grad.contiguous();
  const Tensor out = empty(x.sizes(), x, x.scalar_type()), table = empty({(both ? 2 : 1) * a.side, a.heads}, x, at::kFloat);
  a.x = data(x); a.grad = data(g); a.out = data(out);
  const size_t bytes = hyc_softmax_relative_bias_workspace_bytes(&a);
  const Tensor ws = empty({(int64_t)bytes}, x, at::kByte);
  check(hyc_softmax_relative_bias_bwd(&a, (float*)data(table), data(ws), bytes, on.stream), "hyc_softmax_relative_bias_bwd");
  return {out, table};
}

// ---- products with bias, activation and residual
// [.., n] as rows of n adjacent elements on 16 bytes with one stride, as it is or as a copy
static Tensor rows_of(const Tensor& t_in, int64_t& ld) {
  const int64_t n = t_in.size(-1);
  auto rows = [&](const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, n}); };
  Tensor t = t_in.numel() == 0 ? t_in.new_empty({t_in.numel() / n, n}) : rows(t_in);
  auto fits = [&]() {
    ld = t.size(0) > 1 ? t.stride(0) : n;
    return t.stride(1) == 1 && ld % 8 == 0 && ld >= n && on16(t);
  };
  if (t.numel() > 0 && !fits()) {
    t = t.clone(at::MemoryFormat::Contiguous);
    fits();
  }
  if (t.numel() == 0) ld = n;
  return t;
}
static void check_linear(const Tensor& x, const Tensor& w, const char* what) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, what, " must be bf16 or fp16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 2 && w.scalar_type() == x.scalar_type(), "weight must be a [out, in] matrix of the type ", x.scalar_type(), ", got ", w.scalar_type(),
                    " ", w.sizes());
  TORCH_CHECK_VALUE(w.size(0) >= 8 && w.size(1) >= 8 && w.size(0) % 8 == 0 && w.size(1) % 8 == 0 && w.size(0) <= (1 << 24) && w.size(1) <= (1 << 24),
                    "both sizes of the weight must be multiples of 8 up to 2^24, got ", w.sizes());
}
static at::DimVector with_last(const Tensor& like, int64_t n) {
  at::DimVector s(like.sizes().begin(), like.sizes().end());
  s.back() = n;
  return s;
}

static std::tuple<Tensor, OptTensor> linear_act_forward(const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t act, const OptTensor& residual,
                                                        bool save_pre) {
  require_cuda({&x, &w, opt(bias), opt(residual)});
  check_linear(x, w, "x");
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x must be [.., ", k, "] for this weight, got ", x.sizes());
  TORCH_CHECK_VALUE(x.numel() / k <= 0x3fffffffll, "more than 2^30 - 1 rows");
  const at::DimVector shape = with_last(x, n);
  TORCH_CHECK_VALUE(!given(bias) || (bias->numel() == n && bias->scalar_type() == x.scalar_type()), "bias must have ", n, " entries of the type ", x.scalar_type());
  TORCH_CHECK_VALUE(!given(residual) || (residual->sizes() == at::IntArrayRef(shape) && residual->scalar_type() == x.scalar_type()),
                    "residual must have the result's shape ", at::IntArrayRef(shape), " and the type ", x.scalar_type());
  OnDevice on(x);
  hyc_linear a = {};
  const Tensor xr = rows_of(x, a.ld_a), wr = rows_of(w, a.ld_b), b = given(bias) ? bias->contiguous() : Tensor();
  Tensor res;
  if (given(residual)) res = rows_of(*residual, a.ld_res);
  const Tensor out = empty(shape, x, x.scalar_type());
  OptTensor pre;
  if (save_pre) pre = empty(shape, x, x.scalar_type());
  a.a = data(xr); a.b = data(wr); a.bias = data(b); a.residual = data(res); a.pre = data(pre); a.out = data(out);
  a.rows = xr.size(0); a.cols = (int)n; a.depth = (int)k; a.type = elem_type(x.scalar_type()); a.act = (int)act;
  check(hyc_linear_act_tcgen05(&a, on.stream), "hyc_linear_act_tcgen05");
  return {out, pre};
}

static std::tuple<OptTensor, OptTensor, OptTensor> linear_act_backward(const Tensor& dy, const Tensor& x, const Tensor& w, int64_t act, const OptTensor& pre,
                                                                       bool need_x, bool need_w, bool need_b) {
  require_cuda({&dy, &x, &w, opt(pre)});
  check_linear(x, w, "x");
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x must be [.., ", k, "] for this weight, got ", x.sizes());
  const at::DimVector shape = with_last(x, n);
  TORCH_CHECK_VALUE(dy.sizes() == at::IntArrayRef(shape) && dy.scalar_type() == x.scalar_type(), "dy must be ", at::IntArrayRef(shape), " of the type ",
                    x.scalar_type(), ", got ", dy.scalar_type(), " ", dy.sizes());
  TORCH_CHECK_VALUE(act == HYC_ACT_NONE || (given(pre) && pre->sizes() == at::IntArrayRef(shape) && pre->scalar_type() == x.scalar_type()),
                    "an activation's backward pass needs pre as forward saved it");
  TORCH_CHECK_VALUE(x.numel() / k <= 0x3fffffffll, "more than 2^30 - 1 rows");
  OnDevice on(x);
  OptTensor dx, dw, db;
  const int64_t rows = x.numel() / k;
  const int type = elem_type(x.scalar_type());
  int64_t ld = 0;
  Tensor g = rows_of(dy, ld);
  if (act != HYC_ACT_NONE || need_b) {
    Tensor d, ws;
    size_t bytes = 0;
    if (act != HYC_ACT_NONE) d = empty({rows, n}, x, x.scalar_type());
    if (need_b) {
      db = empty({n}, x, x.scalar_type());
      bytes = hyc_linear_act_dpre_workspace_bytes((int)n);
      ws = empty({(int64_t)bytes}, x, at::kByte);
    }
    const Tensor p = act != HYC_ACT_NONE ? pre->contiguous() : Tensor();
    const Tensor pa = p.defined() && p.numel() > 0 && !on16(p) ? p.clone() : p;
    check(hyc_linear_act_dpre(data(g), ld, data(pa), data(d), data(db), rows, (int)n, type, (int)act, data(ws), bytes, on.stream), "hyc_linear_act_dpre");
    if (d.defined()) { g = d; ld = n; }
  }
  hyc_linear a = {};
  a.a = data(g); a.ld_a = ld; a.b_mn = 1; a.type = type;
  if (need_x) {
    dx = empty(x.sizes(), x, x.scalar_type());
    const Tensor wr = rows_of(w, a.ld_b);
    a.b = data(wr); a.out = data(dx); a.rows = rows; a.cols = (int)k; a.depth = (int)n;
    check(hyc_linear_act_tcgen05(&a, on.stream), "hyc_linear_act_tcgen05");
  }
  if (need_w) {
    dw = empty(w.sizes(), w, w.scalar_type());
    if (rows == 0) {
      dw->zero_();
    } else {
      const Tensor xr = rows_of(x, a.ld_b);
      a.a_mn = 1; a.b = data(xr); a.out = data(dw); a.rows = n; a.cols = (int)k; a.depth = (int)rows;
      check(hyc_linear_act_tcgen05(&a, on.stream), "hyc_linear_act_tcgen05");
    }
  }
  return {dx, dw, db};
}

void bind_forms(pybind11::module_& m) {
  m.def("linear_act_forward", &linear_act_forward);
  m.def("linear_act_backward", &linear_act_backward);
  m.def("linear_status", [](int64_t device) {
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    int status = 0;
    check(hyc_linear_status(&status), "hyc_linear_status");
    return status;
  });
  m.def("softmax_relative_bias_forward", &softmax_relative_bias_forward);
  m.def("softmax_relative_bias_backward", &softmax_relative_bias_backward);
  m.def("qk_norm_rope_forward", &qk_norm_rope_forward);
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward);
}

}  // namespace hyc_host

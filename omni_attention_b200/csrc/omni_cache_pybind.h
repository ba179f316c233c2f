// The part of the extension module behind omni_rotary, omni_cache_append and omni_cache_attention: argument checks,
// results and workspaces, the C-ABI call and, for omni_rotary, the autograd node. Included by omni_attn_pybind.cc inside
// its unnamed namespace. Shapes and types are checked before devices, so that a refusal needs no GPU.

using Optional = std::optional<torch::Tensor>;

int dtype_code(const torch::Tensor& t) {
  return t.scalar_type() == torch::kBFloat16 ? OMNI_DTYPE_BF16 : t.scalar_type() == torch::kHalf ? OMNI_DTYPE_F16 : OMNI_DTYPE_F32;
}

// The text is put together only for a refusal.
#define OMNI_REQUIRE(ok, msg)  \
  do {                         \
    if (!(ok)) refuse(std::string(msg)); \
  } while (0)

std::string shape_of(const torch::Tensor& t) {
  std::ostringstream os;
  os << t.sizes();
  return os.str();
}

void check_heads(const torch::Tensor& t, const char* name, bool f32) {
  OMNI_REQUIRE(t.dim() == 4, std::string(name) + " must be [B, H, N, D], got " + shape_of(t));
  const auto d = t.size(3);
  if (d != 32 && d != 64 && d != 128) {
    pybind11::gil_scoped_acquire gil;
    throw pybind11::value_error("Unsupported head_dim=" + std::to_string(d) + ". Supported: 32, 64, 128.");
  }
  const auto ty = t.scalar_type();
  OMNI_REQUIRE(ty == torch::kHalf || ty == torch::kBFloat16 || (f32 && ty == torch::kFloat32),
          std::string("unsupported dtype of ") + name + (f32 ? ": fp16, bf16 or fp32" : ": fp16 or bf16"));
  for (int i = 0; i < 3; ++i) OMNI_REQUIRE(t.size(i) > 0, std::string(name) + " has an empty dimension: " + shape_of(t));
}

// The device that the call runs on, and that every tensor of it must be on.
void check_device(const torch::Tensor& first, std::initializer_list<const torch::Tensor*> rest) {
  OMNI_REQUIRE(first.is_cuda(), "needs CUDA tensors (there is no CPU path)");
  for (const torch::Tensor* t : rest) {
    OMNI_REQUIRE(!t->defined() || t->device() == first.device(), "all tensors must be on one device");
  }
}

torch::Tensor or_none(const Optional& t) { return t.has_value() ? *t : torch::Tensor(); }

// Rows must be contiguous along head_dim; anything else is copied once.
torch::Tensor with_rows(const torch::Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); }

omni_attn_heads heads_arg(const torch::Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), static_cast<int>(t.size(1))};
}

[[noreturn]] void refuse_rc(int rc) { refuse(rc); }

// What omni_rotary and omni_cache_append are told about norm and rotation.
struct RotaryArgs {
  torch::Tensor inv_freq, positions, q_weight, k_weight;
  bool half = false;
  double factor = 1.0, eps = 0.0;
};

void check_weight(const torch::Tensor& w, const char* name, const torch::Tensor& x) {
  if (!w.defined()) return;
  const bool shape = (w.dim() == 1 && w.size(0) == x.size(3)) || (w.dim() == 2 && w.size(0) == x.size(1) && w.size(1) == x.size(3));
  OMNI_REQUIRE(shape, std::string(name) + " must be [D] or [heads, D], got " + shape_of(w));
  OMNI_REQUIRE(w.scalar_type() == torch::kFloat32 || w.scalar_type() == x.scalar_type(), std::string(name) + " must be fp32 or of the data's dtype");
}

// x: one of the tensors to be rotated ([B, H, N, D]).
void check_rotary_args(const RotaryArgs& r, const torch::Tensor& q, const torch::Tensor& k) {
  const torch::Tensor& x = q.defined() ? q : k;
  if (r.inv_freq.defined()) {
    OMNI_REQUIRE(r.inv_freq.dim() == 1 && r.inv_freq.scalar_type() == torch::kFloat64 && r.inv_freq.is_contiguous(),
            "inv_freq must be a contiguous float64 tensor [rotary_dim / 2]");
    OMNI_REQUIRE(2 * r.inv_freq.size(0) <= x.size(3), "rotary_dim is larger than head_dim");
  }
  if (r.positions.defined()) {
    const auto& p = r.positions;
    OMNI_REQUIRE(p.scalar_type() == torch::kInt32 || p.scalar_type() == torch::kInt64, "positions must be int32 or int64");
    OMNI_REQUIRE((p.dim() == 1 && p.size(0) == x.size(2)) || (p.dim() == 2 && (p.size(0) == x.size(0) || p.size(0) == 1) && p.size(1) == x.size(2)),
            "positions must be [N], [1, N] or [B, N], got " + shape_of(p));
  }
  OMNI_REQUIRE(std::isfinite(static_cast<float>(r.factor)), "the rotary factor must be finite");
  OMNI_REQUIRE(r.eps >= 0.0 && std::isfinite(static_cast<float>(r.eps)), "eps must be finite and not negative");
  if (r.q_weight.defined() && q.defined()) check_weight(r.q_weight, "q_weight", q);
  if (r.k_weight.defined() && k.defined()) check_weight(r.k_weight, "k_weight", k);
  OMNI_REQUIRE(!r.q_weight.defined() || q.defined(), "q_weight without q");
  OMNI_REQUIRE(!r.k_weight.defined() || k.defined(), "k_weight without k");
  if (r.q_weight.defined() && r.k_weight.defined()) {
    OMNI_REQUIRE(r.q_weight.dim() == r.k_weight.dim() && r.q_weight.scalar_type() == r.k_weight.scalar_type(),
            "q_weight and k_weight must be of one form and dtype");
  }
}

omni_attn_rotary rotary_arg(const RotaryArgs& r) {
  omni_attn_rotary a{};
  a.factor = static_cast<float>(r.factor);
  a.eps = static_cast<float>(r.eps);
  a.half_layout = r.half;
  if (r.inv_freq.defined() && r.inv_freq.numel() > 0) {
    a.inv_freq = r.inv_freq.data_ptr<double>();
    a.rotary_dim = static_cast<int>(2 * r.inv_freq.size(0));
  }
  if (r.positions.defined()) {
    a.positions = r.positions.data_ptr();
    a.positions_64 = r.positions.scalar_type() == torch::kInt64;
    a.pos_stride_b = r.positions.dim() == 2 && r.positions.size(0) > 1 ? r.positions.stride(0) : 0;
    a.pos_stride_n = r.positions.stride(-1);
  }
  const torch::Tensor& w = r.q_weight.defined() ? r.q_weight : r.k_weight;
  if (w.defined()) {
    a.weight_f32 = w.scalar_type() == torch::kFloat32;
    a.weight_per_head = w.dim() == 2;
  }
  a.q_weight = r.q_weight.defined() ? r.q_weight.data_ptr() : nullptr;
  a.k_weight = r.k_weight.defined() ? r.k_weight.data_ptr() : nullptr;
  return a;
}

torch::Tensor dense(const torch::Tensor& t) { return t.defined() ? t.contiguous() : t; }

// q, k -> q', k'; either may be undefined, and its result is then too.
std::pair<torch::Tensor, torch::Tensor> rotate(const torch::Tensor& q, const torch::Tensor& k, const RotaryArgs& r, bool inverse) {
  const torch::Tensor& x = q.defined() ? q : k;
  c10::cuda::CUDAGuard guard(x.device());
  torch::Tensor q_out, k_out;
  omni_attn_heads hq{}, hk{};
  if (q.defined()) {
    q_out = at::empty(q.sizes(), q.options());
    hq = heads_arg(q);
  }
  if (k.defined()) {
    k_out = at::empty(k.sizes(), k.options());
    hk = heads_arg(k);
  }
  const omni_attn_rotary a = rotary_arg(r);
  const int rc = library.rotary(q.defined() ? &hq : nullptr, k.defined() ? &hk : nullptr, q.defined() ? q_out.data_ptr() : nullptr,
                                k.defined() ? k_out.data_ptr() : nullptr, &a, static_cast<int>(x.size(0)), static_cast<int>(x.size(2)),
                                static_cast<int>(x.size(3)), dtype_code(x), inverse ? 1 : 0, at::cuda::getCurrentCUDAStream().stream());
  if (rc != OMNI_OK) refuse_rc(rc);
  return {q_out, k_out};
}

// A backward that is being captured, into leaves whose accumulators belong to the default stream (made by a graph outside the
// capture that is still alive): autograd would make the default stream wait for the captured one, which fails inside its
// engine and can end the process. Said here instead, while the capture is still sound.
void refuse_leaves_outside_the_capture() {
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(at::cuda::getCurrentCUDAStream().stream(), &capturing) != cudaSuccess) {
    (void)cudaGetLastError();   // the launch will say it
    return;
  }
  const auto node = torch::autograd::get_current_node();
  if (!node || capturing == cudaStreamCaptureStatusNone) return;
  for (const auto& edge : node->next_edges()) {
    if (!edge.function || dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get()) == nullptr) continue;
    const auto stream = edge.function->stream();
    if (stream && stream->device_type() == c10::DeviceType::CUDA && c10::cuda::CUDAStream(*stream).stream() == nullptr) {
      refuse("omni_rotary: this backward is captured into a CUDA graph, but a leaf's gradient accumulator belongs to the default stream: "
             "drop every graph of the same leaves that was built outside the capture (warm up on a side stream)");
    }
  }
}

struct OmniRotaryFn : torch::autograd::Function<OmniRotaryFn> {
  // The result of q, if there is a q, then that of k.
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Optional& q_in, const Optional& k_in,
                                                const Optional& q_weight, const Optional& k_weight, const Optional& inv_freq,
                                                const Optional& positions, bool half, double factor, double eps) {
    const torch::Tensor q = or_none(q_in), k = or_none(k_in);
    const RotaryArgs r{or_none(inv_freq), or_none(positions), dense(or_none(q_weight)), dense(or_none(k_weight)), half, factor, eps};
    const auto out = rotate(q, k, r, false);
    // what the backward reads: the inputs only where there is a norm
    ctx->save_for_backward({r.q_weight.defined() ? q : torch::Tensor(), r.k_weight.defined() ? k : torch::Tensor(), r.q_weight, r.k_weight,
                            r.inv_freq, r.positions});
    ctx->saved_data["q"] = q.defined();
    ctx->saved_data["k"] = k.defined();
    ctx->saved_data["half"] = half;
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["eps"] = eps;
    torch::autograd::variable_list list;
    if (q.defined()) list.push_back(out.first);
    if (k.defined()) list.push_back(out.second);
    return list;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    // The kernels' results have no graph of their own: what create_graph=True asks for would be missing, silently.
    if (at::GradMode::is_enabled()) refuse("omni_rotary has no second derivative (create_graph=True)");
    refuse_leaves_outside_the_capture();
    const auto saved = ctx->get_saved_variables();
    RotaryArgs r{saved[4], saved[5], saved[2], saved[3], ctx->saved_data["half"].toBool(), ctx->saved_data["factor"].toDouble(),
                 ctx->saved_data["eps"].toDouble()};
    torch::Tensor g[2], dx[2], dw[2];
    size_t next = 0;
    for (int i = 0; i < 2; ++i) {
      if (!ctx->saved_data[i == 0 ? "q" : "k"].toBool()) continue;
      if (grads[next].defined()) g[i] = with_rows(grads[next]);
      ++next;
    }
    const torch::Tensor w[2] = {r.q_weight, r.k_weight};
    torch::Tensor plain[2];   // gradients whose way back is the rotation alone
    for (int i = 0; i < 2; ++i) {
      if (g[i].defined() && !w[i].defined()) plain[i] = g[i];
    }
    if (plain[0].defined() || plain[1].defined()) {
      RotaryArgs back = r;
      back.q_weight = back.k_weight = torch::Tensor();
      std::tie(dx[0], dx[1]) = rotate(plain[0], plain[1], back, true);
    }
    bool normed[2] = {g[0].defined() && w[0].defined(), g[1].defined() && w[1].defined()};
    if (normed[0] || normed[1]) {
      omni_attn_heads hx[2], hg[2];
      const torch::Tensor& any = normed[0] ? saved[0] : saved[1];
      c10::cuda::CUDAGuard guard(any.device());
      for (int i = 0; i < 2; ++i) {
        if (!normed[i]) continue;
        hx[i] = heads_arg(saved[i]);
        hg[i] = heads_arg(g[i]);
        dx[i] = at::empty(saved[i].sizes(), saved[i].options());
        dw[i] = at::empty(w[i].sizes(), w[i].options());
      }
      const int B = static_cast<int>(any.size(0)), N = static_cast<int>(any.size(2)), D = static_cast<int>(any.size(3));
      const omni_attn_rotary a = rotary_arg(r);
      const long long need = library.rotary_bwd_workspace(normed[0] ? hx[0].heads : 0, normed[1] ? hx[1].heads : 0, B, N, D, a.weight_per_head);
      auto workspace = at::empty({need}, any.options().dtype(torch::kUInt8));
      auto at_if = [&](bool yes, const torch::Tensor& t) { return yes ? t.data_ptr() : nullptr; };
      const int rc = library.rotary_bwd(normed[0] ? &hx[0] : nullptr, normed[1] ? &hx[1] : nullptr, normed[0] ? &hg[0] : nullptr,
                                        normed[1] ? &hg[1] : nullptr, at_if(normed[0], dx[0]), at_if(normed[1], dx[1]),
                                        at_if(normed[0], dw[0]), at_if(normed[1], dw[1]), &a, B, N, D, dtype_code(any),
                                        workspace.data_ptr(), need, at::cuda::getCurrentCUDAStream().stream());
      if (rc != OMNI_OK) refuse_rc(rc);
    }
    return {dx[0], dx[1], dw[0], dw[1], torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

bool wants_grad(std::initializer_list<const torch::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const torch::Tensor* t : ts) {
    if (t->defined() && t->requires_grad()) return true;
  }
  return false;
}

// A tangent of forward-mode differentiation would be dropped: the kernels' results have none.
void check_no_tangent(const char* what, std::initializer_list<const torch::Tensor*> ts) {
  for (const torch::Tensor* t : ts) {
    OMNI_REQUIRE(!t->defined() || !t->_fw_grad(0).defined(), std::string(what) + " has no forward-mode derivative: an input carries a tangent");
  }
}

pybind11::object result(const torch::Tensor& t) { return t.defined() ? pybind11::cast(t) : pybind11::object(pybind11::none()); }

pybind11::tuple rotary(const Optional& q_in, const Optional& k_in, const Optional& inv_freq, bool half, double factor,
                       const Optional& positions, const Optional& q_weight, const Optional& k_weight, double eps) {
  torch::Tensor q = or_none(q_in), k = or_none(k_in);
  RotaryArgs r{or_none(inv_freq), or_none(positions), or_none(q_weight), or_none(k_weight), half, factor, eps};
  std::pair<torch::Tensor, torch::Tensor> out;
  {
    pybind11::gil_scoped_release nogil;
    OMNI_REQUIRE(q.defined() || k.defined(), "omni_rotary needs q or k");
    if (q.defined()) check_heads(q, "q", true);
    if (k.defined()) check_heads(k, "k", true);
    if (q.defined() && k.defined()) {
      OMNI_REQUIRE(q.scalar_type() == k.scalar_type() && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
              "q and k must share dtype, batch, length and head_dim: " + shape_of(q) + " and " + shape_of(k));
    }
    check_rotary_args(r, q, k);
    OMNI_REQUIRE(!wants_grad({&r.inv_freq}), "omni_rotary has no gradient of inv_freq: detach it, or call it under torch.no_grad()");
    check_no_tangent("omni_rotary", {&q, &k, &r.q_weight, &r.k_weight, &r.inv_freq});
    check_device(q.defined() ? q : k, {&q, &k, &r.inv_freq, &r.positions, &r.q_weight, &r.k_weight});
    if (q.defined()) q = with_rows(q);
    if (k.defined()) k = with_rows(k);
    if (wants_grad({&q, &k, &r.q_weight, &r.k_weight})) {
      auto given = [](const torch::Tensor& t) { return t.defined() ? Optional(t) : Optional(); };
      const auto list = OmniRotaryFn::apply(given(q), given(k), given(r.q_weight), given(r.k_weight), given(r.inv_freq), given(r.positions),
                                            half, factor, eps);
      if (q.defined()) out.first = list.front();
      if (k.defined()) out.second = list.back();
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      r.q_weight = dense(r.q_weight);
      r.k_weight = dense(r.k_weight);
      out = rotate(q, k, r, false);
    }
  }
  return pybind11::make_tuple(result(out.first), result(out.second));
}

// The tensors of a paged cache, as the C ABI takes them.
omni_attn_paged_cache cache_arg(const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& table,
                                const torch::Tensor& lengths, int64_t B, int64_t D, c10::ScalarType dtype) {
  OMNI_REQUIRE(k_pages.dim() == 4 && v_pages.sizes() == k_pages.sizes(), "k_pages and v_pages must be [num_pages, heads, page_size, D] of one shape");
  OMNI_REQUIRE(k_pages.scalar_type() == dtype && v_pages.scalar_type() == dtype, "the cache and the new tokens must share a dtype");
  OMNI_REQUIRE(k_pages.size(3) == D, "the cache's head_dim is not that of the new tokens");
  OMNI_REQUIRE(k_pages.is_contiguous() && v_pages.is_contiguous(), "k_pages and v_pages must be contiguous");
  OMNI_REQUIRE(table.dim() == 2 && table.size(0) == B && table.scalar_type() == torch::kInt32 && (table.size(1) <= 1 || table.stride(1) == 1),
          "page_table must be int32 [B, max_pages]");
  OMNI_REQUIRE(lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == torch::kInt32 && (B == 1 || lengths.stride(0) == 1),
          "lengths must be int32 [B]");
  OMNI_REQUIRE(k_pages.size(0) <= INT_MAX && table.size(1) <= INT_MAX, "too many pages");
  return {k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr<int32_t>(), B > 1 ? table.stride(0) : 0, lengths.data_ptr<int32_t>(),
          static_cast<int>(k_pages.size(0)), static_cast<int>(table.size(1)), static_cast<int>(k_pages.size(2)),
          static_cast<int>(k_pages.size(1))};
}

const int32_t* int32_or_null(const torch::Tensor& t, c10::IntArrayRef shape, const char* what) {
  if (!t.defined()) return nullptr;
  OMNI_REQUIRE(t.scalar_type() == torch::kInt32 && t.sizes() == shape && t.is_contiguous(), what);
  return t.data_ptr<int32_t>();
}

pybind11::object cache_append(const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& table,
                              const torch::Tensor& lengths, torch::Tensor k, torch::Tensor v, const Optional& q_in,
                              const Optional& inv_freq, bool half, double factor, const Optional& positions, const Optional& counts_in,
                              const Optional& q_weight, const Optional& k_weight, double eps, const Optional& status_in) {
  torch::Tensor q = or_none(q_in), counts = or_none(counts_in), status = or_none(status_in), q_out;
  RotaryArgs r{or_none(inv_freq), or_none(positions), or_none(q_weight), or_none(k_weight), half, factor, eps};
  {
    pybind11::gil_scoped_release nogil;
    check_heads(k, "k", false);
    check_heads(v, "v", false);
    OMNI_REQUIRE(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "k and v must share shape and dtype");
    if (q.defined()) {
      check_heads(q, "q", false);
      OMNI_REQUIRE(q.scalar_type() == k.scalar_type() && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
              "q and k must share dtype, batch, length and head_dim: " + shape_of(q) + " and " + shape_of(k));
    }
    check_rotary_args(r, q, k);
    const int64_t B = k.size(0), N = k.size(2), D = k.size(3);
    const omni_attn_paged_cache cache = cache_arg(k_pages, v_pages, table, lengths, B, D, k.scalar_type());
    OMNI_REQUIRE(cache.heads == k.size(1), "the cache's heads are not those of k");
    const int32_t* counts_ptr = int32_or_null(counts, {B}, "counts must be contiguous int32 [B]");
    int32_t* status_ptr = const_cast<int32_t*>(int32_or_null(status, {1}, "status must be int32 [1]"));
    OMNI_REQUIRE(!wants_grad({&q, &k, &v, &r.q_weight, &r.k_weight, &r.inv_freq, &k_pages, &v_pages}),
            "omni_cache_append has no backward: call it under torch.no_grad(), or on tensors that need no gradient");
    check_no_tangent("omni_cache_append", {&q, &k, &v, &r.q_weight, &r.k_weight, &r.inv_freq, &k_pages, &v_pages});
    check_device(k, {&v, &q, &k_pages, &v_pages, &table, &lengths, &counts, &status, &r.inv_freq, &r.positions, &r.q_weight, &r.k_weight});
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(k.device());
    k = with_rows(k);
    v = with_rows(v);
    r.q_weight = dense(r.q_weight);
    r.k_weight = dense(r.k_weight);
    omni_attn_heads hq{}, hk = heads_arg(k), hv = heads_arg(v);
    if (q.defined()) {
      q = with_rows(q);
      hq = heads_arg(q);
      q_out = at::empty(q.sizes(), q.options());
    }
    const omni_attn_rotary a = rotary_arg(r);
    const int rc = library.cache_append(q.defined() ? &hq : nullptr, &hk, &hv, q.defined() ? q_out.data_ptr() : nullptr, &cache, counts_ptr,
                                        &a, static_cast<int>(B), static_cast<int>(N), static_cast<int>(D), dtype_code(k),
                                        at::cuda::getCurrentCUDAStream().stream(), status_ptr);
    if (rc != OMNI_OK) refuse_rc(rc);
    // A backward that saved the pages before this write must not use them after it, as behind any operation in place.
    for (const torch::Tensor* t : {&k_pages, &v_pages}) {
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
  }
  return result(q_out);
}

pybind11::object cache_attention(torch::Tensor q, const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& table,
                                 const torch::Tensor& lengths, const Optional& counts_in, bool causal, const Optional& limits_in,
                                 double scale, double softcap, bool want_lse, int64_t shared_prefix, const Optional& status_in) {
  torch::Tensor counts = or_none(counts_in), limits = or_none(limits_in), status = or_none(status_in), out, lse;
  {
    pybind11::gil_scoped_release nogil;
    check_heads(q, "q", false);
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
    const omni_attn_paged_cache cache = cache_arg(k_pages, v_pages, table, lengths, B, D, q.scalar_type());
    OMNI_REQUIRE(cache.heads > 0 && H % cache.heads == 0, "the cache's heads must divide the queries' heads");
    const int32_t* counts_ptr = int32_or_null(counts, {B}, "counts must be contiguous int32 [B]");
    const int32_t* limits_ptr = int32_or_null(limits, {B, T}, "limits must be contiguous int32 [B, T]");
    int32_t* status_ptr = const_cast<int32_t*>(int32_or_null(status, {1}, "status must be int32 [1]"));
    OMNI_REQUIRE(std::isfinite(static_cast<float>(scale)) && std::isfinite(static_cast<float>(softcap)) && scale >= 0.0, "scale and softcap must be finite, scale not negative");
    const double scale_used = scale > 0.0 ? scale : 1.0 / std::sqrt(static_cast<double>(D));
    OMNI_REQUIRE(!(softcap > 0.0) || (softcap >= 1.1e-6 * scale_used && softcap <= 0.9e30 * scale_used && softcap <= 0.9e37),
                 "softcap must be between 1e-6 and 1e30 times the scale, and below 1e37 (None or 0: no soft-cap)");
    OMNI_REQUIRE(shared_prefix >= 0 && shared_prefix <= table.size(1) * k_pages.size(2), "shared_prefix must be from 0 to the tokens that the page table holds");
    OMNI_REQUIRE(!wants_grad({&q, &k_pages, &v_pages}),
            "omni_cache_attention has no backward: call it under torch.no_grad(), or on tensors that need no gradient");
    check_no_tangent("omni_cache_attention", {&q, &k_pages, &v_pages});
    check_device(q, {&k_pages, &v_pages, &table, &lengths, &counts, &limits, &status});
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(q.device());
    // 16-byte loads of whole rows
    const bool aligned = q.stride(3) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && q.stride(2) % 8 == 0 &&
                         reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
    if (!aligned) q = q.clone(at::MemoryFormat::Contiguous);
    out = at::empty(q.sizes(), q.options());
    if (want_lse) lse = at::empty({B, H, T}, q.options().dtype(torch::kFloat32));
    const long long need = library.cache_attention_workspace(static_cast<int>(B), static_cast<int>(H), cache.heads, static_cast<int>(T),
                                                             static_cast<int>(D), shared_prefix > 0,
                                                             static_cast<long long>(cache.max_pages) * cache.page_size);
    torch::Tensor workspace;
    if (need > 0) workspace = at::empty({need}, q.options().dtype(torch::kUInt8));
    const omni_attn_heads hq = heads_arg(q);
    const int rc = library.cache_attention(&hq, out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr, &cache, counts_ptr, limits_ptr,
                                           causal ? 1 : 0, static_cast<int>(B), static_cast<int>(T), static_cast<int>(D), dtype_code(q),
                                           static_cast<float>(scale), static_cast<float>(softcap > 0 ? softcap : 0.0),
                                           static_cast<int>(shared_prefix), need > 0 ? workspace.data_ptr() : nullptr, need,
                                           at::cuda::getCurrentCUDAStream().stream(), status_ptr);
    if (rc != OMNI_OK) refuse_rc(rc);
  }
  if (want_lse) return pybind11::make_tuple(out, lse);
  return pybind11::cast(out);
}

#undef OMNI_REQUIRE

void define_cache(pybind11::module_& m) {
  m.def("rotary", &rotary, "norms and rotation of queries and keys");
  m.def("cache_append", &cache_append, "new tokens into a paged cache");
  m.def("cache_attention", &cache_attention, "attention of new tokens over a paged cache");
}

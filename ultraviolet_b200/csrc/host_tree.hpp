// Host paths of the drafted-token, cache-copy and logit operators: argument checks, argument blocks, launches.  Part of host.cpp.
// With `force` unset a function returns None (fork: false) where something watches the call or a gradient is wanted, and the caller
// goes through its torch operator, which calls back with `force` set.
#pragma once

// Tensors of one call, all on the first one's device; None stands for an undefined one.  What take and list hand out is the caller's own
// tensor: its reference is held by the argument, or by the sequence that `held` keeps.
using Tensors = std::vector<const Tensor*>;
struct Call {
  bool force, direct = true;
  std::optional<c10::Device> dev;
  std::vector<py::object> held;
  Call(bool f) : force(f) { direct = f || modes_off(); }
  const Tensor& take(py::handle h, const char* name) {
    const Tensor* t = exact(h);
    if (!t) {
      if (!THPVariable_Check(h.ptr())) throw py::type_error(std::string(name) + " has to be a tensor");
      direct = false;                     // a subclass: its own rules apply
      return THPVariable_Unpack(h.ptr());
    }
    if (!direct) return *t;
    TORCH_CHECK(t->is_cuda(), "ultraviolet_b200 kernels run on CUDA tensors only (no CPU fallback); got a ", t->device(), " tensor (", name,
                ")");
    if (!dev) dev = t->device();
    TORCH_CHECK(t->device() == *dev, "tensors on different devices: ", *dev, " and ", t->device(), " (", name, ")");
    if (!force && !plain(*t, *dev)) direct = false;
    return *t;
  }
  const Tensor& maybe(py::handle h, const char* name) {
    static const Tensor none;
    return h.is_none() ? none : take(h, name);
  }
  Tensors list(const py::sequence& s, const char* name) {
    PyObject* fast = PySequence_Fast(s.ptr(), "one tensor per layer has to be given as a sequence");
    if (!fast) throw py::error_already_set();
    held.push_back(py::reinterpret_steal<py::object>(fast));
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    PyObject** items = PySequence_Fast_ITEMS(fast);
    Tensors v;
    v.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) v.push_back(&take(items[i], name));
    return v;
  }
};

bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
const char* half_types = "takes float16 and bfloat16";

// int64 (B,), contiguous
Tensor index_of(const Tensor& t, int64_t B, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == B, name, " has to hold one value for each of ", B, " rows; got ", t.sizes());
  TORCH_CHECK_VALUE(at::isIntegralType(t.scalar_type(), false), name, " has to hold integers; got ", t.scalar_type());
  return t.scalar_type() == at::kLong && t.is_contiguous() ? t : t.to(at::kLong).contiguous();
}
// Integers of any type as int32, those beyond lo .. hi (which name nothing either) as the nearer of the two.
Tensor int32_of(const Tensor& t, int64_t lo, int64_t hi) {
  if (t.scalar_type() == at::kInt) return t;
  // (narrower types may not hold the bounds, and fit as they are)
  return t.element_size() < 4 ? t.to(at::kInt) : t.to(at::kLong).clamp(lo, hi).to(at::kInt);
}
// parents (B, T) or (T,) as int32 with unit stride along T
Tensor parents_of(const Tensor& p, int64_t B, int64_t T, int64_t& stride) {
  TORCH_CHECK_VALUE((p.dim() == 2 && p.size(0) == B && p.size(1) == T) || (p.dim() == 1 && p.size(0) == T), "parents have to be (", B, ", ", T,
                    ") or (", T, ",); got ", p.sizes());
  TORCH_CHECK_VALUE(at::isIntegralType(p.scalar_type(), false), "parents have to be integers; got ", p.scalar_type());
  TORCH_CHECK_VALUE(T <= 64, "a tree has at most 64 nodes; got ", T);
  Tensor q = int32_of(p, -2, 64);
  if (T > 1 && q.stride(-1) != 1) q = q.contiguous();
  stride = q.dim() == 2 ? q.stride(0) : 0;
  return q;
}
// 16-byte pieces of the inner dimension can be read
bool has_vectors(const Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int64_t i = 0; ok && i + 1 < t.dim(); ++i) ok = t.size(i) == 1 || t.stride(i) % 8 == 0;
  return ok;
}
// stride of a dimension; of one element, whose stride counts for nothing, none where it would not be a multiple of what kernels ask for
int64_t step_of(const Tensor& t, int64_t i, int64_t multiple = 8) { return t.size(i) == 1 && t.stride(i) % multiple ? 0 : t.stride(i); }
Tensor vectors_of(const Tensor& t) { return has_vectors(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

struct Cache {
  int64_t rows, KH, S, hd;
};
Cache cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && k.scalar_type() == at::kChar && v.scalar_type() == at::kChar,
                    "the caches have to be int8 tensors (rows, kv heads, slots, head_dim); got ", k.sizes(), " ", k.scalar_type(), " and ",
                    v.sizes(), " ", v.scalar_type());
  TORCH_CHECK_VALUE(ks.sizes() == k.sizes().slice(0, 3) && vs.sizes() == ks.sizes() && ks.scalar_type() == at::kHalf &&
                        vs.scalar_type() == at::kHalf,
                    "the scales have to be float16 tensors (rows, kv heads, slots); got ", ks.sizes(), " and ", vs.sizes());
  return {k.size(0), k.size(1), k.size(2), k.size(3)};
}
void check_head_dim(int64_t hd) {
  TORCH_CHECK_VALUE(hd == 16 || hd == 32 || hd == 64 || hd == 128, "head_dim has to be 16, 32, 64 or 128; got ", hd);
}

std::optional<Tensor> tree_positions(py::handle hparents, py::handle hpos, bool force) {
  Call c(force);
  const Tensor p_ = c.take(hparents, "parents"), pos_ = c.take(hpos, "pos");
  if (!c.direct) return std::nullopt;
  TORCH_CHECK_VALUE(pos_.dim() == 1 && p_.dim() >= 1, "tree_positions takes parents (B, T) or (T,) and pos (B,)");
  const int64_t B = pos_.size(0), T = p_.size(-1);
  c10::cuda::CUDAGuard guard(*c.dev);
  int64_t stride;
  const Tensor parents = parents_of(p_, B, T, stride), pos = index_of(pos_, B, "pos");
  Tensor out = at::empty({B, T}, pos.options());
  check(L.tree_positions(parents.const_data_ptr<int32_t>(), stride, pos.const_data_ptr<int64_t>(), (int)B, (int)T,
                         out.mutable_data_ptr<int64_t>(), at::cuda::getCurrentCUDAStream().stream()),
        "uv_tree_positions");
  return out;
}

std::optional<Tensor> tree_attention(py::handle hq, py::handle hk, py::handle hv, py::handle hkc, py::handle hvc, py::handle hpos,
                                     py::handle hstarts, py::handle hparents, double scale, py::handle hks, py::handle hvs,
                                     int64_t window, int64_t ring, py::handle hrow_map, int64_t splits, py::handle hxsa, double xsa_eps,
                                     py::handle hgate, py::handle hout, py::handle hstatus, bool force) {
  Call c(force);
  Tensor q = c.take(hq, "q"), k = c.take(hk, "k"), v = c.take(hv, "v");
  const Tensor kc = c.take(hkc, "k_cache"), vc = c.take(hvc, "v_cache"), pos_ = c.take(hpos, "pos"), starts_ = c.take(hstarts, "starts");
  const Tensor parents_ = c.take(hparents, "parents"), ks = c.take(hks, "k_scale"), vs = c.take(hvs, "v_scale");
  const Tensor rm_ = c.maybe(hrow_map, "row_map"), xsa = c.maybe(hxsa, "xsa_alpha"), gate = c.maybe(hgate, "gate_vals");
  Tensor out = c.maybe(hout, "out");
  const Tensor status = c.maybe(hstatus, "status");
  if (!c.direct) return std::nullopt;
  TORCH_CHECK_VALUE(q.dim() == 4, "q has to be (B, T, heads, head_dim); got ", q.sizes());
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), hd = q.size(3);
  const Cache y = cache_of(kc, vc, ks, vs);
  TORCH_CHECK_VALUE(half_type(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "tree_attention ", half_types,
                    ", one of them for q, k and v; got ", q.scalar_type(), ", ", k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(k.dim() == 4 && k.size(0) == B && k.size(1) == T && k.size(2) == y.KH && k.size(3) == hd && v.sizes() == k.sizes() &&
                        y.hd == hd,
                    "k and v have to be (B, T, kv heads, head_dim) of q ", q.sizes(), " and the cache ", kc.sizes(), "; got ", k.sizes(), " and ",
                    v.sizes());
  check_head_dim(hd);
  TORCH_CHECK_VALUE(y.KH > 0 && H > 0 && H % y.KH == 0 && H / y.KH <= 16, "each kv head serves 1 to 16 query heads; got ", H, " and ", y.KH);
  TORCH_CHECK_VALUE(window >= 0 && splits >= 0 && y.S >= 1, "window and num_splits cannot be negative, nor a cache without slots");
  TORCH_CHECK_VALUE(rm_.defined() || y.rows >= B, "the cache has ", y.rows, " rows for a batch of ", B);
  TORCH_CHECK_VALUE(kc.stride(3) == 1 && vc.stride(3) == 1 && (y.S == 1 || (ks.stride(2) == 1 && vs.stride(2) == 1)),
                    "the caches need unit stride along head_dim, the scales along the slots");
  if (xsa.defined()) TORCH_CHECK_VALUE(xsa.scalar_type() == at::kFloat && xsa.is_contiguous() && xsa.numel() == H, "xsa_alpha has to be float32 (heads,)");
  if (gate.defined())
    TORCH_CHECK_VALUE(gate.scalar_type() == at::kFloat && gate.is_contiguous() && gate.numel() == B * T * H, "gate_vals have to be float32 (B * T, heads)");
  if (status.defined()) TORCH_CHECK_VALUE(status.scalar_type() == at::kInt && status.numel() >= 1, "status has to be an int32 word");
  c10::cuda::CUDAGuard guard(*c.dev);
  int64_t pstride;
  const Tensor parents = parents_of(parents_, B, T, pstride), pos = index_of(pos_, B, "pos"), starts = index_of(starts_, B, "starts");
  const Tensor rm = rm_.defined() ? index_of(rm_, B, "row_map") : rm_;
  if (out.defined()) {
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && has_vectors(out),
                      "out has to be like q, with 16-byte aligned vectors");
  } else {
    out = at::empty({B, T, H, hd}, q.options());
  }
  if (B == 0 || T == 0) return out;
  q = vectors_of(q), k = vectors_of(k), v = vectors_of(v);
  uv_tree_attn_args a{};
  a.q = ro(q), a.k = ro(k), a.v = ro(v), a.dtype = code_of(q.scalar_type());
  a.sqb = step_of(q, 0), a.sqt = step_of(q, 1), a.sqh = step_of(q, 2);
  a.snkb = step_of(k, 0), a.snkt = step_of(k, 1), a.snkh = step_of(k, 2), a.snvb = step_of(v, 0), a.snvt = step_of(v, 1), a.snvh = step_of(v, 2);
  a.parents = parents.const_data_ptr<int32_t>(), a.parents_stride = pstride;
  a.k_cache = kc.const_data_ptr<int8_t>(), a.v_cache = vc.const_data_ptr<int8_t>();
  a.skb = step_of(kc, 0, 16), a.skh = step_of(kc, 1, 16), a.sks = step_of(kc, 2, 16);
  a.svb = step_of(vc, 0, 16), a.svh = step_of(vc, 1, 16), a.svs = step_of(vc, 2, 16);
  a.k_scale = static_cast<const uint16_t*>(ro(ks)), a.v_scale = static_cast<const uint16_t*>(ro(vs));
  a.ssb = step_of(ks, 0), a.ssh = step_of(ks, 1), a.stb = step_of(vs, 0), a.sth = step_of(vs, 1);
  a.pos = pos.const_data_ptr<int64_t>(), a.starts = starts.const_data_ptr<int64_t>();
  a.row_map = rm.defined() ? rm.const_data_ptr<int64_t>() : nullptr, a.n_rows = (int)y.rows;
  a.out = out.mutable_data_ptr(), a.sob = step_of(out, 0), a.sot = step_of(out, 1), a.soh = step_of(out, 2);
  a.B = (int)B, a.T = (int)T, a.H = (int)H, a.KH = (int)y.KH, a.hd = (int)hd, a.S = (int)y.S;
  a.S_alloc = (int)row_alloc(kc, vc, ks, vs, y.S), a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.ring = ring < 0 ? window > 0 : ring != 0, a.scale = (float)scale, a.num_splits = (int)std::min<int64_t>(splits, INT32_MAX);
  a.xsa_alpha = xsa.defined() ? xsa.const_data_ptr<float>() : nullptr, a.xsa_eps = (float)xsa_eps;
  a.gate_vals = gate.defined() ? gate.const_data_ptr<float>() : nullptr;
  a.status = status.defined() ? status.mutable_data_ptr<int>() : nullptr;
  Tensor ws;
  if (const size_t n = L.tree_attn_workspace(&a)) {
    ws = at::empty({(int64_t)n}, q.options().dtype(at::kByte));
    a.workspace = ws.mutable_data_ptr(), a.workspace_bytes = n;
  }
  check(L.tree_attn(&a, at::cuda::getCurrentCUDAStream().stream()), "uv_tree_attn");
  return out;
}

// the layers' caches: (rows, KH, S, hd) views of contiguous (rows, KH, S_alloc, hd) memory
struct Layers {
  std::vector<uv_tree_layer> y;
  int64_t rows = 0, KH = 0, hd = 0;
};
Layers layers_of(const Tensors& hk, const Tensors& hv, const Tensors& hks, const Tensors& hvs, const std::vector<bool>& rings) {
  const size_t n = hk.size();
  TORCH_CHECK_VALUE(n >= 1 && n <= 32 && hv.size() == n && hks.size() == n && hvs.size() == n && rings.size() == n,
                    "one cache, one scale and one ring flag per layer, 1 to 32 layers; got ", n, ", ", hv.size(), ", ", hks.size(), ", ", hvs.size(),
                    " and ", rings.size());
  Layers r;
  r.y.reserve(n);
  for (size_t l = 0; l < n; ++l) {
    const Tensor &k = *hk[l], &v = *hv[l], &ks = *hks[l], &vs = *hvs[l];
    const Cache c = cache_of(k, v, ks, vs);
    if (l == 0) r.rows = c.rows, r.KH = c.KH, r.hd = c.hd;
    TORCH_CHECK_VALUE(c.rows == r.rows && c.KH == r.KH && c.hd == r.hd, "the layers' caches differ in rows, kv heads or head_dim");
    const int64_t alloc = c.KH > 1 ? ks.stride(1) : c.rows > 1 ? ks.stride(0) / std::max<int64_t>(c.KH, 1) : row_alloc(k, v, ks, vs, c.S);
    auto fits = [&](const Tensor& t, int64_t inner) {
      return (t.size(0) <= 1 || t.stride(0) == c.KH * alloc * inner) && (c.KH <= 1 || t.stride(1) == alloc * inner) &&
             (c.S <= 1 || t.stride(2) == inner) && (inner == 1 || t.stride(3) == 1);
    };
    TORCH_CHECK_VALUE(c.S >= 1 && alloc >= c.S && fits(k, c.hd) && fits(v, c.hd) && fits(ks, 1) && fits(vs, 1),
                      "the caches of layer ", l, " have to be views [:, :, :S] of contiguous (rows, kv heads, slots, head_dim) tensors");
    uv_tree_layer y{};
    y.k_cache = k.mutable_data_ptr<int8_t>(), y.v_cache = v.mutable_data_ptr<int8_t>();
    y.k_scale = static_cast<uint16_t*>(ks.mutable_data_ptr()), y.v_scale = static_cast<uint16_t*>(vs.mutable_data_ptr());
    y.S = (int)c.S, y.S_alloc = (int)alloc, y.ring = rings[l];
    r.y.push_back(y);
  }
  return r;
}

std::optional<std::tuple<Tensor, Tensor, Tensor>> tree_advance(const py::sequence& hk, const py::sequence& hv, const py::sequence& hkc,
                                                               const py::sequence& hvc, const py::sequence& hks, const py::sequence& hvs,
                                                               const std::vector<bool>& rings, py::handle hparents, py::handle htokens,
                                                               py::handle htarget, py::handle hpos, py::handle hrow_map,
                                                               py::handle hpos_out, py::handle hoob, bool force) {
  Call c(force);
  const Tensors tk = c.list(hk, "k"), tv = c.list(hv, "v");
  const Tensors kc = c.list(hkc, "k_caches"), vc = c.list(hvc, "v_caches"), ks = c.list(hks, "k_scales"), vs = c.list(hvs, "v_scales");
  const Tensor parents_ = c.take(hparents, "parents"), tokens_ = c.take(htokens, "tokens"), target_ = c.take(htarget, "target");
  const Tensor pos_ = c.take(hpos, "pos"), rm_ = c.maybe(hrow_map, "row_map"), pos_out = c.take(hpos_out, "pos_out"), oob = c.maybe(hoob, "oob");
  if (!c.direct) return std::nullopt;
  Layers y = layers_of(kc, vc, ks, vs, rings);
  const size_t n = y.y.size();
  TORCH_CHECK_VALUE(tk.size() == n && tv.size() == n && tk[0]->dim() == 4, "one k and one v (B, T, kv heads, head_dim) per layer");
  const Tensor* k0 = tk[0];
  const Tensor* v0 = tv[0];
  const int64_t B = k0->size(0), T = k0->size(1);
  check_head_dim(y.hd);
  TORCH_CHECK_VALUE(T >= 1, "a tree has at least one node");
  TORCH_CHECK_VALUE(half_type(*k0), "tree_advance ", half_types, "; got ", k0->scalar_type());
  TORCH_CHECK_VALUE(rm_.defined() || y.rows >= B, "the caches have ", y.rows, " rows for a batch of ", B);
  for (const Tensor* t : {&tokens_, &target_})
    TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == B && t->size(1) == T && at::isIntegralType(t->scalar_type(), false),
                      "tokens and target have to be integers (", B, ", ", T, "); got ", t->sizes(), " ", t->scalar_type());
  TORCH_CHECK_VALUE(pos_out.dim() == 1 && pos_out.size(0) == B && pos_out.scalar_type() == at::kLong && pos_out.is_contiguous(),
                    "pos_out has to be a contiguous int64 tensor (", B, ",)");
  if (oob.defined()) TORCH_CHECK_VALUE(oob.scalar_type() == at::kInt && oob.numel() >= 1, "oob has to be an int32 word");
  c10::cuda::CUDAGuard guard(*c.dev);
  bool copy = false;
  for (size_t l = 0; l < n; ++l) {
    for (const Tensor* t : {tk[l], tv[l]}) {
      TORCH_CHECK_VALUE(t->dim() == 4 && t->size(0) == B && t->size(1) == T && t->size(2) == y.KH && t->size(3) == y.hd &&
                            t->scalar_type() == k0->scalar_type(),
                        "k and v have to be (", B, ", ", T, ", ", y.KH, ", ", y.hd, ") of one type in every layer; got ", t->sizes());
      copy |= !has_vectors(*t);
    }
    // one set of strides serves all layers
    copy |= tk[l]->strides() != k0->strides() || tv[l]->strides() != v0->strides();
  }
  std::vector<Tensor> copies;
  if (copy) copies.reserve(2 * n);
  for (size_t l = 0; l < n; ++l) {
    const Tensor *k = tk[l], *v = tv[l];
    if (copy) {
      copies.push_back(k->clone(at::MemoryFormat::Contiguous)), k = &copies.back();
      copies.push_back(v->clone(at::MemoryFormat::Contiguous)), v = &copies.back();
      if (l == 0) k0 = k, v0 = v;
    }
    y.y[l].k = ro(*k), y.y[l].v = ro(*v);
  }
  int64_t pstride;
  const Tensor parents = parents_of(parents_, B, T, pstride), pos = index_of(pos_, B, "pos");
  const Tensor rm = rm_.defined() ? index_of(rm_, B, "row_map") : rm_;
  const Tensor tokens = tokens_.to(at::kLong).contiguous(), target = target_.to(at::kLong).contiguous();
  Tensor path = at::empty({B, T}, parents.options()), count = at::empty({B}, parents.options()), drawn = at::empty({B, T}, pos.options());
  uv_tree_advance_args a{};
  a.dtype = code_of(k0->scalar_type()), a.B = (int)B, a.T = (int)T, a.KH = (int)y.KH, a.hd = (int)y.hd, a.n_layers = (int)n;
  a.skb = step_of(*k0, 0), a.skt = step_of(*k0, 1), a.skh = step_of(*k0, 2);
  a.svb = step_of(*v0, 0), a.svt = step_of(*v0, 1), a.svh = step_of(*v0, 2);
  a.parents = parents.const_data_ptr<int32_t>(), a.parents_stride = pstride;
  a.tokens = tokens.const_data_ptr<int64_t>(), a.target = target.const_data_ptr<int64_t>(), a.pos = pos.const_data_ptr<int64_t>();
  a.row_map = rm.defined() ? rm.const_data_ptr<int64_t>() : nullptr, a.n_rows = (int)y.rows;
  a.path = path.mutable_data_ptr<int32_t>(), a.count = count.mutable_data_ptr<int32_t>(), a.drawn = drawn.mutable_data_ptr<int64_t>();
  a.pos_out = pos_out.mutable_data_ptr<int64_t>(), a.oob_count = oob.defined() ? oob.mutable_data_ptr<int>() : nullptr;
  a.h_layers = y.y.data();
  check(L.tree_advance(&a, at::cuda::getCurrentCUDAStream().stream()), "uv_tree_advance");
  return std::make_tuple(path, count, drawn);
}

bool kv_fork(const py::sequence& hkc, const py::sequence& hvc, const py::sequence& hks, const py::sequence& hvs,
             const std::vector<bool>& rings, py::handle hsrc, py::handle hdst, py::handle hpos, py::handle hstarts, py::handle hoob, bool force) {
  Call c(force);
  const Tensors kc = c.list(hkc, "k_caches"), vc = c.list(hvc, "v_caches"), ks = c.list(hks, "k_scales"), vs = c.list(hvs, "v_scales");
  const Tensor src_ = c.take(hsrc, "src"), dst_ = c.take(hdst, "dst"), pos = c.take(hpos, "pos"), starts = c.take(hstarts, "starts");
  const Tensor oob = c.maybe(hoob, "oob");
  if (!c.direct) return false;
  const Layers y = layers_of(kc, vc, ks, vs, rings);
  TORCH_CHECK_VALUE(src_.dim() == 1, "src has to be (n,); got ", src_.sizes());
  for (const Tensor* t : {&pos, &starts})
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == y.rows && t->scalar_type() == at::kLong && t->is_contiguous(),
                      "pos and starts have to be contiguous int64 tensors with one value for each of ", y.rows, " cache rows");
  if (oob.defined()) TORCH_CHECK_VALUE(oob.scalar_type() == at::kInt && oob.numel() >= 1, "oob has to be an int32 word");
  c10::cuda::CUDAGuard guard(*c.dev);
  const Tensor src = index_of(src_, src_.size(0), "src"), dst = index_of(dst_, src_.size(0), "dst");
  check(L.kv_fork(y.y.data(), (int)y.y.size(), (int)y.KH, (int)y.hd, (int)y.rows, src.const_data_ptr<int64_t>(), dst.const_data_ptr<int64_t>(),
                  (int)src.size(0), pos.mutable_data_ptr<int64_t>(), starts.mutable_data_ptr<int64_t>(),
                  oob.defined() ? oob.mutable_data_ptr<int>() : nullptr, at::cuda::getCurrentCUDAStream().stream()),
        "uv_kv_fork");
  return true;
}

std::optional<Tensor> adjust_logits(py::handle hx, const std::optional<std::tuple<double, double, double>>& cap, py::handle hhistory,
                                    py::handle hlengths, py::handle hprompt, py::handle hparents, py::handle htokens, py::handle hrep,
                                    py::handle hfreq, py::handle hpres, py::handle hids, py::handle hbias, py::handle hallowed,
                                    py::handle hout, bool force) {
  Call c(force);
  Tensor x = c.take(hx, "x");
  Tensor history = c.maybe(hhistory, "history"), allowed = c.maybe(hallowed, "allowed"), out = c.maybe(hout, "out");
  const Tensor lengths_ = c.maybe(hlengths, "lengths"), prompt_ = c.maybe(hprompt, "prompt_lengths"), parents_ = c.maybe(hparents, "parents");
  const Tensor tokens_ = c.maybe(htokens, "tokens"), rep = c.maybe(hrep, "repetition"), freq = c.maybe(hfreq, "frequency");
  const Tensor pres = c.maybe(hpres, "presence"), ids_ = c.maybe(hids, "bias_ids"), bias_ = c.maybe(hbias, "bias");
  if (!c.direct) return std::nullopt;
  TORCH_CHECK_VALUE(x.dim() == 2 || x.dim() == 3, "x has to be (B, V) or (B, T, V); got ", x.sizes());
  const bool flat = x.dim() == 2;
  const int64_t B = x.size(0), T = flat ? 1 : x.size(1), V = x.size(-1);
  auto float_code = [](const Tensor& t, const char* name) {
    const int code = code_of(t.scalar_type());
    TORCH_CHECK_VALUE(code >= 0 && code != UV_I8, name, " has to be float32, float16 or bfloat16; got ", t.scalar_type());
    return code;
  };
  uv_adjust_args a{};
  a.x_dtype = float_code(x, "x");
  c10::cuda::CUDAGuard guard(*c.dev);
  if (V > 1 && x.stride(-1) != 1) x = x.contiguous();
  if (out.defined()) {
    TORCH_CHECK_VALUE(out.sizes() == x.sizes() && (V <= 1 || out.stride(-1) == 1), "out has to be like x, with unit stride along the vocabulary");
  } else {
    out = at::empty(x.sizes(), x.options().dtype(at::kFloat));
  }
  a.out_dtype = float_code(out, "out");
  a.x = ro(x), a.out = out.mutable_data_ptr(), a.B = (int)B, a.T = (int)T, a.V = (int)V;
  a.sxb = x.stride(0), a.sxt = flat ? 0 : x.stride(1), a.sob = out.stride(0), a.sot = flat ? 0 : out.stride(1);
  if (cap) a.softcap = 1, a.cap_a = (float)std::get<0>(*cap), a.cap_b = (float)std::get<1>(*cap), a.cap_c = (float)std::get<2>(*cap);
  Tensor lengths, prompt, parents, tokens, ids, bias;
  if (history.defined()) {
    TORCH_CHECK_VALUE(history.dim() == 2 && history.size(0) == B && (history.scalar_type() == at::kInt || history.scalar_type() == at::kLong),
                      "history has to be int32 or int64 (", B, ", n); got ", history.sizes(), " ", history.scalar_type());
    if (history.size(1) > 1 && history.stride(1) != 1) history = history.contiguous();
    a.history = ro(history), a.hist_bytes = (int)history.element_size(), a.history_stride = history.stride(0), a.history_len = history.size(1);
    if (lengths_.defined()) lengths = index_of(lengths_, B, "lengths"), a.lengths = lengths.const_data_ptr<int64_t>();
    if (prompt_.defined()) prompt = index_of(prompt_, B, "prompt_lengths"), a.prompt_lengths = prompt.const_data_ptr<int64_t>();
  } else {
    TORCH_CHECK_VALUE(!lengths_.defined() && !prompt_.defined(), "lengths and prompt_lengths belong to a history");
  }
  TORCH_CHECK_VALUE(parents_.defined() == tokens_.defined(), "a tree is given by parents and tokens");
  if (parents_.defined()) {
    parents = parents_of(parents_, B, T, a.parents_stride), a.parents = parents.const_data_ptr<int32_t>();
    TORCH_CHECK_VALUE(tokens_.dim() == 2 && tokens_.size(0) == B && tokens_.size(1) == T && at::isIntegralType(tokens_.scalar_type(), false),
                      "tokens have to be integers (", B, ", ", T, "); got ", tokens_.sizes(), " ", tokens_.scalar_type());
    tokens = tokens_.to(at::kLong).contiguous(), a.tokens = tokens.const_data_ptr<int64_t>();
  }
  auto per_row = [&](const Tensor& t, const char* name) -> const float* {
    if (!t.defined()) return nullptr;
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == B && t.scalar_type() == at::kFloat && t.is_contiguous(), name, " has to be contiguous float32 (", B, ",)");
    return t.const_data_ptr<float>();
  };
  a.repetition = per_row(rep, "repetition"), a.frequency = per_row(freq, "frequency"), a.presence = per_row(pres, "presence");
  TORCH_CHECK_VALUE(ids_.defined() == bias_.defined(), "a bias is given by bias_ids and bias");
  if (ids_.defined()) {
    TORCH_CHECK_VALUE(ids_.sizes() == bias_.sizes() && (ids_.dim() == 1 || (ids_.dim() == 2 && ids_.size(0) == B)),
                      "bias_ids and bias have to be (", B, ", n) or (n,); got ", ids_.sizes(), " and ", bias_.sizes());
    TORCH_CHECK_VALUE(at::isIntegralType(ids_.scalar_type(), false) && bias_.scalar_type() == at::kFloat, "bias_ids have to be integers, bias float32");
    ids = int32_of(ids_, -1, INT32_MAX).contiguous(), bias = bias_.contiguous();
    a.bias_ids = ids.const_data_ptr<int32_t>(), a.bias = bias.const_data_ptr<float>(), a.n_bias = (int)ids.size(-1);
    a.bias_stride = ids.dim() == 1 ? 0 : ids.size(-1);
  }
  if (allowed.defined()) {
    const int64_t W = (V + 31) / 32;
    const bool rows = allowed.dim() == 2, nodes = allowed.dim() == 3 && !flat;
    TORCH_CHECK_VALUE(allowed.scalar_type() == at::kInt && (rows || nodes) && allowed.size(0) == B && allowed.size(-1) >= W &&
                          (rows || allowed.size(1) == T),
                      "allowed has to be int32 (", B, ", words) or (", B, ", ", T, ", words) with at least ", W, " words; got ", allowed.sizes(), " ",
                      allowed.scalar_type());
    if (allowed.size(-1) > 1 && allowed.stride(-1) != 1) allowed = allowed.contiguous();
    a.allowed = allowed.const_data_ptr<int32_t>(), a.sab = allowed.stride(0), a.sat = nodes ? allowed.stride(1) : 0;
  }
  check(L.adjust_logits(&a, at::cuda::getCurrentCUDAStream().stream()), "uv_adjust_logits");
  return out;
}

// The Python calls of the cache operators, in C++: checks of the operands, the output and the launch through
// libmtpk's C entry points. In Python these took 9 to 19 us a call, of which the launch is 3: more than
// the small calls' kernels. The module holds no second copy of the library: `bind` gets the entry points'
// addresses from the loaded one (_mtpk.py), and a call before that raises.
//
// Streams come as handles from the caller (torch's current stream of the tensors' device). Errors in the
// arguments are ValueErrors, as _mtpk.check raises them.

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/util/StringUtil.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <vector>

#include "mtpk.h"

namespace py = pybind11;
using at::Tensor;

namespace {

constexpr int64_t kBlock = 16;  // rows of a cache block

struct Entries {
  decltype(&mtpk_status_string) status_string = nullptr;
  decltype(&mtpk_rotate) rotate = nullptr;
  decltype(&mtpk_rotate_to_cache) rotate_to_cache = nullptr;
  decltype(&mtpk_attention_masked_splits) splits = nullptr;
  decltype(&mtpk_attention_masked_workspace_bytes) workspace = nullptr;
  decltype(&mtpk_paged_attention_masked) attention = nullptr;
  decltype(&mtpk_copy_blocks) copy_blocks = nullptr;
  decltype(&mtpk_attention_tree_splits) tree_splits = nullptr;
  decltype(&mtpk_attention_tree_workspace_bytes) tree_workspace = nullptr;
  decltype(&mtpk_paged_attention_tree) tree_attention = nullptr;
  decltype(&mtpk_deltanet_prep_tree) prep_tree = nullptr;
  decltype(&mtpk_delta_rule_tree) rule_tree = nullptr;
  decltype(&mtpk_deltanet_commit_path) commit_path = nullptr;
  decltype(&mtpk_tree_accept) tree_accept = nullptr;
  decltype(&mtpk_keep_path) keep_path = nullptr;
} lib;

template <typename... A>
void need(bool ok, const A&... text) {
  if (!ok) throw py::value_error(c10::str(text...));
}

void check(int status, const char* what) {
  if (status == 0) return;
  const std::string text = std::string(what) + ": " + lib.status_string(status);
  if (status == MTPK_EINVAL || status == MTPK_ETOOBIG) throw py::value_error(text);
  throw std::runtime_error(text + " (status " + std::to_string(status) + ")");
}

void on(const c10::Device& device, const Tensor& t) {
  need(t.device() == device, "all tensors must be on the same device, got ", t.device(), " and ", device);
}
c10::Device hip_device(const Tensor& t) {
  need(t.is_cuda(), "libmtpk entry points take device tensors");
  need(lib.status_string != nullptr, "the native calls are not bound to libmtpk");
  return t.device();
}

int float_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return MTPK_F32;
  need(t.scalar_type() == at::kBFloat16, "unsupported float dtype ", t.scalar_type(), " (float32 or bfloat16)");
  return MTPK_BF16;
}
bool index_type(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
int index_code(const Tensor& t) { return t.scalar_type() == at::kInt ? MTPK_I32 : MTPK_I64; }

const void* ptr(const std::optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

// Whether every row along the last dim is contiguous and starts on 16 bytes.
bool rows16(const Tensor& t) {
  const int64_t unit = 16 / t.element_size(), n = t.dim();
  if (t.stride(n - 1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.stride(i) % unit) return false;
  return true;
}
Tensor on16(const Tensor& t) { return rows16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

struct Strides {  // (lane, head, step) of [B, t, heads, hd]
  int64_t s[3];
  explicit Strides(const Tensor& t) : s{t.stride(0), t.stride(2), t.stride(1)} {}
};

int check_rates(const Tensor& rates, int64_t dim) {
  need(rates.scalar_type() == at::kDouble && rates.dim() == 1 && rates.is_contiguous(),
       "rates must be a contiguous float64 [pairs] tensor");
  const int64_t rot = 2 * rates.size(0);
  need(rot >= 2 && rot <= dim, rates.size(0), " pairs do not fit heads of ", dim, " channels");
  need(dim % 8 == 0 && dim <= 512, "head dim must be a multiple of 8 up to 512, got ", dim);
  return (int)rot;
}

std::optional<Tensor> check_norm(const std::optional<Tensor>& w, int64_t dim, const c10::Device& device) {
  if (!w) return w;
  need(w->dim() == 1 && w->size(0) == dim, "a norm's weight must be a [", dim, "] tensor, got ", w->sizes());
  on(device, *w);
  float_code(*w);
  return on16(*w);
}

// `x` as [tokens, heads, dim] with rows on 16 bytes, or nothing where its leading dims have no one stride.
std::optional<Tensor> tokens_of(const Tensor& x) {
  Tensor y = x;
  if (x.dim() != 3) {
    const int64_t heads = x.size(-2), dim = x.size(-1);
    if (x.numel() == 0) return x.reshape({0, heads, dim});
    int64_t n = 1, stride = -1;
    for (int64_t i = x.dim() - 3; i >= 0; --i) {  // collapse from the inside; a size-1 dim's stride is arbitrary
      if (x.size(i) == 1) continue;
      if (stride >= 0 && x.stride(i) != stride * n) return std::nullopt;
      if (stride < 0) stride = x.stride(i);
      n *= x.size(i);
    }
    y = x.as_strided({n, heads, dim}, {stride < 0 ? heads * dim : stride, x.stride(-2), x.stride(-1)});
  }
  if (!rows16(y)) return std::nullopt;
  return y;
}

Tensor rotate(const Tensor& x, const Tensor& positions, const Tensor& rates, double magnitude, bool interleaved,
              const std::optional<Tensor>& weight, double eps, const std::optional<Tensor>& given, int64_t stream) {
  const c10::Device device = hip_device(x);
  on(device, positions);
  on(device, rates);
  need(x.dim() >= 2 && positions.sizes() == x.sizes().slice(0, x.dim() - 2), "positions must be ",
       x.sizes().slice(0, x.dim() >= 2 ? x.dim() - 2 : 0), " for heads ", x.sizes(), ", got ", positions.sizes());
  const int64_t heads = x.size(-2), dim = x.size(-1);
  const int rot = check_rates(rates, dim), dtype = float_code(x);
  const std::optional<Tensor> w = check_norm(weight, dim, device);
  need(at::isIntegralType(positions.scalar_type(), false), "positions must be integers");
  const Tensor pos = positions.to(at::kLong).contiguous();
  if (given)
    need(given->sizes() == x.sizes() && given->scalar_type() == x.scalar_type() && given->device() == device, "out must be ",
         x.sizes(), " ", x.scalar_type(), " on ", device);
  const Tensor out = given ? *given : at::empty_like(x, x.options(), at::MemoryFormat::Contiguous);
  std::optional<Tensor> src = tokens_of(x), dst = tokens_of(out);
  if (!src) src = tokens_of(x.clone(at::MemoryFormat::Contiguous));
  need(src && dst, "out's rows must lie on 16 bytes and its leading dims at one stride");
  if (src->size(0) == 0 || heads == 0) return out;
  const int64_t xs[2] = {src->stride(0), src->stride(1)}, os[2] = {dst->stride(0), dst->stride(1)};
  const c10::DeviceGuard guard(device);
  check(lib.rotate(src->data_ptr(), dtype, xs, src->size(0), heads, dim, ptr(w), w ? float_code(*w) : 0, (float)eps,
                   pos.data_ptr<int64_t>(), rates.data_ptr<double>(), rot, interleaved, (float)magnitude, dst->data_ptr(), os,
                   (void*)stream),
        "mtpk_rotate");
  return out;
}

// The cache's operands as the kernels read them: pools checked, table int32, base int64, contiguous.
struct Cache {
  uint16_t *k, *v;
  int64_t rows;
  Tensor table, base;
  Cache(const Tensor& k_pool, const Tensor& v_pool, const Tensor& block_table, const Tensor& base_pos, int64_t batch,
        int64_t kv_heads, int64_t head_dim, const c10::Device& device)
      : table(block_table), base(base_pos) {
    for (const Tensor* t : {&k_pool, &v_pool, &block_table, &base_pos}) on(device, *t);
    rows = k_pool.dim() == 3 ? k_pool.size(0) : 0;
    need(rows > 0 && rows % kBlock == 0 && k_pool.size(1) == kv_heads && k_pool.size(2) == head_dim, "k_pool must be [rows, ",
         kv_heads, ", ", head_dim, "] of ", kBlock, "-row blocks, got ", k_pool.sizes());
    need(v_pool.dim() == 4 && v_pool.size(0) == rows / kBlock && v_pool.size(1) == kv_heads && v_pool.size(2) == head_dim &&
             v_pool.size(3) == kBlock,
         "v_pool must be [", rows / kBlock, ", ", kv_heads, ", ", head_dim, ", ", kBlock, "] (V transposed per block), got ",
         v_pool.sizes());
    need(k_pool.scalar_type() == at::kBFloat16 && v_pool.scalar_type() == at::kBFloat16 && k_pool.is_contiguous() &&
             v_pool.is_contiguous(),
         "pools must be contiguous bf16");
    need(table.dim() == 2 && table.size(0) == batch && base.dim() == 1 && base.size(0) == batch, "block_table must be [", batch,
         ", blocks] and base_pos [", batch, "], got ", table.sizes(), " and ", base.sizes());
    need(index_type(table) && index_type(base), "block_table and base_pos must be int32 or int64, got ", table.scalar_type(),
         " and ", base.scalar_type());
    table = table.to(at::kInt).contiguous();
    base = base.to(at::kLong).contiguous();
    k = (uint16_t*)k_pool.data_ptr();
    v = (uint16_t*)v_pool.data_ptr();
  }
};

Tensor rotate_to_cache(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& rates, const Tensor& k_pool,
                       const Tensor& v_pool, const Tensor& block_table, const Tensor& base_pos, double magnitude,
                       bool interleaved, const std::optional<Tensor>& q_weight, const std::optional<Tensor>& k_weight, double eps,
                       const std::optional<Tensor>& keep, const std::optional<Tensor>& positions, int64_t stream) {
  const c10::Device device = hip_device(q_in);
  for (const Tensor* t : {&k_in, &v_in, &rates}) on(device, *t);
  need(q_in.dim() == 4 && k_in.dim() == 4, "q and k must be [B, t, heads, hd], got ", q_in.sizes(), " and ", k_in.sizes());
  const int64_t b = q_in.size(0), t = q_in.size(1), heads = q_in.size(2), hd = q_in.size(3), kvh = k_in.size(2);
  need(k_in.size(0) == b && k_in.size(1) == t && k_in.size(3) == hd && v_in.sizes() == k_in.sizes(), "k and v must be [", b, ", ",
       t, ", kv_heads, ", hd, "], got ", k_in.sizes(), " and ", v_in.sizes());
  for (const Tensor* x : {&q_in, &k_in, &v_in}) need(x->scalar_type() == at::kBFloat16, "q, k and v must be bf16");
  const int rot = check_rates(rates, hd);
  const Cache cache(k_pool, v_pool, block_table, base_pos, b, kvh, hd, device);
  const std::optional<Tensor> qw = check_norm(q_weight, hd, device), kw = check_norm(k_weight, hd, device);
  need(!qw || !kw || qw->scalar_type() == kw->scalar_type(), "q_norm and k_norm must be of one type");
  const std::optional<Tensor>& norm = qw ? qw : kw;
  std::optional<Tensor> pos = positions;
  if (pos) {
    need(pos->dim() == 2 && pos->size(0) == b && pos->size(1) == t && pos->scalar_type() == at::kLong, "positions must be int64 [", b,
         ", ", t, "]");
    on(device, *pos);
    pos = pos->contiguous();
  }
  if (keep) {
    const bool flags = keep->scalar_type() == at::kBool || keep->scalar_type() == at::kByte;
    need(flags && keep->dim() == 2 && keep->size(0) == b && keep->size(1) == t, "keep must be bool [", b, ", ", t, "]");
    on(device, *keep);
  }
  need(heads > 0 && kvh > 0, "q and k must have heads, got ", q_in.sizes(), " and ", k_in.sizes());
  const Tensor out = at::empty_like(q_in, q_in.options(), at::MemoryFormat::Contiguous);
  if (out.numel() == 0) return out;  // no rows
  const Tensor q = on16(q_in), k = on16(k_in), v = on16(v_in);
  const Strides qs(q), ks(k), vs(v), os(out);
  const c10::DeviceGuard guard(device);
  check(lib.rotate_to_cache((const uint16_t*)q.data_ptr(), qs.s, (const uint16_t*)k.data_ptr(), ks.s, (const uint16_t*)v.data_ptr(),
                            vs.s, ptr(qw), ptr(kw), norm ? float_code(*norm) : 0, (float)eps, rates.data_ptr<double>(), rot,
                            interleaved, (float)magnitude, cache.k, cache.v, cache.rows, cache.table.data_ptr<int32_t>(),
                            cache.table.size(1), cache.base.data_ptr<int64_t>(), (const int64_t*)ptr(pos), (const uint8_t*)ptr(keep),
                            keep ? keep->stride(0) : 0, keep ? keep->stride(1) : 0, b, t, heads, kvh, hd, (uint16_t*)out.data_ptr(),
                            os.s, (void*)stream),
        "mtpk_rotate_to_cache");
  return out;
}

std::optional<Tensor> check_integers(const std::optional<Tensor>& x, const char* name, at::IntArrayRef shape,
                                     const c10::Device& device) {
  if (!x) return x;
  need(x->sizes() == shape && index_type(*x), name, " must be int32 or int64 ", shape, ", got ", x->scalar_type(), " ", x->sizes());
  on(device, *x);
  return x->contiguous();
}

Tensor paged_attention_masked(const Tensor& q_in, const Tensor& k_pool, const Tensor& v_pool, const Tensor& block_table,
                              const Tensor& base_pos, int64_t ctx_len, double scale, double softcap, int64_t window,
                              const std::optional<Tensor>& slopes_in, const std::optional<Tensor>& prefix_in,
                              const std::optional<Tensor>& first_in, const std::optional<Tensor>& gate_in, int64_t stream) {
  const c10::Device device = hip_device(q_in);
  need(q_in.dim() == 4 && q_in.scalar_type() == at::kBFloat16, "q must be bf16 [B, t, heads, hd], got ", q_in.scalar_type(), " ",
       q_in.sizes());
  const int64_t b = q_in.size(0), t = q_in.size(1), heads = q_in.size(2), hd = q_in.size(3);
  need(hd == 64 || hd == 128 || hd == 256, "head_dim must be one of (64, 128, 256), got ", hd);
  need(k_pool.dim() == 3, "k_pool must be [rows, kv_heads, ", hd, "], got ", k_pool.sizes());
  const int64_t kvh = k_pool.size(1);
  const Cache cache(k_pool, v_pool, block_table, base_pos, b, kvh, hd, device);
  need(heads > 0 && kvh > 0 && heads % kvh == 0, heads, " q heads are not a multiple of ", kvh, " kv heads");
  need(ctx_len >= 0 && ctx_len <= cache.table.size(1) * kBlock, "context bound ", ctx_len, " exceeds the table's ",
       cache.table.size(1), " blocks");
  need(scale > 0 && std::isfinite(scale) && softcap >= 0 && std::isfinite(softcap) && window >= 0,
       "scale must be positive, softcap and window not negative, got ", scale, ", ", softcap, " and ", window);
  need(softcap == 0 || (float)softcap > 0, "softcap ", softcap, " is below float32's range, where 0 means none");
  std::optional<Tensor> gate, slopes;
  if (gate_in) {
    need(gate_in->sizes() == q_in.sizes() && gate_in->scalar_type() == at::kBFloat16, "gate must be bf16 of q's shape");
    on(device, *gate_in);
    gate = on16(*gate_in);
  }
  if (slopes_in) {
    need(slopes_in->dim() == 1 && slopes_in->size(0) == heads && slopes_in->scalar_type() == at::kFloat, "slopes must be float32 [",
         heads, "]");
    on(device, *slopes_in);
    slopes = slopes_in->contiguous();
  }
  const std::optional<Tensor> prefix = check_integers(prefix_in, "prefix", {b}, device);
  const std::optional<Tensor> first = check_integers(first_in, "first", {b, t}, device);
  const Tensor out = at::empty_like(q_in, q_in.options(), at::MemoryFormat::Contiguous);
  if (out.numel() == 0) return out;
  const Tensor q = on16(q_in);
  const c10::DeviceGuard guard(device);
  const int n_split = lib.splits(b, t, heads, kvh, hd, ctx_len, window);
  Tensor ws;
  int64_t ws_bytes = 0;
  if (n_split > 1) {
    ws_bytes = lib.workspace(b, t, heads, kvh, hd, n_split);
    ws = at::empty({ws_bytes}, q.options().dtype(at::kByte));
  }
  const Strides qs(q), os(out);
  const Strides gs(gate ? *gate : out);
  check(lib.attention((const uint16_t*)q.data_ptr(), qs.s, (const uint16_t*)ptr(gate), gs.s, b, t, heads, kvh, hd, cache.k, cache.v,
                      cache.rows, cache.table.data_ptr<int32_t>(), cache.table.size(1), cache.base.data_ptr<int64_t>(), (float)scale,
                      (float)softcap, window, (const float*)ptr(slopes), ptr(prefix), prefix ? index_code(*prefix) : 0, ptr(first),
                      first ? index_code(*first) : 0, n_split, n_split > 1 ? ws.data_ptr() : nullptr, ws_bytes,
                      (uint16_t*)out.data_ptr(), os.s, (void*)stream),
        "mtpk_paged_attention_masked");
  return out;
}

// Blocks of the pools, one number for all of them: K caches [rows, kv_heads, hd], V caches [blocks, kv_heads, hd, block].
int64_t pool_blocks(const std::vector<Tensor>& pools, int64_t block) {
  need(!pools.empty(), "copy_blocks takes at least one pool");
  need(block > 0, "a block has at least one row");
  const auto device = pools[0].device();
  const int64_t n = pools[0].dim() > 0 ? pools[0].size(0) / (pools[0].dim() == 4 ? 1 : block) : 0;
  for (const Tensor& p : pools)
    need(((p.dim() == 3 && p.size(0) == n * block) || (p.dim() == 4 && p.size(0) == n)) && p.numel() > 0 && p.is_contiguous() &&
             p.device() == device,
         "pools must be contiguous K caches [rows, kv_heads, hd] and V caches [blocks, kv_heads, hd, ", block,
         "] of one number of blocks on one device, got ", p.sizes(), " on ", p.device());
  return n;
}

void copy_blocks(const std::vector<Tensor>& pools, const Tensor& src_in, const Tensor& dst_in, int64_t block, int64_t stream) {
  const int64_t n = pool_blocks(pools, block);
  const c10::Device device = hip_device(pools[0]);
  on(device, src_in);
  on(device, dst_in);
  need(src_in.dim() == 1 && src_in.sizes() == dst_in.sizes() && index_type(src_in) && src_in.scalar_type() == dst_in.scalar_type(),
       "src and dst must be int32 or int64 vectors of one length and type");
  const Tensor src = src_in.contiguous(), dst = dst_in.contiguous();
  std::vector<void*> at(pools.size());
  std::vector<int64_t> bytes(pools.size());
  for (size_t i = 0; i < pools.size(); ++i) {
    at[i] = pools[i].data_ptr();
    bytes[i] = pools[i].numel() / n * pools[i].element_size();
  }
  const c10::DeviceGuard guard(device);
  check(lib.copy_blocks(at.data(), bytes.data(), (int)pools.size(), n, src.data_ptr(), dst.data_ptr(), index_code(src), src.size(0),
                        (void*)stream),
        "mtpk_copy_blocks (blocks of a multiple of 16 bytes, pools on 16 bytes)");
}

// A call's outputs in one allocation, each from 16 bytes on: an allocation of its own takes the host about 1.1 us.
std::vector<Tensor> together(const at::TensorOptions& options, std::initializer_list<at::IntArrayRef> shapes) {
  const int64_t unit = 16 / (int64_t)options.dtype().itemsize();
  int64_t total = 0;
  for (const at::IntArrayRef& s : shapes) total += (c10::multiply_integers(s) + unit - 1) / unit * unit;
  const Tensor all = at::empty({total}, options);
  const at::AutoDispatchBelowADInplaceOrView plain;  // outputs of a call, not views of a tensor that anyone else holds
  std::vector<Tensor> out;
  out.reserve(shapes.size());
  int64_t at = 0;
  for (const at::IntArrayRef& s : shapes) {
    int64_t strides[4], step = 1;
    for (size_t i = s.size(); i-- > 0; step *= s[i]) strides[i] = step;
    out.push_back(all.as_strided(s, at::IntArrayRef(strides, s.size()), at));
    at += (step + unit - 1) / unit * unit;
  }
  return out;
}

// A tree's parents, read where they lie.
struct Tree {
  const void* p;
  int dtype;
  int64_t s[2];
  Tree(const Tensor& parents, int64_t batch, int64_t t, const c10::Device& device) {
    need(parents.dim() == 2 && parents.size(0) == batch && parents.size(1) == t && index_type(parents), "parents must be int32 or int64 [",
         batch, ", ", t, "], got ", parents.scalar_type(), " ", parents.sizes());
    need(t >= 1 && t <= 64, "a tree has 1 to 64 nodes, got ", t);
    on(device, parents);
    p = parents.data_ptr();
    dtype = index_code(parents);
    s[0] = parents.stride(0);
    s[1] = parents.stride(1);
  }
};

Tensor as_long(const Tensor& x, const char* name, at::IntArrayRef shape, const c10::Device& device) {
  need(x.sizes() == shape && index_type(x), name, " must be int32 or int64 ", shape, ", got ", x.scalar_type(), " ", x.sizes());
  on(device, x);
  return x.to(at::kLong).contiguous();
}
Tensor as_float(const Tensor& x, const char* name, at::IntArrayRef shape, const c10::Device& device) {
  need(x.sizes() == shape, name, " must be ", shape, ", got ", x.sizes());
  need(at::isFloatingType(x.scalar_type()), name, " must be of floats, got ", x.scalar_type());
  on(device, x);
  return x.to(at::kFloat).contiguous();
}

Tensor paged_attention_tree(const Tensor& q_in, const Tensor& k_pool, const Tensor& v_pool, const Tensor& block_table,
                            const Tensor& base_pos, int64_t ctx_len, double scale, const Tensor& parents,
                            const std::optional<Tensor>& gate_in, int64_t stream) {
  const c10::Device device = hip_device(q_in);
  need(q_in.dim() == 4 && q_in.scalar_type() == at::kBFloat16, "q must be bf16 [B, t, heads, hd], got ", q_in.scalar_type(), " ",
       q_in.sizes());
  const int64_t b = q_in.size(0), t = q_in.size(1), heads = q_in.size(2), hd = q_in.size(3);
  need(hd == 64 || hd == 128 || hd == 256, "head_dim must be one of (64, 128, 256), got ", hd);
  need(k_pool.dim() == 3, "k_pool must be [rows, kv_heads, ", hd, "], got ", k_pool.sizes());
  const int64_t kvh = k_pool.size(1);
  const Tree tree(parents, b, t, device);
  const Cache cache(k_pool, v_pool, block_table, base_pos, b, kvh, hd, device);
  need(heads > 0 && kvh > 0 && heads % kvh == 0, heads, " q heads are not a multiple of ", kvh, " kv heads");
  need(ctx_len >= 0 && ctx_len <= cache.table.size(1) * kBlock, "context bound ", ctx_len, " exceeds the table's ",
       cache.table.size(1), " blocks");
  need((float)scale > 0 && std::isfinite((float)scale), "scale must be positive, got ", scale);
  std::optional<Tensor> gate;
  if (gate_in) {
    need(gate_in->sizes() == q_in.sizes() && gate_in->scalar_type() == at::kBFloat16, "gate must be bf16 of q's shape");
    on(device, *gate_in);
    gate = on16(*gate_in);
  }
  const Tensor out = at::empty_like(q_in, q_in.options(), at::MemoryFormat::Contiguous);
  if (out.numel() == 0) return out;
  const Tensor q = on16(q_in);
  const c10::DeviceGuard guard(device);
  const int n_split = lib.tree_splits(b, t, heads, kvh, hd, ctx_len);
  Tensor ws;
  int64_t ws_bytes = 0;
  if (n_split > 1) {
    ws_bytes = lib.tree_workspace(b, t, heads, kvh, hd, n_split);
    ws = at::empty({ws_bytes}, q.options().dtype(at::kByte));
  }
  const Strides qs(q), os(out);
  const Strides gs(gate ? *gate : out);
  check(lib.tree_attention((const uint16_t*)q.data_ptr(), qs.s, (const uint16_t*)ptr(gate), gs.s, b, t, heads, kvh, hd, cache.k,
                           cache.v, cache.rows, cache.table.data_ptr<int32_t>(), cache.table.size(1),
                           cache.base.data_ptr<int64_t>(), (float)scale, tree.p, tree.dtype, tree.s, n_split,
                           n_split > 1 ? ws.data_ptr() : nullptr, ws_bytes, (uint16_t*)out.data_ptr(), os.s, (void*)stream),
        "mtpk_paged_attention_tree");
  return out;
}

// The in-projection's rows [B, t, P], which lie at one stride.
Tensor proj_rows(const Tensor& proj, int64_t* stride) {
  need(proj.dim() == 3, "proj must be [B, t, P], got ", proj.sizes());
  float_code(proj);
  const int64_t b = proj.size(0), t = proj.size(1);
  const bool rows = proj.stride(2) == 1 && (t == 1 || b <= 1 || proj.stride(0) == t * proj.stride(1)) &&
                    (t == 1 ? proj.stride(0) : proj.stride(1)) >= proj.size(2);
  const Tensor out = rows ? proj : proj.contiguous();
  *stride = b * t <= 1 ? proj.size(2) : t == 1 ? out.stride(0) : out.stride(1);
  return out;
}

std::vector<Tensor> prep_tree(const Tensor& proj_in, const Tensor& conv_state, const Tensor& slots_in, const Tensor& conv_w,
                              const Tensor& a_log_in, const Tensor& dt_bias_in, int64_t k_heads, int64_t k_dim, int64_t v_heads,
                              int64_t v_dim, const Tensor& parents, double eps, int64_t stream) {
  const c10::Device device = hip_device(proj_in);
  int64_t stride = 0;
  const Tensor proj = proj_rows(proj_in, &stride);
  const int64_t b = proj.size(0), t = proj.size(1);
  need(k_heads > 0 && v_heads > 0 && k_dim > 0 && v_dim > 0 && k_dim <= 256 && v_dim <= 256,
       "heads must be of 1 to 256 channels, got ", k_heads, " of ", k_dim, " and ", v_heads, " of ", v_dim);
  const int64_t channels = 2 * k_heads * k_dim + v_heads * v_dim, width = channels + v_heads * v_dim + 2 * v_heads;
  need(proj.size(2) >= width, "proj's rows must hold ", width, " values, got ", proj.size(2));
  const Tree tree(parents, b, t, device);
  need(conv_w.dim() == 2 && conv_w.size(0) == channels && conv_w.size(1) >= 2 && conv_w.size(1) <= 9, "conv_w must be [", channels,
       ", 2 to 9], got ", conv_w.sizes());
  need(conv_state.dim() == 3 && conv_state.size(0) > 0 && conv_state.size(1) == channels && conv_state.size(2) == conv_w.size(1) - 1,
       "conv_state must be [slots, ", channels, ", ", conv_w.size(1) - 1, "], got ", conv_state.sizes());
  for (const Tensor* x : {&conv_state, &conv_w}) {
    need(x->scalar_type() == proj.scalar_type() && x->is_contiguous(), "conv_state and conv_w must be contiguous and of proj's type");
    on(device, *x);
  }
  const c10::DeviceGuard guard(device);
  const Tensor slots = as_long(slots_in, "slots", {b}, device);
  const Tensor a_log = as_float(a_log_in, "a_log", {v_heads}, device), dt_bias = as_float(dt_bias_in, "dt_bias", {v_heads}, device);
  const int64_t qk_shape[4] = {b, t, k_heads, k_dim}, v_shape[4] = {b, t, v_heads, v_dim}, g_shape[3] = {b, t, v_heads};
  const std::vector<Tensor> out = together(proj.options().dtype(at::kFloat), {qk_shape, qk_shape, v_shape, g_shape, g_shape});
  const Tensor &q = out[0], &k = out[1], &v = out[2], &g = out[3], &beta = out[4];
  check(lib.prep_tree(proj.data_ptr(), float_code(proj), stride, conv_state.data_ptr(), slots.data_ptr<int64_t>(), conv_state.size(0),
                      conv_w.data_ptr(), a_log.data_ptr<float>(), dt_bias.data_ptr<float>(), tree.p, tree.dtype, tree.s, b, t, k_heads,
                      k_dim, v_heads, v_dim, conv_w.size(1), (float)eps, (float)(1.0 / std::sqrt((double)k_dim)), q.data_ptr<float>(),
                      k.data_ptr<float>(), v.data_ptr<float>(), g.data_ptr<float>(), beta.data_ptr<float>(), (void*)stream),
        "mtpk_deltanet_prep_tree");
  return out;
}

// The delta rule's operands of a call's rows: fp32, contiguous.
struct RuleRows {
  int64_t b, t, heads, qk_heads, k_dim, v_dim, slots;
  Tensor q, k, v, g, beta;
  RuleRows(const Tensor& state, const Tensor* q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& g_in, const Tensor& beta_in,
           const c10::Device& device) {
    need(state.dim() == 4 && state.scalar_type() == at::kFloat && state.is_contiguous(),
         "state must be a contiguous f32 [slots, heads, k_dim, v_dim] tensor");
    slots = state.size(0), heads = state.size(1), k_dim = state.size(2), v_dim = state.size(3);
    need(k_dim == 16 || k_dim == 32 || k_dim == 64 || k_dim == 128, "k_dim must be 16, 32, 64 or 128, got ", k_dim);
    need(k_in.dim() == 4 && k_in.size(3) == k_dim, "k must be [B, t, heads, ", k_dim, "], got ", k_in.sizes());
    b = k_in.size(0), t = k_in.size(1), qk_heads = k_in.size(2);
    need(t >= 1 && t <= 64, "a tree has 1 to 64 nodes, got ", t);
    need(qk_heads > 0 && heads > 0 && heads % qk_heads == 0, "state heads ", heads, " is not a multiple of q/k heads ", qk_heads);
    if (q_in) q = as_float(*q_in, "q", k_in.sizes(), device);
    k = as_float(k_in, "k", k_in.sizes(), device);
    v = as_float(v_in, "v", {b, t, heads, v_dim}, device);
    g = as_float(g_in, "g", {b, t, heads}, device);
    beta = as_float(beta_in, "beta", {b, t, heads}, device);
  }
};

Tensor delta_rule_tree(const Tensor& state, const std::optional<Tensor>& slots_in, const Tensor& q, const Tensor& k, const Tensor& v,
                       const Tensor& g, const Tensor& beta, const Tensor& parents, int64_t stream) {
  const c10::Device device = hip_device(state);
  const c10::DeviceGuard guard(device);
  const RuleRows r(state, &q, k, v, g, beta, device);
  const Tree tree(parents, r.b, r.t, device);
  std::optional<Tensor> slots;
  if (slots_in)
    slots = as_long(*slots_in, "slots", {r.b}, device);
  else
    need(r.slots >= r.b, r.b, " rows need ", r.b, " state slots, the pool has ", r.slots);
  const Tensor out = at::empty({r.b, r.t, r.heads, r.v_dim}, state.options());
  if (out.numel() == 0) return out;
  check(lib.rule_tree(state.data_ptr<float>(), r.slots, (const int64_t*)ptr(slots), r.b, r.t, r.heads, r.qk_heads, r.k_dim, r.v_dim,
                      r.q.data_ptr<float>(), r.k.data_ptr<float>(), r.v.data_ptr<float>(), r.g.data_ptr<float>(),
                      r.beta.data_ptr<float>(), tree.p, tree.dtype, tree.s, out.data_ptr<float>(), (void*)stream),
        "mtpk_delta_rule_tree");
  return out;
}

void commit_path(const Tensor& state, const Tensor& conv_state, const Tensor& slots_in, const Tensor& k, const Tensor& v,
                 const Tensor& g, const Tensor& beta, const Tensor& path_in, const Tensor& lengths_in, const Tensor& proj_in,
                 int64_t channels, int64_t stream) {
  const c10::Device device = hip_device(state);
  const c10::DeviceGuard guard(device);
  const RuleRows r(state, nullptr, k, v, g, beta, device);
  int64_t stride = 0;
  const Tensor proj = proj_rows(proj_in, &stride);
  on(device, proj);
  on(device, conv_state);
  need(proj.size(0) == r.b && proj.size(1) == r.t && channels > 0 && proj.size(2) >= channels, "proj must be [", r.b, ", ", r.t,
       ", at least ", channels, "], got ", proj.sizes());
  need(conv_state.dim() == 3 && conv_state.size(0) > 0 && conv_state.size(1) == channels && conv_state.size(2) >= 1 &&
           conv_state.size(2) <= 8,
       "conv_state must be [slots, ", channels, ", 1 to 8], got ", conv_state.sizes());
  need(conv_state.scalar_type() == proj.scalar_type() && conv_state.is_contiguous(), "conv_state must be contiguous and of proj's type");
  const Tensor slots = as_long(slots_in, "slots", {r.b}, device), path = as_long(path_in, "path", {r.b, r.t}, device),
               lengths = as_long(lengths_in, "lengths", {r.b}, device);
  if (r.b == 0) return;
  check(lib.commit_path(state.data_ptr<float>(), r.slots, slots.data_ptr<int64_t>(), r.b, r.t, r.heads, r.qk_heads, r.k_dim, r.v_dim,
                        r.k.data_ptr<float>(), r.v.data_ptr<float>(), r.g.data_ptr<float>(), r.beta.data_ptr<float>(),
                        path.data_ptr<int64_t>(), lengths.data_ptr<int64_t>(), conv_state.data_ptr(), float_code(conv_state),
                        conv_state.size(0), proj.data_ptr(), stride, channels, conv_state.size(2), (void*)stream),
        "mtpk_deltanet_commit_path");
}

std::vector<Tensor> tree_accept(const Tensor& argmax_in, const Tensor& tokens_in, const Tensor& parents, const Tensor& active_in,
                                const Tensor& pos_in, const Tensor& budget_in, const Tensor& stops_in, int64_t stream) {
  const c10::Device device = hip_device(argmax_in);
  need(argmax_in.dim() == 2, "step_argmax must be [B, t], got ", argmax_in.sizes());
  const int64_t b = argmax_in.size(0), t = argmax_in.size(1);
  const Tree tree(parents, b, t, device);
  need(active_in.dim() == 1 && active_in.size(0) == b && active_in.scalar_type() == at::kBool, "active must be bool [", b, "]");
  need(stops_in.dim() == 2 && stops_in.size(0) == b && stops_in.scalar_type() == at::kLong, "stops must be int64 [", b, ", stop ids]");
  for (const Tensor* x : {&argmax_in, &tokens_in, &pos_in, &budget_in})
    need(x->scalar_type() == at::kLong, "step_argmax, tokens, pos and budget must be int64");
  need(tokens_in.sizes() == argmax_in.sizes() && pos_in.dim() == 1 && pos_in.size(0) == b && budget_in.sizes() == pos_in.sizes(),
       "tokens must be [", b, ", ", t, "], pos and budget [", b, "]");
  for (const Tensor* x : {&tokens_in, &active_in, &pos_in, &budget_in, &stops_in}) on(device, *x);
  const c10::DeviceGuard guard(device);
  const Tensor best = argmax_in.stride(1) == 1 ? argmax_in : argmax_in.contiguous(),
               tokens = tokens_in.stride(1) == 1 ? tokens_in : tokens_in.contiguous();
  const Tensor active = active_in.contiguous(), pos = pos_in.contiguous(), budget = budget_in.contiguous(), stops = stops_in.contiguous();
  const int64_t lanes[1] = {b}, rows[2] = {b, t};
  const std::vector<Tensor> n = together(best.options(), {lanes, lanes, lanes, lanes, lanes, lanes, rows});
  const std::vector<Tensor> flags = together(best.options().dtype(at::kBool), {lanes, rows});
  const Tensor &path = n[6], &keep = flags[1], &live = flags[0];
  auto at64 = [](const Tensor& x) { return x.data_ptr<int64_t>(); };
  check(lib.tree_accept(at64(best), best.stride(0), at64(tokens), tokens.stride(0), tree.p, tree.dtype, tree.s,
                        (const uint8_t*)active.data_ptr(), at64(pos), at64(budget), at64(stops), stops.size(1), b, t, at64(path),
                        at64(n[0]), at64(n[1]), (uint8_t*)keep.data_ptr(), at64(n[2]), at64(n[3]), at64(n[4]),
                        (uint8_t*)live.data_ptr(), at64(n[5]), (void*)stream),
        "mtpk_tree_accept");
  return {path, n[0], n[1], keep, n[2], n[3], n[4], live, n[5]};
}

void keep_path(const std::vector<Tensor>& pools, const Tensor& block_table, const Tensor& base_pos, const Tensor& path_in,
               const Tensor& lengths_in, int64_t stream) {
  const int64_t n = pool_blocks(pools, kBlock);
  const c10::Device device = hip_device(pools[0]);
  const c10::DeviceGuard guard(device);
  need(path_in.dim() == 2 && path_in.size(1) >= 1 && path_in.size(1) <= 64, "path must be [B, 1 to 64], got ", path_in.sizes());
  const int64_t b = path_in.size(0), t = path_in.size(1);
  const Tensor path = as_long(path_in, "path", {b, t}, device), lengths = as_long(lengths_in, "lengths", {b}, device),
               base = as_long(base_pos, "base_pos", {b}, device);
  need(block_table.dim() == 2 && block_table.size(0) == b && block_table.size(1) > 0 && index_type(block_table),
       "block_table must be int32 or int64 [", b, ", blocks], got ", block_table.scalar_type(), " ", block_table.sizes());
  on(device, block_table);
  const Tensor table = block_table.to(at::kInt).contiguous();
  std::vector<void*> at(pools.size());
  std::vector<int64_t> channels(pools.size());
  std::vector<int> size(pools.size()), transposed(pools.size());
  for (size_t i = 0; i < pools.size(); ++i) {
    const Tensor& p = pools[i];
    need(p.dim() == 3 || p.size(3) == kBlock, "V caches must be [blocks, kv_heads, hd, ", kBlock, "], got ", p.sizes());
    at[i] = p.data_ptr();
    channels[i] = p.size(1) * p.size(2);
    size[i] = (int)p.element_size();
    transposed[i] = p.dim() == 4;
  }
  check(lib.keep_path(at.data(), channels.data(), size.data(), transposed.data(), (int)pools.size(), n, table.data_ptr<int32_t>(),
                      table.size(1), base.data_ptr<int64_t>(), path.data_ptr<int64_t>(), lengths.data_ptr<int64_t>(), b, t,
                      (void*)stream),
        "mtpk_keep_path (elements of 2 or 4 bytes, K rows of a multiple of 16 bytes, pools on 16 bytes, no two of one memory)");
}

template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
  f = (F)(uintptr_t)addresses[name].cast<uint64_t>();
}

void bind(const py::dict& a) {
  take(lib.rotate, a, "mtpk_rotate");
  take(lib.rotate_to_cache, a, "mtpk_rotate_to_cache");
  take(lib.splits, a, "mtpk_attention_masked_splits");
  take(lib.workspace, a, "mtpk_attention_masked_workspace_bytes");
  take(lib.attention, a, "mtpk_paged_attention_masked");
  take(lib.copy_blocks, a, "mtpk_copy_blocks");
  take(lib.tree_splits, a, "mtpk_attention_tree_splits");
  take(lib.tree_workspace, a, "mtpk_attention_tree_workspace_bytes");
  take(lib.tree_attention, a, "mtpk_paged_attention_tree");
  take(lib.prep_tree, a, "mtpk_deltanet_prep_tree");
  take(lib.rule_tree, a, "mtpk_delta_rule_tree");
  take(lib.commit_path, a, "mtpk_deltanet_commit_path");
  take(lib.tree_accept, a, "mtpk_tree_accept");
  take(lib.keep_path, a, "mtpk_keep_path");
  take(lib.status_string, a, "mtpk_status_string");
}

}  // namespace

PYBIND11_MODULE(_mtpk_torch, m) {
  m.attr("abi_version") = MTPK_ABI_VERSION;
  m.def("bind", &bind);
  m.def("rotate", &rotate);
  m.def("rotate_to_cache", &rotate_to_cache);
  m.def("paged_attention_masked", &paged_attention_masked);
  m.def("pool_blocks", &pool_blocks);
  m.def("copy_blocks", &copy_blocks);
  m.def("paged_attention_tree", &paged_attention_tree);
  m.def("prep_tree", &prep_tree);
  m.def("delta_rule_tree", &delta_rule_tree);
  m.def("commit_path", &commit_path);
  m.def("tree_accept", &tree_accept);
  m.def("keep_path", &keep_path);
}

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
}

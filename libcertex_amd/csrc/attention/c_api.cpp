// C API of the attention operators: checks of the arguments, then one launch each. Every entry point
// turns C++ exceptions into CUVS_ERROR and the last-error text of the calling thread.

#include <cuvs/neighbors/certex_attention.h>

#include "../certex_state.hpp"
#include "attention.hpp"
#include "overlap.hpp"

#include <cfloat>
#include <cmath>
#include <exception>
#include <string>
#include <vector>

namespace {

namespace ops = certex_amd::attention;

template <typename Fn>
cuvsError_t translate(Fn fn)
{
  try {
    fn();
    cuvsSetLastErrorText(nullptr);
    return CUVS_SUCCESS;
  } catch (std::exception const& e) {
    cuvsSetLastErrorText(e.what());
  } catch (...) {
    cuvsSetLastErrorText("unknown exception");
  }
  return CUVS_ERROR;
}

[[noreturn]] void refuse(std::string const& message) { throw std::invalid_argument("certex: " + message); }

/** The message is only put together where the check fails. */
#define EXPECTS(ok, message)         \
  do {                               \
    if (!(ok)) { refuse(message); }  \
  } while (0)

constexpr int kMaxDims = 4;

/** A borrowed tensor: extents, and strides in elements. */
struct tensor {
  void* p = nullptr;
  int ndim = 0;
  DLDataType type{};
  DLDevice device{};
  int64_t shape[kMaxDims]  = {};
  int64_t stride[kMaxDims] = {};
  const char* name         = "";

  [[nodiscard]] int64_t size() const
  {
    int64_t n = 1;
    for (int i = 0; i < ndim; ++i) { n *= shape[i]; }
    return n;
  }
  [[nodiscard]] bool is(uint8_t code, uint8_t bits) const
  {
    return type.code == code && type.bits == bits && type.lanes == 1;
  }
};

auto tensor_of(DLManagedTensor* m, const char* name) -> tensor
{
  EXPECTS(m != nullptr, std::string(name) + " is NULL");
  DLTensor const& t = m->dl_tensor;
  tensor v;
  v.name = name;
  v.ndim = t.ndim;
  EXPECTS(t.ndim >= 1 && t.ndim <= kMaxDims, std::string(name) + " has the wrong number of dimensions");
  EXPECTS(t.shape != nullptr, std::string(name) + " has no shape");
  v.p      = static_cast<char*>(t.data) + t.byte_offset;
  v.type   = t.dtype;
  v.device = t.device;
  EXPECTS(t.device.device_type == kDLROCM || t.device.device_type == kDLCUDA || t.device.device_type == kDLCUDAManaged,
          std::string(name) + " must be in device memory");
  int64_t dense = 1;
  for (int i = t.ndim - 1; i >= 0; --i) {
    EXPECTS(t.shape[i] >= 0, std::string(name) + " has a negative extent");
    v.shape[i]  = t.shape[i];
    v.stride[i] = t.strides != nullptr ? t.strides[i] : dense;
    EXPECTS(v.stride[i] >= 0, std::string(name) + " has a negative stride");
    if (v.shape[i] <= 1) { v.stride[i] = dense; }  // never stepped: keeps alignment rules simple
    dense *= std::max<int64_t>(1, t.shape[i]);
  }
  EXPECTS(v.size() == 0 || t.data != nullptr, std::string(name) + " has no data");
  EXPECTS(reinterpret_cast<uintptr_t>(v.p) % std::max(1, t.dtype.bits / 8) == 0,
          std::string(name) + " must begin at a multiple of its element size");
  return v;
}

void expects_shape(tensor const& t, std::initializer_list<int64_t> shape)
{
  bool ok = t.ndim == int(shape.size());
  int i   = 0;
  for (int64_t n : shape) {
    ok = ok && t.shape[i++] == n;
  }
  if (ok) { return; }
  std::string text;
  for (int64_t n : shape) { text += (text.empty() ? "" : ", ") + std::to_string(n); }
  refuse(std::string(t.name) + " must have shape (" + text + ")");
}

void expects_ndim(tensor const& t, int ndim)
{
  EXPECTS(t.ndim == ndim, std::string(t.name) + " must have " + std::to_string(ndim) + " dimensions");
}

auto dense(tensor t) -> tensor
{
  int64_t expect = 1;
  for (int i = t.ndim - 1; i >= 0; --i) {
    EXPECTS(t.stride[i] == expect || t.size() == 0, std::string(t.name) + " must be dense and row major");
    expect *= t.shape[i];
  }
  return t;
}

/** A row tensor of the elements `type` (or any, which it sets). */
auto rows(tensor t, ops::elem* type, bool first) -> tensor
{
  ops::elem e;
  if (t.is(kDLFloat, 32)) {
    e = ops::elem::f32;
  } else if (t.is(kDLFloat, 16)) {
    e = ops::elem::f16;
  } else if (t.is(kDLBfloat, 16)) {
    e = ops::elem::bf16;
  } else {
    throw std::invalid_argument(std::string("certex: ") + t.name + " must be float32, float16 or bfloat16");
  }
  EXPECTS(first || e == *type, std::string(t.name) + " must have the element type of the other tensors");
  *type = e;
  EXPECTS(t.stride[t.ndim - 1] == 1 || t.size() == 0, std::string(t.name) + " must be dense in its last dimension");
  return t;
}

struct dimensions {
  ops::dimension d[kMaxDims];
  explicit dimensions(tensor const& t)
  {
    for (int i = 0; i < t.ndim; ++i) { d[i] = {t.shape[i], t.stride[i]}; }
  }
};

/** A row tensor that is written: no two of its elements may be one in memory. */
auto written(tensor t) -> tensor
{
  if (t.size() == 0) { return t; }
  for (int i = 0; i < t.ndim; ++i) {
    EXPECTS(t.stride[i] > 0, std::string(t.name) + " is written and must not be broadcast");
  }
  EXPECTS(!ops::shares_itself(dimensions(t).d, t.ndim),
          std::string(t.name) + " is written and none of its elements may share memory");
  return t;
}

/** That b, which is written, shares no memory with a of the same element type, which is read or written by others. */
void expects_apart(tensor const& a, tensor const& b)
{
  if (a.size() == 0 || b.size() == 0) { return; }
  const int64_t distance = (static_cast<char const*>(b.p) - static_cast<char const*>(a.p)) / (b.type.bits / 8);
  EXPECTS(!ops::shares(dimensions(a).d, a.ndim, dimensions(b).d, b.ndim, distance),
          std::string(a.name) + " and " + b.name + " must not share memory in part");
}

/** The same, or that b is a, element for element. */
void expects_same_or_apart(tensor const& a, tensor const& b)
{
  if (a.p == b.p && a.ndim == b.ndim && std::equal(a.shape, a.shape + a.ndim, b.shape) &&
      std::equal(a.stride, a.stride + a.ndim, b.stride)) {
    return;
  }
  expects_apart(a, b);
}

auto integers(DLManagedTensor* m, const char* name) -> tensor
{
  tensor t = dense(tensor_of(m, name));
  EXPECTS(t.is(kDLInt, 32) || t.is(kDLInt, 64), std::string(name) + " must be int32 or int64");
  return t;
}

auto int_vector_of(tensor const& t) -> ops::int_vector { return {t.p, t.is(kDLInt, 64)}; }

auto res_of(cuvsResources_t res) -> cuvs::resources&
{
  EXPECTS(res != 0, "the resources handle is NULL");
  return *reinterpret_cast<cuvs::resources*>(res);
}

template <typename... Ts>
void expects_device(cuvs::resources const& r, Ts const&... ts)
{
  for (tensor const* t : {&ts...}) {
    EXPECTS(t->p == nullptr || t->size() == 0 || t->device.device_id == r.device(),
            std::string(t->name) + " is on another device than the resources");
  }
}

auto stream_of(cuvs::resources const& r) -> hipStream_t { return static_cast<hipStream_t>(r.stream()); }

/** The launch's own status (an invalid configuration); later faults surface on the stream. */
void check_launch() { CERTEX_HIP_TRY(hipGetLastError()); }

auto page_map_of(tensor const& table, int64_t sequences, tensor const& pages) -> ops::page_map
{
  EXPECTS(table.is(kDLInt, 32), std::string(table.name) + " must be int32");
  const int64_t width = table.shape[table.ndim - 1], page = pages.shape[1], n_pages = pages.shape[0];
  EXPECTS(page >= 1, "pages must hold at least one position");
  EXPECTS(n_pages < (int64_t(1) << 31) && page < (int64_t(1) << 31) && width < (int64_t(1) << 31) &&
            (page == 0 || width <= ((int64_t(1) << 31) - 1) / page),
          "a sequence's pages hold fewer than 2^31 positions");
  return {static_cast<const int32_t*>(table.p), sequences, int32_t(width), int32_t(n_pages), int32_t(page)};
}

struct rotary {
  int device       = 0;
  int rotary_dim   = 0;
  bool interleaved = false;
  float magnitude  = 1.0f;
  cuvs::detail::device_buffer frequencies;
};

auto rotary_of(cuvsCertexRotary_t r) -> rotary&
{
  EXPECTS(r != 0, "the rotary handle is NULL");
  return *reinterpret_cast<rotary*>(r);
}

/** The scaled frequencies and the magnitude. */
auto frequencies_of(cuvsCertexRotaryParams const& p, double* magnitude) -> std::vector<double>
{
  EXPECTS(p.rotary_dim >= 2 && p.rotary_dim % 2 == 0, "rotary_dim must be even and at least 2");
  EXPECTS(p.layout == CERTEX_ROTARY_HALF || p.layout == CERTEX_ROTARY_INTERLEAVED, "unknown rotary layout");
  EXPECTS(p.scaling >= CERTEX_ROTARY_NONE && p.scaling <= CERTEX_ROTARY_RAMP, "unknown rotary scaling");
  EXPECTS(std::isfinite(p.base) && p.base >= 1.0, "the rotary base must be at least 1");
  EXPECTS(p.scaling == CERTEX_ROTARY_NONE || (std::isfinite(p.factor) && p.factor >= 1.0),
          "the rotary factor must be at least 1");
  EXPECTS(std::isfinite(p.magnitude) && p.magnitude >= 0.0, "the rotary magnitude must not be negative");
  const int pairs = p.rotary_dim / 2;
  double base     = p.base;
  if (p.scaling == CERTEX_ROTARY_BASE) {
    EXPECTS(p.rotary_dim > 2, "scaling the base needs more than one pair");
    base *= std::pow(p.factor, double(p.rotary_dim) / (p.rotary_dim - 2));
  }
  const double two_pi = 2.0 * M_PI;
  std::vector<double> f(pairs);
  if (p.scaling == CERTEX_ROTARY_RAMP) {
    EXPECTS(std::isfinite(p.original_length) && p.original_length > 0.0, "the ramp needs the original length");
    EXPECTS(std::isfinite(p.ramp_low) && std::isfinite(p.ramp_high) && p.ramp_low < p.ramp_high,
            "the ramp must rise");
  }
  for (int i = 0; i < pairs; ++i) {
    f[i] = std::pow(base, -2.0 * i / p.rotary_dim);
    if (p.scaling == CERTEX_ROTARY_LINEAR) {
      f[i] /= p.factor;
    } else if (p.scaling == CERTEX_ROTARY_RAMP) {
      const double turns = p.original_length * f[i] / two_pi;
      const double g     = std::min(1.0, std::max(0.0, (turns - p.ramp_low) / (p.ramp_high - p.ramp_low)));
      f[i] *= g + (1.0 - g) / p.factor;
    }
  }
  *magnitude = p.magnitude > 0.0                          ? p.magnitude
               : p.scaling == CERTEX_ROTARY_RAMP ? 0.1 * std::log(p.factor) + 1.0
                                                  : 1.0;
  return f;
}

/** The window, cut to 2^32, which holds all positions: what the kernels add to it and take from it stays far from 64 bits' ends. */
auto window_of(int64_t window) -> int64_t
{
  EXPECTS(window >= 0, "the window must not be negative");
  return std::min(window, int64_t(1) << 32);
}

/** Queries, pages and table of an attention call, checked against each other. With `prompts` the queries are tokens of
 *  any of the table's sequences, else one of each. */
template <typename Args>
auto paged_args_of(DLManagedTensor* q_, DLManagedTensor* k_, DLManagedTensor* v_, DLManagedTensor* table_,
                   int64_t window, bool prompts, ops::elem* type, tensor* q, tensor* k, tensor* v, tensor* table) -> Args
{
  *q     = rows(tensor_of(q_, "q"), type, true);
  *k     = rows(tensor_of(k_, "k_pages"), type, false);
  *v     = rows(tensor_of(v_, "v_pages"), type, false);
  *table = dense(tensor_of(table_, "page_table"));
  expects_ndim(*q, 3);
  expects_ndim(*k, 4);
  expects_ndim(*v, 4);
  Args a;
  a.heads    = int32_t(q->shape[1]);
  a.kv_heads = int32_t(k->shape[2]);
  a.dim      = int32_t(q->shape[2]);
  a.vdim     = int32_t(v->shape[3]);
  EXPECTS(q->shape[1] >= 1 && q->shape[1] <= 65535 && k->shape[2] >= 1 && q->shape[1] % k->shape[2] == 0,
          "the query heads must be a multiple of the key heads (and at most 65535)");
  EXPECTS(a.dim >= 1 && k->shape[3] == a.dim, "q and k_pages must have the same head dimension");
  EXPECTS(q->shape[2] <= ops::kMaxHeadDim && v->shape[3] >= 1 && v->shape[3] <= ops::kMaxHeadDim,
          "head dimensions must be between 1 and " + std::to_string(ops::kMaxHeadDim));
  expects_shape(*v, {k->shape[0], k->shape[1], k->shape[2], v->shape[3]});
  expects_ndim(*table, 2);
  EXPECTS(prompts || table->shape[0] == q->shape[0], "page_table must have one row per sequence");
  EXPECTS(table->shape[0] <= 65535, "at most 65535 sequences");
  EXPECTS(k->shape[1] % ops::kPageUnit == 0 && k->shape[1] >= ops::kPageUnit,
          "the page size must be a multiple of " + std::to_string(ops::kPageUnit));
  a.window = window_of(window);
  a.pages  = page_map_of(*table, table->shape[0], *k);
  a.q      = q->p;
  a.q_head = q->stride[1];
  a.k      = k->p;
  a.k_page = k->stride[0];
  a.k_slot = k->stride[1];
  a.k_head = k->stride[2];
  a.v      = v->p;
  a.v_page = v->stride[0];
  a.v_slot = v->stride[1];
  a.v_head = v->stride[2];
  return a;
}

auto attend_args_of(DLManagedTensor* q_, DLManagedTensor* k_, DLManagedTensor* v_, DLManagedTensor* table_,
                    int64_t window, ops::elem* type, tensor* q, tensor* k, tensor* v, tensor* table)
  -> ops::attend_args
{
  auto a  = paged_args_of<ops::attend_args>(q_, k_, v_, table_, window, false, type, q, k, v, table);
  a.q_seq = q->stride[0];
  return a;
}

auto prompt_args_of(DLManagedTensor* q_, DLManagedTensor* k_, DLManagedTensor* v_, DLManagedTensor* table_,
                    int64_t window, ops::elem* type, tensor* q, tensor* k, tensor* v, tensor* table)
  -> ops::prompt_args
{
  auto a    = paged_args_of<ops::prompt_args>(q_, k_, v_, table_, window, true, type, q, k, v, table);
  a.q_token = q->stride[0];
  a.tokens  = q->shape[0];
  const int64_t group = a.heads / a.kv_heads;
  // rows of a key head, and blocks of 256 threads that a launch may have
  EXPECTS(a.tokens < (int64_t(1) << 29) && a.tokens * group < (int64_t(1) << 29) &&
            (a.tokens * group / 128 + std::min(a.tokens, table->shape[0])) * a.kv_heads < (int64_t(1) << 23),
          "too many tokens in one call");
  EXPECTS(int64_t(a.pages.width) * a.pages.page <= (int64_t(1) << 31) - 64, "a sequence's pages hold at most 2^31 - 64 positions");
  return a;
}

/** The bent scores' parameters: a cap of 0 and no slopes leave the scores as they are. */
auto shape_of(cuvs::resources const& r, float scale, float cap, DLManagedTensor* slopes, int64_t heads) -> ops::score_shape
{
  EXPECTS(std::isfinite(scale), "the scale must be finite");
  EXPECTS(std::isfinite(cap) && cap >= 0.0f, "the cap must be finite and not negative");
  EXPECTS(cap == 0.0f || std::abs(scale / cap) < 1e37f, "the cap is too small for the scale");
  // scores are taken as fractions of it, which float32 has to hold
  EXPECTS(cap <= 1e30f && (cap == 0.0f || scale == 0.0f || std::abs(scale / cap) >= FLT_MIN), "the cap is too large");
  ops::score_shape s;
  s.cap = cap;
  if (slopes != nullptr) {
    const tensor t = dense(tensor_of(slopes, "slopes"));
    EXPECTS(t.is(kDLFloat, 32), "slopes must be float32");
    expects_shape(t, {heads});
    expects_device(r, t);
    s.slopes = static_cast<const float*>(t.p);
  }
  return s;
}

/** 4-bit pages of heads of dim and vdim elements, and the table over them. */
auto packed_pages_of(DLManagedTensor* pages_, DLManagedTensor* table_, int64_t dim, int64_t vdim, tensor* pages, tensor* table)
  -> ops::packed_pages
{
  *pages = dense(tensor_of(pages_, "pages"));
  *table = dense(tensor_of(table_, "page_table"));
  expects_ndim(*pages, 4);
  expects_ndim(*table, 2);
  EXPECTS(pages->is(kDLUInt, 8), "pages must be uint8");
  EXPECTS(dim >= 1 && dim <= ops::kMaxHeadDim && vdim >= 1 && vdim <= ops::kMaxHeadDim,
          "head dimensions must be between 1 and " + std::to_string(ops::kMaxHeadDim));
  EXPECTS(pages->shape[1] >= 1 && pages->shape[1] <= 65535, "pages must have between 1 and 65535 heads");
  EXPECTS(pages->shape[2] >= 1 && pages->shape[2] < (int64_t(1) << 28), "pages must hold a multiple of 8 positions");
  EXPECTS(reinterpret_cast<uintptr_t>(pages->p) % 16 == 0, "pages must be aligned to 16 bytes");
  EXPECTS(table->shape[0] <= 65535, "at most 65535 sequences");
  ops::packed_pages p;
  p.p        = static_cast<uint8_t*>(pages->p);
  p.kv_heads = int32_t(pages->shape[1]);
  p.dim      = int32_t(dim);
  p.vdim     = int32_t(vdim);
  EXPECTS(pages->shape[3] == p.record(), "pages of heads of these dimensions have records of " + std::to_string(p.record()) +
                                           " bytes, not " + std::to_string(pages->shape[3]));
  tensor slots   = *pages;  // as the pages of other types are described: positions in their second extent
  slots.shape[1] = pages->shape[2] * 8;
  p.map          = page_map_of(*table, table->shape[0], slots);
  return p;
}

auto packed_args_of(DLManagedTensor* q_, DLManagedTensor* pages_, int64_t vdim, DLManagedTensor* table_, int64_t window,
                    ops::elem* type, tensor* q, tensor* pages, tensor* table) -> ops::packed_args
{
  *q = rows(tensor_of(q_, "q"), type, true);
  expects_ndim(*q, 3);
  ops::packed_args args;
  args.pages = packed_pages_of(pages_, table_, q->shape[2], vdim, pages, table);
  auto& a    = args.a;
  EXPECTS(q->shape[1] >= 1 && q->shape[1] <= 65535 && q->shape[1] % args.pages.kv_heads == 0,
          "the query heads must be a multiple of the key heads (and at most 65535)");
  EXPECTS(table->shape[0] == q->shape[0], "page_table must have one row per sequence");
  a.heads    = int32_t(q->shape[1]);
  a.kv_heads = args.pages.kv_heads;
  a.dim      = int32_t(q->shape[2]);
  a.vdim     = int32_t(vdim);
  a.pages    = args.pages.map;
  a.q        = q->p;
  a.q_seq    = q->stride[0];
  a.q_head   = q->stride[1];
  a.window   = window_of(window);
  return args;
}

auto select_args_of(DLManagedTensor* scores_, DLManagedTensor* values_, DLManagedTensor* table_, ops::elem* type,
                    tensor* scores, tensor* values, tensor* table) -> ops::select_args
{
  *scores = dense(tensor_of(scores_, "scores"));
  *values = rows(tensor_of(values_, "values"), type, true);
  EXPECTS(scores->is(kDLFloat, 32), "scores must be float32");
  expects_ndim(*scores, 3);
  ops::select_args a;
  const bool paged = table_ != nullptr;
  expects_ndim(*values, paged ? 4 : 3);
  const int64_t kv_heads = values->shape[paged ? 2 : 0], vdim = values->shape[paged ? 3 : 2];
  if (paged) {
    *table = dense(tensor_of(table_, "page_table"));
    expects_ndim(*table, 1);
    a.pages  = page_map_of(*table, 1, *values);
    a.n      = int64_t(a.pages.width) * a.pages.page;
    a.v_page = values->stride[0];
    a.v_slot = values->stride[1];
    a.v_head = values->stride[2];
  } else {
    a.n      = values->shape[1];
    a.v_head = values->stride[0];
    a.v_slot = values->stride[1];
    EXPECTS(a.n < (int64_t(1) << 31), "values hold fewer than 2^31 rows a head");
  }
  EXPECTS(scores->shape[0] >= 1 && kv_heads >= 1 && scores->shape[0] % kv_heads == 0,
          "the query heads must be a multiple of the value heads");
  EXPECTS(vdim >= 1 && vdim <= ops::kMaxHeadDim,
          "head dimensions must be between 1 and " + std::to_string(ops::kMaxHeadDim));
  EXPECTS(scores->shape[0] * scores->shape[1] <= (int64_t(1) << 23), "at most 2^23 queries over all heads");
  EXPECTS(scores->shape[2] < (int64_t(1) << 31), "fewer than 2^31 selected rows a query");
  a.heads    = int32_t(scores->shape[0]);
  a.kv_heads = int32_t(kv_heads);
  a.vdim     = int32_t(vdim);
  a.queries  = scores->shape[1];
  a.k        = scores->shape[2];
  a.scores   = static_cast<const float*>(scores->p);
  a.v        = values->p;
  return a;
}

/** The workspace argument: NULL, or a dense uint8 vector of enough bytes, 16-byte aligned. */
auto workspace_of(cuvs::resources const& r, DLManagedTensor* m, size_t bytes) -> void*
{
  if (bytes == 0) { return nullptr; }
  EXPECTS(m != nullptr, "this call needs a workspace");
  tensor t = dense(tensor_of(m, "workspace"));
  expects_ndim(t, 1);
  EXPECTS(t.is(kDLUInt, 8), "workspace must be uint8");
  EXPECTS(size_t(t.shape[0]) >= bytes, "the workspace is too small");
  EXPECTS(reinterpret_cast<uintptr_t>(t.p) % 16 == 0, "the workspace must be aligned to 16 bytes");
  expects_device(r, t);
  return t.p;
}

auto lse_of(cuvs::resources const& r, DLManagedTensor* m, int64_t rows_, int64_t cols) -> float*
{
  if (m == nullptr) { return nullptr; }
  tensor t = dense(tensor_of(m, "lse"));
  EXPECTS(t.is(kDLFloat, 32), "lse must be float32");
  expects_shape(t, {rows_, cols});
  expects_device(r, t);
  return static_cast<float*>(t.p);
}

}  // namespace

extern "C" {

cuvsError_t cuvsCertexRotaryParamsCreate(cuvsCertexRotaryParams_t* params)
{
  return translate([=] {
    EXPECTS(params != nullptr, "NULL argument");
    *params = new cuvsCertexRotaryParams{128, CERTEX_ROTARY_HALF, 10000.0, CERTEX_ROTARY_NONE, 1.0, 8192.0,
                                         1.0, 32.0, 0.0};
  });
}

cuvsError_t cuvsCertexRotaryParamsDestroy(cuvsCertexRotaryParams_t params)
{
  return translate([=] { delete params; });
}

cuvsError_t cuvsCertexRotaryFrequencies(cuvsCertexRotaryParams_t params, double* frequencies, double* magnitude)
{
  return translate([=] {
    EXPECTS(params != nullptr && frequencies != nullptr && magnitude != nullptr, "NULL argument");
    const auto f = frequencies_of(*params, magnitude);
    std::copy(f.begin(), f.end(), frequencies);
  });
}

cuvsError_t cuvsCertexRotaryCreate(cuvsResources_t res, cuvsCertexRotaryParams_t params, cuvsCertexRotary_t* out)
{
  return translate([=] {
    EXPECTS(params != nullptr && out != nullptr, "NULL argument");
    auto& r          = res_of(res);
    double magnitude = 1.0;
    const auto f     = frequencies_of(*params, &magnitude);
    // turns per position in 64-bit fixed point (at most 1 / (2 pi) of a turn)
    std::vector<uint64_t> turns(f.size());
    for (size_t i = 0; i < f.size(); ++i) { turns[i] = uint64_t(std::llround(std::ldexp(f[i] / (2.0 * M_PI), 64))); }
    auto h         = std::make_unique<rotary>();
    h->device      = r.device();
    h->rotary_dim  = params->rotary_dim;
    h->interleaved = params->layout == CERTEX_ROTARY_INTERLEAVED;
    h->magnitude   = float(magnitude);
    h->frequencies.resize_discard(turns.size() * sizeof(uint64_t));
    CERTEX_HIP_TRY(hipMemcpy(h->frequencies.p, turns.data(), turns.size() * sizeof(uint64_t), hipMemcpyHostToDevice));
    *out = reinterpret_cast<cuvsCertexRotary_t>(h.release());
  });
}

cuvsError_t cuvsCertexRotaryDestroy(cuvsCertexRotary_t rotary_)
{
  return translate([=] { delete reinterpret_cast<rotary*>(rotary_); });
}

cuvsError_t cuvsCertexRotate(cuvsResources_t res,
                             cuvsCertexRotary_t rotary_,
                             DLManagedTensor* x_,
                             DLManagedTensor* positions_,
                             DLManagedTensor* y_,
                             bool transpose)
{
  return translate([=] {
    auto& r = res_of(res);
    auto& h = rotary_of(rotary_);
    ops::elem type{};
    const tensor x = rows(tensor_of(x_, "x"), &type, true);
    const tensor y = written(rows(tensor_of(y_, "y"), &type, false));
    const tensor p = integers(positions_, "positions");
    EXPECTS(x.ndim == 3 || x.ndim == 4, "x must have 3 or 4 dimensions");
    const int o = x.ndim - 3;  // 1: a batch dimension
    EXPECTS(y.ndim == x.ndim && std::equal(x.shape, x.shape + x.ndim, y.shape), "y must have the shape of x");
    EXPECTS(p.ndim == 1 + o && std::equal(x.shape, x.shape + 1 + o, p.shape), "positions must have one entry per token");
    EXPECTS(h.rotary_dim <= x.shape[2 + o], "the rotation is wider than the heads");
    expects_device(r, x, y, p);
    EXPECTS(h.device == r.device(), "the rotary handle is on another device than the resources");
    EXPECTS(x.shape[1 + o] < (1 << 30) && x.shape[2 + o] < (1 << 30), "x is too large");
    if (x.size() == 0) { return; }
    expects_same_or_apart(x, y);
    ops::turn_args a;
    a.frequencies = h.frequencies.as<uint64_t>();
    a.magnitude   = h.magnitude;
    a.interleaved = h.interleaved;
    a.transpose   = transpose;
    a.positions   = int_vector_of(p);
    a.tokens      = p.size();
    a.inner       = x.shape[o];
    auto& j       = a.job[0];
    a.jobs        = 1;
    j.src         = x.p;
    j.dst         = y.p;
    j.src_outer   = o == 1 ? x.stride[0] : 0;
    j.dst_outer   = o == 1 ? y.stride[0] : 0;
    j.src_token   = x.stride[o];
    j.dst_token   = y.stride[o];
    j.src_head    = x.stride[1 + o];
    j.dst_head    = y.stride[1 + o];
    j.heads       = int32_t(x.shape[1 + o]);
    j.dim         = int32_t(x.shape[2 + o]);
    j.rotary      = h.rotary_dim;
    ops::turn(type, a, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexAppendPages(cuvsResources_t res,
                                  cuvsCertexRotary_t rotary_,
                                  DLManagedTensor* k_,
                                  DLManagedTensor* v_,
                                  DLManagedTensor* k_pages_,
                                  DLManagedTensor* v_pages_,
                                  DLManagedTensor* page_table_,
                                  DLManagedTensor* positions_,
                                  DLManagedTensor* sequences_,
                                  DLManagedTensor* q_,
                                  DLManagedTensor* q_out_)
{
  return translate([=] {
    auto& r  = res_of(res);
    auto* h  = rotary_ != 0 ? &rotary_of(rotary_) : nullptr;
    ops::elem type{};
    const tensor k = rows(tensor_of(k_, "k"), &type, true), v = rows(tensor_of(v_, "v"), &type, false);
    const tensor kp = written(rows(tensor_of(k_pages_, "k_pages"), &type, false));
    const tensor vp = written(rows(tensor_of(v_pages_, "v_pages"), &type, false));
    const tensor table = dense(tensor_of(page_table_, "page_table"));
    const tensor p     = integers(positions_, "positions");
    expects_ndim(k, 3);
    expects_ndim(kp, 4);
    expects_ndim(table, 2);
    const int64_t tokens = k.shape[0], heads = k.shape[1];
    EXPECTS(v.ndim == 3 && v.shape[0] == tokens && v.shape[1] == heads, "v must have the tokens and heads of k");
    expects_shape(kp, {kp.shape[0], kp.shape[1], heads, k.shape[2]});
    expects_shape(vp, {kp.shape[0], kp.shape[1], heads, v.shape[2]});
    expects_shape(p, {tokens});
    expects_device(r, k, v, kp, vp, table, p);
    EXPECTS(heads < (1 << 30) && k.shape[2] < (1 << 30) && v.shape[2] < (1 << 30), "k or v is too large");
    if (h != nullptr) {
      EXPECTS(h->rotary_dim <= k.shape[2], "the rotation is wider than the heads");
      EXPECTS(h->device == r.device(), "the rotary handle is on another device than the resources");
    }
    ops::turn_args a;
    a.positions = int_vector_of(p);
    if (sequences_ != nullptr) {
      const tensor s = integers(sequences_, "sequences");
      expects_shape(s, {tokens});
      expects_device(r, s);
      a.sequences = int_vector_of(s);
    } else {
      EXPECTS(table.shape[0] >= tokens, "without sequences, page_table must have one row per token");
    }
    if (h != nullptr) {
      a.frequencies = h->frequencies.as<uint64_t>();
      a.magnitude   = h->magnitude;
      a.interleaved = h->interleaved;
    }
    a.tokens = tokens;
    a.inner  = std::max<int64_t>(1, tokens);
    a.pages  = page_map_of(table, table.shape[0], kp);
    const auto add = [&](tensor const& src, tensor const& dst, int rotated, bool paged) {
      if (src.size() == 0) { return; }
      auto& j     = a.job[a.jobs++];
      j.src       = src.p;
      j.dst       = dst.p;
      j.src_token = src.stride[0];
      j.src_head  = src.stride[1];
      j.heads     = int32_t(src.shape[1]);
      j.dim       = int32_t(src.shape[2]);
      j.rotary    = rotated;
      j.paged     = paged;
      if (paged) { j.dst_outer = dst.stride[0]; }
      j.dst_token = dst.stride[paged ? 1 : 0];
      j.dst_head  = dst.stride[paged ? 2 : 1];
    };
    const int rotated = h != nullptr ? h->rotary_dim : 0;
    if (kp.size() > 0) { add(k, kp, rotated, true); }
    if (vp.size() > 0) { add(v, vp, 0, true); }
    if (q_ != nullptr) {
      const tensor q  = rows(tensor_of(q_, "q"), &type, false);
      const tensor qo = written(rows(tensor_of(q_out_, "q_out"), &type, false));
      EXPECTS(q.ndim == 3 && q.shape[0] == tokens && q.shape[2] == k.shape[2], "q must have the tokens and head dimension of k");
      expects_shape(qo, {q.shape[0], q.shape[1], q.shape[2]});
      expects_device(r, q, qo);
      expects_same_or_apart(q, qo);
      for (tensor const* t : {&k, &v, &kp, &vp}) { expects_apart(*t, qo); }
      add(q, qo, rotated, false);
    }
    if (a.jobs == 0) { return; }
    ops::turn(type, a, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexPagedAttentionWorkspace(DLManagedTensor* q_,
                                              DLManagedTensor* k_pages_,
                                              DLManagedTensor* v_pages_,
                                              DLManagedTensor* page_table_,
                                              int64_t window,
                                              int64_t* bytes)
{
  return translate([=] {
    EXPECTS(bytes != nullptr, "NULL argument");
    ops::elem type{};
    tensor q, k, v, table;
    const auto a = attend_args_of(q_, k_pages_, v_pages_, page_table_, window, &type, &q, &k, &v, &table);
    *bytes       = int64_t(ops::attend_workspace(type, a));
  });
}

cuvsError_t cuvsCertexPagedAttentionShaped(cuvsResources_t res,
                                           DLManagedTensor* q_,
                                           DLManagedTensor* k_pages_,
                                           DLManagedTensor* v_pages_,
                                           DLManagedTensor* page_table_,
                                           DLManagedTensor* lengths_,
                                           float scale,
                                           float cap,
                                           DLManagedTensor* slopes_,
                                           int64_t window,
                                           DLManagedTensor* workspace_,
                                           DLManagedTensor* out_,
                                           DLManagedTensor* lse_)
{
  return translate([=] {
    auto& r = res_of(res);
    ops::elem type{};
    tensor q, k, v, table;
    auto a = attend_args_of(q_, k_pages_, v_pages_, page_table_, window, &type, &q, &k, &v, &table);
    const tensor lengths = integers(lengths_, "lengths");
    expects_shape(lengths, {q.shape[0]});
    const tensor out = dense(rows(tensor_of(out_, "out"), &type, false));
    expects_shape(out, {q.shape[0], q.shape[1], v.shape[3]});
    expects_device(r, q, k, v, table, lengths, out);
    EXPECTS(std::isfinite(scale), "the scale must be finite");
    const auto shape = shape_of(r, scale, cap, slopes_, q.shape[1]);
    a.lse = lse_of(r, lse_, q.shape[0], q.shape[1]);
    if (q.shape[0] == 0) { return; }
    a.lengths   = int_vector_of(lengths);
    a.scale     = scale;
    a.shape     = shape;
    a.out       = out.p;
    a.workspace = workspace_of(r, workspace_, ops::attend_workspace(type, a));
    ops::attend(type, a, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexPagedAttention(cuvsResources_t res,
                                     DLManagedTensor* q_,
                                     DLManagedTensor* k_pages_,
                                     DLManagedTensor* v_pages_,
                                     DLManagedTensor* page_table_,
                                     DLManagedTensor* lengths_,
                                     float scale,
                                     int64_t window,
                                     DLManagedTensor* workspace_,
                                     DLManagedTensor* out_,
                                     DLManagedTensor* lse_)
{
  return cuvsCertexPagedAttentionShaped(res, q_, k_pages_, v_pages_, page_table_, lengths_, scale, 0.0f, nullptr, window,
                                        workspace_, out_, lse_);
}

cuvsError_t cuvsCertexPromptAttentionWorkspace(DLManagedTensor* q_,
                                               DLManagedTensor* k_pages_,
                                               DLManagedTensor* v_pages_,
                                               DLManagedTensor* page_table_,
                                               int64_t window,
                                               int64_t* bytes)
{
  return translate([=] {
    EXPECTS(bytes != nullptr, "NULL argument");
    ops::elem type{};
    tensor q, k, v, table;
    const auto a = prompt_args_of(q_, k_pages_, v_pages_, page_table_, window, &type, &q, &k, &v, &table);
    *bytes       = int64_t(ops::prompt_workspace(type, a));
  });
}

cuvsError_t cuvsCertexPromptAttention(cuvsResources_t res,
                                      DLManagedTensor* q_,
                                      DLManagedTensor* k_pages_,
                                      DLManagedTensor* v_pages_,
                                      DLManagedTensor* page_table_,
                                      DLManagedTensor* lengths_,
                                      DLManagedTensor* first_,
                                      DLManagedTensor* prefix_,
                                      float scale,
                                      float cap,
                                      DLManagedTensor* slopes_,
                                      int64_t window,
                                      DLManagedTensor* workspace_,
                                      DLManagedTensor* out_,
                                      DLManagedTensor* lse_)
{
  return translate([=] {
    auto& r = res_of(res);
    ops::elem type{};
    tensor q, k, v, table;
    auto a = prompt_args_of(q_, k_pages_, v_pages_, page_table_, window, &type, &q, &k, &v, &table);
    const int64_t sequences = table.shape[0];
    const tensor lengths = integers(lengths_, "lengths"), first = integers(first_, "first");
    expects_shape(lengths, {sequences});
    expects_shape(first, {sequences + 1});
    const tensor out = dense(rows(tensor_of(out_, "out"), &type, false));
    expects_shape(out, {q.shape[0], q.shape[1], v.shape[3]});
    expects_device(r, q, k, v, table, lengths, first, out);
    EXPECTS(std::isfinite(scale), "the scale must be finite");
    if (prefix_ != nullptr) {
      const tensor prefix = integers(prefix_, "prefix");
      expects_shape(prefix, {sequences});
      expects_device(r, prefix);
      a.prefix = int_vector_of(prefix);
    }
    a.shape = shape_of(r, scale, cap, slopes_, q.shape[1]);
    a.lse   = lse_of(r, lse_, q.shape[0], q.shape[1]);
    if (q.shape[0] == 0) { return; }
    a.lengths   = int_vector_of(lengths);
    a.first     = int_vector_of(first);
    a.scale     = scale;
    a.out       = out.p;
    a.workspace = workspace_of(r, workspace_, ops::prompt_workspace(type, a));
    ops::prompt(type, a, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexPackedRecord(int64_t dim, int64_t vdim, int64_t* bytes)
{
  return translate([=] {
    EXPECTS(bytes != nullptr, "NULL argument");
    EXPECTS(dim >= 1 && dim <= ops::kMaxHeadDim && vdim >= 1 && vdim <= ops::kMaxHeadDim,
            "head dimensions must be between 1 and " + std::to_string(ops::kMaxHeadDim));
    ops::packed_pages p;
    p.dim  = int32_t(dim);
    p.vdim = int32_t(vdim);
    *bytes = p.record();
  });
}

cuvsError_t cuvsCertexPackPages(cuvsResources_t res,
                                cuvsCertexRotary_t rotary_,
                                DLManagedTensor* k_,
                                DLManagedTensor* v_,
                                DLManagedTensor* pages_,
                                DLManagedTensor* page_table_,
                                DLManagedTensor* positions_,
                                DLManagedTensor* sequences_)
{
  return translate([=] {
    auto& r = res_of(res);
    auto* h = rotary_ != 0 ? &rotary_of(rotary_) : nullptr;
    ops::elem type{};
    const tensor k = rows(tensor_of(k_, "k"), &type, true), v = rows(tensor_of(v_, "v"), &type, false);
    expects_ndim(k, 3);
    expects_ndim(v, 3);
    tensor pages, table;
    ops::pack_args a;
    a.pages             = packed_pages_of(pages_, page_table_, k.shape[2], v.shape[2], &pages, &table);
    const int64_t tokens = k.shape[0];
    EXPECTS(k.shape[1] == a.pages.kv_heads, "k must have the heads of the pages");
    EXPECTS(v.shape[0] == tokens && v.shape[1] == k.shape[1], "v must have the tokens and heads of k");
    a.tokens = tokens;
    const tensor positions = integers(positions_, "positions");
    expects_shape(positions, {tokens});
    a.positions = int_vector_of(positions);
    expects_device(r, k, v, pages, table, positions);
    if (sequences_ != nullptr) {
      const tensor s = integers(sequences_, "sequences");
      expects_shape(s, {tokens});
      expects_device(r, s);
      a.sequences = int_vector_of(s);
    } else {
      EXPECTS(table.shape[0] >= tokens, "without sequences, page_table must have one row per token");
    }
    if (h != nullptr) {
      EXPECTS(h->rotary_dim <= k.shape[2], "the rotation is wider than the heads");
      EXPECTS(h->device == r.device(), "the rotary handle is on another device than the resources");
      a.frequencies = h->frequencies.as<uint64_t>();
      a.magnitude   = h->magnitude;
      a.interleaved = h->interleaved;
      a.rotary      = h->rotary_dim;
    }
    if (tokens == 0 || pages.size() == 0) { return; }
    a.k = {k.p, nullptr, k.stride[0], k.stride[1]};
    a.v = {v.p, nullptr, v.stride[0], v.stride[1]};
    ops::pack_pages(type, a, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexUnpackPages(cuvsResources_t res,
                                  DLManagedTensor* pages_,
                                  DLManagedTensor* page_table_,
                                  DLManagedTensor* positions_,
                                  DLManagedTensor* sequences_,
                                  DLManagedTensor* k_,
                                  DLManagedTensor* v_)
{
  return translate([=] {
    auto& r = res_of(res);
    ops::elem type{};
    const tensor k = written(rows(tensor_of(k_, "k"), &type, true)), v = written(rows(tensor_of(v_, "v"), &type, false));
    expects_ndim(k, 3);
    expects_ndim(v, 3);
    tensor pages, table;
    ops::pack_args a;
    a.pages             = packed_pages_of(pages_, page_table_, k.shape[2], v.shape[2], &pages, &table);
    const int64_t tokens = k.shape[0];
    EXPECTS(k.shape[1] == a.pages.kv_heads, "k must have the heads of the pages");
    EXPECTS(v.shape[0] == tokens && v.shape[1] == k.shape[1], "v must have the tokens and heads of k");
    a.tokens = tokens;
    const tensor positions = integers(positions_, "positions");
    expects_shape(positions, {tokens});
    a.positions = int_vector_of(positions);
    expects_device(r, k, v, pages, table, positions);
    expects_apart(k, v);
    if (sequences_ != nullptr) {
      const tensor s = integers(sequences_, "sequences");
      expects_shape(s, {tokens});
      expects_device(r, s);
      a.sequences = int_vector_of(s);
    } else {
      EXPECTS(table.shape[0] >= tokens, "without sequences, page_table must have one row per token");
    }
    if (tokens == 0) { return; }
    a.k = {nullptr, k.p, k.stride[0], k.stride[1]};
    a.v = {nullptr, v.p, v.stride[0], v.stride[1]};
    ops::unpack_pages(type, a, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexPackedAttentionWorkspace(DLManagedTensor* q_,
                                               DLManagedTensor* pages_,
                                               int64_t vdim,
                                               DLManagedTensor* page_table_,
                                               int64_t window,
                                               int64_t* bytes)
{
  return translate([=] {
    EXPECTS(bytes != nullptr, "NULL argument");
    ops::elem type{};
    tensor q, pages, table;
    const auto args = packed_args_of(q_, pages_, vdim, page_table_, window, &type, &q, &pages, &table);
    *bytes          = int64_t(ops::packed_workspace(type, args));
  });
}

cuvsError_t cuvsCertexPackedAttention(cuvsResources_t res,
                                      DLManagedTensor* q_,
                                      DLManagedTensor* pages_,
                                      int64_t vdim,
                                      DLManagedTensor* page_table_,
                                      DLManagedTensor* lengths_,
                                      float scale,
                                      float cap,
                                      DLManagedTensor* slopes_,
                                      int64_t window,
                                      DLManagedTensor* workspace_,
                                      DLManagedTensor* out_,
                                      DLManagedTensor* lse_)
{
  return translate([=] {
    auto& r = res_of(res);
    ops::elem type{};
    tensor q, pages, table;
    auto args            = packed_args_of(q_, pages_, vdim, page_table_, window, &type, &q, &pages, &table);
    auto& a              = args.a;
    const tensor lengths = integers(lengths_, "lengths");
    expects_shape(lengths, {q.shape[0]});
    const tensor out = dense(rows(tensor_of(out_, "out"), &type, false));
    expects_shape(out, {q.shape[0], q.shape[1], vdim});
    expects_device(r, q, pages, table, lengths, out);
    EXPECTS(std::isfinite(scale), "the scale must be finite");
    a.shape = shape_of(r, scale, cap, slopes_, q.shape[1]);
    a.lse   = lse_of(r, lse_, q.shape[0], q.shape[1]);
    if (q.shape[0] == 0) { return; }
    a.lengths   = int_vector_of(lengths);
    a.scale     = scale;
    a.out       = out.p;
    a.workspace = workspace_of(r, workspace_, ops::packed_workspace(type, args));
    ops::packed_attend(type, args, stream_of(r));
    check_launch();
  });
}

cuvsError_t cuvsCertexSelectedAttentionWorkspace(DLManagedTensor* scores_,
                                                 DLManagedTensor* values_,
                                                 DLManagedTensor* page_table_,
                                                 int64_t* bytes)
{
  return translate([=] {
    EXPECTS(bytes != nullptr, "NULL argument");
    ops::elem type{};
    tensor scores, values, table;
    const auto a = select_args_of(scores_, values_, page_table_, &type, &scores, &values, &table);
    *bytes       = int64_t(ops::select_workspace(type, a));
  });
}

cuvsError_t cuvsCertexSelectedAttention(cuvsResources_t res,
                                        DLManagedTensor* scores_,
                                        DLManagedTensor* ids_,
                                        DLManagedTensor* values_,
                                        DLManagedTensor* page_table_,
                                        float scale,
                                        DLManagedTensor* workspace_,
                                        DLManagedTensor* out_,
                                        DLManagedTensor* lse_)
{
  return translate([=] {
    auto& r = res_of(res);
    ops::elem type{};
    tensor scores, values, table;
    auto a = select_args_of(scores_, values_, page_table_, &type, &scores, &values, &table);
    const tensor ids = integers(ids_, "ids");
    expects_shape(ids, {scores.shape[0], scores.shape[1], scores.shape[2]});
    const tensor out = dense(rows(tensor_of(out_, "out"), &type, false));
    expects_shape(out, {scores.shape[0], scores.shape[1], int64_t(a.vdim)});
    expects_device(r, scores, ids, values, table, out);
    EXPECTS(std::isfinite(scale), "the scale must be finite");
    a.lse = lse_of(r, lse_, scores.shape[0], scores.shape[1]);
    if (a.queries == 0) { return; }
    a.ids       = int_vector_of(ids);
    a.scale     = scale;
    a.out       = out.p;
    a.workspace = workspace_of(r, workspace_, ops::select_workspace(type, a));
    ops::select(type, a, stream_of(r));
    check_launch();
  });
}

}  // extern "C"

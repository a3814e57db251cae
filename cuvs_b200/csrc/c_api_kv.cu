// C interface of attention over a paged cache (include/cuvs_kv_cache.h): descriptions of tensors, checks, calls.
#include "../../include/cuvs_kv_cache.h"

#include "c_api_util.hpp"
#include "kv_cache.hpp"
#include "tensor_exchange.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

using namespace cuvs_b200;
using namespace cuvs_b200::capi;
using kv::tensor;

namespace {

tensor describe(const DLTensor& d, const char* name)
{
  tensor t;
  CUVS_EXPECTS(d.ndim >= 1 && d.ndim <= 4, "%s: 1 to 4 dimensions, not %d", name, int(d.ndim));
  CUVS_EXPECTS(d.dtype.lanes == 1, "More than 1 DLTensor lanes not supported");
  t.data        = static_cast<char*>(d.data) + d.byte_offset;
  t.code        = d.dtype.code;
  t.bits        = d.dtype.bits;
  t.ndim        = d.ndim;
  t.device_type = int(d.device.device_type);
  t.device_id   = d.device.device_id;
  int64_t dense = 1;
  for (int i = d.ndim - 1; i >= 0; i--) {
    t.shape[i]  = d.shape[i];
    t.stride[i] = d.strides ? d.strides[i] : dense;
    dense *= d.shape[i];
  }
  return t;
}
tensor describe(const DLManagedTensor* mt, const char* name) { return mt == nullptr ? tensor{} : describe(mt->dl_tensor, name); }

// From words: ndim | type code << 32 | bits << 40 (0: not given), address, device, shape, strides.
tensor describe(const int64_t*& w, const int64_t* end, const char* name)
{
  tensor t;
  CUVS_EXPECTS(w < end, "the words do not describe the call");
  const int64_t kind = *w++;
  if (kind == 0) { return t; }
  t.ndim = int(kind & 0xFF);
  CUVS_EXPECTS(t.ndim >= 1 && t.ndim <= 4, "%s: 1 to 4 dimensions, not %d", name, t.ndim);
  CUVS_EXPECTS(end - w >= 2 + 2 * t.ndim, "the words do not describe the call");
  t.code        = int((kind >> 32) & 0xFF);
  t.bits        = int((kind >> 40) & 0xFF);
  t.data        = reinterpret_cast<char*>(w[0]);
  t.device_type = int(w[1] & 0xFFFFFFFF);
  t.device_id   = int(w[1] >> 32);
  std::copy(w + 2, w + 2 + t.ndim, t.shape);
  std::copy(w + 2 + t.ndim, w + 2 + 2 * t.ndim, t.stride);
  w += 2 + 2 * t.ndim;
  return t;
}

struct device_scope {  // the handle's device for the length of a call, whatever the caller's current one is
  int before = 0;
  int device;
  explicit device_scope(int d) : device(d)
  {
    CUDA_TRY(cudaGetDevice(&before));
    if (before != device) { CUDA_TRY(cudaSetDevice(device)); }
  }
  ~device_scope()
  {
    if (before != device) { cudaSetDevice(before); }
  }
};

// A given tensor on the handle's device; extents are not negative, strides of extents of one do not matter.
void check_place(int device, tensor& t, int ndim, const char* name)
{
  CUVS_EXPECTS(t.given(), "%s: null tensor", name);
  CUVS_EXPECTS(t.ndim == ndim, "%s: %d dimensions, not %d", name, ndim, t.ndim);
  CUVS_EXPECTS(t.device_type == kDLCUDA || t.device_type == kDLCUDAManaged, "%s: device_type mismatch: expected a CUDA tensor", name);
  CUVS_EXPECTS(t.device_type != kDLCUDA || t.device_id == device, "%s: on device %d, but the handle is for device %d", name,
               t.device_id, device);
  bool empty = false;
  for (int i = 0; i < ndim; i++) {
    CUVS_EXPECTS(t.shape[i] >= 0 && t.stride[i] >= 0, "%s: negative extent or stride", name);
    CUVS_EXPECTS(t.shape[i] <= (int64_t(1) << 48) && t.stride[i] <= (int64_t(1) << 48), "%s: too large", name);
    if (t.shape[i] <= 1) { t.stride[i] = 0; }
    empty = empty || t.shape[i] == 0;
  }
  CUVS_EXPECTS(empty || t.data != nullptr, "%s: null tensor", name);
  CUVS_EXPECTS(empty || t.bits < 8 || reinterpret_cast<uintptr_t>(t.data) % (t.bits / 8) == 0, "%s: not on a boundary of its elements", name);
  if (empty) {  // no element has a place: as if it were dense
    int64_t dense = 1;
    for (int i = ndim - 1; i >= 0; i--) {
      t.stride[i] = t.shape[i] <= 1 ? 0 : dense;
      dense *= t.shape[i];
    }
  }
}

kv::elem elem_of(const tensor& t, const char* name)
{
  if (t.code == kDLFloat && t.bits == 16) { return kv::elem::f16; }
  if (t.code == kDLBfloat && t.bits == 16) { return kv::elem::bf16; }
  if (t.code == kDLFloat && t.bits == 32) { return kv::elem::f32; }
  fail("%s: unsupported element type (code %d, %d bits): f16, bf16 and f32 are supported", name, t.code, t.bits);
}

void check_type(const tensor& t, int code, int bits, const char* name)
{
  CUVS_EXPECTS(t.code == code && t.bits == bits, "%s: expected %s%d elements, not code %d with %d bits", name,
               code == kDLInt ? "int" : code == kDLUInt ? "uint" : "float", bits, t.code, t.bits);
}

// The tensors' strides of given extents in ascending order never step into what lies between: no element twice.
void check_distinct(const tensor& t, const char* name)
{
  int order[4], n = 0;
  for (int i = 0; i < t.ndim; i++) {
    if (t.shape[i] == 0) { return; }
    if (t.shape[i] > 1) { order[n++] = i; }
  }
  std::sort(order, order + n, [&](int a, int b) { return t.stride[a] < t.stride[b]; });
  int64_t reach = 1;
  for (int i = 0; i < n; i++) {
    CUVS_EXPECTS(t.stride[order[i]] >= reach, "%s: its elements overlap, it cannot be written", name);
    reach = t.stride[order[i]] * t.shape[order[i]];
  }
}

// Rows of `dim` contiguous elements, each on a 16-byte boundary.
void check_rows(int device, tensor& t, int ndim, kv::elem type, const char* name)
{
  check_place(device, t, ndim, name);
  CUVS_EXPECTS(elem_of(t, name) == type, "%s: the element type of keys and values is another", name);
  const int64_t size = t.bits / 8, dim = t.shape[ndim - 1];
  CUVS_EXPECTS(dim >= 1 && dim <= 256, "%s: rows of 1 to 256 elements, not %lld", name, (long long)dim);
  CUVS_EXPECTS(t.stride[ndim - 1] == (dim == 1 ? 0 : 1), "%s: the elements of a row must be contiguous", name);
  bool aligned = (dim * size) % 16 == 0 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0;
  for (int i = 0; i + 1 < ndim; i++) { aligned = aligned && (t.stride[i] * size) % 16 == 0; }
  CUVS_EXPECTS(aligned, "%s: rows must be a multiple of 16 bytes long and start on 16-byte boundaries", name);
}

kv::cache_view cache_of(int device, tensor& keys, tensor& values, const tensor& filter_given, kv::elem& type)
{
  CUVS_EXPECTS(keys.given(), "keys: null tensor");
  type = elem_of(keys, "keys");
  check_rows(device, keys, 4, type, "keys");
  check_rows(device, values, 4, type, "values");
  CUVS_EXPECTS(std::equal(keys.shape, keys.shape + 4, values.shape), "keys and values must have the same shape");
  kv::cache_view c{};
  CUVS_EXPECTS(keys.shape[0] < (int64_t(1) << 31) && keys.shape[1] < (int64_t(1) << 31) && keys.shape[2] < 65536,
               "keys: too many pages, tokens of a page or heads");
  CUVS_EXPECTS(keys.shape[1] >= 1 && keys.shape[2] >= 1, "keys: pages of at least one token and one head");
  c.keys       = keys.data;
  c.values     = values.data;
  c.k_page     = keys.stride[0];
  c.k_token    = keys.stride[1];
  c.k_head     = keys.stride[2];
  c.v_page     = values.stride[0];
  c.v_token    = values.stride[1];
  c.v_head     = values.stride[2];
  c.n_pages    = int32_t(keys.shape[0]);
  c.page       = kv::divisor_of(uint32_t(keys.shape[1]));
  c.n_heads    = uint32_t(keys.shape[2]);
  c.dim        = uint32_t(keys.shape[3]);
  c.n_slots    = keys.shape[0] * keys.shape[1];
  // the largest unit that all strides are multiples of; 16 bytes at least
  const int64_t size     = keys.bits / 8;
  const int64_t strides[] = {c.k_page * size, c.k_token * size, c.v_page * size, c.v_token * size};
  c.unit_shift           = 4;
  while (c.unit_shift < 16 && std::all_of(strides, strides + 4, [&](int64_t x) { return x % (int64_t(2) << c.unit_shift) == 0; })) { c.unit_shift++; }
  for (int i = 0; i < 4; i += 2) {
    const auto reach = [&](int64_t n, int64_t stride) { return unsigned(n > 0 ? n - 1 : 0) * (unsigned __int128)(stride >> c.unit_shift); };
    CUVS_EXPECTS(reach(c.n_pages, strides[i]) + reach(c.page.size, strides[i + 1]) < ((unsigned __int128)1 << 32),
                 "%s: too large for rows at multiples of %u bytes", i == 0 ? "keys" : "values", 1u << c.unit_shift);
  }
  c.k_page_units  = uint32_t(strides[0] >> c.unit_shift);
  c.k_token_units = uint32_t(strides[1] >> c.unit_shift);
  c.v_page_units  = uint32_t(strides[2] >> c.unit_shift);
  c.v_token_units = uint32_t(strides[3] >> c.unit_shift);
  if (filter_given.given()) {
    tensor f = filter_given;
    check_place(device, f, 1, "filter");
    check_type(f, kDLUInt, 32, "filter");
    CUVS_EXPECTS(f.shape[0] <= 1 || f.stride[0] == 1, "filter: must be contiguous");
    CUVS_EXPECTS(f.shape[0] >= (c.n_slots + 31) / 32, "filter: %lld words cannot hold a bit for each of %lld slots", (long long)f.shape[0],
                 (long long)c.n_slots);
    if (c.n_slots > 0) { c.filter = reinterpret_cast<const uint32_t*>(f.data); }
  }
  return c;
}

tensor filter_of(const cuvsFilter& f)
{
  if (f.type == NO_FILTER) { return {}; }
  CUVS_EXPECTS(f.type == BITSET, "Unsupported sample filter type");
  CUVS_EXPECTS(f.addr != 0, "filter: null tensor");
  return describe(reinterpret_cast<const DLManagedTensor*>(f.addr), "filter");
}

const int32_t* ints_of(int device, tensor& t, const char* name, int64_t n, const char* what)
{
  check_place(device, t, 1, name);
  check_type(t, kDLInt, 32, name);
  CUVS_EXPECTS(t.shape[0] <= 1 || t.stride[0] == 1, "%s: must be contiguous", name);
  CUVS_EXPECTS(n < 0 || t.shape[0] == n, "%s: one for each %s", name, what);
  return reinterpret_cast<const int32_t*>(t.data);
}

// [n, n_heads, dim] rows that go with the cache
kv::rows_view rows_of(int device, tensor& t, kv::elem type, const kv::cache_view& c, int64_t n, int64_t n_heads, const char* name)
{
  check_rows(device, t, 3, type, name);
  CUVS_EXPECTS(t.shape[2] == int64_t(c.dim), "%s: rows of %u elements, not %lld", name, c.dim, (long long)t.shape[2]);
  CUVS_EXPECTS((n < 0 || t.shape[0] == n) && (n_heads < 0 || t.shape[1] == n_heads), "%s: expected %lld rows of %lld heads, not %lld of %lld",
               name, (long long)n, (long long)n_heads, (long long)t.shape[0], (long long)t.shape[1]);
  return {t.data, t.stride[0], t.stride[1]};
}

uint32_t query_heads_of(const tensor& queries, const kv::cache_view& c)
{
  CUVS_EXPECTS(queries.shape[1] >= 1 && queries.shape[1] % c.n_heads == 0 && queries.shape[1] < 65536,
               "queries: their %lld heads are no multiple of the cache's %u", (long long)queries.shape[1], c.n_heads);
  CUVS_EXPECTS(queries.shape[0] * queries.shape[1] < (int64_t(1) << 31), "queries: too many rows");
  return uint32_t(queries.shape[1]);
}

float* lse_of(int device, tensor& t, int64_t n, int64_t n_heads)
{
  check_place(device, t, 2, "lse");
  check_type(t, kDLFloat, 32, "lse");
  CUVS_EXPECTS(t.shape[0] == n && t.shape[1] == n_heads, "lse: expected shape [%lld, %lld]", (long long)n, (long long)n_heads);
  CUVS_EXPECTS((n_heads <= 1 || t.stride[1] == 1) && (n <= 1 || t.stride[0] == n_heads), "lse: must be contiguous");
  return reinterpret_cast<float*>(t.data);
}

void pages_of(int device, tensor& t, uint32_t& n_sequences, uint32_t& width, int64_t& stride)
{
  check_place(device, t, 2, "pages");
  check_type(t, kDLInt, 32, "pages");
  CUVS_EXPECTS(t.shape[0] < (int64_t(1) << 31) && t.shape[1] < (int64_t(1) << 31), "pages: too large");
  CUVS_EXPECTS(t.shape[1] <= 1 || t.stride[1] == 1, "pages: the entries of a sequence must be contiguous");
  n_sequences = uint32_t(t.shape[0]);
  width       = uint32_t(t.shape[1]);
  stride      = t.stride[0];
}

kv::append_args append_of(int device, tensor* t, bool interleaved)
{
  enum { KEYS, VALUES, NEW_KEYS, NEW_VALUES, PAGES, POSITIONS, SEQUENCES, QUERIES, FREQUENCIES, SLOTS, ROTATED };
  kv::append_args a{};
  a.cache = cache_of(device, t[KEYS], t[VALUES], {}, a.type);
  check_distinct(t[KEYS], "keys");
  check_distinct(t[VALUES], "values");
  const kv::rows_view k = rows_of(device, t[NEW_KEYS], a.type, a.cache, -1, a.cache.n_heads, "new_keys");
  const int64_t n       = t[NEW_KEYS].shape[0];
  const kv::rows_view v = rows_of(device, t[NEW_VALUES], a.type, a.cache, n, a.cache.n_heads, "new_values");
  CUVS_EXPECTS(n < (int64_t(1) << 31), "new_keys: too many tokens");
  a.n_tokens = uint32_t(n);
  a.keys     = k.data;
  a.k_row    = k.row;
  a.k_head   = k.head;
  a.values   = v.data;
  a.v_row    = v.row;
  a.v_head   = v.head;
  pages_of(device, t[PAGES], a.n_sequences, a.table_width, a.table_stride);
  a.pages     = reinterpret_cast<const int32_t*>(t[PAGES].data);
  a.positions = ints_of(device, t[POSITIONS], "positions", n, "token");
  if (t[SEQUENCES].given()) {
    a.sequences = ints_of(device, t[SEQUENCES], "sequences", n, "token");
  } else {
    CUVS_EXPECTS(int64_t(a.n_sequences) == n, "without `sequences` there must be one token for each of the %u sequences, not %lld", a.n_sequences,
                 (long long)n);
  }
  if (t[FREQUENCIES].given()) {
    tensor& f = t[FREQUENCIES];
    check_place(device, f, 1, "frequencies");
    CUVS_EXPECTS(f.code == kDLFloat && (f.bits == 64 || f.bits == 32), "frequencies: expected float64 or float32 elements");
    CUVS_EXPECTS(f.shape[0] <= 1 || f.stride[0] == 1, "frequencies: must be contiguous");
    CUVS_EXPECTS(2 * f.shape[0] <= int64_t(a.cache.dim), "frequencies: %lld pairs do not fit rows of %u elements", (long long)f.shape[0],
                 a.cache.dim);
    a.frequencies     = f.data;
    a.frequencies_f32 = f.bits == 32;
    a.n_pairs         = uint32_t(f.shape[0]);
  }
  a.interleaved = interleaved;
  CUVS_EXPECTS(t[QUERIES].given() == t[ROTATED].given(), "queries and rotated are given together");
  if (t[QUERIES].given()) {
    a.queries       = rows_of(device, t[QUERIES], a.type, a.cache, n, -1, "queries");
    a.n_query_heads = uint32_t(t[QUERIES].shape[1]);
    CUVS_EXPECTS(t[QUERIES].shape[1] < 65536, "queries: too many heads");
    a.rotated = rows_of(device, t[ROTATED], a.type, a.cache, n, t[QUERIES].shape[1], "rotated");
    check_distinct(t[ROTATED], "rotated");
  }
  check_place(device, t[SLOTS], 1, "slots");
  check_type(t[SLOTS], kDLInt, 64, "slots");
  CUVS_EXPECTS(t[SLOTS].shape[0] == n && (n <= 1 || t[SLOTS].stride[0] == 1), "slots: a contiguous one for each token");
  a.slots = reinterpret_cast<int64_t*>(t[SLOTS].data);
  return a;
}

kv::attention_args attention_of(int device, tensor* t, float scale, int64_t window)
{
  enum { KEYS, VALUES, QUERIES, PAGES, LENGTHS, FILTER, OUT, LSE, WORKSPACE };
  kv::attention_args a{};
  a.cache   = cache_of(device, t[KEYS], t[VALUES], t[FILTER], a.type);
  a.queries = rows_of(device, t[QUERIES], a.type, a.cache, -1, -1, "queries");
  const int64_t n = t[QUERIES].shape[0];
  a.n_query_heads = query_heads_of(t[QUERIES], a.cache);
  pages_of(device, t[PAGES], a.n_sequences, a.table_width, a.table_stride);
  CUVS_EXPECTS(int64_t(a.n_sequences) == n, "pages: a row for each of the %lld queries, not %u", (long long)n, a.n_sequences);
  a.pages   = reinterpret_cast<const int32_t*>(t[PAGES].data);
  a.lengths = ints_of(device, t[LENGTHS], "lengths", n, "sequence");
  CUVS_EXPECTS(std::isfinite(scale), "scale must be finite");
  CUVS_EXPECTS(window >= 0, "window must not be negative");
  a.scale  = scale;
  a.window = window;
  a.out    = rows_of(device, t[OUT], a.type, a.cache, n, a.n_query_heads, "out");
  check_distinct(t[OUT], "out");
  a.lse = lse_of(device, t[LSE], n, a.n_query_heads);
  if (t[WORKSPACE].given()) {
    check_place(device, t[WORKSPACE], 1, "workspace");
    check_type(t[WORKSPACE], kDLUInt, 8, "workspace");
    CUVS_EXPECTS(t[WORKSPACE].shape[0] <= 1 || t[WORKSPACE].stride[0] == 1, "workspace: must be contiguous");
    CUVS_EXPECTS(reinterpret_cast<uintptr_t>(t[WORKSPACE].data) % 16 == 0, "workspace: must start on a 16-byte boundary");
    a.workspace       = t[WORKSPACE].data;
    a.workspace_bytes = size_t(t[WORKSPACE].shape[0]);
  }
  return a;
}

// With the workspace that the caller gave, or the handle's own for the stream.  False: the stream is being captured, and the call needs one
// to itself.
bool attention_call(resources& res, cudaStream_t stream, kv::attention_args a)
{
  const size_t need = kv::attention_workspace(res, a.type, a.n_sequences, a.n_query_heads, a.cache.n_heads, a.cache.dim,
                                              uint64_t(a.table_width) * a.cache.page.size, a.window);
  std::unique_lock<std::mutex> held;
  if (need > 0 && a.workspace != nullptr) {
    CUVS_EXPECTS(a.workspace_bytes >= need, "workspace: %zu bytes, but %zu are needed", a.workspace_bytes, need);
  } else if (need > 0) {
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    CUDA_TRY(cudaStreamIsCapturing(stream, &capturing));
    if (capturing != cudaStreamCaptureStatusNone) { return false; }
    held = res.stream_workspace(stream, need, &a.workspace);
  }
  kv::attention(res, stream, a);
  return true;
}
constexpr const char* kOwnWorkspace = "a call that is captured needs a workspace of its own";

kv::candidates_args candidates_of(int device, tensor* t, float scale)
{
  enum { KEYS, VALUES, QUERIES, CANDIDATES, FILTER, OUT, LSE };
  kv::candidates_args a{};
  a.cache   = cache_of(device, t[KEYS], t[VALUES], t[FILTER], a.type);
  a.queries = rows_of(device, t[QUERIES], a.type, a.cache, -1, -1, "queries");
  const int64_t n = t[QUERIES].shape[0];
  a.n_query_heads = query_heads_of(t[QUERIES], a.cache);
  a.n_tokens      = uint32_t(n);
  tensor& c       = t[CANDIDATES];
  check_place(device, c, 3, "candidates");
  check_type(c, kDLInt, 64, "candidates");
  CUVS_EXPECTS(c.shape[0] == n && c.shape[1] == int64_t(a.n_query_heads), "candidates: a list for each of %lld tokens and %u heads", (long long)n,
               a.n_query_heads);
  CUVS_EXPECTS(c.shape[2] < (int64_t(1) << 31), "candidates: too many");
  CUVS_EXPECTS((c.shape[2] <= 1 || c.stride[2] == 1) && (c.shape[1] <= 1 || c.stride[1] == c.shape[2]) &&
                 (c.shape[0] <= 1 || c.stride[0] == c.shape[1] * c.shape[2]),
               "candidates: must be contiguous");
  a.n_candidates = uint32_t(c.shape[2]);
  a.candidates   = reinterpret_cast<const int64_t*>(c.data);
  CUVS_EXPECTS(std::isfinite(scale), "scale must be finite");
  a.scale = scale;
  a.out   = rows_of(device, t[OUT], a.type, a.cache, n, a.n_query_heads, "out");
  check_distinct(t[OUT], "out");
  a.lse = lse_of(device, t[LSE], n, a.n_query_heads);
  return a;
}

kv::merge_args merge_of(int device, tensor* t)
{
  enum { PARTS, PARTS_LSE, OUT, LSE };
  kv::merge_args a{};
  CUVS_EXPECTS(t[PARTS].given(), "parts: null tensor");
  a.type = elem_of(t[PARTS], "parts");
  check_rows(device, t[PARTS], 4, a.type, "parts");
  check_place(device, t[PARTS_LSE], 3, "parts_lse");
  check_type(t[PARTS_LSE], kDLFloat, 32, "parts_lse");
  CUVS_EXPECTS(std::equal(t[PARTS].shape, t[PARTS].shape + 3, t[PARTS_LSE].shape), "parts_lse: one for each row of the parts");
  const int64_t n = t[PARTS].shape[1], h = t[PARTS].shape[2];
  CUVS_EXPECTS(t[PARTS].shape[0] < (int64_t(1) << 31) && n * h < (int64_t(1) << 31), "parts: too many rows");
  check_rows(device, t[OUT], 3, a.type, "out");
  CUVS_EXPECTS(std::equal(t[OUT].shape, t[OUT].shape + 3, t[PARTS].shape + 1), "out: the shape of one part");
  check_distinct(t[OUT], "out");
  a.lse       = lse_of(device, t[LSE], n, h);
  a.n_parts   = uint32_t(t[PARTS].shape[0]);
  a.n_tokens  = uint32_t(n);
  a.n_heads   = uint32_t(h);
  a.dim       = uint32_t(t[PARTS].shape[3]);
  a.parts     = t[PARTS].data;
  a.p_part    = t[PARTS].stride[0];
  a.p_row     = t[PARTS].stride[1];
  a.p_head    = t[PARTS].stride[2];
  a.parts_lse = reinterpret_cast<const float*>(t[PARTS_LSE].data);
  a.l_part    = t[PARTS_LSE].stride[0];
  a.l_row     = t[PARTS_LSE].stride[1];
  a.l_head    = t[PARTS_LSE].stride[2];
  a.out       = {t[OUT].data, t[OUT].stride[0], t[OUT].stride[1]};
  return a;
}

void workspace_of(resources& res, tensor* t, int64_t window, size_t* bytes)
{
  enum { KEYS, QUERIES, PAGES };
  CUVS_EXPECTS(bytes != nullptr, "null output pointer");
  kv::elem type;
  tensor values          = t[KEYS];
  const kv::cache_view c = cache_of(res.device, t[KEYS], values, {}, type);
  rows_of(res.device, t[QUERIES], type, c, -1, -1, "queries");
  uint32_t n, width;
  int64_t stride;
  pages_of(res.device, t[PAGES], n, width, stride);
  CUVS_EXPECTS(window >= 0, "window must not be negative");
  *bytes = kv::attention_workspace(res, type, n, query_heads_of(t[QUERIES], c), c.n_heads, c.dim, uint64_t(width) * c.page.size, window);
}

resources& single_device(cuvsResources_t res)
{
  resources* r = res_of(res);
  CUVS_EXPECTS(r->kind == 0, "the handle must be for one device");
  return *r;
}

}  // namespace

extern "C" cuvsError_t cuvsKvCacheAppend(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* values, DLManagedTensor* new_keys,
                                         DLManagedTensor* new_values, DLManagedTensor* pages, DLManagedTensor* positions,
                                         DLManagedTensor* sequences, DLManagedTensor* queries, DLManagedTensor* frequencies, bool interleaved,
                                         DLManagedTensor* slots, DLManagedTensor* rotated)
{
  return translate_exceptions([=] {
    resources& r = single_device(res);
    device_scope on(r.device);
    tensor t[] = {describe(keys, "keys"),           describe(values, "values"),       describe(new_keys, "new_keys"),
                  describe(new_values, "new_values"), describe(pages, "pages"),       describe(positions, "positions"),
                  describe(sequences, "sequences"), describe(queries, "queries"),     describe(frequencies, "frequencies"),
                  describe(slots, "slots"),         describe(rotated, "rotated")};
    kv::append(r, r.stream, append_of(r.device, t, interleaved));
  });
}

extern "C" cuvsError_t cuvsKvCacheAttention(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* values, DLManagedTensor* queries,
                                            DLManagedTensor* pages, DLManagedTensor* lengths, float scale, int64_t window, cuvsFilter filter,
                                            DLManagedTensor* out, DLManagedTensor* lse, DLManagedTensor* workspace)
{
  return translate_exceptions([=] {
    resources& r = single_device(res);
    device_scope on(r.device);
    tensor t[] = {describe(keys, "keys"),       describe(values, "values"), describe(queries, "queries"),
                  describe(pages, "pages"),     describe(lengths, "lengths"), filter_of(filter),
                  describe(out, "out"),         describe(lse, "lse"),       describe(workspace, "workspace")};
    CUVS_EXPECTS(attention_call(r, r.stream, attention_of(r.device, t, scale, window)), kOwnWorkspace);
  });
}

extern "C" cuvsError_t cuvsKvCacheAttentionWorkspace(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* queries,
                                                     DLManagedTensor* pages, int64_t window, size_t* bytes)
{
  return translate_exceptions([=] {
    tensor t[] = {describe(keys, "keys"), describe(queries, "queries"), describe(pages, "pages")};
    workspace_of(single_device(res), t, window, bytes);
  });
}

extern "C" cuvsError_t cuvsKvCacheAttendCandidates(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* values,
                                                   DLManagedTensor* queries, DLManagedTensor* candidates, float scale, cuvsFilter filter,
                                                   DLManagedTensor* out, DLManagedTensor* lse)
{
  return translate_exceptions([=] {
    resources& r = single_device(res);
    device_scope on(r.device);
    tensor t[] = {describe(keys, "keys"), describe(values, "values"), describe(queries, "queries"), describe(candidates, "candidates"),
                  filter_of(filter),      describe(out, "out"),       describe(lse, "lse")};
    kv::attend_candidates(r, r.stream, candidates_of(r.device, t, scale));
  });
}

extern "C" cuvsError_t cuvsKvCacheMergeParts(cuvsResources_t res, DLManagedTensor* parts, DLManagedTensor* parts_lse, DLManagedTensor* out,
                                             DLManagedTensor* lse)
{
  return translate_exceptions([=] {
    resources& r = single_device(res);
    device_scope on(r.device);
    tensor t[] = {describe(parts, "parts"), describe(parts_lse, "parts_lse"), describe(out, "out"), describe(lse, "lse")};
    kv::merge_parts(r, r.stream, merge_of(r.device, t));
  });
}

namespace {

constexpr int kMost = 11;  // tensors of a call
const int n_tensors[]            = {11, 9, 7, 4};
const int n_scalars[]            = {1, 2, 1, 0};
const char* const names[][kMost] = {
  {"keys", "values", "new_keys", "new_values", "pages", "positions", "sequences", "queries", "frequencies", "slots", "rotated"},
  {"keys", "values", "queries", "pages", "lengths", "filter", "out", "lse", "workspace"},
  {"keys", "values", "queries", "candidates", "filter", "out", "lse"},
  {"parts", "parts_lse", "out", "lse"}};

struct call {
  tensor t[kMost];
  bool interleaved = false;
  float scale      = 0.0f;
  int64_t window   = 0;
  call() = default;
  call(int op, const int64_t* words, int64_t n_words)
  {
    CUVS_EXPECTS(op >= 0 && op < 4 && words != nullptr, "unknown call %d", op);
    const int64_t* end = words + n_words;
    for (int i = 0; i < n_tensors[op]; i++) { t[i] = describe(words, end, names[op][i]); }
    CUVS_EXPECTS(end - words == n_scalars[op], "the words do not describe the call");
    if (op == 0) { interleaved = words[0] != 0; }
    if (op == 1) { window = words[0]; }
    if (op == 1 || op == 2) {
      const uint32_t bits = uint32_t(words[op == 1 ? 1 : 0]);
      std::memcpy(&scale, &bits, 4);
    }
  }
  // False: it needs a workspace to itself.  The handle's stream stays what it is: another thread may be in the middle of a search that reads it.
  bool run(cuvsResources_t res, cudaStream_t stream, int op, bool sync)
  {
    resources& r = single_device(res);
    device_scope on(r.device);
    if (sync) {
      cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
      CUDA_TRY(cudaStreamIsCapturing(stream, &capturing));
      CUVS_EXPECTS(capturing == cudaStreamCaptureStatusNone, "a call that is captured cannot wait for its work: pass sync=False");
    }
    switch (op) {
      case 0: kv::append(r, stream, append_of(r.device, t, interleaved)); break;
      case 1:
        if (!attention_call(r, stream, attention_of(r.device, t, scale, window))) { return false; }
        break;
      case 2: kv::attend_candidates(r, stream, candidates_of(r.device, t, scale)); break;
      default: kv::merge_parts(r, stream, merge_of(r.device, t));
    }
    return true;
  }
};

constexpr int kNeedsWorkspace = 2;  // beside the values of cuvsError_t: nothing was done, the call needs a workspace to itself

const tensor_exchange* g_exchange = nullptr;  // set once, when the Python module is imported
const void* g_none                = nullptr;

}  // namespace

extern "C" int cuvsB200KvCacheArrays(cuvsResources_t res, cudaStream_t stream, int op, const int64_t* words, int64_t n_words, bool sync)
{
  int status = CUVS_ERROR;
  const auto raised = translate_exceptions([&] {
    status = call(op, words, n_words).run(res, stream, op, sync) ? CUVS_SUCCESS : kNeedsWorkspace;
    if (sync && status == CUVS_SUCCESS) { CUDA_TRY(cudaStreamSynchronize(stream)); }
  });
  return raised == CUVS_SUCCESS ? status : CUVS_ERROR;
}

extern "C" cuvsError_t cuvsB200SetTensorExchange(const void* table, const void* none)
{
  return translate_exceptions([=] {
    const auto* x = static_cast<const tensor_exchange*>(table);
    CUVS_EXPECTS(x != nullptr && x->major == 1 && x->from_python != nullptr, "no DLPack 1.x table of exchange functions");
    g_exchange = x;
    g_none     = none;
  });
}

extern "C" int cuvsB200KvCacheTensors(cuvsResources_t res, cudaStream_t stream, int op, void* t0, void* t1, void* t2, void* t3, void* t4, void* t5,
                                      void* t6, void* t7, void* t8, void* t9, void* t10, int64_t integer, float scale, bool sync)
{
  int status = CUVS_ERROR;
  const auto raised = translate_exceptions([&] {
    CUVS_EXPECTS(g_exchange != nullptr && op >= 0 && op < 4, "unknown call %d", op);
    void* const objects[kMost] = {t0, t1, t2, t3, t4, t5, t6, t7, t8, t9, t10};
    call c;
    for (int i = 0; i < n_tensors[op]; i++) {
      if (objects[i] == g_none) { continue; }
      DLTensor d{};
      CUVS_EXPECTS(g_exchange->from_python(objects[i], &d) == 0, "%s: cannot be described", names[op][i]);
      c.t[i] = describe(d, names[op][i]);
    }
    c.interleaved = integer != 0;
    c.window      = integer;
    c.scale       = scale;
    status        = c.run(res, stream, op, sync) ? CUVS_SUCCESS : kNeedsWorkspace;
  });
  return raised == CUVS_SUCCESS ? status : CUVS_ERROR;
}

extern "C" cuvsError_t cuvsB200KvCacheWait(cuvsResources_t res, cudaStream_t stream)
{
  return translate_exceptions([=] {
    device_scope on(single_device(res).device);
    CUDA_TRY(cudaStreamSynchronize(stream));
  });
}

extern "C" cuvsError_t cuvsB200KvCacheWorkspaceArrays(cuvsResources_t res, const int64_t* words, int64_t n_words, size_t* bytes)
{
  return translate_exceptions([=] {
    CUVS_EXPECTS(words != nullptr, "null words");
    const int64_t *at = words, *end = words + n_words;
    tensor t[3];
    static const char* const names[] = {"keys", "queries", "pages"};
    for (int i = 0; i < 3; i++) { t[i] = describe(at, end, names[i]); }
    CUVS_EXPECTS(end - at == 1, "the words do not describe the call");
    workspace_of(single_device(res), t, *at, bytes);
  });
}

extern "C" cuvsError_t cuvsB200KvCacheCheck(int device, int op, const int64_t* words, int64_t n_words)
{
  return translate_exceptions([=] {
    call c(op, words, n_words);
    switch (op) {
      case 0: append_of(device, c.t, c.interleaved); break;
      case 1: attention_of(device, c.t, c.scale, c.window); break;
      case 2: candidates_of(device, c.t, c.scale); break;
      default: merge_of(device, c.t);
    }
  });
}

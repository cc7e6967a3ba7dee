// C ABI of the stream operators: argument checks, then the launches of
// fav_conv.cu, fav_scan.cu, fav_norm.cu and fav_int4.cu. Declarations and
// contracts: include/fast_audiovae_cuda.h.
#include <initializer_list>

#include "fav_ops.cuh"

namespace fav {

cudaError_t launch_causal_conv(const fav_conv_args&, const Sequences&, cudaStream_t);
size_t scan_workspace_bytes(const fav_scan_args&, const Sequences&);
cudaError_t launch_selective_scan(const fav_scan_args&, const Sequences&, cudaStream_t);
cudaError_t launch_group_norm(const fav_norm_args&, const Sequences&, cudaStream_t);
cudaError_t launch_project_int4(const fav_int4_args&, cudaStream_t);

namespace {

constexpr long long kMaxRows = 0x7fff0000;
constexpr int kMaxChannels = 1 << 20;

// Rows, channels and sequences that index arithmetic and grids can hold.
int32_t check_rows(int32_t type, int32_t channels, int32_t n, int32_t length, int32_t rows, const int32_t* offsets) {
  if (type < FAV_TYPE_F32 || type > FAV_TYPE_F16) return fail(FAV_UNSUPPORTED, "unsupported element type %d", type);
  if (channels < 1 || channels > kMaxChannels) return fail(FAV_INVALID_ARGUMENT, "channels must be in 1..%d", kMaxChannels);
  if (n < 0 || rows < 0 || rows > kMaxRows) return fail(FAV_INVALID_ARGUMENT, "bad sequence or row count");
  if (!offsets && (length < 1 || (long long)n * length != rows))
    return fail(FAV_INVALID_ARGUMENT, "rows must be n * length with length >= 1 when offsets is NULL");
  return FAV_OK;
}

int32_t check_states(const void* pool, const int32_t* codes, int32_t n, int32_t num_slots) {
  if (!pool != !codes) return fail(FAV_INVALID_ARGUMENT, "a state pool and slot codes go together");
  if (pool && (num_slots < n || num_slots > (1 << 29)))
    return fail(FAV_INVALID_ARGUMENT, "num_slots >= n sequences required");
  return FAV_OK;
}

// A strided array of `rows` rows of `width` elements.
struct View {
  const char* p;
  long long stride, width, rows;  // bytes
};

View view(const void* p, long long stride, long long width, long long rows, int elem) {
  return {static_cast<const char*>(p), stride * elem, width * elem, rows};
}

// Consecutive elements.
View flat(const void* p, long long count, int elem) { return view(p, count, count, 1, elem); }

// Whether two views share a byte. Views of one row stride may interleave (two
// column ranges of one buffer), and a single row with the rows of a view; any other
// crossing counts as an overlap.
bool overlap(const View& a, const View& b) {
  if (!a.p || !b.p || a.rows == 0 || b.rows == 0) return false;
  const char *a_end = a.p + (a.rows - 1) * a.stride + a.width, *b_end = b.p + (b.rows - 1) * b.stride + b.width;
  if (a_end <= b.p || b_end <= a.p) return false;
  if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) return true;
  const long long stride = a.rows > 1 ? a.stride : b.stride;
  if ((a.rows == 1 && b.rows == 1) || stride <= 0) return true;
  const long long at = ((b.p - a.p) % stride + stride) % stride;
  return at < a.width || at + b.width > stride;
}

// Every array that a call writes is apart from the others and from what it reads.
int32_t check_apart(std::initializer_list<View> written, std::initializer_list<View> read) {
  for (const View* w = written.begin(); w != written.end(); ++w) {
    for (const View& r : read)
      if (overlap(*w, r)) return fail(FAV_OVERLAP, "outputs, state pool and workspace must not overlap the inputs");
    for (const View* v = written.begin(); v != w; ++v)
      if (overlap(*w, *v)) return fail(FAV_OVERLAP, "outputs, state pool and workspace must not overlap");
  }
  return FAV_OK;
}

int32_t check_stride(const char* name, int64_t stride, int32_t width, int32_t rows) {
  // Rows may not overlap, and byte offsets must stay far inside 64 bits.
  if (rows > 1 && (stride < width || stride > (1LL << 30) || rows * stride > (1LL << 56)))
    return fail(FAV_INVALID_ARGUMENT, "%s row stride %lld outside [%d, 2^30], or array too large", name,
                (long long)stride, width);
  return FAV_OK;
}

// A load from an address that is no multiple of its size would fault on the device.
int32_t check_aligned(int bytes, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % bytes)
      return fail(FAV_INVALID_ARGUMENT, "array at %p is not aligned to its elements of %d bytes", p, bytes);
  return FAV_OK;
}

int32_t launched(cudaError_t e, const char* what) {
  if (e == cudaErrorInvalidValue) return fail(FAV_SIZE_OVERFLOW, "%s too large", what);
  return e == cudaSuccess ? FAV_OK : cuda_fail(e, what);
}

Sequences sequences(const int32_t* offsets, const int32_t* codes, int n, int length, int rows, int num_slots,
                    uint32_t* status) {
  return {offsets, codes, n, length, rows, num_slots, status};
}

int32_t check_scan_sizes(const fav_scan_args& c) {
  int32_t st = check_rows(c.type, c.channels, c.n, c.length, c.rows, c.offsets);
  if (st != FAV_OK) return st;
  if (c.states < 1 || c.states > 128) return fail(FAV_INVALID_ARGUMENT, "states must be in 1..128");
  if (c.groups < 1 || c.channels % c.groups) return fail(FAV_INVALID_ARGUMENT, "groups must divide channels");
  return FAV_OK;
}

}  // namespace
}  // namespace fav

using namespace fav;

extern "C" {

int32_t fav_causal_conv(const fav_conv_args* args, void* cuda_stream) {
  clear_error();
  if (!args) return fail(FAV_INVALID_ARGUMENT, "args is NULL");
  const fav_conv_args& c = *args;
  int32_t st = check_rows(c.type, c.channels, c.n, c.length, c.rows, c.offsets);
  if (st != FAV_OK) return st;
  if (c.taps < 2 || c.taps > 8) return fail(FAV_INVALID_ARGUMENT, "taps must be in 2..8");
  if (c.activation != FAV_ACTIVATION_NONE && c.activation != FAV_ACTIVATION_SILU)
    return fail(FAV_UNSUPPORTED, "unsupported activation %d", c.activation);
  if ((st = check_states(c.state_pool, c.slot_codes, c.n, c.num_slots)) != FAV_OK) return st;
  if (c.n == 0) return FAV_OK;
  if (!c.weight || (c.rows && (!c.x || !c.y))) return fail(FAV_INVALID_ARGUMENT, "NULL x, y or weight");
  if ((st = check_stride("x", c.x_stride, c.channels, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("y", c.y_stride, c.channels, c.rows)) != FAV_OK) return st;
  const int e = elem_bytes(c.type);
  if ((st = check_aligned(e, {c.x, c.y, c.state_pool})) != FAV_OK ||
      (st = check_aligned(4, {c.weight, c.bias, c.slot_codes, c.offsets, c.status})) != FAV_OK)
    return st;
  const long long state = 2LL * (c.taps - 1) * c.channels;
  st = check_apart({view(c.y, c.y_stride, c.channels, c.rows, e), view(c.state_pool, state, state, c.num_slots, e),
                    flat(c.status, 1, 4)},
                   {view(c.x, c.x_stride, c.channels, c.rows, e), flat(c.weight, (long long)c.channels * c.taps, 4),
                    flat(c.bias, c.channels, 4), flat(c.slot_codes, c.n, 4), flat(c.offsets, c.n + 1LL, 4)});
  if (st != FAV_OK) return st;
  return launched(launch_causal_conv(c, sequences(c.offsets, c.slot_codes, c.n, c.length, c.rows, c.num_slots, c.status),
                                     static_cast<cudaStream_t>(cuda_stream)),
                  "convolution");
}

size_t fav_selective_scan_workspace_bytes(const fav_scan_args* args) {
  if (!args || check_scan_sizes(*args) != FAV_OK || args->n == 0) return 0;
  return scan_workspace_bytes(*args, sequences(args->offsets, nullptr, args->n, args->length, args->rows, 0, nullptr));
}

int32_t fav_selective_scan(const fav_scan_args* args, void* cuda_stream) {
  clear_error();
  if (!args) return fail(FAV_INVALID_ARGUMENT, "args is NULL");
  const fav_scan_args& c = *args;
  int32_t st = check_scan_sizes(c);
  if (st != FAV_OK) return st;
  if ((st = check_states(c.state_pool, c.slot_codes, c.n, c.num_slots)) != FAV_OK) return st;
  if (c.n == 0) return FAV_OK;
  if (!c.a || (c.rows && (!c.x || !c.dt || !c.b || !c.c || !c.y)))
    return fail(FAV_INVALID_ARGUMENT, "NULL x, dt, a, b, c or y");
  if ((st = check_stride("x", c.x_stride, c.channels, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("dt", c.dt_stride, c.channels, c.rows)) != FAV_OK) return st;
  if (c.z && (st = check_stride("z", c.z_stride, c.channels, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("y", c.y_stride, c.channels, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("b", c.b_stride, 1, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("c", c.c_stride, 1, c.rows)) != FAV_OK) return st;
  if (c.groups > 1 && (c.b_group_stride < c.states || c.c_group_stride < c.states || c.b_group_stride > (1LL << 30) ||
                       c.c_group_stride > (1LL << 30)))
    return fail(FAV_INVALID_ARGUMENT, "b and c group strides must be in [states, 2^30]");
  const Sequences q = sequences(c.offsets, c.slot_codes, c.n, c.length, c.rows, c.num_slots, c.status);
  const size_t need = scan_workspace_bytes(c, q);
  if (need && (!c.workspace || c.workspace_bytes < need))
    return fail(FAV_INVALID_ARGUMENT, "workspace too small: %zu < %zu bytes", c.workspace ? c.workspace_bytes : 0, need);
  const int e = elem_bytes(c.type);
  if ((st = check_aligned(e, {c.x, c.dt, c.z, c.b, c.c, c.y})) != FAV_OK ||
      (st = check_aligned(4, {c.a, c.d, c.dt_bias, c.state_pool, c.slot_codes, c.offsets, c.status, c.workspace})) != FAV_OK)
    return st;
  const long long state = 2LL * c.states * c.channels;
  const long long b_width = (c.groups - 1) * (c.groups > 1 ? c.b_group_stride : 0) + c.states;
  const long long c_width = (c.groups - 1) * (c.groups > 1 ? c.c_group_stride : 0) + c.states;
  st = check_apart({view(c.y, c.y_stride, c.channels, c.rows, e), view(c.state_pool, state, state, c.num_slots, 4),
                    flat(need ? c.workspace : nullptr, (long long)need, 1), flat(c.status, 1, 4)},
                   {view(c.x, c.x_stride, c.channels, c.rows, e), view(c.dt, c.dt_stride, c.channels, c.rows, e),
                    view(c.z, c.z_stride, c.channels, c.rows, e), view(c.b, c.b_stride, b_width, c.rows, e),
                    view(c.c, c.c_stride, c_width, c.rows, e), flat(c.a, (long long)c.states * c.channels, 4),
                    flat(c.d, c.channels, 4), flat(c.dt_bias, c.channels, 4), flat(c.slot_codes, c.n, 4),
                    flat(c.offsets, c.n + 1LL, 4)});
  if (st != FAV_OK) return st;
  return launched(launch_selective_scan(c, q, static_cast<cudaStream_t>(cuda_stream)), "scan");
}

int32_t fav_group_norm(const fav_norm_args* args, void* cuda_stream) {
  clear_error();
  if (!args) return fail(FAV_INVALID_ARGUMENT, "args is NULL");
  const fav_norm_args& c = *args;
  int32_t st = check_rows(c.type, c.channels, c.n, c.length, c.rows, c.offsets);
  if (st != FAV_OK) return st;
  if (c.groups < 1 || c.channels % c.groups) return fail(FAV_INVALID_ARGUMENT, "groups must divide channels");
  if (c.activation < FAV_ACTIVATION_NONE || c.activation > FAV_ACTIVATION_SNAKE)
    return fail(FAV_UNSUPPORTED, "unsupported activation %d", c.activation);
  if (c.activation == FAV_ACTIVATION_SNAKE && (!c.alpha || !c.reciprocal))
    return fail(FAV_INVALID_ARGUMENT, "Snake needs alpha and reciprocal");
  if (!(c.eps >= 0.f)) return fail(FAV_INVALID_ARGUMENT, "eps must not be negative");
  if (c.n == 0) return FAV_OK;
  if (c.rows && (!c.x || !c.y)) return fail(FAV_INVALID_ARGUMENT, "NULL x or y");
  if ((st = check_stride("x", c.x_stride, c.channels, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("y", c.y_stride, c.channels, c.rows)) != FAV_OK) return st;
  const int e = elem_bytes(c.type);
  if ((st = check_aligned(e, {c.x, c.y})) != FAV_OK ||
      (st = check_aligned(4, {c.weight, c.bias, c.alpha, c.reciprocal, c.offsets, c.status})) != FAV_OK)
    return st;
  st = check_apart({view(c.y, c.y_stride, c.channels, c.rows, e), flat(c.status, 1, 4)},
                   {view(c.x, c.x_stride, c.channels, c.rows, e), flat(c.weight, c.channels, 4), flat(c.bias, c.channels, 4),
                    flat(c.alpha, c.channels, 4), flat(c.reciprocal, c.channels, 4), flat(c.offsets, c.n + 1LL, 4)});
  if (st != FAV_OK) return st;
  return launched(launch_group_norm(c, sequences(c.offsets, nullptr, c.n, c.length, c.rows, 0, c.status),
                                    static_cast<cudaStream_t>(cuda_stream)),
                  "group norm");
}

int32_t fav_project_int4(const fav_int4_args* args, void* cuda_stream) {
  clear_error();
  if (!args) return fail(FAV_INVALID_ARGUMENT, "args is NULL");
  const fav_int4_args& c = *args;
  int32_t st = check_rows(c.type, c.depth, c.rows, 1, c.rows, nullptr);
  if (st != FAV_OK) return st;
  if (c.out < 1 || c.out > kMaxChannels) return fail(FAV_INVALID_ARGUMENT, "out must be in 1..%d", kMaxChannels);
  if (c.depth % 32 || c.group < 32 || c.group % 32)
    return fail(FAV_INVALID_ARGUMENT, "depth and group must be multiples of 32");
  if (c.rows == 0) return FAV_OK;
  if (!c.x || !c.y || !c.weight || !c.scales) return fail(FAV_INVALID_ARGUMENT, "NULL x, y, weight or scales");
  if ((st = check_stride("x", c.x_stride, c.depth, c.rows)) != FAV_OK) return st;
  if ((st = check_stride("y", c.y_stride, c.out, c.rows)) != FAV_OK) return st;
  if (reinterpret_cast<uintptr_t>(c.weight) % 16) return fail(FAV_INVALID_ARGUMENT, "weight must be 16-byte aligned");
  const int e = elem_bytes(c.type);
  if ((st = check_aligned(e, {c.x, c.y})) != FAV_OK || (st = check_aligned(4, {c.scales, c.bias})) != FAV_OK) return st;
  const long long groups = ((long long)c.depth + c.group - 1) / c.group;
  st = check_apart({view(c.y, c.y_stride, c.out, c.rows, e)},
                   {view(c.x, c.x_stride, c.depth, c.rows, e), flat(c.weight, (long long)c.out * c.depth / 2, 1),
                    flat(c.scales, c.out * groups, 4), flat(c.bias, c.out, 4)});
  if (st != FAV_OK) return st;
  return launched(launch_project_int4(c, static_cast<cudaStream_t>(cuda_stream)), "projection");
}

}  // extern "C"

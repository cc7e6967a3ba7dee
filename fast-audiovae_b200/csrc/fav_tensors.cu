// The stream operators on Python tensor objects: reads each tensor through the
// producer's DLPack C exchange functions, checks it, and calls the C ABI on the
// current stream. Reading a tensor takes some tens of nanoseconds here and most of
// a microsecond from Python, where a step's call would cost more time than its
// kernel. Anything out of the ordinary is left to the caller (kAsk), which
// checks again and says what is wrong.
#include "../../include/fast_audiovae_cuda.h"
#include "fav_internal.h"

#include <dlfcn.h>

#include <algorithm>
#include <initializer_list>

namespace fav {
namespace {

constexpr int32_t kAsk = -1;
constexpr size_t kMinWorkspace = 256;  // what a scan asks for at least: above every status

// DLPack 1.x: the structures of its C interface that are used here.
struct DlTensor {
  void* data;
  int32_t device_type, device_id;
  int32_t ndim;
  uint8_t code, bits;
  uint16_t lanes;
  int64_t* shape;
  int64_t* strides;
  uint64_t byte_offset;
};
struct DlExchange {
  uint32_t major, minor;
  void* previous;
  void *allocate, *export_managed, *import_managed;
  int (*view)(void* object, DlTensor* out);
  int (*current_stream)(int32_t device_type, int32_t device_id, void** out);
};
constexpr int32_t kDlCuda = 2;
constexpr uint8_t kDlInt = 0, kDlUInt = 1, kDlFloat = 2, kDlBfloat = 4;

const DlExchange* g_exchange = nullptr;
void* g_none = nullptr;

// The interpreter's lock, which a launch gives back meanwhile: it waits while the
// device's queue is full, and the program's other threads need not. The functions
// are the running interpreter's own.
void* (*g_save)() = nullptr;
void (*g_restore)(void*) = nullptr;
int (*g_locked)() = nullptr;

struct Unlocked {
  void* thread = g_save && g_restore && g_locked && g_locked() ? g_save() : nullptr;
  ~Unlocked() {
    if (thread) g_restore(thread);
  }
};

struct Tensor {
  DlTensor t;
  bool read(void* object) {  // false of None too, which the exchange must not be given
    return object != g_none && g_exchange->view(object, &t) == 0 && t.device_type == kDlCuda && t.strides &&
           t.lanes == 1 && !may_be_negated();
  }
  // The exchange does not tell whether a tensor stands for the negative of its memory. Such
  // a one is the imaginary part of conjugated numbers, every second value of a row: with
  // adjacent channels it has one channel, and lies apart or is a single value. The caller
  // looks closer.
  bool may_be_negated() const {
    if (t.ndim == 0 || t.shape[t.ndim - 1] != 1 || (t.code != kDlFloat && t.code != kDlBfloat)) return false;
    int64_t count = 1;
    for (int i = 0; i < t.ndim; ++i) count *= t.shape[i];
    return count == 1 || !contiguous();
  }
  const char* data() const { return static_cast<const char*>(t.data) + t.byte_offset; }
  bool is(uint8_t code, uint8_t bits) const { return t.code == code && t.bits == bits; }
  int type() const {
    return is(kDlFloat, 32) ? FAV_TYPE_F32 : is(kDlBfloat, 16) ? FAV_TYPE_BF16 : is(kDlFloat, 16) ? FAV_TYPE_F16 : -1;
  }
  bool contiguous() const {
    int64_t expect = 1;
    for (int i = t.ndim - 1; i >= 0; --i) {
      if (t.shape[i] != 1 && t.strides[i] != expect) return false;
      expect *= t.shape[i];
    }
    return true;
  }
  bool has_shape(std::initializer_list<int64_t> shape) const {
    if ((size_t)t.ndim != shape.size()) return false;
    int i = 0;
    for (int64_t s : shape)
      if (t.shape[i++] != s) return false;
    return true;
  }
};

// Rows [rows, channels] or [n, length, channels] with adjacent channels and one
// stride between rows; false leaves the case to the caller.
struct Rows {
  int64_t n, length, rows, channels, stride;
};
bool rows_of(const DlTensor& t, Rows* r) {
  if (t.ndim != 2 && t.ndim != 3) return false;
  r->channels = t.shape[t.ndim - 1];
  if (r->channels < 1 || (t.strides[t.ndim - 1] != 1 && r->channels != 1)) return false;
  r->n = t.shape[0];
  r->length = t.ndim == 3 ? t.shape[1] : 1;
  r->rows = r->n * r->length;
  if (r->n < 1 || r->length < 1 || r->rows > 0x7fffffff || r->channels > 0x7fffffff) return false;
  if (t.ndim == 2 || r->length == 1)
    r->stride = t.strides[0];
  else if (r->n == 1 || t.strides[0] == r->length * t.strides[1])
    r->stride = t.strides[1];
  else
    return false;
  if (r->rows == 1) r->stride = r->channels;
  return true;
}
bool like(const Tensor& a, const Tensor& x) {
  if (a.t.ndim != x.t.ndim || a.t.code != x.t.code || a.t.bits != x.t.bits || a.t.device_id != x.t.device_id) return false;
  for (int i = 0; i < x.t.ndim; ++i)
    if (a.t.shape[i] != x.t.shape[i]) return false;
  return true;
}
// A tensor shaped like x: its address and row stride.
template <typename P>
bool same_rows(void* object, const Tensor& x, P** address, int64_t* stride) {
  Tensor a;
  Rows r;
  if (!a.read(object) || !like(a, x) || !rows_of(a.t, &r)) return false;
  *address = (P*)a.data();
  *stride = r.stride;
  return true;
}
// A contiguous fp32 array of this shape; None gives a null address.
bool coefficients(void* object, const Tensor& x, std::initializer_list<int64_t> shape, const float** address) {
  *address = nullptr;
  if (object == g_none) return true;
  Tensor a;
  if (!a.read(object) || !a.is(kDlFloat, 32) || a.t.device_id != x.t.device_id || !a.has_shape(shape) || !a.contiguous())
    return false;
  *address = reinterpret_cast<const float*>(a.data());
  return true;
}
template <typename P>
bool indices(void* object, const Tensor& x, int64_t count, P** address) {
  *address = nullptr;
  if (object == g_none) return true;
  Tensor a;
  if (!a.read(object) || !a.is(kDlInt, 32) || a.t.device_id != x.t.device_id || !a.has_shape({count}) || !a.contiguous())
    return false;
  *address = (P*)a.data();
  return true;
}
// A state pool [slots, 2, rows, channels] with its codes, or neither.
template <typename P>
bool states(void* pool, void* codes, const Tensor& x, uint8_t code, uint8_t bits, int64_t n, int64_t rows,
            int64_t channels, P** address, const int32_t** codes_at, int32_t* slots) {
  *address = nullptr;
  *codes_at = nullptr;
  *slots = 0;
  if ((pool == g_none) != (codes == g_none)) return false;
  if (pool == g_none) return true;
  Tensor a;
  if (!a.read(pool) || !a.is(code, bits) || a.t.device_id != x.t.device_id || a.t.ndim != 4 || a.t.shape[0] < n ||
      a.t.shape[0] > 0x7fffffff || !a.has_shape({a.t.shape[0], 2, rows, channels}) || !a.contiguous())
    return false;
  *address = (P*)a.data();
  *slots = (int32_t)a.t.shape[0];
  return indices(codes, x, n, codes_at) && *codes_at;
}

// An input or output map [..., groups, states] over x's rows.
bool map_of(const Tensor& m, const Tensor& x, const Rows& r, int64_t states, const void** address, int64_t* stride,
            int64_t* group_stride) {
  const int lead = x.t.ndim - 1;
  if (m.t.ndim != lead + 2 || m.t.code != x.t.code || m.t.bits != x.t.bits || m.t.device_id != x.t.device_id) return false;
  for (int i = 0; i < lead; ++i)
    if (m.t.shape[i] != x.t.shape[i]) return false;
  const int64_t groups = m.t.shape[lead];
  if (groups < 1 || r.channels % groups || m.t.shape[lead + 1] != states || (m.t.strides[lead + 1] != 1 && states != 1))
    return false;
  if (lead == 1 || r.length == 1)
    *stride = m.t.strides[0];
  else if (r.n == 1 || m.t.strides[0] == r.length * m.t.strides[1])
    *stride = m.t.strides[1];
  else
    return false;
  if (r.rows == 1) *stride = groups * states;
  *group_stride = groups > 1 ? m.t.strides[lead] : 0;
  *address = m.data();
  return true;
}

// Sequences of x: packed by `offsets`, or of its shape.
bool sequences_of(void* offsets, const Tensor& x, const Rows& r, const int32_t** address, int32_t* n, int32_t* length) {
  *address = nullptr;
  *n = (int32_t)r.n;
  *length = (int32_t)r.length;
  if (offsets == g_none) return true;
  Tensor o;
  if (x.t.ndim != 2 || !o.read(offsets) || o.t.ndim != 1 || o.t.shape[0] < 2 || o.t.shape[0] > 0x7fffffff ||
      !indices(offsets, x, o.t.shape[0], address))
    return false;
  *n = (int32_t)o.t.shape[0] - 1;
  *length = 0;
  return true;
}

// The current stream of x's device, which must be the current device.
bool stream_of(const Tensor& x, void** stream) {
  int device = -1;
  return cudaGetDevice(&device) == cudaSuccess && device == x.t.device_id &&
         g_exchange->current_stream(kDlCuda, x.t.device_id, stream) == 0;
}

}  // namespace
}  // namespace fav

using namespace fav;

extern "C" {

int32_t fav_bind_tensors(const void* exchange, void* none) {
  clear_error();
  const DlExchange* e = static_cast<const DlExchange*>(exchange);
  if (!e || !none) return fail(FAV_INVALID_ARGUMENT, "exchange and none must be non-null");
  if (e->major != 1 || !e->view || !e->current_stream) return fail(FAV_UNSUPPORTED, "DLPack 1.x exchange required");
  g_exchange = e;
  g_none = none;
  g_save = reinterpret_cast<void* (*)()>(dlsym(RTLD_DEFAULT, "PyEval_SaveThread"));
  g_restore = reinterpret_cast<void (*)(void*)>(dlsym(RTLD_DEFAULT, "PyEval_RestoreThread"));
  g_locked = reinterpret_cast<int (*)()>(dlsym(RTLD_DEFAULT, "PyGILState_Check"));
  return FAV_OK;
}

int32_t fav_causal_conv_tensors(void* x, void* weight, void* bias, void* offsets, void* state, void* codes, void* status,
                                void* y, int32_t activation) {
  if (!g_exchange) return kAsk;
  Tensor xt, wt;
  Rows r;
  fav_conv_args a{};
  if (!xt.read(x) || (a.type = xt.type()) < 0 || !rows_of(xt.t, &r)) return kAsk;
  if (!wt.read(weight) || wt.t.ndim != 2 || wt.t.shape[1] < 2 || wt.t.shape[1] > 8) return kAsk;
  const int64_t taps = wt.t.shape[1];
  if (!sequences_of(offsets, xt, r, &a.offsets, &a.n, &a.length)) return kAsk;
  void* stream = nullptr;
  if (!coefficients(weight, xt, {r.channels, taps}, &a.weight) || !coefficients(bias, xt, {r.channels}, &a.bias) ||
      !states(state, codes, xt, xt.t.code, xt.t.bits, a.n, taps - 1, r.channels, &a.state_pool, &a.slot_codes, &a.num_slots) ||
      !indices(status, xt, 1, &a.status) || !same_rows(y, xt, &a.y, &a.y_stride) || !stream_of(xt, &stream))
    return kAsk;
  a.x = xt.data();
  a.x_stride = r.stride;
  a.channels = (int32_t)r.channels;
  a.taps = (int32_t)taps;
  a.activation = activation;
  a.rows = (int32_t)r.rows;
  Unlocked meanwhile;
  return fav_causal_conv(&a, stream);
}

int64_t fav_selective_scan_tensors(void* x, void* dt, void* a_, void* b, void* c, void* d, void* z, void* dt_bias,
                                   void* offsets, void* state, void* codes, void* status, void* workspace, void* y,
                                   int32_t softplus) {
  if (!g_exchange) return kAsk;
  Tensor xt, at, bt, ct;
  Rows r;
  fav_scan_args a{};
  if (!xt.read(x) || (a.type = xt.type()) < 0 || !rows_of(xt.t, &r)) return kAsk;
  if (!at.read(a_) || at.t.ndim != 2 || at.t.shape[0] < 1 || at.t.shape[0] > 128) return kAsk;
  if (!bt.read(b) || !ct.read(c) || !map_of(bt, xt, r, at.t.shape[0], &a.b, &a.b_stride, &a.b_group_stride) ||
      !map_of(ct, xt, r, at.t.shape[0], &a.c, &a.c_stride, &a.c_group_stride) ||
      bt.t.shape[bt.t.ndim - 2] != ct.t.shape[ct.t.ndim - 2])
    return kAsk;
  const int64_t states_ = at.t.shape[0], groups = bt.t.shape[bt.t.ndim - 2];
  void* stream = nullptr;
  if (!sequences_of(offsets, xt, r, &a.offsets, &a.n, &a.length) ||
      !coefficients(a_, xt, {states_, r.channels}, &a.a) || !coefficients(d, xt, {r.channels}, &a.d) ||
      !coefficients(dt_bias, xt, {r.channels}, &a.dt_bias) || !same_rows(dt, xt, &a.dt, &a.dt_stride) ||
      (z != g_none && !same_rows(z, xt, &a.z, &a.z_stride)) ||
      !states(state, codes, xt, kDlFloat, 32, a.n, states_, r.channels, &a.state_pool, &a.slot_codes, &a.num_slots) ||
      !indices(status, xt, 1, &a.status) || !same_rows(y, xt, &a.y, &a.y_stride) || !stream_of(xt, &stream))
    return kAsk;
  a.x = xt.data();
  a.x_stride = r.stride;
  a.channels = (int32_t)r.channels;
  a.states = (int32_t)states_;
  a.groups = (int32_t)groups;
  a.softplus = softplus;
  a.rows = (int32_t)r.rows;
  if (a.length != 1) {
    const size_t need = fav_selective_scan_workspace_bytes(&a);
    if (need) {
      if (workspace == g_none) return (int64_t)std::max(need, kMinWorkspace);
      Tensor w;
      if (!w.read(workspace) || w.t.device_id != xt.t.device_id || w.t.ndim != 1 || !w.is(kDlUInt, 8) || !w.contiguous())
        return kAsk;
      a.workspace = (void*)w.data();
      a.workspace_bytes = (size_t)w.t.shape[0];
    }
  }
  Unlocked meanwhile;
  return fav_selective_scan(&a, stream);
}

int32_t fav_group_norm_tensors(void* x, void* weight, void* bias, void* alpha, void* reciprocal, void* offsets,
                               void* status, void* y, int32_t groups, float eps, int32_t activation) {
  if (!g_exchange) return kAsk;
  Tensor xt;
  Rows r;
  fav_norm_args a{};
  void* stream = nullptr;
  if (!xt.read(x) || (a.type = xt.type()) < 0 || !rows_of(xt.t, &r) || groups < 1 || r.channels % groups ||
      (activation == FAV_ACTIVATION_SNAKE) != (alpha != g_none) || (alpha != g_none) != (reciprocal != g_none) ||
      !coefficients(weight, xt, {r.channels}, &a.weight) ||
      !coefficients(bias, xt, {r.channels}, &a.bias) || !coefficients(alpha, xt, {r.channels}, &a.alpha) ||
      !coefficients(reciprocal, xt, {r.channels}, &a.reciprocal) ||
      !sequences_of(offsets, xt, r, &a.offsets, &a.n, &a.length) || !indices(status, xt, 1, &a.status) ||
      !same_rows(y, xt, &a.y, &a.y_stride) || !stream_of(xt, &stream))
    return kAsk;
  a.x = xt.data();
  a.x_stride = r.stride;
  a.eps = eps;
  a.channels = (int32_t)r.channels;
  a.groups = groups;
  a.activation = activation;
  a.rows = (int32_t)r.rows;
  Unlocked meanwhile;
  return fav_group_norm(&a, stream);
}

int32_t fav_project_int4_tensors(void* x, void* weight, void* scales, void* bias, void* y, int32_t group) {
  if (!g_exchange) return kAsk;
  Tensor xt, wt, yt;
  Rows r, o;
  fav_int4_args a{};
  void* stream = nullptr;
  if (!xt.read(x) || (a.type = xt.type()) < 0 || xt.t.ndim != 2 || !rows_of(xt.t, &r) || group < 32 || group % 32 ||
      r.channels % 32 || !wt.read(weight) || !wt.is(kDlUInt, 8) || wt.t.device_id != xt.t.device_id || wt.t.ndim != 2 ||
      wt.t.shape[0] < 1 || wt.t.shape[0] > 0x7fffffff || wt.t.shape[1] != r.channels / 2 || !wt.contiguous())
    return kAsk;
  const int64_t out = wt.t.shape[0];
  if (scales == g_none || !coefficients(scales, xt, {out, (r.channels + group - 1) / group}, &a.scales) ||
      !coefficients(bias, xt, {out}, &a.bias) || !yt.read(y) || yt.t.code != xt.t.code || yt.t.bits != xt.t.bits ||
      yt.t.device_id != xt.t.device_id || !yt.has_shape({r.rows, out}) || !rows_of(yt.t, &o) || !stream_of(xt, &stream))
    return kAsk;
  a.x = xt.data();
  a.x_stride = r.stride;
  a.y = (void*)yt.data();
  a.y_stride = o.stride;
  a.weight = reinterpret_cast<const uint8_t*>(wt.data());
  a.rows = (int32_t)r.rows;
  a.depth = (int32_t)r.channels;
  a.out = (int32_t)out;
  a.group = group;
  Unlocked meanwhile;
  return fav_project_int4(&a, stream);
}

}  // extern "C"

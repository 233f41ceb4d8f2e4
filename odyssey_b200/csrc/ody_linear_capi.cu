// ody_linear_capi.cu -- C entry points of the quantised linear layer
// (include/odyssey_mp.h): argument checks, staging for host callers, and the
// launches of ody_linear.cu.
#include <exception>

#include "ody_host.h"
#include "ody_linear.h"
#include "ody_linear_gemm.h"
#include "ody_linear_rows.h"

using namespace ody;

namespace {

constexpr int64_t kMaxDim = INT32_MAX - 1024;  // of rows, features and (with padding) row pitches

// no C++ exception leaves a C entry point
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return fail(ODY_ERR_STATE, std::string("host error: ") + e.what());
  }
}

int check_shape(int64_t rows, int64_t out, int64_t in) {
  if (rows <= 0 || out <= 0 || in <= 0) return fail(ODY_ERR_SHAPE, "linear: rows and features must be positive");
  if (rows > kMaxDim || out > kMaxDim || in > kMaxDim) return fail(ODY_ERR_SHAPE, "linear: a dimension is too large");
  return ODY_OK;
}

int check_pitch(int64_t ld, int64_t cols, const char* what) {
  if (ld < cols || ld > ((int64_t)1 << 38))
    return fail(ODY_ERR_SHAPE, std::string("the row pitch of ") + what + " is smaller than its columns, or too large");
  return ODY_OK;
}

bool is_w4(int kind) {
  return kind == ODY_Q_MXFP4 || kind == ODY_Q_NVFP4 || kind == ODY_Q_NVFP4_TENSOR || kind == ODY_Q_MXFP4_OCP;
}

// what both forms of a product check, and its arguments for the launcher
int product(LinearArgs& a, int op, int32_t kind, int64_t rows, int64_t out, int64_t in, const void* act, int32_t adt,
            int64_t lda, const void* q, const void* scales, void* c, int32_t cdt, int64_t ldc) {
  if (op == LIN_WGRAD ? (kind != ODY_A8_E4M3 && kind != ODY_A8_E5M2) : !is_w4(kind))
    return fail(ODY_ERR_ARG, op == LIN_WGRAD ? "unknown 8-bit activation format " + std::to_string(kind)
                                             : "the weight must be one of the 4-bit kinds, not " + std::to_string(kind));
  if (check_dtype(adt) || check_dtype(cdt)) return ODY_ERR_DTYPE;
  if (int rc = check_shape(rows, out, in)) return rc;
  if (int rc = check_pitch(lda, op == LIN_FORWARD ? in : out, op == LIN_FORWARD ? "x" : "dy")) return rc;
  if (int rc = check_pitch(ldc, op == LIN_FORWARD ? out : in, op == LIN_FORWARD ? "y" : (op == LIN_DGRAD ? "dx" : "dw")))
    return rc;
  if (!act || !q || !c || (op == LIN_WGRAD && !scales)) return fail(ODY_ERR_ARG, "null pointer");
  a = LinearArgs{};
  a.op = op;
  a.rows = rows, a.out = out, a.in = in;
  a.a = act, a.a_dtype = adt, a.lda = lda;
  a.kind = kind;
  a.q = (const uint8_t*)q, a.scales = (const uint8_t*)scales;
  a.o.c = c, a.o.dtype = cdt, a.o.ld = ldc;
  a.o.alpha = 1.0f;
  return ODY_OK;
}

int aligned_to(const void* p, int dtype, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % dtype_size(dtype))
    return fail(ODY_ERR_ARG, std::string(what) + " is not aligned to its element type");
  return ODY_OK;
}

// A buffer as its rows: `n` of `bytes`, `pitch` bytes apart.
struct Span {
  const void* p;
  int64_t n, bytes, pitch;
};
Span flat(const void* p, int64_t bytes) { return {p, 1, bytes, bytes}; }

// Whether two buffers share a byte.  Rows may interleave: at one pitch
// (columns of one wide buffer) their places in it tell; else, where the
// extents meet, each row of the buffer with fewer is compared with the first
// row of the other that ends behind its begin.
bool meet(const Span& u, const Span& v) {
  if (!u.p || !v.p) return false;
  using Wide = __int128;  // a pitch times a number of rows may pass 64 bits
  const Span &x = u.n <= v.n ? u : v, &y = u.n <= v.n ? v : u;
  const Wide a = (Wide)(uintptr_t)x.p, b = (Wide)(uintptr_t)y.p;
  const Wide a_end = a + (Wide)(x.n - 1) * x.pitch + x.bytes, b_end = b + (Wide)(y.n - 1) * y.pitch + y.bytes;
  if (a_end <= b || b_end <= a) return false;
  if (x.pitch == y.pitch) {
    const Wide d = b >= a ? (b - a) % x.pitch : x.pitch - 1 - (a - b - 1) % x.pitch;  // y's place in x's pitch
    if (d >= x.bytes && d + y.bytes <= x.pitch) return false;
  }
  for (int64_t i = 0; i < x.n; i++) {
    const Wide s = a + (Wide)i * x.pitch, e = s + x.bytes;
    const Wide j = s - b < y.bytes ? 0 : (s - b - y.bytes) / y.pitch + 1;
    if (j < y.n && b + j * y.pitch < e) return true;
  }
  return false;
}

constexpr const char* kOverlap = "the output must not be or overlap an operand";

// the rows of a product's buffers
struct Spans {
  Span a, c, q, scales;
  explicit Spans(const LinearArgs& l) {
    const int64_t es = dtype_size(l.a_dtype), cs = dtype_size(l.o.dtype), groups = (l.in + kA8Group - 1) / kA8Group;
    a = {l.a, l.rows, (l.op == LIN_FORWARD ? l.in : l.out) * es, l.lda * es};
    c = {l.o.c, l.op == LIN_WGRAD ? l.out : l.rows, (l.op == LIN_FORWARD ? l.out : l.in) * cs, l.o.ld * cs};
    q = flat(l.q, l.op == LIN_WGRAD ? l.rows * groups * kA8Group : ody_quant_bytes(l.kind, l.out * l.in));
    scales = flat(l.scales, l.rows * groups);
  }
};

// an error of the launcher itself is ours to report, not the next caller's to find
int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return ODY_OK;
  cudaGetLastError();
  return fail(ODY_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

int launch(const LinearArgs& a, void* ws, cudaStream_t st) {
  if (aligned_to(a.a, a.a_dtype, "an operand") || aligned_to(a.o.c, a.o.dtype, "the output") ||
      (a.o.add && aligned_to(a.o.add, a.o.dtype, "add")))
    return ODY_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(a.o.tscale) % 4)
    return fail(ODY_ERR_ARG, "the tensor scale is not aligned to its element type");
  const Spans s(a);
  const Span add = {a.o.add == a.o.c ? nullptr : a.o.add, s.c.n, s.c.bytes, s.c.pitch};
  if (meet(s.c, s.a) || meet(s.c, s.q) || meet(s.c, s.scales) || meet(s.c, flat(a.o.tscale, 4)) || meet(s.c, add))
    return fail(ODY_ERR_ARG, kOverlap);
  return launched(launch_linear(a, ws, st), "launch_linear");
}

int on_stream(const LinearArgs& a, void* ws, size_t ws_bytes, void* stream, const char* name) {
  const int64_t need = linear_workspace(a);
  if (need > 0 && (!ws || (int64_t)ws_bytes < need))
    return fail(ODY_ERR_ARG, std::string(name) + ": needs " + std::to_string(need) + " bytes of workspace");
  int cur = 0;
  cudaGetDevice(&cur);
  const void* const ptrs[] = {a.a, a.q, a.o.c, a.scales, a.o.tscale, a.o.add == a.o.c ? nullptr : a.o.add,
                              need > 0 ? ws : nullptr};
  bool here = true;
  for (const void* p : ptrs)
    if (p) {
      const int d = device_of(p);
      here = here && (d == cur || d == INT32_MAX);
    }
  if (!here)
    return fail(ODY_ERR_ARG, std::string(name) + " takes memory of the current GPU only");
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(ODY_ERR_ARG, std::string(name) + ": the workspace must be 256-byte aligned");
  return launch(a, ws, (cudaStream_t)stream);
}

// waits for the stream; whether a bounded wait on the device ran out
int status(cudaStream_t st) {
  bool ran_out = false;
  ODY_CUDA(gemm_wait_error(st, &ran_out));
  return ran_out ? fail(ODY_ERR_DEVICE_BOUNDS, "a bounded wait inside a linear kernel ran out") : ODY_OK;
}

// Host or device buffers, contiguous; waits for the result.  (Host buffers
// are copied, so the output's copy never meets another one: the caller's own
// addresses are compared first.)
int staged(LinearArgs a, float alpha) {
  if (a.o.c == a.a || a.o.c == a.q || a.o.c == a.scales) return fail(ODY_ERR_ARG, kOverlap);
  const Spans s(a);
  const int64_t asz = s.a.n * s.a.pitch, csz = s.c.n * s.c.pitch, qsz = s.q.bytes;
  a.o.alpha = alpha;
  Scope S;
  S.bufs.reserve(8);
  void *da, *dq, *dc, *ds = nullptr, *dadd = nullptr, *ws = nullptr;
  void* const c = a.o.c;
  ODY_STAGE(S, a.a, (size_t)asz, true, &da);
  ODY_STAGE(S, a.q, (size_t)qsz, true, &dq);
  if (a.scales) ODY_STAGE(S, a.scales, (size_t)s.scales.bytes, true, &ds);
  if (a.o.add && a.o.add != c) ODY_STAGE(S, a.o.add, (size_t)csz, true, &dadd);
  ODY_STAGE(S, c, (size_t)csz, a.o.add == c, &dc);
  if (a.o.add == c) dadd = dc;
  const int64_t need = linear_workspace(a);
  if (need > 0) {
    ODY_CUDA(cudaMallocAsync(&ws, (size_t)need, S.st));
    S.bufs.push_back({nullptr, ws, 0, true});
  }
  a.a = da, a.q = (const uint8_t*)dq, a.scales = (const uint8_t*)ds, a.o.c = dc, a.o.add = dadd;
  if (int rc = launch(a, ws, S.st)) return rc;
  ODY_CUDA(S.copy_out(c));
  return status(S.st);
}

int act8_args(int32_t fmt, const void* x, int32_t dt, int64_t rows, int64_t cols, int64_t ld, const void* codes,
              const void* scales) {
  if (fmt != ODY_A8_E4M3 && fmt != ODY_A8_E5M2)
    return fail(ODY_ERR_ARG, "unknown 8-bit activation format " + std::to_string(fmt));
  if (check_dtype(dt)) return ODY_ERR_DTYPE;
  if (rows <= 0 || cols <= 0) return fail(ODY_ERR_SHAPE, "cannot save an empty activation");
  if (rows > kMaxDim || cols > kMaxDim) return fail(ODY_ERR_SHAPE, "linear: a dimension is too large");
  if (int rc = check_pitch(ld, cols, "the activation")) return rc;
  if (!x || !codes || !scales) return fail(ODY_ERR_ARG, "null pointer");
  if (x == codes || x == scales || codes == scales) return fail(ODY_ERR_ARG, kOverlap);
  return ODY_OK;
}

int act8_device(const void* x, int32_t dt, int64_t rows, int64_t cols, int64_t ld, const void* codes, const void* scales,
                const char* name) {
  const int64_t es = dtype_size(dt), groups = ody_act8_groups(cols);
  const Span sx = {x, rows, cols * es, ld * es}, sc = flat(codes, rows * groups * kA8Group), ss = flat(scales, rows * groups);
  if (!is_device_ptr(x) || !is_device_ptr(codes) || !is_device_ptr(scales))
    return fail(ODY_ERR_ARG, std::string(name) + " takes memory of the current GPU only");
  if (reinterpret_cast<uintptr_t>(codes) & 15u)
    return fail(ODY_ERR_ARG, std::string(name) + ": codes must be 16-byte aligned");
  if (meet(sx, sc) || meet(sx, ss) || meet(sc, ss)) return fail(ODY_ERR_ARG, kOverlap);
  return aligned_to(x, dt, "the activation");
}

}  // namespace

extern "C" int64_t ody_act8_groups(int64_t cols) { return cols > 0 ? (cols + kA8Group - 1) / kA8Group : 0; }

extern "C" int ody_act8_save_on_stream(int32_t fmt, const void* x, int32_t dt, int64_t rows, int64_t cols, int64_t ldx,
                                       uint8_t* codes, uint8_t* scales, void* stream) {
  return guarded([&]() -> int {
    if (int rc = act8_args(fmt, x, dt, rows, cols, ldx, codes, scales)) return rc;
    if (int rc = act8_device(x, dt, rows, cols, ldx, codes, scales, "ody_act8_save_on_stream")) return rc;
    return launched(launch_act8_save(fmt, x, dt, rows, cols, ldx, codes, scales, (cudaStream_t)stream), "launch_act8_save");
  });
}

extern "C" int ody_act8_load_on_stream(int32_t fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                       int64_t cols, void* out, int32_t dt, int64_t ldo, void* stream) {
  return guarded([&]() -> int {
    if (int rc = act8_args(fmt, out, dt, rows, cols, ldo, codes, scales)) return rc;
    if (int rc = act8_device(out, dt, rows, cols, ldo, codes, scales, "ody_act8_load_on_stream")) return rc;
    return launched(launch_act8_load(fmt, codes, scales, rows, cols, out, dt, ldo, (cudaStream_t)stream), "launch_act8_load");
  });
}

extern "C" int ody_act8_save(int32_t fmt, const void* x, int32_t dt, int64_t rows, int64_t cols, uint8_t* codes,
                             uint8_t* scales) {
  return guarded([&]() -> int {
    if (int rc = act8_args(fmt, x, dt, rows, cols, cols, codes, scales)) return rc;
    const int64_t groups = ody_act8_groups(cols);
    Scope S;
    S.bufs.reserve(4);
    void *dx, *dc, *ds;
    ODY_STAGE(S, x, (size_t)(rows * cols) * dtype_size(dt), true, &dx);
    ODY_STAGE(S, codes, (size_t)(rows * groups * kA8Group), false, &dc);
    ODY_STAGE(S, scales, (size_t)(rows * groups), false, &ds);
    if (int rc = act8_device(dx, dt, rows, cols, cols, dc, ds, "ody_act8_save")) return rc;
    if (int rc = launched(launch_act8_save(fmt, dx, dt, rows, cols, cols, (uint8_t*)dc, (uint8_t*)ds, S.st), "launch_act8_save"))
      return rc;
    ODY_CUDA(S.copy_out(codes));
    ODY_CUDA(S.copy_out(scales));
    ODY_CUDA(cudaStreamSynchronize(S.st));
    return ODY_OK;
  });
}

extern "C" int ody_act8_load(int32_t fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols,
                             void* out, int32_t dt) {
  return guarded([&]() -> int {
    if (int rc = act8_args(fmt, out, dt, rows, cols, cols, codes, scales)) return rc;
    const int64_t groups = ody_act8_groups(cols);
    Scope S;
    S.bufs.reserve(4);
    void *dx, *dc, *ds;
    ODY_STAGE(S, codes, (size_t)(rows * groups * kA8Group), true, &dc);
    ODY_STAGE(S, scales, (size_t)(rows * groups), true, &ds);
    ODY_STAGE(S, out, (size_t)(rows * cols) * dtype_size(dt), false, &dx);
    if (int rc = act8_device(dx, dt, rows, cols, cols, dc, ds, "ody_act8_load")) return rc;
    if (int rc = launched(launch_act8_load(fmt, (const uint8_t*)dc, (const uint8_t*)ds, rows, cols, dx, dt, cols, S.st),
                          "launch_act8_load"))
      return rc;
    ODY_CUDA(S.copy_out(out));
    ODY_CUDA(cudaStreamSynchronize(S.st));
    return ODY_OK;
  });
}

extern "C" int64_t ody_linear_workspace_of(int32_t op, int32_t kind, int64_t rows, int64_t out, int64_t in,
                                           int32_t act_dtype) {
  LinearArgs a{};
  if (op < LIN_FORWARD || op > LIN_WGRAD || (op != LIN_WGRAD && !is_w4(kind)) || rows <= 0 || out <= 0 || in <= 0 ||
      rows > kMaxDim || out > kMaxDim || in > kMaxDim || act_dtype < DT_F32 || act_dtype > DT_BF16)
    return -1;
  a.op = op;
  a.rows = rows, a.out = out, a.in = in;
  a.a_dtype = act_dtype;
  a.kind = kind;
  return linear_workspace(a);
}

// the kind that fewest widths are whole blocks of asks for the most
extern "C" int64_t ody_linear_workspace(int32_t op, int64_t rows, int64_t out, int64_t in, int32_t act_dtype) {
  return ody_linear_workspace_of(op, ODY_Q_MXFP4, rows, out, in, act_dtype);
}

#define ODY_W4_PAIR(NAME, OP, ACT, OUT, ACOLS, CCOLS)                                                               \
  extern "C" int NAME##_on_stream(int32_t kind, const void* q, const float* tensor_scale, float alpha,              \
                                  int64_t out_features, int64_t in_features, const void* ACT, int32_t act_dtype,    \
                                  int64_t rows, int64_t lda, void* OUT, int32_t out_dtype, int64_t ldo,             \
                                  void* workspace, size_t workspace_bytes, void* stream) {                          \
    return guarded([&]() -> int {                                                                                   \
      LinearArgs a;                                                                                                 \
      if (int rc = product(a, OP, kind, rows, out_features, in_features, ACT, act_dtype, lda, q, nullptr, OUT,      \
                           out_dtype, ldo))                                                                         \
        return rc;                                                                                                  \
      a.o.alpha = alpha;                                                                                            \
      a.o.tscale = tensor_scale;                                                                                    \
      return on_stream(a, workspace, workspace_bytes, stream, #NAME "_on_stream");                                  \
    });                                                                                                             \
  }                                                                                                                 \
  extern "C" int NAME(int32_t kind, const void* q, float tensor_scale, int64_t out_features, int64_t in_features,   \
                      const void* ACT, int32_t act_dtype, int64_t rows, void* OUT, int32_t out_dtype) {             \
    return guarded([&]() -> int {                                                                                   \
      LinearArgs a;                                                                                                 \
      if (int rc = product(a, OP, kind, rows, out_features, in_features, ACT, act_dtype, ACOLS, q, nullptr, OUT,    \
                           out_dtype, CCOLS))                                                                       \
        return rc;                                                                                                  \
      return staged(a, kind == ODY_Q_NVFP4_TENSOR ? tensor_scale : 1.0f);                                           \
    });                                                                                                             \
  }

ODY_W4_PAIR(ody_fp4_linear, LIN_FORWARD, x, y, in_features, out_features)
ODY_W4_PAIR(ody_fp4_linear_dgrad, LIN_DGRAD, dy, dx, out_features, in_features)
#undef ODY_W4_PAIR

extern "C" int ody_linear_wgrad8_on_stream(int32_t fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                           int64_t in_features, const void* dy, int32_t dy_dtype, int64_t out_features,
                                           int64_t lddy, float alpha, const void* add, void* dw, int32_t dw_dtype,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    LinearArgs a;
    if (int rc = product(a, LIN_WGRAD, fmt, rows, out_features, in_features, dy, dy_dtype, lddy, codes, scales, dw,
                         dw_dtype, in_features))
      return rc;
    a.o.alpha = alpha;
    a.o.add = add;
    if (reinterpret_cast<uintptr_t>(codes) & 15u)
      return fail(ODY_ERR_ARG, "ody_linear_wgrad8_on_stream: codes must be 16-byte aligned");
    return on_stream(a, workspace, workspace_bytes, stream, "ody_linear_wgrad8_on_stream");
  });
}

extern "C" int ody_linear_wgrad8(int32_t fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                 int64_t in_features, const void* dy, int32_t dy_dtype, int64_t out_features,
                                 float alpha, const void* add, void* dw, int32_t dw_dtype) {
  return guarded([&]() -> int {
    LinearArgs a;
    if (int rc = product(a, LIN_WGRAD, fmt, rows, out_features, in_features, dy, dy_dtype, out_features, codes, scales,
                         dw, dw_dtype, in_features))
      return rc;
    a.o.add = add;
    if (is_device_ptr(codes) && (reinterpret_cast<uintptr_t>(codes) & 15u))
      return fail(ODY_ERR_ARG, "ody_linear_wgrad8: codes must be 16-byte aligned");
    return staged(a, alpha);
  });
}

extern "C" int ody_linear_status(void* stream) {
  return guarded([&]() -> int { return status((cudaStream_t)stream); });
}

// Test hook (not part of include/odyssey_mp.h): a device-side wait that runs
// out after so many cycles.
extern "C" int odyx_linear_wait_selftest(int64_t cycles, void* stream) {
  ODY_CUDA(launch_wait_selftest(cycles, (cudaStream_t)stream));
  return ODY_OK;
}

// Test hook (not part of include/odyssey_mp.h): what a few-row kernel may take
// of shared memory, as the calls so far have set it.
extern "C" int odyx_linear_rows_limit(int32_t* bytes) {
  ODY_CUDA(rows_shared_limit(bytes));
  return ODY_OK;
}

// The layer's host path: one call per autograd node.  Allocates every output and workspace with
// torch's caching allocator, enqueues the kernels of libmomoe_hip.so on the current stream and
// records the autograd nodes.  It is native because a call makes a dozen launches: driven from
// Python (a wrapper, an allocation or two and a foreign-function call per launch) the host needed
// 84 us for a forward and 240 us for a training step of any size, longer than the GPU works on a
// decode call or on a small step.
//
// Nothing here synchronises with the device (unless the caller asks for the routing check): every
// launch is sized from static upper bounds and the routing-dependent tile list lives in device
// memory.
#include <ATen/autocast_mode.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <atomic>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/momoe_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- launch timing (kernel_timer in _hip.py): an event pair around every library call ---------
struct TimedCall {
  std::string name;
  hipEvent_t begin, end;
};
std::mutex g_timing_mutex;
std::atomic<bool> g_timing{false};  // read by every thread that launches; a stale read only skips a record
std::vector<TimedCall> g_calls;

void timing_start() { g_timing.store(true, std::memory_order_relaxed); }
void timing_stop() { g_timing.store(false, std::memory_order_relaxed); }
// durations in ms of the calls recorded so far; the device must be idle
std::vector<std::pair<std::string, double>> timing_take() {
  std::lock_guard<std::mutex> lock(g_timing_mutex);
  std::vector<std::pair<std::string, double>> out;
  for (auto& c : g_calls) {
    float ms = 0.0f;
    const bool ok = hipEventElapsedTime(&ms, c.begin, c.end) == hipSuccess;
    (void)hipEventDestroy(c.begin);
    (void)hipEventDestroy(c.end);
    if (ok) out.emplace_back(c.name, (double)ms);
  }
  g_calls.clear();
  return out;
}

// fn(), with an event pair around it on `st` while launches are timed
template <class Fn>
auto timed(const char* name, hipStream_t st, Fn fn) {
  if (!g_timing.load(std::memory_order_relaxed)) return fn();
  TimedCall t{name, nullptr, nullptr};
  const bool begun = hipEventCreate(&t.begin) == hipSuccess && hipEventCreate(&t.end) == hipSuccess &&
                     hipEventRecord(t.begin, st) == hipSuccess;
  auto result = fn();
  if (begun && hipEventRecord(t.end, st) == hipSuccess) {
    std::lock_guard<std::mutex> lock(g_timing_mutex);
    g_calls.push_back(std::move(t));
  } else {
    if (t.begin) (void)hipEventDestroy(t.begin);
    if (t.end) (void)hipEventDestroy(t.end);
  }
  return result;
}

template <class Fn, class... Args>
void call(const char* name, hipStream_t st, Fn fn, Args... args) {
  const int code = timed(name, st, [&] { return fn(args..., (void*)st); });
  TORCH_CHECK(code == MOMOE_OK, name, " failed: status ", code, " (", momoe_status_string(code), ")");
}
#define MOMOE_CALL(fn, st, ...) call(#fn, st, fn, __VA_ARGS__)

hipStream_t stream_of(const at::Device& dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

Tensor empty_bf16(at::IntArrayRef size, const at::Device& dev) {
  return at::empty(size, at::TensorOptions().dtype(at::kBFloat16).device(dev));
}
Tensor empty_i32(int64_t n, const at::Device& dev) {
  return at::empty({n}, at::TensorOptions().dtype(at::kInt).device(dev));
}
Tensor empty_f32(at::IntArrayRef size, const at::Device& dev) {
  return at::empty(size, at::TensorOptions().dtype(at::kFloat).device(dev));
}

// Buffers that live no longer than the call: pieces of one allocation where they are few bytes in all, since an
// allocation takes the host a microsecond and a small call is as long as its host work (in us of the host, a forward of 7 tokens
// with its router 37.2 -> 34.8, the backward of 128 tokens 88 -> 81); allocations of their own, given back as soon as they are
// done with, where their size counts.  The line is torch's own between small allocations and large ones; forwards in a row below
// it, us, in several -> in one: 7 tokens, D = 256, H = 128, N = 16, K = 2 19.8 -> 18.2; 128, 512, 128, 32, 2 21.9 -> 21.6; 150, 512, 128, 48, 4
// 22.3 -> 22.1; 300, 512, 256, 16, 2 25.9 -> 25.4; 200, 256, 256, 96, 4 26.7 -> 26.6; 400, 384, 128, 64, 2 24.2 -> 24.1.
class Transients {
  const at::Device dev_;
  Tensor block_;
  int64_t used_ = 0;
  static int64_t up(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }

 public:
  Transients(const at::Device& dev, std::initializer_list<int64_t> sizes) : dev_(dev) {
    constexpr int64_t kMost = 1 << 20;
    int64_t all = 0;
    for (int64_t bytes : sizes) all += bytes <= kMost ? up(bytes) : 2 * kMost;
    if (all <= kMost) block_ = bytes_of(all);
  }
  Tensor bytes_of(int64_t bytes) const { return at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(dev_)); }
  // the next of those sizes; `own` holds it if it is an allocation of its own
  void* take(int64_t bytes, Tensor& own) {
    if (!block_.defined()) return (own = bytes_of(bytes)).data_ptr();
    TORCH_INTERNAL_ASSERT(used_ + bytes <= block_.numel());
    void* const p = (char*)block_.data_ptr() + used_;
    used_ += up(bytes);
    return p;
  }
};

// A Python exception of the given type, raised when the binding returns
[[noreturn]] void throw_python(PyObject* type, const std::string& what) {
  py::gil_scoped_acquire gil;
  PyErr_SetString(type, what.c_str());
  throw py::error_already_set();
}

// Whether a call has to go through its autograd function.  A forward-mode tangent counts: the
// function refuses it, where the plain forward would drop it without a word.
bool wants_autograd(std::initializer_list<const Tensor*> inputs) {
  bool any = false;
  for (const Tensor* t : inputs)
    any = any || (at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined();
  return any;
}

// A call under torch.jit.trace, made again through the operator momoe::`name` (TORCH_LIBRARY
// below), whose kernel is the calling function itself: the tracer records operators that pass
// the dispatcher.  Of a plain call it would see the allocations only and record a graph that
// returns unwritten memory.
template <class Result, class... Args>
Result call_recorded(const char* name, Args... args) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Result(Args...)>().call(
      std::forward<Args>(args)...);
}

// A tensor that a backward hands to kernels by pointer, as the forward saved it.  A saved-tensor hook
// may have put any other in its place: one on the host, of another type or shorter would be read
// past its end on the device.  `packed`: contiguous and on a 16-byte boundary.
const Tensor& as_saved(const Tensor& t, const char* name, const at::Device& dev, at::ScalarType type,
                       at::IntArrayRef sizes, bool packed = true) {
  TORCH_CHECK(t.defined() && t.device() == dev && t.scalar_type() == type && t.sizes() == sizes &&
                  (!packed || (t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0)),
              "backward: the saved tensor ", name, " came back from its hook as something else than ", type, " ", sizes,
              " on ", dev, packed ? ", contiguous" : "");
  return t;
}

// ---- experts -----------------------------------------------------------------------------------
// What the index build leaves for the rest of the forward and for the backward, in one allocation:
// [cumsums N+1 | idx Msum | inv Msum | tile table | table of tiles of at most 256 rows], every part
// on a 16-byte boundary.  The parts are found again from the sizes alone.
struct Index {
  int64_t M, N, K, tile_rows;
  bool with_rc;  // with the second table; the first one is then of the library's choice
  int64_t off_idx, off_inv, off_table, off_rc, ints;
  Index(int64_t M_, int64_t N_, int64_t K_, int64_t tile_rows_, bool with_rc_)
      : M(M_), N(N_), K(K_), tile_rows(tile_rows_), with_rc(with_rc_) {
    auto up = [](int64_t n) { return (n + 3) & ~(int64_t)3; };
    off_idx = up(N + 1);
    off_inv = off_idx + up(M * K);
    off_table = off_inv + up(M * K);
    off_rc = off_table + up(momoe_tile_table_ints(M, N, K, (int)tile_rows));
    ints = off_rc + (with_rc ? up(momoe_tile_table_ints(M, N, K, MOMOE_RECOMPUTE_TILE_ROWS)) : 0);
  }
  int32_t* base = nullptr;
  int32_t* cumsums() const { return base; }
  int32_t* idx() const { return base + off_idx; }
  int32_t* inv() const { return base + off_inv; }
  int32_t* table() const { return base + off_table; }
  int32_t* table_rc() const { return with_rc ? base + off_rc : nullptr; }
  // the one that suits a GEMM of `cols` output columns
  int32_t* table_for(int64_t cols, int64_t contraction) const {
    return with_rc && momoe_gemm_tile_rows(M * K, N, cols, contraction) != 0 ? table_rc() : table();
  }
};

struct Forward {
  Tensor y, sizes;                     // results
  Tensor x, W1, W2, s, index, ab_save; // for the backward
};

Forward experts_forward(const Tensor& x_BSD, const Tensor& Wl1, const Tensor& Wl2, const Tensor& mask_NM,
                        const Tensor& s_NM, int64_t K, int64_t msave, bool want_rc, int64_t tile_rows,
                        bool check) {
  const at::Device dev = Wl1.device();
  const int64_t B = x_BSD.size(0), S = x_BSD.size(1), D = x_BSD.size(2), M = B * S;
  const int64_t N = Wl1.size(0), H = Wl1.size(2) / 2, msum = M * K;
  const c10::DeviceGuard guard(dev);
  const hipStream_t st = stream_of(dev);
  Forward f;
  f.x = x_BSD.reshape({M, D}).to(dev, at::kBFloat16).contiguous();
  f.W1 = Wl1.to(at::kBFloat16).contiguous();
  f.W2 = Wl2.to(at::kBFloat16).contiguous();
  const Tensor mask = mask_NM.to(dev, at::kInt);
  f.s = s_NM.to(dev, at::kFloat);
  TORCH_CHECK(mask.dim() == 2 && mask.size(0) == N && mask.size(1) == M, "mask_NM must be [", N, ", ", M, "]");
  TORCH_CHECK(f.s.dim() == 2 && f.s.size(0) == N && f.s.size(1) == M, "s_NM must be [", N, ", ", M, "]");

  Index ib(M, N, K, tile_rows, want_rc);
  f.index = empty_i32(ib.ints, dev);
  ib.base = f.index.data_ptr<int32_t>();
  f.sizes = at::empty({N}, at::TensorOptions().dtype(at::kLong).device(dev));
  const int64_t ws_bytes = momoe_index_workspace_bytes(M, N);
  // only the build itself needs these: its panel counts, the slot of every pair, and the counter
  // of tokens with another number of experts than K, which starts from zero if it is to be read
  const int64_t scratch_bytes = (4 + ((msum + 3) & ~(int64_t)3) + (ws_bytes + 3) / 4) * 4;
  Transients transients(dev, {scratch_bytes, msum * H * 2, msum * D * 2});
  Tensor counter, scratch, h_own, ys_own;
  int32_t* const build = (int32_t*)transients.take(scratch_bytes, scratch);
  int32_t* violations = build;
  if (check) {
    counter = at::zeros({4}, at::TensorOptions().dtype(at::kInt).device(dev));
    violations = counter.data_ptr<int32_t>();
  }
  MOMOE_CALL(momoe_index_build, st, mask.data_ptr<int32_t>(), mask.stride(0), mask.stride(1), M, N, K,
             f.sizes.data_ptr<int64_t>(), ib.cumsums(), ib.idx(), build + 4, ib.inv(), ib.table(),
             (int)tile_rows, ib.table_rc(), (void*)(build + 4 + ((msum + 3) & ~(int64_t)3)), ws_bytes,
             violations);

  if (msave > 0) f.ab_save = empty_bf16({msave, 2 * H}, dev);
  // h in blocks of 32 hidden columns, [H/32][Msum][32]: the layout the down projection reads
  void* const h = transients.take(msum * H * 2, h_own);
  MOMOE_CALL(momoe_lin1_swiglu_fwd, st, f.x.data_ptr(), f.W1.data_ptr(), ib.idx(), ib.table_for(2 * H, D), h,
             msave > 0 ? f.ab_save.data_ptr() : nullptr, (int64_t)0, msave, M, D, H, N, msum);
  void* const ys = transients.take(msum * D * 2, ys_own);
  MOMOE_CALL(momoe_lin2_scale_fwd, st, h, f.W2.data_ptr(), f.s.data_ptr<float>(), f.s.stride(0),
             f.s.stride(1), ib.idx(), ib.table_for(D, H), ys, M, D, H, N, msum);
  h_own.reset();
  f.y = empty_bf16({B, S, D}, dev);
  MOMOE_CALL(momoe_combine, st, ys, ib.inv(), f.y.data_ptr(), M, D, K, msum);
  if (check) {
    const int v = counter.narrow(0, 0, 1).item<int32_t>();
    TORCH_CHECK(v == 0, "mask_NM: ", v, " tokens do not have exactly K = ", K,
                " experts (or the mask holds more than M*K pairs)");
  }
  if (x_BSD.device() != dev) f.y = f.y.to(x_BSD.device());
  return f;
}

// Tile height left to the library (tile_rows = 0): one table of 256 rows if that suits all these GEMMs (output
// columns, contraction), else the library's choice, and that one next to it if any wants it.
void choose_tables(std::initializer_list<std::pair<int64_t, int64_t>> gemms, int64_t msum, int64_t N, int64_t& tile_rows,
                   bool& with_rc) {
  if (tile_rows != 0) {
    with_rc = false;
    return;
  }
  bool all = true;
  for (const auto& g : gemms) {
    const bool short_tiles = momoe_gemm_tile_rows(msum, N, g.first, g.second) != 0;
    all = all && short_tiles;
    with_rc = with_rc || short_tiles;
  }
  if (!all) return;
  tile_rows = MOMOE_RECOMPUTE_TILE_ROWS;
  with_rc = false;
}

struct ExpertsFn : torch::autograd::Function<ExpertsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& W1, const Tensor& W2,
                               const Tensor& mask, const Tensor& s, int64_t K, int64_t msave, int64_t tile_rows,
                               bool check) {
    // the recomputing GEMM's tiles have at most 256 rows
    bool want_rc = msave < x.size(0) * x.size(1) * K;
    const int64_t D = W1.size(1), H = W2.size(1);
    choose_tables({{2 * H, D}, {D, H}, {H, D}, {D, 2 * H}}, x.size(0) * x.size(1) * K, W1.size(0), tile_rows, want_rc);
    Forward f = experts_forward(x, W1, W2, mask, s, K, msave, want_rc, tile_rows, check);
    // (one entry: each takes the host 0.3 us to make and 0.2 to find)
    ctx->saved_data["call"] = std::vector<int64_t>{K, msave, tile_rows, want_rc, f.W1.device().index(), f.W1.size(1), f.W2.size(0), f.W2.size(1)};
    ctx->save_for_backward({f.x, f.s, f.W1, f.W2, f.index, f.ab_save});
    ctx->mark_non_differentiable({f.sizes});
    ctx->set_materialize_grads(false);
    return {f.y, f.sizes};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const std::vector<int64_t> call_of = ctx->saved_data["call"].toIntVector();
    const int64_t K = call_of[0], msave = call_of[1], tile_rows = call_of[2], D = call_of[5], N = call_of[6], H = call_of[7];
    const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(1),
               need_w2 = ctx->needs_input_grad(2), need_s = ctx->needs_input_grad(4);
    variable_list out(9);
    if (!grads[0].defined()) return out;
    const at::Device dev(at::kCUDA, (at::DeviceIndex)call_of[4]), gdev = grads[0].device();
    const int64_t B = grads[0].size(0), S = grads[0].size(1), M = B * S, msum = M * K;
    Index ib(M, N, K, tile_rows, call_of[3] != 0);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& x = as_saved(saved[0], "x", dev, at::kBFloat16, {M, D});
    const Tensor& s = as_saved(saved[1], "s", dev, at::kFloat, {N, M}, /*packed=*/false);
    const Tensor& W1 = as_saved(saved[2], "Wl1", dev, at::kBFloat16, {N, D, 2 * H});
    const Tensor& W2 = as_saved(saved[3], "Wl2", dev, at::kBFloat16, {N, H, D});
    ib.base = as_saved(saved[4], "index", dev, at::kInt, {ib.ints}).data_ptr<int32_t>();
    const Tensor& ab_save = saved[5];
    if (msave > 0) as_saved(ab_save, "a|b", dev, at::kBFloat16, {msave, 2 * H});
    const c10::DeviceGuard guard(dev);
    const hipStream_t st = stream_of(dev);
    const Tensor Gy = grads[0].reshape({M, D}).to(dev, at::kBFloat16).contiguous();

    // dL/dh before the gate weight, in sorted order
    // few tiles and no row saved: made on the way by the launch that needs it
    const bool joined = msave == 0 && momoe_dgrad_h_lin1_bwd_fits(M, D, H, N, msum) != 0;
    const int64_t u_bytes = msum * H * 2, gz_bytes = 2 * u_bytes, hst_bytes = momoe_padded_rows(msum, N) * H * 2;
    const int64_t nparts = momoe_gs_parts(H, N, msum), parts_bytes = nparts * msum * 4, gxs_bytes = need_x ? msum * D * 2 : 0;
    // scratch for the weight gradients of experts with many rows: what the library can use, but no
    // more than u occupied (just freed, so the peak does not move)
    auto scratch_bytes = [&](bool need, int64_t X, int64_t Y) {
      return need ? std::min(u_bytes, momoe_wgrad_workspace_bytes(N, X, Y, msum)) : 0;
    };
    // small: both weight gradients and dL/dx in one launch
    const bool tail = need_w1 && need_w2 && need_x && momoe_backward_tail_fits(M, D, H, N, msum) != 0;
    const int64_t ws2_bytes = scratch_bytes(need_w2 && !tail, H, D), ws1_bytes = scratch_bytes(need_w1 && !tail, D, 2 * H);
    Transients transients(dev, {u_bytes, gz_bytes, hst_bytes, parts_bytes, ws2_bytes, ws1_bytes, gxs_bytes});
    Tensor u_own, gz_own, hst_own, parts_own;
    void* const u = transients.take(u_bytes, u_own);
    if (!joined) MOMOE_CALL(momoe_dgrad_h, st, Gy.data_ptr(), W2.data_ptr(), ib.idx(), ib.table_for(H, D), u, M, D, H, N, msum);
    // SwiGLU backward: rows with saved a|b read them; the others recompute a|b = x.Wl1 and consume
    // them straight from the GEMM's accumulators.
    // G_a|G_b in blocks of 32 columns, [2H/32][Msum][32]: the layout dL/dx contracts over
    void* const gz = transients.take(gz_bytes, gz_own);
    // s*h in groups of 32 padded sorted rows, feature-major inside a group: the layout the Wl2
    // gradient reads fastest
    void* const hst = transients.take(hst_bytes, hst_own);
    float* const gs_part = (float*)transients.take(parts_bytes, parts_own);
    if (msave > 0)
      MOMOE_CALL(momoe_swiglu_bwd_saved, st, ab_save.data_ptr(), u, s.data_ptr<float>(), s.stride(0),
                 s.stride(1), ib.idx(), ib.cumsums(), msave, gz, hst, H,
                 gs_part, nparts, M, H, N, msum);
    if (msave < msum) {
      // the recomputing GEMM takes no taller tiles: a table of its own where another height was given
      Tensor own;
      const int32_t* table_rc = ib.with_rc ? ib.table_rc() : ib.table();
      if (tile_rows != 0 && tile_rows != MOMOE_RECOMPUTE_TILE_ROWS) {
        own = empty_i32(momoe_tile_table_ints(M, N, K, MOMOE_RECOMPUTE_TILE_ROWS), dev);
        MOMOE_CALL(momoe_tile_table_build, st, ib.cumsums(), N, msum, MOMOE_RECOMPUTE_TILE_ROWS,
                   own.data_ptr<int32_t>());
        table_rc = own.data_ptr<int32_t>();
      }
      if (joined)
        MOMOE_CALL(momoe_dgrad_h_lin1_bwd, st, Gy.data_ptr(), W2.data_ptr(), x.data_ptr(), W1.data_ptr(), (const int32_t*)ib.idx(),
                   table_rc, (const float*)s.data_ptr<float>(), s.stride(0), s.stride(1), u, gz, hst, H, gs_part, nparts, M, D, H, N, msum);
      else
        call("momoe_lin1_swiglu_bwd", st, momoe_lin1_swiglu_bwd_parts, x.data_ptr(), W1.data_ptr(), ib.idx(), table_rc,
           u, s.data_ptr<float>(), s.stride(0), s.stride(1), msave, gz, hst, H,
           gs_part, nparts, M, D, H, N, msum);
    }
    u_own.reset();
    float* gs_tail = nullptr;
    if (need_s) {
      // in the layout of s, where autograd keeps it without a copy
      if (s.stride(0) == 1 && s.stride(1) == N) {
        out[4] = at::empty_strided({N, M}, {1, N}, at::TensorOptions().dtype(at::kFloat).device(dev));
        if (tail)
          gs_tail = out[4].data_ptr<float>();
        else
          call("momoe_gs_scatter", st, momoe_gs_scatter_tokens, gs_part, nparts, (const int32_t*)ib.idx(),
               (const int32_t*)ib.cumsums(), out[4].data_ptr<float>(), M, N, msum);
      } else {
        out[4] = empty_f32({N, M}, dev);
        MOMOE_CALL(momoe_gs_scatter, st, gs_part, nparts, ib.idx(), ib.cumsums(),
                   out[4].data_ptr<float>(), M, N, msum);
      }
    }
    if (!tail) parts_own.reset();
    // (what the joined launch reads and writes is all there at once: the peak is the weight gradients, gz, s*h, the partial sums and
    // gxs, where one launch after the other has dL/dx in the place of s*h: 11.6 MiB more at 700 tokens, D = 2048, H = 768, N = 128,
    // K = 8, and always less than the 64 MiB of momoe_backward_tail_fits)
    if (need_w2) out[2] = at::empty_like(W2);
    if (need_w1 && tail) out[1] = at::empty_like(W1);
    Tensor gxs_own;
    void* gxs = nullptr;
    if (tail) {
      gxs = transients.take(gxs_bytes, gxs_own);
      MOMOE_CALL(momoe_backward_tail, st, hst, H, Gy.data_ptr(), x.data_ptr(), gz, W1.data_ptr(), (const int32_t*)ib.idx(),
                 (const int32_t*)ib.cumsums(), (const int32_t*)ib.table_for(D, 2 * H), out[2].data_ptr(), out[1].data_ptr(), gxs,
                 (const float*)gs_part, nparts, gs_tail, M, D, H, N, msum);
      parts_own.reset();
      gz_own.reset();
    }
    if (need_w2 && !tail) {
      Tensor ws_own;
      void* const ws = ws2_bytes > 0 ? transients.take(ws2_bytes, ws_own) : nullptr;
      MOMOE_CALL(momoe_wgrad, st, hst, H, MOMOE_LAYOUT_TRANSPOSED, (const int32_t*)nullptr, Gy.data_ptr(),
                 D, MOMOE_LAYOUT_ROWS, (const int32_t*)ib.idx(), ib.cumsums(), out[2].data_ptr(), M, N, H, D, msum,
                 ws, ws2_bytes);
    }
    hst_own.reset();
    if (need_w1 && !tail) {
      out[1] = at::empty_like(W1);
      Tensor ws_own;
      void* const ws = ws1_bytes > 0 ? transients.take(ws1_bytes, ws_own) : nullptr;
      MOMOE_CALL(momoe_wgrad, st, x.data_ptr(), D, MOMOE_LAYOUT_ROWS, (const int32_t*)ib.idx(), gz, msum,
                 MOMOE_LAYOUT_KBLOCKED, (const int32_t*)nullptr, ib.cumsums(), out[1].data_ptr(), M, N, D, 2 * H, msum,
                 ws, ws1_bytes);
    }
    if (need_x) {
      if (!tail) {
        gxs = transients.take(gxs_bytes, gxs_own);
        MOMOE_CALL(momoe_dgrad_x, st, gz, W1.data_ptr(), ib.table_for(D, 2 * H), gxs, M, D, H, N, msum);
      }
      Tensor Gx = empty_bf16({B, S, D}, dev);
      MOMOE_CALL(momoe_combine, st, gxs, ib.inv(), Gx.data_ptr(), M, D, K, msum);
      out[0] = gdev == dev ? Gx : Gx.to(gdev);
    }
    return out;
  }
};

std::tuple<Tensor, Tensor> experts(const Tensor& x, const Tensor& W1, const Tensor& W2, const Tensor& mask,
                                   const Tensor& s, int64_t K, double save_percent, int64_t tile_rows, bool check) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<std::tuple<Tensor, Tensor>, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                         const Tensor&, int64_t, double, int64_t, bool>("momoe::experts", x, W1, W2, mask, s, K,
                                                                        save_percent, tile_rows, check);
  if (W1.device() != W2.device())
    throw_python(PyExc_AssertionError, "All weights must be on the same device, but got: Wl1_ND2H.device = " +
                                    W1.device().str() + ", Wl2_NHD.device = " + W2.device().str());
  TORCH_CHECK(W1.is_cuda(), "MoMoE weights must live on the GPU: there is no CPU compute path");
  if (x.dim() != 3 || W1.dim() != 3 || W2.dim() != 3 || W1.size(1) != x.size(2) || W2.size(0) != W1.size(0) ||
      W2.size(1) != W1.size(2) / 2 || W2.size(2) != x.size(2))
    throw_python(PyExc_AssertionError, "x_BSD [B,S,D], Wl1_ND2H [N,D,2H] and Wl2_NHD [N,H,D] do not fit together");
  const int64_t msum = x.size(0) * x.size(1) * K;
  if (!wants_autograd({&x, &W1, &W2, &s})) {  // nothing is kept for a backward that cannot happen
    bool with_rc = false;
    choose_tables({{2 * W2.size(1), W1.size(1)}, {W1.size(1), W2.size(1)}}, msum, W1.size(0), tile_rows, with_rc);
    Forward f = experts_forward(x, W1, W2, mask, s, K, 0, with_rc, tile_rows, check);
    return {f.y, f.sizes};
  }
  // the Wl1 gradient addresses the eight 32-column blocks of a gz tile with 32-bit byte offsets
  // (momoe_wgrad, k-blocked operand): say so now rather than in the backward
  TORCH_CHECK(!W1.requires_grad() || 8 * msum * 64 < (1ll << 32),
              "MoMoE backward supports fewer than 8388608 (token, expert) pairs per call, got ", msum,
              ": split the batch");
  const int64_t msave = (int64_t)((double)msum * save_percent / 100.0);  // momoe/momoe.py:251
  variable_list r = ExpertsFn::apply(x, W1, W2, mask, s, K, msave, tile_rows, check);
  return {r[0], r[1]};
}

// ---- experts in 8-bit floating point ----------------------------------------------------------
int type_of(at::ScalarType t) {
  return t == at::kBFloat16 ? MOMOE_TYPE_BF16 : t == at::kFloat ? MOMOE_TYPE_F32 : t == at::kHalf ? MOMOE_TYPE_F16 : -1;
}

// x [B, S, D]; W1, W2 packed, S1, S2 the bits of their scales, int32 (a trace cannot hold the view between the two); forward only
std::tuple<Tensor, Tensor> experts_fp8(const Tensor& x_BSD, const Tensor& W1, const Tensor& S1, const Tensor& W2, const Tensor& S2,
                                       const Tensor& mask_NM, const Tensor& s_NM, int64_t K, int64_t H, bool check) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<std::tuple<Tensor, Tensor>, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                         const Tensor&, const Tensor&, int64_t, int64_t, bool>("momoe::experts_fp8", x_BSD, W1, S1, W2, S2, mask_NM,
                                                                              s_NM, K, H, check);
  TORCH_CHECK(W1.is_cuda(), "MoMoEFP8 weights must live on the GPU: there is no CPU compute path");
  TORCH_CHECK(!wants_autograd({&x_BSD, &s_NM}),
              "MoMoEFP8 has no backward, and an input requires a gradient: call it under torch.no_grad()");
  const at::Device dev = W1.device();
  if (x_BSD.dim() != 3) throw_python(PyExc_AssertionError, "x_BSD must be [B, S, D]");
  const int64_t B = x_BSD.size(0), S = x_BSD.size(1), D = x_BSD.size(2), M = B * S;
  TORCH_CHECK(K >= 1, "K, the experts of a token, must be at least 1, got ", K);
  const int64_t N = S1.dim() == 4 ? S1.size(0) : 0, msum = M * K, DB = (D + 127) / 128, HB = (H + 127) / 128;
  const auto held = [&](const Tensor& t, at::ScalarType type) {
    return t.device() == dev && t.scalar_type() == type && t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0;
  };
  const bool fit = S1.dim() == 4 && S2.dim() == 3 && S1.sizes() == at::IntArrayRef({N, DB, 2, HB}) &&
                   S2.sizes() == at::IntArrayRef({N, HB, DB}) && W1.numel() == momoe_fp8_weight_bytes(N, D, 2 * H) &&
                   W2.numel() == momoe_fp8_weight_bytes(N, H, D) && held(W1, at::kByte) && held(W2, at::kByte) && held(S1, at::kInt) &&
                   held(S2, at::kInt);
  if (!fit) throw_python(PyExc_AssertionError, "x_BSD [B,S,D] and the packed weights do not fit together");
  const c10::DeviceGuard guard(dev);
  const hipStream_t st = stream_of(dev);
  const Tensor mask = mask_NM.to(dev, at::kInt), s = s_NM.to(dev, at::kFloat);
  TORCH_CHECK(mask.dim() == 2 && mask.size(0) == N && mask.size(1) == M, "mask_NM must be [", N, ", ", M, "]");
  TORCH_CHECK(s.dim() == 2 && s.size(0) == N && s.size(1) == M, "s_NM must be [", N, ", ", M, "]");
  Tensor y = empty_bf16({B, S, D}, dev), sizes = at::empty({N}, at::TensorOptions().dtype(at::kLong).device(dev));
  if (M == 0) return {x_BSD.device() == dev ? y : y.to(x_BSD.device()), sizes.zero_()};
  // rows in 8 bits from the type they come in; any other type as bf16
  Tensor x = x_BSD.reshape({M, D}).to(dev);
  if (type_of(x.scalar_type()) < 0) x = x.to(at::kBFloat16);
  x = x.contiguous();
  if ((uintptr_t)x.data_ptr() % 16 != 0) x = x.clone();

  // (the tall tiles gather their rows in 8 bits at 32-bit offsets)
  const bool far = M * DB * 128 >= (1ll << 32);
  Index ib(M, N, K, far ? MOMOE_FP8_FEW_ROWS : momoe_fp8_tile_rows(msum, D, H, N), false);
  const bool few = ib.tile_rows == MOMOE_FP8_FEW_ROWS;  // the products bring their rows to 8 bits themselves
  const int64_t ws_bytes = momoe_index_workspace_bytes(M, N), index_bytes = ib.ints * 4;
  const int64_t scratch_bytes = (4 + ((msum + 3) & ~(int64_t)3) + (ws_bytes + 3) / 4) * 4;
  const int64_t xq_bytes = few ? 0 : M * DB * 128, xs_bytes = few ? 0 : M * momoe_fp8_code_bytes(D);
  const int64_t h_bytes = few ? msum * H * 4 : msum * HB * 128, hs_bytes = few ? 0 : msum * momoe_fp8_code_bytes(H);
  Transients transients(dev, {index_bytes, scratch_bytes, xq_bytes, xs_bytes, h_bytes, hs_bytes, msum * D * 2});
  Tensor index_own, scratch, xq_own, xs_own, h_own, hs_own, ys_own, counter;
  ib.base = (int32_t*)transients.take(index_bytes, index_own);
  int32_t* const build = (int32_t*)transients.take(scratch_bytes, scratch);
  int32_t* violations = build;
  if (check) {
    counter = at::zeros({4}, at::TensorOptions().dtype(at::kInt).device(dev));
    violations = counter.data_ptr<int32_t>();
  }
  MOMOE_CALL(momoe_index_build, st, mask.data_ptr<int32_t>(), mask.stride(0), mask.stride(1), M, N, K, sizes.data_ptr<int64_t>(),
             ib.cumsums(), ib.idx(), build + 4, ib.inv(), ib.table(), (int)ib.tile_rows, (int32_t*)nullptr,
             (void*)(build + 4 + ((msum + 3) & ~(int64_t)3)), ws_bytes, violations);
  void *h, *ys;
  const int type = type_of(x.scalar_type());
  if (few) {
    h = transients.take(h_bytes, h_own);
    MOMOE_CALL(momoe_fp8_few_lin1_swiglu_fwd, st, x.data_ptr(), type, D, W1.data_ptr(), (const float*)S1.data_ptr(), ib.idx(), ib.table(),
               (float*)h, M, D, H, N, msum);
    ys = transients.take(msum * D * 2, ys_own);
    MOMOE_CALL(momoe_fp8_few_lin2_scale_fwd, st, (const float*)h, W2.data_ptr(), (const float*)S2.data_ptr(), s.data_ptr<float>(), s.stride(0),
               s.stride(1), ib.idx(), ib.table(), ys, M, D, H, N, msum);
  } else {
    void* const xq = transients.take(xq_bytes, xq_own);
    void* const xs = transients.take(xs_bytes, xs_own);
    MOMOE_CALL(momoe_fp8_quantize_rows, st, x.data_ptr(), type, D, M, D, xq, xs);
    h = transients.take(h_bytes, h_own);
    void* const hs = transients.take(hs_bytes, hs_own);
    MOMOE_CALL(momoe_fp8_lin1_swiglu_fwd, st, xq, xs, W1.data_ptr(), (const float*)S1.data_ptr(), ib.idx(), ib.table(), h, hs, M, D, H, N, msum);
    ys = transients.take(msum * D * 2, ys_own);
    MOMOE_CALL(momoe_fp8_lin2_scale_fwd, st, h, hs, W2.data_ptr(), (const float*)S2.data_ptr(), s.data_ptr<float>(), s.stride(0), s.stride(1),
               ib.idx(), ib.table(), ys, M, D, H, N, msum);
  }
  MOMOE_CALL(momoe_fp8_combine, st, ys, ib.inv(), y.data_ptr(), M, D, K, msum);
  if (check) {
    const int v = counter.narrow(0, 0, 1).item<int32_t>();
    TORCH_CHECK(v == 0, "mask_NM: ", v, " tokens do not have exactly K = ", K, " experts (or the mask holds more than M*K pairs)");
  }
  return {x_BSD.device() == dev ? y : y.to(x_BSD.device()), sizes};
}

// ---- dense block ---------------------------------------------------------------------------------
// [M, D] bf16 rows on a 16-byte boundary, of the device the weights are on; any other type is rounded to bf16
Tensor rows_in_bf16(const Tensor& x, int64_t M, int64_t D, const at::Device& dev) {
  Tensor rows = x.reshape({M, D}).to(dev, at::kBFloat16);
  // (pitches that the kernels take, and momoe_wgrad of a gradient)
  const int64_t ld = M > 1 ? rows.stride(0) : D;
  if (rows.stride(1) != 1 || ld < D || ld % 8 != 0 || ld >= (1 << 22) || (ld > D && M * ld * 2 >= (1ll << 32))) rows = rows.contiguous();
  if ((uintptr_t)rows.data_ptr() % 16 != 0) rows = rows.clone(at::MemoryFormat::Contiguous);
  return rows;
}
int64_t pitch_of_rows(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
// a weight as the kernels read it
Tensor packed_bf16(const Tensor& W) {
  const Tensor w = W.to(at::kBFloat16).contiguous();
  return (uintptr_t)w.data_ptr() % 16 != 0 ? w.clone() : w;
}
Tensor fragments(int64_t rows, int64_t cols, const at::Device& dev) { return empty_f32({momoe_ffn_fragment_floats(rows, cols)}, dev); }

struct FeedForward {
  Tensor y;
  Tensor x, W1, W2, ab;  // for the backward
};

// a | b of the first `msave` rows are kept
FeedForward feed_forward_forward(const Tensor& x, const Tensor& W1, const Tensor& W2, int64_t msave) {
  const at::Device dev = W1.device();
  const int64_t D = W1.size(0), H = W2.size(0), M = x.numel() / D;
  const c10::DeviceGuard guard(dev);
  const hipStream_t st = stream_of(dev);
  FeedForward f;
  f.y = empty_bf16(x.sizes(), dev);
  f.x = rows_in_bf16(x, M, D, dev);
  f.W1 = packed_bf16(W1);
  f.W2 = packed_bf16(W2);
  if (M > 0) {
    if (msave > 0) f.ab = fragments(msave, 2 * H, dev);
    const int64_t ws_bytes = momoe_ffn_workspace_bytes(M, D, H);
    const int64_t ldm = momoe_ffn_h_rows(M), h_bytes = ldm * H * 2;
    Transients transients(dev, {h_bytes, ws_bytes});
    Tensor h_own, ws_own;
    void* const h = transients.take(h_bytes, h_own);
    MOMOE_CALL(momoe_ffn_lin1_fwd, st, f.x.data_ptr(), pitch_of_rows(f.x), f.W1.data_ptr(), h, msave > 0 ? f.ab.data_ptr<float>() : nullptr,
               (msave + 31) / 32 * 32, M, ldm, D, H);
    void* const ws = ws_bytes > 0 ? transients.take(ws_bytes, ws_own) : nullptr;
    MOMOE_CALL(momoe_ffn_lin2_fwd, st, (const void*)h, f.W2.data_ptr(), f.y.data_ptr(), M, ldm, D, H, ws, ws_bytes);
  }
  if (x.device() != dev) f.y = f.y.to(x.device());
  return f;
}

struct FeedForwardFn : torch::autograd::Function<FeedForwardFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& W1, const Tensor& W2, int64_t msave) {
    FeedForward f = feed_forward_forward(x, W1, W2, msave);
    ctx->save_for_backward({f.x, f.W1, f.W2, f.ab});
    ctx->saved_data["call"] = std::vector<int64_t>{msave, f.W1.device().index(), f.x.size(0), W1.size(0), W2.size(0)};
    return {f.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "FeedForward has no second derivative: call backward without create_graph");
    const std::vector<int64_t> call_of = ctx->saved_data["call"].toIntVector();
    const int64_t msave = call_of[0], M = call_of[2], D = call_of[3], H = call_of[4];
    const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(1), need_w2 = ctx->needs_input_grad(2);
    const at::Device dev(at::kCUDA, (at::DeviceIndex)call_of[1]);
    const c10::DeviceGuard guard(dev);
    const hipStream_t st = stream_of(dev);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& W1 = as_saved(saved[1], "Wl1", dev, at::kBFloat16, {D, 2 * H});
    const Tensor& W2 = as_saved(saved[2], "Wl2", dev, at::kBFloat16, {H, D});
    // (a hook may have brought x back with other strides)
    const Tensor x = rows_in_bf16(as_saved(saved[0], "x", dev, at::kBFloat16, {M, D}, /*packed=*/false), M, D, dev);
    if (msave > 0) as_saved(saved[3], "a|b", dev, at::kFloat, {momoe_ffn_fragment_floats(msave, 2 * H)});
    if (need_w1) out[1] = empty_bf16({D, 2 * H}, dev);
    if (need_w2) out[2] = empty_bf16({H, D}, dev);
    if (M == 0) {
      if (need_x) out[0] = at::empty(grads[0].sizes(), grads[0].options().dtype(at::kBFloat16));
      if (need_w1) out[1].zero_();
      if (need_w2) out[2].zero_();
      return out;
    }
    const Tensor Gy = rows_in_bf16(grads[0], M, D, dev);
    const int64_t ldx = pitch_of_rows(x), ldgy = pitch_of_rows(Gy);
    const int64_t rest = M - msave, ldm = (M + 31) / 32 * 32, gz_bytes = 4 * H * ldm, ht_bytes = need_w2 ? momoe_padded_rows(M, 1) * H * 2 : 0;
    const int64_t u_bytes = rest > 0 ? momoe_ffn_fragment_floats(rest, H) * 4 : 0;
    const int64_t ws_bytes = momoe_ffn_gradients_workspace_bytes(M, D, H, need_x, need_w1, need_w2);
    Transients transients(dev, {16, gz_bytes, ht_bytes, u_bytes, ws_bytes});
    Tensor counts_own, gz_own, ht_own, u_own, ws_own;
    const auto scratch = [&](int64_t bytes, Tensor& own) { return bytes > 0 ? transients.take(bytes, own) : nullptr; };
    int32_t* const counts = (int32_t*)transients.take(16, counts_own);
    void* const gz = transients.take(gz_bytes, gz_own);
    void* const ht = scratch(ht_bytes, ht_own);
    // what lies behind row msave, a multiple of 32
    const auto behind = [&](const void* p, int64_t pitch) { return p ? (void*)((char*)p + msave * pitch * 2) : nullptr; };
    if (msave > 0)
      MOMOE_CALL(momoe_ffn_dgrad_h_saved, st, Gy.data_ptr(), ldgy, W2.data_ptr(), (const float*)saved[3].data_ptr<float>(), gz, ht, counts,
                 M, msave, ldm, D, H);
    if (rest > 0) {
      float* const u = (float*)transients.take(u_bytes, u_own);
      MOMOE_CALL(momoe_ffn_dgrad_h, st, behind(Gy.data_ptr(), ldgy), ldgy, W2.data_ptr(), u, rest, D, H);
      MOMOE_CALL(momoe_ffn_swiglu_bwd, st, behind(x.data_ptr(), ldx), ldx, W1.data_ptr(), (const float*)u, behind(gz, 32), behind(ht, H), counts,
                 M, rest, ldm, D, H);
      u_own.reset();
    }
    Tensor Gx;
    if (need_x) Gx = empty_bf16({M, D}, dev);
    const auto result = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    MOMOE_CALL(momoe_ffn_gradients, st, x.data_ptr(), ldx, Gy.data_ptr(), ldgy, (const void*)gz, (const void*)ht, W1.data_ptr(), (const int32_t*)counts,
               result(Gx), result(out[1]), result(out[2]), scratch(ws_bytes, ws_own), ws_bytes, M, ldm, D, H);
    if (need_x) out[0] = Gx.view(grads[0].sizes()).to(grads[0].device());
    return out;
  }
};

Tensor feed_forward(const Tensor& x, const Tensor& W1, const Tensor& W2, double save_percent) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<Tensor, const Tensor&, const Tensor&, const Tensor&, double>("momoe::feed_forward", x, W1, W2, save_percent);
  if (W1.device() != W2.device())
    throw_python(PyExc_AssertionError, "All weights must be on the same device, but got: Wl1_D2H.device = " + W1.device().str() +
                                           ", Wl2_HD.device = " + W2.device().str());
  TORCH_CHECK(W1.is_cuda(), "FeedForward weights must live on the GPU: there is no CPU compute path");
  if (x.dim() < 1 || W1.dim() != 2 || W2.dim() != 2 || W1.size(0) != x.size(-1) || W2.size(1) != x.size(-1) || W1.size(1) != 2 * W2.size(0))
    throw_python(PyExc_AssertionError, "x [.., D], Wl1_D2H [D,2H] and Wl2_HD [H,D] do not fit together");
  const int64_t D = W1.size(0), H = W2.size(0);
  TORCH_CHECK(D > 0 && H > 0 && D % 32 == 0 && H % 32 == 0 && D < (1 << 22) && H < (1 << 22) && D * H * 4 < (1ll << 32),
              "FeedForward takes D and H that are multiples of 32 and below 4194304 with weights below 4 GiB, got ", D, " and ", H);
  TORCH_CHECK(save_percent >= 0 && save_percent <= 100, "save_percent must be between 0 and 100, got ", save_percent);
  const int64_t M = x.numel() / D;
  if (!wants_autograd({&x, &W1, &W2})) return feed_forward_forward(x, W1, W2, 0).y;
  // what the gradients of the weights do not take (momoe_wgrad): say so now rather than in the backward.  Their rows and columns,
  // and tokens at 32-bit offsets
  TORCH_CHECK(momoe_ffn_gradients_take(D, H, W1.requires_grad(), W2.requires_grad()),
              "FeedForward backward supports weights with gradients of up to 1048576 rows and columns, got D = ", D, " and H = ", H);
  TORCH_CHECK(!(W1.requires_grad() || W2.requires_grad()) || ((M + 31) * D * 2 < (1ll << 32) && 8 * (M + 31) * 64 < (1ll << 32)),
              "FeedForward backward supports batches of less than 4 GiB and 8388608 tokens per call, got ", M, " tokens: split the batch");
  const int64_t part = (int64_t)((double)M * save_percent / 100.0), msave = part == M ? M : part / 32 * 32;
  return FeedForwardFn::apply(x, W1, W2, msave)[0];
}

// ---- blocks with weights in 4 bits --------------------------------------------------------------
bool held_int4(const Tensor& W, const Tensor& S, const at::Device& dev, int64_t N, int64_t R, int64_t C, int64_t group) {
  const auto held = [&](const Tensor& t, at::ScalarType type, int64_t n) {
    return t.device() == dev && t.scalar_type() == type && t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0 && t.numel() == n;
  };
  return held(W, at::kByte, momoe_int4_weight_bytes(N, R, C)) && held(S, at::kInt, momoe_int4_scale_words(N, R, C, (int)group));
}

// x [B, S, D]; W1, W2 packed, S1, S2 words of their scales and zeros; forward only
std::tuple<Tensor, Tensor> experts_int4(const Tensor& x_BSD, const Tensor& W1, const Tensor& S1, const Tensor& W2, const Tensor& S2,
                                        const Tensor& mask_NM, const Tensor& s_NM, int64_t K, int64_t H, int64_t group, bool check) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<std::tuple<Tensor, Tensor>, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                         const Tensor&, const Tensor&, int64_t, int64_t, int64_t, bool>("momoe::experts_int4", x_BSD, W1, S1, W2, S2,
                                                                                       mask_NM, s_NM, K, H, group, check);
  TORCH_CHECK(W1.is_cuda(), "MoMoEInt4 weights must live on the GPU: there is no CPU compute path");
  TORCH_CHECK(!wants_autograd({&x_BSD, &s_NM}),
              "MoMoEInt4 has no backward, and an input requires a gradient: call it under torch.no_grad()");
  const at::Device dev = W1.device();
  if (x_BSD.dim() != 3) throw_python(PyExc_AssertionError, "x_BSD must be [B, S, D]");
  const int64_t B = x_BSD.size(0), S = x_BSD.size(1), D = x_BSD.size(2), M = B * S;
  TORCH_CHECK(K >= 1, "K, the experts of a token, must be at least 1, got ", K);
  const int64_t N = mask_NM.dim() == 2 ? mask_NM.size(0) : 0, msum = M * K;
  if (!held_int4(W1, S1, dev, N, D, 2 * H, group) || !held_int4(W2, S2, dev, N, H, D, group))
    throw_python(PyExc_AssertionError, "x_BSD [B,S,D], mask_NM [N,M] and the packed weights do not fit together");
  const c10::DeviceGuard guard(dev);
  const hipStream_t st = stream_of(dev);
  const Tensor mask = mask_NM.to(dev, at::kInt), s = s_NM.to(dev, at::kFloat);
  TORCH_CHECK(mask.size(1) == M, "mask_NM must be [", N, ", ", M, "]");
  TORCH_CHECK(s.dim() == 2 && s.size(0) == N && s.size(1) == M, "s_NM must be [", N, ", ", M, "]");
  Tensor y = empty_bf16({B, S, D}, dev), sizes = at::empty({N}, at::TensorOptions().dtype(at::kLong).device(dev));
  if (M == 0) return {x_BSD.device() == dev ? y : y.to(x_BSD.device()), sizes.zero_()};
  const Tensor x = rows_in_bf16(x_BSD, M, D, dev);

  // (the taller tiles gather their rows at 32-bit offsets)
  const int tile_rows = M * pitch_of_rows(x) * 2 >= (1ll << 32) ? 32 : momoe_int4_tile_rows(msum, D, H, N);
  const int64_t slices1 = momoe_int4_slices(msum, N, 2 * H, D, tile_rows), slices2 = momoe_int4_slices(msum, N, D, H, tile_rows);
  const int64_t ws1_bytes = slices1 > 1 ? slices1 * msum * 2 * H * 4 : 0, ys_bytes = slices2 * msum * D * 4;
  Index ib(M, N, K, tile_rows, false);
  const int64_t ws_bytes = momoe_index_workspace_bytes(M, N), index_bytes = ib.ints * 4;
  const int64_t scratch_bytes = (4 + ((msum + 3) & ~(int64_t)3) + (ws_bytes + 3) / 4) * 4;
  const int64_t h_bytes = momoe_int4_h_rows(msum, N) * H * 2;
  Transients transients(dev, {index_bytes, scratch_bytes, h_bytes, ws1_bytes, ys_bytes});
  Tensor index_own, scratch, h_own, ws_own, ys_own, counter;
  ib.base = (int32_t*)transients.take(index_bytes, index_own);
  int32_t* const build = (int32_t*)transients.take(scratch_bytes, scratch);
  int32_t* violations = build;
  if (check) {
    counter = at::zeros({4}, at::TensorOptions().dtype(at::kInt).device(dev));
    violations = counter.data_ptr<int32_t>();
  }
  MOMOE_CALL(momoe_index_build, st, mask.data_ptr<int32_t>(), mask.stride(0), mask.stride(1), M, N, K, sizes.data_ptr<int64_t>(),
             ib.cumsums(), ib.idx(), build + 4, ib.inv(), ib.table(), tile_rows, (int32_t*)nullptr,
             (void*)(build + 4 + ((msum + 3) & ~(int64_t)3)), ws_bytes, violations);
  void* const h = transients.take(h_bytes, h_own);
  void* const ws1 = ws1_bytes > 0 ? transients.take(ws1_bytes, ws_own) : nullptr;
  MOMOE_CALL(momoe_int4_lin1_swiglu_fwd, st, x.data_ptr(), pitch_of_rows(x), W1.data_ptr(), S1.data_ptr(), (int)group,
             (const int32_t*)ib.idx(), (const int32_t*)ib.table(), tile_rows, h, ws1, ws1_bytes, M, D, H, N, msum);
  ws_own.reset();
  float* const ys = (float*)transients.take(ys_bytes, ys_own);
  MOMOE_CALL(momoe_int4_lin2_scale_fwd, st, h, W2.data_ptr(), S2.data_ptr(), (int)group, (const float*)s.data_ptr<float>(), s.stride(0),
             s.stride(1), (const int32_t*)ib.idx(), (const int32_t*)ib.table(), tile_rows, ys, M, D, H, N, msum);
  MOMOE_CALL(momoe_int4_combine, st, (const float*)ys, (int)slices2, (const int32_t*)ib.inv(), y.data_ptr(), M, D, K, msum);
  if (check) {
    const int v = counter.narrow(0, 0, 1).item<int32_t>();
    TORCH_CHECK(v == 0, "mask_NM: ", v, " tokens do not have exactly K = ", K, " experts (or the mask holds more than M*K pairs)");
  }
  return {x_BSD.device() == dev ? y : y.to(x_BSD.device()), sizes};
}

// x [.., D]; a dense block
Tensor feed_forward_int4(const Tensor& x, const Tensor& W1, const Tensor& S1, const Tensor& W2, const Tensor& S2, int64_t H,
                         int64_t group) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<Tensor, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, int64_t>(
        "momoe::feed_forward_int4", x, W1, S1, W2, S2, H, group);
  TORCH_CHECK(W1.is_cuda(), "FeedForwardInt4 weights must live on the GPU: there is no CPU compute path");
  TORCH_CHECK(!wants_autograd({&x}), "FeedForwardInt4 has no backward, and x requires a gradient: call it under torch.no_grad()");
  const at::Device dev = W1.device();
  if (x.dim() < 1) throw_python(PyExc_AssertionError, "x must be [.., D]");
  const int64_t D = x.size(-1);
  if (!held_int4(W1, S1, dev, 1, D, 2 * H, group) || !held_int4(W2, S2, dev, 1, H, D, group))
    throw_python(PyExc_AssertionError, "x [.., D] and the packed weights do not fit together");
  const int64_t M = x.numel() / D;
  const c10::DeviceGuard guard(dev);
  const hipStream_t st = stream_of(dev);
  Tensor y = empty_bf16(x.sizes(), dev);
  if (M > 0) {
    const Tensor rows = rows_in_bf16(x, M, D, dev);
    const int64_t ws_bytes = momoe_int4_ffn_workspace_bytes(M, D, H);
    const int64_t h_bytes = momoe_int4_h_rows(M, 1) * H * 2;
    Transients transients(dev, {h_bytes, ws_bytes});
    Tensor h_own, ws_own;
    void* const h = transients.take(h_bytes, h_own);
    void* const ws = ws_bytes > 0 ? transients.take(ws_bytes, ws_own) : nullptr;
    MOMOE_CALL(momoe_int4_ffn_fwd, st, rows.data_ptr(), pitch_of_rows(rows), W1.data_ptr(), S1.data_ptr(), W2.data_ptr(),
               S2.data_ptr(), (int)group, h, y.data_ptr(), ws, ws_bytes, M, D, H);
  }
  return x.device() == dev ? y : y.to(x.device());
}

// ---- router ------------------------------------------------------------------------------------
struct Routed {
  Tensor x_MD, mask, s_MN, p_sel, norms;
  Tensor logits;  // of `keep_logits`
};
Routed router_forward(const Tensor& x_BSD, const Tensor& Wg, const Tensor& biases, int64_t N, int64_t K, int64_t Ks,
                      bool keep_logits = false) {
  const at::Device dev = Wg.device();
  const int64_t D = x_BSD.size(2), M = x_BSD.size(0) * x_BSD.size(1);
  const c10::DeviceGuard guard(dev);
  Routed r;
  r.x_MD = x_BSD.reshape({M, D}).to(dev, at::kBFloat16);
  // Few tokens: the product in the library's kernel, whose launch alone takes the host 18 us
  const int64_t ws_bytes = momoe_gate_router_workspace_bytes(M, D, N);
  const auto aligned = [](const Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0; };
  const bool own = ws_bytes >= 0 && !at::autocast::is_autocast_enabled(at::kCUDA) && Wg.dim() == 2 && Wg.size(0) == D &&
                   Wg.size(1) == N && Wg.is_contiguous() && aligned(Wg) && aligned(r.x_MD) && r.x_MD.stride(1) == 1 &&
                   r.x_MD.stride(0) >= D && r.x_MD.stride(0) % 8 == 0;
  // Other products come first of all: the GPU has work while the host allocates
  Tensor logits;
  if (!own) {
    // autocast may give the product another type than its operands'; the kernel reads two of them
    logits = at::mm(r.x_MD, Wg).contiguous();
    if (logits.scalar_type() != at::kBFloat16 && logits.scalar_type() != at::kFloat)
      throw_python(PyExc_AssertionError, std::string("the gate logits must be bfloat16 or float32, got ") +
                                             c10::toString(logits.scalar_type()));
    TORCH_CHECK(logits.size(1) == N, "Wg_DN must have N = ", N, " columns");
  }
  const Tensor bias = biases.to(dev, at::kFloat).contiguous();
  TORCH_CHECK(bias.numel() == N, "biases_N must have N = ", N, " elements");
  r.mask = at::empty({N, M}, at::TensorOptions().dtype(at::kInt).device(dev));
  r.s_MN = empty_f32({M, N}, dev);
  r.p_sel = empty_f32({M, N}, dev);
  r.norms = empty_f32({2, M}, dev);  // per token: sum over the selected, over the shared experts
  float* norms = r.norms.data_ptr<float>();
  const hipStream_t st = stream_of(dev);
  if (own) {
    const Tensor ws = empty_f32({ws_bytes / 4}, dev);
    if (keep_logits) r.logits = empty_bf16({M, N}, dev);
    call("momoe_gate_router_fwd", st, momoe_gate_router_fwd_logits, r.x_MD.data_ptr(), r.x_MD.stride(0), Wg.data_ptr(),
         bias.data_ptr<float>(), M, D, N, K, Ks, r.mask.data_ptr<int32_t>(), r.s_MN.data_ptr<float>(), r.p_sel.data_ptr<float>(), norms,
         norms + M, keep_logits ? r.logits.data_ptr() : nullptr, ws.data_ptr(), ws_bytes);
    return r;
  }
  MOMOE_CALL(momoe_router_fwd, st, logits.data_ptr(), logits.scalar_type() == at::kFloat, bias.data_ptr<float>(), M, N, K, Ks,
             r.mask.data_ptr<int32_t>(), r.s_MN.data_ptr<float>(), r.p_sel.data_ptr<float>(), norms, norms + M);
  if (keep_logits) r.logits = logits;
  return r;
}

// x^T . G_logits [D, N].  (The library's product has few tiles and one long contraction for each, and takes the host 18 us where
// two launches take 8: 300 tokens, D = 512, N = 64 9.0 us of the GPU against 9.6; 1024, 1024, 32 9.3, 8.9; 2000, 1120, 48 19.6, 9.4;
// 8192, 2048, 128 60, 22.)  The own kernel's partial sums are D * N at the least, written and read for each range of tokens:
// it takes more than 2^18 results only from a token for 1024 of them on, and up to 2^20, where the library's tiles
// fill the chip.  Us, 300 tokens, D = 2048, N = 128 10.3, 11.6; 1000, 2048, 256 14.7, 15.9; 4096, 2048, 256 29.9, 21.3;
// 4096, 2048, 512 31.3, 30.3; past the line 300, 2048, 256 9.2, 12.8; 1000, 2048, 512 15.4, 21.9; 4096, 4096, 512 38.5, 47.1; 8192,
// 8192, 512 91, 147 (though 32768, 4096, 512 302, 276).  And the library's where autograd records it.
Tensor gate_gradient(const Tensor& x, const Tensor& G_logit) {
  const int64_t M = x.size(0), D = x.size(1), N = G_logit.size(1);
  const int64_t bytes = momoe_gate_wgrad_workspace_bytes(M, D, N);
  const bool sizes = bytes >= 0 && (D * N <= 1 << 18 || (D * N <= 1 << 20 && D * N <= 1024 * M));
  const bool rows = x.stride(1) == 1 && x.stride(0) >= D && x.stride(0) % 8 == 0 && (uintptr_t)x.data_ptr() % 16 == 0;
  if (!sizes || !rows || at::GradMode::is_enabled() || at::autocast::is_autocast_enabled(at::kCUDA)) return at::mm(x.t(), G_logit);
  const Tensor out = empty_bf16({D, N}, x.device()), ws = empty_f32({bytes / 4}, x.device());
  MOMOE_CALL(momoe_gate_wgrad, stream_of(x.device()), x.data_ptr(), x.stride(0), G_logit.data_ptr(), out.data_ptr(), M, D, N,
             ws.data_ptr(), bytes);
  return out;
}

// G_x + G_logits . Wg^T [M, D]; G_x may be undefined.  (The library copies G_x in front of its product, and takes the host 14 us
// more.)  The own kernel reloads both operands for every 32 experts and waits for each: with more than 128 experts it takes
// products of up to 2^31 terms.  In a graph, us, the library's -> own: 8192 tokens, D = 2048, N = 128 32.4 -> 26.1; 32768, 4096, 128
// 232 -> 198; 1000, 1024, 256 9.9 -> 12.3; 8192, 1024, 256 25.8 -> 22.9; 4096, 1024, 512 20.4 -> 20.8; 1000, 2048, 512 14.2 -> 19.7;
// past the line 4096, 2048, 512 29.7 -> 36.6; 8192, 2048, 256 35.3 -> 39.7; 32768, 4096, 512 299 -> 511.
Tensor gate_input_gradient(const Tensor& G_x, const Tensor& G_logit, const Tensor& Wg) {
  const int64_t M = G_logit.size(0), N = G_logit.size(1), D = Wg.size(0);
  const auto packed = [](const Tensor& t) { return t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0; };
  const bool sizes = momoe_gate_wgrad_workspace_bytes(M, D, N) >= 0 && M < 65535 * 128 && (N <= 128 || M * D * N <= (1ll << 31));
  if (!sizes || !packed(Wg) || (G_x.defined() && !packed(G_x)) || at::GradMode::is_enabled() ||
      at::autocast::is_autocast_enabled(at::kCUDA))
    return G_x.defined() ? at::addmm(G_x, G_logit, Wg.t()) : at::mm(G_logit, Wg.t());
  const Tensor out = empty_bf16({M, D}, G_logit.device());
  MOMOE_CALL(momoe_gate_dgrad, stream_of(G_logit.device()), G_logit.data_ptr(), Wg.data_ptr(),
             G_x.defined() ? (const void*)G_x.data_ptr() : nullptr, out.data_ptr(), M, D, N);
  return out;
}

// Gradient of the gate logits, bf16 [M, N], from that of the gate weights; `saved`: x, Wg, mask, p, s, norms
Tensor router_gradient(const variable_list& saved, const at::Device& dev, const Tensor& G_s_NM, int64_t M, int64_t N, int64_t Ks) {
  const Tensor& mask = as_saved(saved[2], "mask", dev, at::kInt, {N, M});
  const Tensor& p_sel = as_saved(saved[3], "p", dev, at::kFloat, {M, N});
  const Tensor& s_MN = as_saved(saved[4], "s", dev, at::kFloat, {M, N});
  const Tensor& norms = as_saved(saved[5], "norms", dev, at::kFloat, {2, M});
  const Tensor G_s = G_s_NM.to(dev, at::kFloat);
  const Tensor G_logit = empty_bf16({M, N}, dev);
  const float* nrm = norms.data_ptr<float>();
  MOMOE_CALL(momoe_router_bwd, stream_of(dev), G_s.data_ptr<float>(), G_s.stride(0), G_s.stride(1),
             p_sel.data_ptr<float>(), s_MN.data_ptr<float>(), nrm, nrm + M, mask.data_ptr<int32_t>(), M, N,
             Ks, G_logit.data_ptr());
  return G_logit;
}
// The gradients that go back through the gate product: of x to out[0] (G_x, what comes back past the gate, may be undefined), of
// Wg to out[1]; without a gradient of the logits that of Wg is zero
void gate_gradients(AutogradContext* ctx, const variable_list& saved, const at::Device& dev, Tensor G_x, const Tensor& G_logit,
                    at::IntArrayRef x_sizes, int64_t N, variable_list& out) {
  const int64_t M = x_sizes[0] * x_sizes[1], D = x_sizes[2];
  const Tensor& x = as_saved(saved[0], "x", dev, at::kBFloat16, {M, D}, /*packed=*/false);
  const Tensor& Wg = as_saved(saved[1], "Wg", dev, at::kBFloat16, {D, N}, /*packed=*/false);
  const bool need_x = ctx->needs_input_grad(0), need_wg = ctx->needs_input_grad(1);
  if (G_logit.defined()) {
    if (need_x) G_x = gate_input_gradient(G_x, G_logit, Wg);
    if (need_wg) out[1] = gate_gradient(x, G_logit);
  } else if (need_wg) {
    out[1] = at::zeros_like(Wg);
  }
  if (need_x && G_x.defined()) out[0] = G_x.reshape(x_sizes);
}

struct RouterFn : torch::autograd::Function<RouterFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& Wg, const Tensor& biases,
                               int64_t N, int64_t K, int64_t Ks) {
    Routed r = router_forward(x, Wg, biases, N, K, Ks);
    ctx->save_for_backward({r.x_MD, Wg, r.mask, r.p_sel, r.s_MN, r.norms});
    ctx->saved_data["call"] = std::vector<int64_t>{Ks, N, Wg.device().index(), x.size(0), x.size(1), x.size(2)};
    ctx->mark_non_differentiable({r.mask});
    ctx->set_materialize_grads(false);
    return {x, r.mask, r.s_MN.t()};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> call_of = ctx->saved_data["call"].toIntVector();
    const at::Device dev(at::kCUDA, (at::DeviceIndex)call_of[2]);
    const int64_t Ks = call_of[0], N = call_of[1], M = call_of[3] * call_of[4], D = call_of[5];
    const c10::DeviceGuard guard(dev);
    const Tensor &G_x_BSD = grads[0], &G_s_NM = grads[2];
    Tensor G_x, G_logit;
    if (G_x_BSD.defined()) G_x = G_x_BSD.reshape({M, D}).to(dev, at::kBFloat16);
    if (G_s_NM.defined()) G_logit = router_gradient(saved, dev, G_s_NM, M, N, Ks);
    variable_list out(6);
    gate_gradients(ctx, saved, dev, G_x, G_logit, {call_of[3], call_of[4], D}, N, out);
    return out;
  }
};

void check_router(const Tensor& x, const Tensor& Wg) {
  if (Wg.scalar_type() != at::kBFloat16) throw_python(PyExc_AssertionError, "Wg_DN must be of type torch.bfloat16");
  TORCH_CHECK(Wg.is_cuda(), "TopKRouter weights must live on the GPU: there is no CPU compute path");
  TORCH_CHECK(x.dim() == 3, "x_BSD must be [B, S, D]");
}

std::tuple<Tensor, Tensor, Tensor> router(const Tensor& x, const Tensor& Wg, const Tensor& biases, int64_t N, int64_t K,
                                          int64_t Ks) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<std::tuple<Tensor, Tensor, Tensor>, const Tensor&, const Tensor&, const Tensor&, int64_t,
                         int64_t, int64_t>("momoe::router", x, Wg, biases, N, K, Ks);
  check_router(x, Wg);
  if (!wants_autograd({&x, &Wg})) {
    Routed r = router_forward(x, Wg, biases, N, K, Ks);
    return {x, r.mask, r.s_MN.t()};
  }
  variable_list r = RouterFn::apply(x, Wg, biases, N, K, Ks);
  return {r[0], r[1], r[2]};
}

// ---- balance loss ------------------------------------------------------------------------------
// Rows that the kernels walk with one pitch: [M, N] of unit column stride
bool has_rows(const Tensor& t) { return t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) == 1 || t.stride(0) >= t.size(1)); }
Tensor rows_of(const Tensor& t, int64_t M, int64_t N) {
  const Tensor rows = t.reshape({M, N});
  return has_rows(rows) ? rows : rows.contiguous();
}
Tensor flags_of(const Tensor& valid, int64_t M) { return valid.reshape({M}).contiguous(); }
int64_t pitch_of(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

struct Balanced {
  Tensor loss, counts;  // results: [], [groups, N]
  // For the backward, with the logits.  `valid` may be undefined, and has the shape that it came in.  `kept`: info, and behind it the
  // counts once more: the others are the caller's, who may sum them over ranks before the backward, which autograd does not see.
  // (One tensor: each takes the host 1.5 us to make, save and find.)
  Tensor valid, kept;
};
// int64 places of info, of which it takes half of one for each group and one for all; kept_of: those of `kept`
int64_t info_of(int64_t groups) { return groups / 2 + 1; }
int64_t kept_of(int64_t groups, int64_t N) { return info_of(groups) + groups * N; }

// logits [.., N] of one of the three types, `groups` of as many tokens each; `valid` as check_valid takes it
Balanced balance_forward(const Tensor& logits, const Tensor& mask_NM, int64_t Ks, const std::optional<Tensor>& valid,
                         int64_t groups, bool for_backward) {
  const at::Device dev = logits.device();
  const int64_t N = logits.size(-1), M = logits.numel() / N;
  const c10::DeviceGuard guard(dev);
  Balanced b;
  const Tensor rows = rows_of(logits, M, N);
  const Tensor mask = mask_NM.to(dev, at::kInt);
  TORCH_CHECK(mask.dim() == 2 && mask.size(0) == N && mask.size(1) == M, "mask_NM must be [", N, ", ", M, "]");
  Tensor flags;
  if (valid.has_value()) {
    b.valid = valid->to(dev);
    flags = flags_of(b.valid, M);
  }
  b.counts = at::empty({groups, N}, at::TensorOptions().dtype(at::kLong).device(dev));
  b.kept = at::empty({for_backward ? kept_of(groups, N) : info_of(groups)}, b.counts.options());
  b.loss = empty_f32({}, dev);
  if (M == 0) {
    b.counts.zero_();
    b.kept.zero_();
    b.loss.zero_();
    return b;
  }
  const int64_t S = M / groups, ws_bytes = momoe_balance_workspace_bytes(groups, S, N);
  TORCH_CHECK(ws_bytes >= 0, "balance loss: [", M, ", ", N, "] logits are past the sizes that it takes (N <= 512)");
  const Tensor ws = empty_f32({ws_bytes / 4}, dev);
  call("momoe_balance_fwd", stream_of(dev), momoe_balance_fwd_kept, rows.data_ptr(), type_of(rows.scalar_type()), pitch_of(rows),
       mask.data_ptr<int32_t>(), mask.stride(0), mask.stride(1), flags.defined() ? (const uint8_t*)flags.data_ptr() : nullptr, groups, S,
       N, Ks, b.loss.data_ptr<float>(), b.counts.data_ptr<int64_t>(), for_backward ? b.kept.data_ptr<int64_t>() + info_of(groups) : nullptr,
       (float*)b.kept.data_ptr(), ws.data_ptr(), ws_bytes);
  return b;
}

// What the forward saved, as balance_gradient takes it: logits, valid, kept from `saved[at]` on
struct BalanceSaved {
  Tensor logits, valid, kept;
  int64_t groups;
  BalanceSaved(const variable_list& saved, size_t at, const at::Device& dev, at::ScalarType type, at::IntArrayRef sizes, int64_t M,
               int64_t N, int64_t groups_)
      : groups(groups_) {
    logits = rows_of(as_saved(saved[at], "logits", dev, type, sizes, /*packed=*/false), M, N);
    if (saved[at + 1].defined()) {
      const Tensor& v = saved[at + 1];
      TORCH_CHECK(v.numel() == M, "backward: the saved tensor valid came back from its hook in another size");
      valid = flags_of(as_saved(v, "valid", dev, at::kBool, v.sizes(), /*packed=*/false), M);
    }
    kept = as_saved(saved[at + 2], "counts", dev, at::kLong, {kept_of(groups, N)});
  }
};

// d loss / d logits, of type `type`, + `add` in its place if that is defined
Tensor balance_gradient(const BalanceSaved& t, const Tensor& G_loss, int64_t Ks, at::ScalarType type, const Tensor& add) {
  const at::Device dev = t.logits.device();
  const int64_t M = t.logits.size(0), N = t.logits.size(1);
  const Tensor g = G_loss.to(dev, at::kFloat).contiguous();
  Tensor out = add.defined() ? add : at::empty({M, N}, at::TensorOptions().dtype(type).device(dev));
  if (M == 0) return out;
  MOMOE_CALL(momoe_balance_bwd, stream_of(dev), t.logits.data_ptr(), type_of(t.logits.scalar_type()), pitch_of(t.logits),
             t.valid.defined() ? (const uint8_t*)t.valid.data_ptr() : nullptr, t.kept.data_ptr<int64_t>() + info_of(t.groups),
             (const float*)t.kept.data_ptr(), g.data_ptr<float>(), add.defined() ? (const void*)add.data_ptr() : nullptr, out.data_ptr(),
             type_of(type), t.groups, M / t.groups, N, Ks);
  return out;
}

struct BalanceFn : torch::autograd::Function<BalanceFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& mask, int64_t Ks,
                               const std::optional<Tensor>& valid, int64_t groups) {
    Balanced b = balance_forward(logits, mask, Ks, valid, groups, /*for_backward=*/true);
    // (logits and valid as they came: a view made here would hide from autograd that they changed since)
    ctx->save_for_backward({logits, b.valid, b.kept});
    ctx->saved_data["call"] = std::vector<int64_t>{Ks, groups, logits.device().index(), (int64_t)logits.scalar_type()};
    ctx->saved_data["sizes"] = logits.sizes().vec();
    ctx->mark_non_differentiable({b.counts});
    ctx->set_materialize_grads(false);
    return {b.loss, b.counts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "balance_loss has no second derivative: call backward without create_graph");
    const std::vector<int64_t> call_of = ctx->saved_data["call"].toIntVector();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const at::ScalarType type = (at::ScalarType)call_of[3];
    const at::Device dev(at::kCUDA, (at::DeviceIndex)call_of[2]);
    const c10::DeviceGuard guard(dev);
    const BalanceSaved t(ctx->get_saved_variables(), 0, dev, type, sizes, c10::multiply_integers(sizes.begin(), sizes.end() - 1),
                         sizes.back(), call_of[1]);
    out[0] = balance_gradient(t, grads[0], call_of[0], type, {}).view(sizes);
    return out;
  }
};

// Groups of a call: its sequences, or all of its tokens
int64_t groups_of(at::IntArrayRef sizes, bool per_sequence) {
  TORCH_CHECK(!per_sequence || sizes.size() == 3, "per_sequence takes [B, S, N] logits or [B, S, D] tokens");
  return per_sequence ? sizes[0] : 1;
}

// One flag a token, in their order: as many in another shape would be those of other tokens.  `sizes`: of the tokens and their
// logits or values, [M, ..] or [B, S, ..]
void check_valid(const std::optional<Tensor>& valid, at::IntArrayRef sizes) {
  if (!valid.has_value()) return;
  const at::IntArrayRef tokens = sizes.slice(0, sizes.size() - 1);
  const int64_t M = c10::multiply_integers(tokens);
  const bool shape = valid->dim() == 1 || (valid->dim() == 2 && (tokens.size() == 1 || valid->sizes() == tokens));
  TORCH_CHECK(valid->scalar_type() == at::kBool && shape && valid->numel() == M, "valid must be a bool tensor with a flag for each of the ",
              tokens, " tokens, in that shape or in one dimension, got ", valid->scalar_type(), " ", valid->sizes());
}

std::tuple<Tensor, Tensor> balance_loss(const Tensor& logits, const Tensor& mask, int64_t Ks, const std::optional<Tensor>& valid,
                                        bool per_sequence) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<std::tuple<Tensor, Tensor>, const Tensor&, const Tensor&, int64_t, const std::optional<Tensor>&, bool>(
        "momoe::balance_loss", logits, mask, Ks, valid, per_sequence);
  TORCH_CHECK(logits.is_cuda(), "balance_loss needs logits on the GPU: there is no CPU compute path");
  if (type_of(logits.scalar_type()) < 0)
    throw_python(PyExc_AssertionError, std::string("the logits must be bfloat16, float32 or float16, got ") +
                                           c10::toString(logits.scalar_type()));
  TORCH_CHECK(logits.dim() == 2 || logits.dim() == 3, "logits must be [M, N] or [B, S, N]");
  const int64_t N = logits.size(-1), groups = groups_of(logits.sizes(), per_sequence);
  TORCH_CHECK(Ks >= 0 && Ks < N, "num_shared_experts must be between 0 and N - 1 = ", N - 1, ", got ", Ks);
  TORCH_CHECK(N <= 512, "balance_loss takes up to 512 experts, got ", N);
  check_valid(valid, logits.sizes());
  Tensor loss, counts;
  if (wants_autograd({&logits})) {
    variable_list r = BalanceFn::apply(logits, mask, Ks, valid, groups);
    loss = r[0], counts = r[1];
  } else {
    Balanced b = balance_forward(logits, mask, Ks, valid, groups, /*for_backward=*/false);
    loss = b.loss, counts = b.counts;
  }
  return {loss, per_sequence ? counts : counts.select(0, 0)};
}

// The router and, of its logits, the balance loss: one gradient of the logits goes back through the gate product
struct BalancedRouterFn : torch::autograd::Function<BalancedRouterFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& Wg, const Tensor& biases, int64_t N, int64_t K,
                               int64_t Ks, const std::optional<Tensor>& valid, int64_t groups) {
    Routed r = router_forward(x, Wg, biases, N, K, Ks, /*keep_logits=*/true);
    Balanced b = balance_forward(r.logits, r.mask, Ks, valid, groups, /*for_backward=*/true);
    ctx->save_for_backward({r.x_MD, Wg, r.mask, r.p_sel, r.s_MN, r.norms, r.logits, b.valid, b.kept});
    ctx->saved_data["call"] = std::vector<int64_t>{Ks, N, Wg.device().index(), x.size(0), x.size(1), x.size(2), groups,
                                                   (int64_t)r.logits.scalar_type()};
    ctx->mark_non_differentiable({r.mask, b.counts});
    ctx->set_materialize_grads(false);
    return {x, r.mask, r.s_MN.t(), b.loss, b.counts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> call_of = ctx->saved_data["call"].toIntVector();
    const at::Device dev(at::kCUDA, (at::DeviceIndex)call_of[2]);
    const c10::DeviceGuard guard(dev);
    const int64_t Ks = call_of[0], N = call_of[1], M = call_of[3] * call_of[4], D = call_of[5];
    const Tensor &G_x_BSD = grads[0], &G_s_NM = grads[2], &G_loss = grads[3];
    Tensor G_x, G_logit;
    if (G_x_BSD.defined()) G_x = G_x_BSD.reshape({M, D}).to(dev, at::kBFloat16);
    if (G_s_NM.defined()) G_logit = router_gradient(saved, dev, G_s_NM, M, N, Ks);
    if (G_loss.defined()) {
      TORCH_CHECK(!at::GradMode::is_enabled(), "the balance loss has no second derivative: call backward without create_graph");
      const BalanceSaved t(saved, 6, dev, (at::ScalarType)call_of[7], {M, N}, M, N, call_of[6]);
      // (where both come back the router's is rounded to bf16 first, as without the loss, and their sum again: two half steps)
      G_logit = balance_gradient(t, G_loss, Ks, at::kBFloat16, G_logit);
    }
    variable_list out(8);
    gate_gradients(ctx, saved, dev, G_x, G_logit, {call_of[3], call_of[4], D}, N, out);
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> router_balanced(const Tensor& x, const Tensor& Wg, const Tensor& biases, int64_t N,
                                                                   int64_t K, int64_t Ks, const std::optional<Tensor>& valid,
                                                                   bool per_sequence) {
  if (torch::jit::tracer::isTracing())
    return call_recorded<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>, const Tensor&, const Tensor&, const Tensor&, int64_t,
                         int64_t, int64_t, const std::optional<Tensor>&, bool>("momoe::router_balanced", x, Wg, biases, N, K, Ks,
                                                                               valid, per_sequence);
  check_router(x, Wg);
  TORCH_CHECK(Ks >= 0 && Ks < N, "the balance loss needs a routed expert: ", N, " experts, ", Ks, " of them shared");
  const int64_t groups = groups_of(x.sizes(), per_sequence);
  check_valid(valid, x.sizes());
  variable_list r;
  if (wants_autograd({&x, &Wg})) {
    r = BalancedRouterFn::apply(x, Wg, biases, N, K, Ks, valid, groups);
  } else {
    Routed t = router_forward(x, Wg, biases, N, K, Ks, /*keep_logits=*/true);
    Balanced b = balance_forward(t.logits, t.mask, Ks, valid, groups, /*for_backward=*/false);
    r = {x, t.mask, t.s_MN.t(), b.loss, b.counts};
  }
  return {r[0], r[1], r[2], r[3], per_sequence ? r[4] : r[4].select(0, 0)};
}

// biases += rate * sign(c_avg - sizes), in place, in fp32
void bias_update(Tensor biases, const Tensor& sizes, double c_avg, double rate) {
  const c10::DeviceGuard guard(biases.device());
  MOMOE_CALL(momoe_bias_update, stream_of(biases.device()), sizes.data_ptr<int64_t>(), (float)c_avg, (float)rate,
             biases.numel(), biases.data_ptr<float>());
  biases.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

// The operators of a traced call.  A graph keeps the integers and flags it was traced with, the sizes
// are those of the tensors it is run on.
TORCH_LIBRARY(momoe, m) {
  m.def("experts(Tensor x_BSD, Tensor Wl1_ND2H, Tensor Wl2_NHD, Tensor mask_NM, Tensor s_NM, int K, "
        "float save_percent, int tile_rows, bool check) -> (Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(experts)));
  m.def("router(Tensor(a) x_BSD, Tensor Wg_DN, Tensor biases_N, int N, int K, int Ks) -> (Tensor(a), Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(router)));
  m.def("experts_fp8(Tensor x_BSD, Tensor Wl1, Tensor Wl1_scale_bits, Tensor Wl2, Tensor Wl2_scale_bits, Tensor mask_NM, Tensor s_NM, int K, "
        "int H, bool check) -> (Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(experts_fp8)));
  m.def("feed_forward(Tensor x, Tensor Wl1_D2H, Tensor Wl2_HD, float save_percent) -> Tensor",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(feed_forward)));
  m.def("experts_int4(Tensor x_BSD, Tensor Wl1, Tensor Wl1_words, Tensor Wl2, Tensor Wl2_words, Tensor mask_NM, Tensor s_NM, int K, int H, "
        "int group, bool check) -> (Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(experts_int4)));
  m.def("feed_forward_int4(Tensor x, Tensor Wl1, Tensor Wl1_words, Tensor Wl2, Tensor Wl2_words, int H, int group) -> Tensor",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(feed_forward_int4)));
  m.def("balance_loss(Tensor logits, Tensor mask_NM, int Ks, Tensor? valid, bool per_sequence) -> (Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(balance_loss)));
  m.def("router_balanced(Tensor(a) x_BSD, Tensor Wg_DN, Tensor biases_N, int N, int K, int Ks, Tensor? valid, bool per_sequence) "
        "-> (Tensor(a), Tensor, Tensor, Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(router_balanced)));
}

PYBIND11_MODULE(_layer, m) {
  m.def("experts", &experts, py::call_guard<py::gil_scoped_release>());
  m.def("experts_fp8", &experts_fp8, py::call_guard<py::gil_scoped_release>());
  m.def("feed_forward", &feed_forward, py::call_guard<py::gil_scoped_release>());
  m.def("experts_int4", &experts_int4, py::call_guard<py::gil_scoped_release>());
  m.def("feed_forward_int4", &feed_forward_int4, py::call_guard<py::gil_scoped_release>());
  m.def("router", &router, py::call_guard<py::gil_scoped_release>());
  m.def("balance_loss", &balance_loss, py::call_guard<py::gil_scoped_release>());
  m.def("router_balanced", &router_balanced, py::call_guard<py::gil_scoped_release>());
  m.def("bias_update", &bias_update, py::call_guard<py::gil_scoped_release>());
  m.def("timing_start", &timing_start);
  m.def("timing_stop", &timing_stop);
  m.def("timing_take", &timing_take);
  // a library call made from Python, recorded like those made here
  m.def("timed", [](const std::string& name, uintptr_t stream, const py::function& fn) {
    return timed(name.c_str(), (hipStream_t)stream, [&] { return py::object(fn()); });
  });
}

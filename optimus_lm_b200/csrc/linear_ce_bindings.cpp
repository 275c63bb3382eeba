// Python bindings of the cross entropy from hidden states: the launch sequences of forward and backward.
//
// The exponentials (bf16, [tokens, V]) are kept within the caller's workspace limit, in one of three ways:
//   they fit                 : forward = product + finish, exponentials and row factors are kept; backward = the two
//                              gradient products, straight to bf16 with the incoming gradient in the row factors.
//   pieces of the batch      : for one scalar loss the incoming gradient is a common factor, so forward runs the gradient
//                              products of each piece too (dX to bf16, dW summed in fp32) and backward scales them (one
//                              more rounding of dX unless the gradient is a power of two); every logit is computed once, 6 T H V
//                              operations in all.  Needs the fp32 dW within the limit as well, or where none is
//                              wanted the exponentials of 256 rows.
//   pieces of the vocabulary : losses per row, whose gradients the forward does not know, or a weight too large for the
//                              fp32 dW.  Forward keeps four floats per row (what its exponentials were relative to, ce_grow,
//                              their sum, 1 / Z); backward computes the same exponentials again, 8 T H V
//                              operations in all, dX summed in fp32 over the pieces, dW's rows finished piece by piece.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <atomic>
#include <limits>

#include "olb_api.h"

namespace {

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Launches of this file so far: their number depends on sizes and limits, and the backward is not called through Python.
std::atomic<int64_t> launches{0};

inline void check(int rc, const char* what, int n = 1) {
  TORCH_CHECK(rc == 0, std::string(what) + " failed with code " + std::to_string(rc));
  launches += n;
}

enum { MEAN = 0, SUM = 1, NONE = 2 };

// What forward leaves to backward: the exponentials and row factors; or the gradients of a scalar loss (dx, and dw in
// fp32; undefined where not wanted); or the rows' sum, 1 / Z, reference and ce_grow, as [4, T].
enum { PIECE = 0, SCALE = 1, AGAIN = 2 };
struct Kept {
  int64_t kind = PIECE;
  at::Tensor a, b;
};

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Problem {
  at::Tensor x, w, targets;
  int64_t T, H, V, lde;
  int* status;
  cudaStream_t stream;
};

Problem make_problem(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, const at::Tensor& status) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() == 2 && x.stride(1) == 1, "x must be a 2D CUDA bf16 tensor with unit inner stride");
  TORCH_CHECK(w.is_cuda() && w.scalar_type() == at::kBFloat16 && w.dim() == 2 && w.stride(1) == 1, "weight must be a 2D CUDA bf16 tensor with unit inner stride");
  TORCH_CHECK(targets.is_cuda() && targets.scalar_type() == at::kLong && targets.dim() == 1 && targets.is_contiguous(), "targets must be a contiguous 1D CUDA int64 tensor");
  TORCH_CHECK(x.device() == w.device() && x.device() == targets.device() && x.device() == status.device(), "x, weight, targets must be on one device");
  TORCH_CHECK(x.size(1) == w.size(1) && x.size(0) == targets.size(0), "shapes of x, weight, targets do not match");
  TORCH_CHECK(x.size(1) % 8 == 0 && x.size(1) > 0 && w.size(0) > 0, "the hidden size must be a positive multiple of 8");
  TORCH_CHECK(x.size(0) < (1ll << 31) - 256 && w.size(0) < (1ll << 31) - 256 && w.size(1) < (1ll << 31), "too many rows");
  return {x, w, targets, x.size(0), x.size(1), w.size(0), round_up(w.size(0), 64), status.data_ptr<int>(), cur_stream()};
}

int64_t piece_rows(int64_t T, int64_t bytes_per_row, int64_t max_bytes) {
  const int64_t most = std::max<int64_t>(256, max_bytes / bytes_per_row / 256 * 256);
  const int64_t n = std::max<int64_t>(1, (T + most - 1) / most);
  return n == 1 ? T : round_up((T + n - 1) / n, 256);
}

const long long* ptr_i64(const at::Tensor& t, int64_t at) { return reinterpret_cast<const long long*>(t.data_ptr<int64_t>()) + at; }
void* row_ptr(const at::Tensor& t, int64_t row) { return static_cast<char*>(t.data_ptr()) + row * t.stride(0) * t.element_size(); }

// Runs an OLB_EPI_ROWSCALE product with the scratch that its last wave wants.
void rowscale_product(const Problem& p, olb_gemm_desc& d, const char* what) {
  d.epilogue = OLB_EPI_ROWSCALE;
  d.wide_tiles = 1;
  d.status = p.status;
  const long long floats = olb_gemm_tail_floats(&d);
  at::Tensor scratch;
  if (floats > 0) {
    scratch = at::empty({floats}, p.x.options().dtype(at::kFloat));
    d.tail_part = scratch.data_ptr<float>();
  } else if (d.row_scale == nullptr) {
    d.epilogue = OLB_EPI_PLAIN;   // neither factors nor a split: 2 to 3 us less for 50304 x 2048
  }
  check(olb_gemm_bf16(&d, p.stream), what, floats > 0 ? 2 : 1);
}

// e = exp(l - ref) of some rows and columns [v0, v0 + cols) of the vocabulary (and the sums of their tiles), then of the
// row blocks that need another reference.
void product(const Problem& p, int64_t r0, int64_t rows, int64_t v0, int64_t cols, const float* ref, const float* grow,
             unsigned* top, int* flags, float* part, int64_t part_ld, void* E, int64_t lde, bool behind_prep) {
  olb_gemm_desc d{};
  d.A = row_ptr(p.x, r0);
  d.B = row_ptr(p.w, v0);
  d.C = E;
  d.lda = p.x.stride(0);
  d.ldb = p.w.stride(0);
  d.ldc = lde;
  d.a_rows = rows;
  d.b_rows = cols;
  d.M = static_cast<int>(rows);
  d.N = static_cast<int>(cols);
  d.K = static_cast<int>(p.H);
  d.ce_v0 = static_cast<int>(v0);
  d.ce_v_total = static_cast<int>(p.V);
  d.epilogue = OLB_EPI_CE;
  d.status = p.status;
  d.ce_targets = ptr_i64(p.targets, r0);
  d.ce_ref = ref;
  d.ce_grow = grow;
  d.ce_max = top;
  d.ce_flags = flags;
  d.ce_part = part;
  d.ce_part_ld = part_ld;
  d.overlap = behind_prep;
  check(olb_gemm_bf16(&d, p.stream), "olb_gemm_bf16 (cross entropy)");
  if (flags) {
    d.overlap = 1;
    d.ce_repair = 1;
    check(olb_gemm_bf16(&d, p.stream), "olb_gemm_bf16 (cross entropy, repair)");
  }
}

// dx[r0 .. r0 + rows) = row_factor * (E W).  behind_factors: the launch before it makes row_factor and not E.
void input_gradient(const Problem& p, int64_t r0, int64_t rows, const void* E, const float* row_factor, at::Tensor& dx,
                    bool behind_factors) {
  olb_gemm_desc d{};
  d.A = E;
  d.B = p.w.data_ptr();
  d.C = row_ptr(dx, r0);
  d.lda = p.lde;
  d.ldb = p.w.stride(0);
  d.ldc = p.H;
  d.a_rows = rows;
  d.b_rows = p.V;
  d.M = static_cast<int>(rows);
  d.N = static_cast<int>(p.H);
  d.K = static_cast<int>(p.V);
  d.b_mn_major = 1;
  d.overlap = behind_factors;
  d.row_scale = row_factor;
  rowscale_product(p, d, "olb_gemm_bf16 (input gradient)");
}

// Rows [v0, v0 + cols) of dw (=, += or, in fp32, reduced into) E^T xs
void weight_gradient(const Problem& p, int64_t rows, int64_t v0, int64_t cols, const void* E, int64_t lde, const void* xs,
                     at::Tensor& dw, bool add) {
  olb_gemm_desc d{};
  d.A = E;
  d.B = xs;
  d.C = row_ptr(dw, v0);
  d.lda = lde;
  d.ldb = p.H;
  d.ldc = dw.stride(0);
  d.a_rows = rows;
  d.b_rows = rows;
  d.M = static_cast<int>(cols);
  d.N = static_cast<int>(p.H);
  d.K = static_cast<int>(rows);
  d.a_mn_major = d.b_mn_major = 1;
  if (dw.scalar_type() == at::kBFloat16) {
    d.accumulate = add;
    rowscale_product(p, d, "olb_gemm_bf16 (weight gradient)");
    return;
  }
  d.wide_tiles = 1;
  d.status = p.status;
  d.out_fp32 = 1;
  d.c_reduce = add;
  check(olb_gemm_bf16(&d, p.stream), "olb_gemm_bf16 (weight gradient)");
}

at::Tensor weight_gradient_out(const Problem& p, const c10::optional<at::Tensor>& dw_out, bool accumulate) {
  if (!dw_out.has_value()) {
    TORCH_CHECK(!accumulate, "nothing to accumulate into");
    return at::empty({p.V, p.H}, p.w.options());
  }
  TORCH_CHECK(dw_out->scalar_type() == at::kBFloat16 && dw_out->device() == p.w.device() && dw_out->is_contiguous() &&
              dw_out->dim() == 2 && dw_out->size(0) == p.V && dw_out->size(1) == p.H, "dw_out must be a contiguous bf16 [V, H] tensor");
  return *dw_out;
}

// The loss: a scalar, or [T] for NONE.
at::Tensor linear_ce_fwd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, int64_t reduction,
                         bool need_dx, bool need_dw, int64_t max_bytes, const at::Tensor& status, Kept& kept) {
  TORCH_CHECK(reduction >= MEAN && reduction <= NONE);
  c10::cuda::CUDAGuard guard(x.device());
  const Problem p = make_problem(x, w, targets, status);
  const bool grad = need_dx || need_dw;
  const auto f32 = x.options().dtype(at::kFloat);
  if (p.T == 0) {
    at::Tensor out = reduction == NONE ? at::empty({0}, f32)
                                       : at::full({}, reduction == MEAN ? std::numeric_limits<double>::quiet_NaN() : 0.0, f32);
    kept = {PIECE, at::empty({0, p.lde}, x.options()), at::empty({0}, f32)};
    return out;
  }
  int64_t rows_max = piece_rows(p.T, grad ? 2 * p.lde : 4 * ((p.V + 15) / 16), max_bytes);
  const bool single = rows_max >= p.T;
  // pieces of the batch: the weight's fp32 gradient fits, or none is wanted and the smallest piece's exponentials fit
  const bool in_pieces = reduction != NONE && (4 * p.V * p.H <= max_bytes || (!need_dw && 2 * p.lde * 256 <= max_bytes));
  const bool store = grad && (single || in_pieces);
  if (grad && !store) rows_max = piece_rows(p.T, 4 * ((p.V + 15) / 16), max_bytes);
  // sums per row, of whole pieces and of a shorter last one
  const int64_t last = p.T - (p.T - 1) / rows_max * rows_max;
  const int64_t ntiles_most = std::max(olb_gemm_ce_slices(static_cast<int>(std::min(rows_max, p.T)), static_cast<int>(p.V)),
                                       olb_gemm_ce_slices(static_cast<int>(last), static_cast<int>(p.V)));

  at::Tensor out = reduction == NONE ? at::empty({p.T}, f32) : at::empty({}, f32);
  // small per-row and per-launch words: (losses,) ref, grow, top, flags, ticket, count, 1 / count
  const int64_t losses = reduction == NONE ? 0 : p.T;
  at::Tensor words = at::empty({losses + 3 * rows_max + (rows_max + 127) / 128 + 1 + 3}, f32);
  float* loss_rows = reduction == NONE ? out.data_ptr<float>() : words.data_ptr<float>();
  float* ref = words.data_ptr<float>() + losses;
  float* grow = ref + rows_max;
  unsigned* top = reinterpret_cast<unsigned*>(grow + rows_max);
  int* flags = reinterpret_cast<int*>(top + rows_max);
  unsigned* ticket = reinterpret_cast<unsigned*>(flags + (rows_max + 127) / 128 + 1);
  float* count = reinterpret_cast<float*>(ticket + 1);
  at::Tensor part = at::empty({ntiles_most, rows_max}, f32);
  at::Tensor E, factor, dx, dw32, stats, xs;
  if (store) {
    E = at::empty({rows_max, p.lde}, x.options());
    factor = at::empty({rows_max}, f32);
  }
  const bool in_forward = store && !single;
  if (in_forward) {
    if (need_dx) dx = at::empty({p.T, p.H}, x.options());
    if (need_dw) {
      dw32 = at::empty({p.V, p.H}, f32);
      xs = at::empty({rows_max, p.H}, x.options());
    }
  }
  if (grad && !store) stats = at::empty({4, p.T}, f32);
  for (int64_t r0 = 0; r0 < p.T; r0 += rows_max) {
    const int64_t rows = std::min(rows_max, p.T - r0);
    if (stats.defined()) grow = stats.data_ptr<float>() + 3 * p.T + r0;
    check(olb_lce_prep(row_ptr(x, r0), x.stride(0), w.data_ptr(), w.stride(0), ptr_i64(p.targets, r0), static_cast<int>(rows),
                       static_cast<int>(p.H), static_cast<int>(p.V), ref, grow, top, flags, ticket, ptr_i64(p.targets, 0), p.T,
                       reduction == MEAN && r0 == 0 ? count : nullptr, p.stream),
          "olb_lce_prep");
    product(p, r0, rows, 0, p.V, ref, grow, top, flags, part.data_ptr<float>(), rows_max, store ? E.data_ptr() : nullptr, p.lde, true);
    olb_lce_finish_desc f{};
    f.part = part.data_ptr<float>();
    f.part_ld = rows_max;
    f.ntiles = olb_gemm_ce_slices(static_cast<int>(rows), static_cast<int>(p.V));
    f.ref = ref;
    f.ce_max = top;
    f.targets = ptr_i64(p.targets, r0);
    f.rows = static_cast<int>(rows);
    f.V = static_cast<int>(p.V);
    f.H = static_cast<int>(p.H);
    f.loss = loss_rows + r0;
    if (stats.defined()) {
      f.sum = stats.data_ptr<float>() + r0;
      f.inv_z = f.sum + p.T;
      f.base = f.inv_z + p.T;
    }
    if (store) {
      f.E = E.data_ptr();
      f.lde = p.lde;
      f.factor = factor.data_ptr<float>();
    }
    if (grad) f.scale = reduction == MEAN ? count + 1 : nullptr;
    if (xs.defined()) {
      f.x = row_ptr(x, r0);
      f.ldx = x.stride(0);
      f.xs = xs.data_ptr();
    }
    if (reduction != NONE && r0 + rows == p.T) {
      f.ticket = ticket;
      f.loss_all = loss_rows;
      f.n_all = p.T;
      f.total = out.data_ptr<float>();
      f.total_scale = reduction == MEAN ? count : nullptr;
    }
    check(olb_lce_finish(&f, p.stream), "olb_lce_finish");
    if (in_forward) {
      if (need_dx) input_gradient(p, r0, rows, E.data_ptr(), factor.data_ptr<float>(), dx, false);
      if (need_dw) weight_gradient(p, rows, 0, p.V, E.data_ptr(), p.lde, xs.data_ptr(), dw32, r0 > 0);
    }
  }
  if (in_forward) kept = {SCALE, dx, dw32};
  else if (store) kept = {PIECE, E, factor};
  else kept = {AGAIN, stats};
  return out;
}

// One piece: E and factor as the forward left them; grad is a scalar or [T].  Returns {dx, dw} (undefined where not
// wanted; dw is dw_out when that is given).
std::vector<at::Tensor> linear_ce_bwd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, const at::Tensor& E,
                                      const at::Tensor& factor, const at::Tensor& grad, bool need_dx, bool need_dw,
                                      const c10::optional<at::Tensor>& dw_out, bool accumulate, const at::Tensor& status) {
  c10::cuda::CUDAGuard guard(x.device());
  const Problem p = make_problem(x, w, targets, status);
  TORCH_CHECK(grad.scalar_type() == at::kFloat && grad.device() == x.device() && grad.is_contiguous() &&
              (grad.numel() == 1 || grad.numel() == p.T), "grad must be one fp32 value or one for each row");
  TORCH_CHECK(E.scalar_type() == at::kBFloat16 && E.size(0) >= p.T && E.size(1) == p.lde && E.is_contiguous() && factor.numel() >= p.T);
  at::Tensor dx, dw;
  if (need_dx) dx = at::empty({p.T, p.H}, x.options());
  if (need_dw) dw = weight_gradient_out(p, dw_out, accumulate);
  if (p.T == 0) {
    if (need_dw && !accumulate) dw.zero_();
    return {dx, dw};
  }
  at::Tensor row_factor = at::empty({p.T}, x.options().dtype(at::kFloat));
  at::Tensor xs = need_dw ? at::empty({p.T, p.H}, x.options()) : at::Tensor();
  check(olb_lce_scale_rows(x.data_ptr(), x.stride(0), factor.data_ptr<float>(), grad.data_ptr<float>(),
                           grad.dim() == 0 ? 0 : 1, static_cast<int>(p.T), static_cast<int>(p.H), row_factor.data_ptr<float>(),
                           need_dw ? xs.data_ptr() : nullptr, p.stream),
        "olb_lce_scale_rows");
  if (need_dx) input_gradient(p, 0, p.T, E.data_ptr(), row_factor.data_ptr<float>(), dx, true);
  if (need_dw) weight_gradient(p, p.T, 0, p.V, E.data_ptr(), p.lde, xs.data_ptr(), dw, accumulate);
  return {dx, dw};
}

// Several pieces of a scalar loss: the gradients of the forward times the incoming gradient.
std::vector<at::Tensor> linear_ce_bwd_scale(const at::Tensor& dx_in, const at::Tensor& dw32, const at::Tensor& grad,
                                            const c10::optional<at::Tensor>& dw_out, bool accumulate) {
  const at::Tensor& any = dx_in.defined() ? dx_in : dw32;
  c10::cuda::CUDAGuard guard(any.device());
  TORCH_CHECK(grad.scalar_type() == at::kFloat && grad.numel() == 1 && grad.device() == any.device());
  at::Tensor dx, dw;
  if (dx_in.defined()) {
    dx = at::empty_like(dx_in);
    check(olb_lce_scale_out(dx_in.data_ptr(), 1, dx.numel(), grad.data_ptr<float>(), dx.data_ptr(), 0, cur_stream()), "olb_lce_scale_out");
  }
  if (dw32.defined()) {
    TORCH_CHECK(!accumulate || dw_out.has_value());
    dw = dw_out.has_value() ? *dw_out : at::empty(dw32.sizes(), dw32.options().dtype(at::kBFloat16));
    TORCH_CHECK(dw.scalar_type() == at::kBFloat16 && dw.is_contiguous() && dw.sizes() == dw32.sizes() && dw.device() == dw32.device());
    check(olb_lce_scale_out(dw32.data_ptr(), 0, dw.numel(), grad.data_ptr<float>(), dw.data_ptr(), accumulate, cur_stream()), "olb_lce_scale_out");
  }
  return {dx, dw};
}

// Pieces of the vocabulary: the forward's exponentials again, against the references that it recorded.
std::vector<at::Tensor> linear_ce_bwd_again(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets,
                                            const at::Tensor& stats, const at::Tensor& grad, bool need_dx, bool need_dw,
                                            int64_t max_bytes, const c10::optional<at::Tensor>& dw_out, bool accumulate,
                                            const at::Tensor& status) {
  c10::cuda::CUDAGuard guard(x.device());
  const Problem p = make_problem(x, w, targets, status);
  TORCH_CHECK(grad.scalar_type() == at::kFloat && grad.device() == x.device() && grad.is_contiguous() &&
              (grad.dim() == 0 || grad.numel() == p.T) && stats.is_contiguous() && stats.numel() == 4 * p.T);
  const float *sum = stats.data_ptr<float>(), *inv_z = sum + p.T, *base = inv_z + p.T, *grow = base + p.T;
  const auto f32 = x.options().dtype(at::kFloat);
  const int64_t most = std::max<int64_t>(256, max_bytes / (2 * p.T) / 256 * 256);
  const int64_t pieces = (p.V + most - 1) / most;
  const int64_t cols_max = pieces == 1 ? p.V : round_up((p.V + pieces - 1) / pieces, 256), lde = round_up(cols_max, 64);
  const int T = static_cast<int>(p.T), H = static_cast<int>(p.H), V = static_cast<int>(p.V);
  at::Tensor E = at::empty({p.T, lde}, x.options());
  at::Tensor factors = at::empty({2, p.T}, f32);
  float *factor = factors.data_ptr<float>(), *row_factor = factor + p.T;
  at::Tensor dx, dx32, dw, xs;
  if (need_dx) dx32 = at::empty({p.T, p.H}, f32);
  if (need_dw) {
    dw = weight_gradient_out(p, dw_out, accumulate);
    xs = at::empty({p.T, p.H}, x.options());
  }
  check(olb_lce_patch(sum, inv_z, ptr_i64(p.targets, 0), T, V, factor, 0, 0, nullptr, 0, p.stream), "olb_lce_patch");
  check(olb_lce_scale_rows(x.data_ptr(), x.stride(0), factor, grad.data_ptr<float>(), grad.dim() == 0 ? 0 : 1, T, H, row_factor,
                           need_dw ? xs.data_ptr() : nullptr, p.stream),
        "olb_lce_scale_rows");
  for (int64_t v0 = 0; v0 < p.V; v0 += cols_max) {
    const int64_t cols = std::min(cols_max, p.V - v0);
    product(p, 0, p.T, v0, cols, base, grow, nullptr, nullptr, nullptr, 0, E.data_ptr(), lde, false);
    check(olb_lce_patch(sum, inv_z, ptr_i64(p.targets, 0), T, V, nullptr, static_cast<int>(v0), static_cast<int>(cols), E.data_ptr(),
                        lde, p.stream),
          "olb_lce_patch");
    if (need_dx) {
      olb_gemm_desc d{};
      d.A = E.data_ptr();
      d.B = row_ptr(p.w, v0);
      d.C = dx32.data_ptr();
      d.lda = lde;
      d.ldb = p.w.stride(0);
      d.ldc = p.H;
      d.a_rows = p.T;
      d.b_rows = cols;
      d.M = T;
      d.N = H;
      d.K = static_cast<int>(cols);
      d.b_mn_major = 1;
      d.wide_tiles = 1;
      d.status = p.status;
      d.out_fp32 = 1;
      d.c_reduce = v0 > 0;
      check(olb_gemm_bf16(&d, p.stream), "olb_gemm_bf16 (input gradient)");
    }
    if (need_dw) weight_gradient(p, p.T, v0, cols, E.data_ptr(), lde, xs.data_ptr(), dw, accumulate);
  }
  if (need_dx) {
    dx = at::empty({p.T, p.H}, x.options());
    check(olb_lce_round_rows(dx32.data_ptr<float>(), T, H, row_factor, dx.data_ptr(), p.stream), "olb_lce_round_rows");
  }
  return {dx, dw};
}

// A gradient buffer of ops/functional.py (DirectGrad): `buf`, and `ready` = it holds a gradient of this step already.
struct GradHolder : torch::CustomClassHolder {
  pybind11::object obj;
  explicit GradHolder(pybind11::object o) : obj(std::move(o)) {}
  ~GradHolder() override {
    if (!Py_IsInitialized()) {  // a graph that outlives the interpreter
      obj.release();
      return;
    }
    pybind11::gil_scoped_acquire gil;
    obj = pybind11::object();
  }
};

// The autograd node lives here rather than in Python: a training step of a small batch is bound by the host, and the
// Python form of the same node took 190 us for 65 us of kernels.
struct LinearCE : torch::autograd::Function<LinearCE> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const at::Tensor& targets, int64_t reduction, bool need_dx, bool need_dw, int64_t max_bytes,
                            const at::Tensor& status, const c10::intrusive_ptr<GradHolder>& holder) {
    Kept kept;
    at::Tensor out = linear_ce_fwd(x, w, targets, reduction, need_dx, need_dw, max_bytes, status, kept);
    ctx->save_for_backward({x, w, targets, kept.a, kept.b});
    ctx->saved_data["status"] = status;  // cleared in place by whoever reads it
    ctx->saved_data["kind"] = kept.kind;
    ctx->saved_data["need"] = static_cast<int64_t>(need_dx) + 2 * static_cast<int64_t>(need_dw);
    ctx->saved_data["max_bytes"] = max_bytes;
    if (holder) ctx->saved_data["holder"] = c10::IValue::make_capsule(holder);
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy cannot be differentiated twice");
    const auto saved = ctx->get_saved_variables();
    const int64_t kind = ctx->saved_data["kind"].toInt(), need = ctx->saved_data["need"].toInt();
    const bool need_dx = need & 1, need_dw = need & 2;
    const at::Tensor grad = grads[0].to(at::kFloat).contiguous();
    c10::optional<at::Tensor> into;
    bool add = false;
    c10::intrusive_ptr<GradHolder> holder;
    if (need_dw && ctx->saved_data.count("holder")) {
      holder = c10::static_intrusive_pointer_cast<GradHolder>(ctx->saved_data["holder"].toCapsule());
      pybind11::gil_scoped_acquire gil;
      into = holder->obj.attr("buf").cast<at::Tensor>();
      add = holder->obj.attr("ready").cast<bool>();
    }
    const at::Tensor &x = saved[0], &w = saved[1], &targets = saved[2], &a = saved[3], &b = saved[4];
    const at::Tensor status = ctx->saved_data["status"].toTensor();
    auto got = kind == PIECE   ? linear_ce_bwd(x, w, targets, a, b, grad, need_dx, need_dw, into, add, status)
               : kind == SCALE ? linear_ce_bwd_scale(a, b, grad, into, add)
                               : linear_ce_bwd_again(x, w, targets, a, grad, need_dx, need_dw, ctx->saved_data["max_bytes"].toInt(),
                                                     into, add, status);
    if (holder) {
      pybind11::gil_scoped_acquire gil;
      holder->obj.attr("ready") = true;
      got[1] = at::Tensor();
    }
    at::Tensor none;
    return {got[0], got[1], none, none, none, none, none, none, none};
  }
};

// Rows that a tensor map can describe: 2D, unit inner stride, 16-byte rows that do not overlap.
at::Tensor as_rows(const at::Tensor& t) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  const bool fits = r.stride(1) == 1 && r.stride(0) % 8 == 0 && r.stride(0) >= r.size(1) &&
                    reinterpret_cast<uintptr_t>(r.const_data_ptr()) % 16 == 0;
  return fits ? r : r.clone(at::MemoryFormat::Contiguous);
}

// The checks of ops/functional.py's plain path, for CUDA tensors; nothing for types and sizes that the kernels do not take.
c10::optional<at::Tensor> linear_ce(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, int64_t reduction,
                                    int64_t max_bytes, const at::Tensor& status, const pybind11::object& holder) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1), "x [..., H] and weight [V, H] do not match");
  TORCH_CHECK_VALUE(targets.sizes() == x.sizes().slice(0, x.dim() - 1), "targets must have the shape of x without its last axis");
  TORCH_CHECK_VALUE(at::isIntegralType(targets.scalar_type(), false), "targets must be integers");
  TORCH_CHECK_VALUE(weight.numel() > 0, "weight is empty");
  TORCH_CHECK_VALUE(x.device() == weight.device() && x.device() == targets.device(), "x, weight and targets are on different devices");
  TORCH_CHECK_VALUE(max_bytes > 0, "max_workspace must be positive");
  if (x.scalar_type() != at::kBFloat16 || weight.scalar_type() != at::kBFloat16 || weight.size(1) % 8) return c10::nullopt;
  // with or without gradients: a call without a node would lose the tangent
  TORCH_CHECK_NOT_IMPLEMENTED(!x._fw_grad(0).defined() && !weight._fw_grad(0).defined(),
                              "linear_cross_entropy has no forward-mode derivative for bf16 CUDA tensors");
  const at::Tensor x2 = as_rows(x), w = as_rows(weight);
  const at::Tensor flat = (targets.dim() == 1 ? targets : targets.reshape({-1})).to(at::kLong).contiguous();
  const bool grad = at::GradMode::is_enabled();
  const bool need_dx = grad && x2.requires_grad(), need_dw = grad && w.requires_grad();
  at::Tensor out;
  if (need_dx || need_dw) {
    c10::intrusive_ptr<GradHolder> h;
    if (!holder.is_none() && weight.is_contiguous() && w.is_same(weight)) h = c10::make_intrusive<GradHolder>(holder);
    out = LinearCE::apply(x2, w, flat, reduction, need_dx, need_dw, max_bytes, status, h);
  } else {
    Kept kept;
    out = linear_ce_fwd(x2, w, flat, reduction, false, false, max_bytes, status, kept);
  }
  return reduction == NONE && targets.dim() != 1 ? out.view(targets.sizes()) : out;
}

}  // namespace

void register_linear_ce(pybind11::module& m) {
  m.def("linear_ce", &linear_ce);
  m.def("linear_ce_launches", [] { return launches.load(); });
}

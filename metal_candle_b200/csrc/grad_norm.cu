// The 2-norm of many gradient tensors taken as one vector, and clipping by it:
//   norm = sqrt(sum g^2);  g <- g min(1, max_norm / (norm + 1e-6))
// Two launches whatever the number of tensors (up to 512 a launch): the first leaves a partial sum of squares of each of its blocks,
// in the second every block adds these up for itself, in their order, and scales its share; an optimiser's update takes the factor
// the same way (adamw.cu).  No atomics, so the same gradients give the same bits.
//
// HBM-bound: the gradients are read twice (the second time from L2 where they fit its 126 MB) and written once.  The tensors are cut into pieces of 4096
// elements that are dealt out over all blocks, so that tensors of a thousand and of a hundred million elements share a launch.
//
// Squares are summed in float32 by a thread (16 elements, then in float64).  Where a thread's largest magnitude is outside [2^-50, 2^50] its squares are
// taken in float64: the norm of gradients near either end of float32 is right.  It is NaN or inf where an element is, and reads inf where it passes the largest
// float32, which does not keep finite gradients from being clipped by it.
#include "grad_norm.cuh"

namespace mcb {
namespace gnorm {
namespace {

constexpr int kThreads = 256, kMaxTensors = 512, kPiece = 4096;

struct Tensor {
  const void* g;
  void* out;
  int64_t n;
  uint32_t first;   // number of its first piece
  int32_t dtype;
};
struct Table {
  Tensor t[kMaxTensors];
  int count;
  uint32_t pieces;
};
static_assert(sizeof(Table) < 32000, "fits the kernel parameters");

__device__ __forceinline__ const Tensor& tensor_of(const Table& tab, uint32_t piece) {
  int lo = 0, hi = tab.count - 1;   // the last tensor whose first piece is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first <= piece) lo = mid;
    else hi = mid - 1;
  }
  return tab.t[lo];
}

// The 16 elements of a thread in its piece, which begins at element `at`: N at a time, N * (tid + 256 k) on.  VEC: N == 1, or g + at is on a 16-byte boundary.
// N > 1 without it reads the N elements one by one: they are the same lines, from L1.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_piece(const T* g, int64_t n, int64_t at, float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 16 / N; ++k) {
    const int64_t i = at + N * (threadIdx.x + kThreads * k);
#pragma unroll
    for (int e = 0; e < N; ++e) v[N * k + e] = 0.0f;
    if (N > 1 && VEC && i + N <= n) {
      if constexpr (N > 1) {
        Vec16<T> x;
        x.raw = *reinterpret_cast<const decltype(x.raw)*>(g + i);
        x.to_float(v + N * k);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e < n) v[N * k + e] = to_f32(g[i + e]);
    }
  }
}

__device__ __forceinline__ double squares(const float (&v)[16]) {
  float top = 0.0f, s = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    top = fmaxf(top, fabsf(v[e]));
    s = fmaf(v[e], v[e], s);
  }
  if (top == 0.0f || (top >= 0x1p-50f && top <= 0x1p50f)) return s;   // (a NaN is in s either way)
  double d = 0.0;
  for (int e = 0; e < 16; ++e) d += static_cast<double>(v[e]) * v[e];
  return d;
}

template <typename T>
__device__ __forceinline__ void load_tensor(const Tensor& t, int64_t at, float (&v)[16]) {
  const T* g = static_cast<const T*>(t.g);
  // (off a boundary neighbouring threads take neighbouring elements, so that a warp's access is whole lines again)
  if ((reinterpret_cast<uintptr_t>(g) & 15u) == 0) load_piece<T, Vec16<T>::N, true>(g, t.n, at, v);
  else load_piece<T, 1, true>(g, t.n, at, v);
}
__device__ __forceinline__ void load_number(const Table& tab, uint32_t piece, float (&v)[16]) {
  const Tensor& t = tensor_of(tab, piece);
  const int64_t at = static_cast<int64_t>(piece - t.first) * kPiece;
  if (t.dtype == MCB_F32) load_tensor<float>(t, at, v);
  else load_tensor<__nv_bfloat16>(t, at, v);
}

__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Table tab, double* part) {
  __shared__ double s[kThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  double sum = 0.0;
  // the next piece is on its way while one is summed
  float v[2][16];
  uint32_t piece = blockIdx.x;
  if (piece < tab.pieces) load_number(tab, piece, v[0]);
  while (piece < tab.pieces) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (piece >= tab.pieces) break;
      if (piece + gridDim.x < tab.pieces) load_number(tab, piece + gridDim.x, v[1 - i]);
      sum += squares(v[i]);
      piece += gridDim.x;
    }
  }
  sum = block_sum(sum, s);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* part, int parts, float* norm) {
  __shared__ double s[kThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const double v = norm_of(part, parts, s);
  if (threadIdx.x == 0) norm[0] = static_cast<float>(v);
}

// Pieces go by the output's 16-byte boundaries, the first few elements of a tensor by themselves: what is written are whole vectors
// (written element by element, 250 M elements that lie off the gradients' alignment took 421 us instead of 350).
template <typename T>
__device__ __forceinline__ int head_of(const Tensor& t) {
  return static_cast<int>((16 - (reinterpret_cast<uintptr_t>(t.out) & 15u)) % 16 / sizeof(T));
}
template <typename T>
__device__ __forceinline__ void load_for_clip(const Tensor& t, int64_t piece, float (&v)[16]) {
  constexpr int N = Vec16<T>::N;
  const T* g = static_cast<const T*>(t.g);
  const int head = head_of<T>(t);
  const int64_t at = head + piece * kPiece;
  if ((reinterpret_cast<uintptr_t>(g + head) & 15u) == 0) load_piece<T, N, true>(g, t.n, at, v);
  else load_piece<T, N, false>(g, t.n, at, v);
}
template <typename T>
__device__ __forceinline__ void clip_piece(const Tensor& t, int64_t piece, float2 f, const float (&v)[16]) {
  constexpr int N = Vec16<T>::N;
  const T* g = static_cast<const T*>(t.g);
  T* out = static_cast<T*>(t.out);
  const int head = head_of<T>(t);
  if (piece == 0 && static_cast<int>(threadIdx.x) < head && threadIdx.x < t.n) out[threadIdx.x] = from_f32<T>(to_f32(g[threadIdx.x]) * f.x * f.y);
  const int64_t at = head + piece * kPiece;
#pragma unroll
  for (int k = 0; k < 16 / N; ++k) {
    const int64_t i = at + N * (threadIdx.x + kThreads * k);
    float w[N];
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = v[N * k + e] * f.x * f.y;
    if (i + N <= t.n) {
      Vec16<T> x;
      x.from_float(w);
      *reinterpret_cast<decltype(x.raw)*>(out + i) = x.raw;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e < t.n) out[i + e] = from_f32<T>(w[e]);
    }
  }
}

__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ Table tab, const double* part, int parts, float max_norm, float* norm) {
  __shared__ double s[kThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  // from the last piece back: what the sums read last is still in L2
  auto tensor = [&](uint32_t i, int64_t& piece) -> const Tensor& {
    const Tensor& t = tensor_of(tab, tab.pieces - 1 - i);
    piece = tab.pieces - 1 - i - t.first;
    return t;
  };
  auto load = [&](uint32_t i, float (&v)[16]) {
    int64_t piece;
    const Tensor& t = tensor(i, piece);
    if (t.dtype == MCB_F32) load_for_clip<float>(t, piece, v);
    else load_for_clip<__nv_bfloat16>(t, piece, v);
  };
  float v[2][16];
  uint32_t i = blockIdx.x;
  const double total = norm_of(part, parts, s);
  const float2 f = clip_factor(total, max_norm, 1.0f);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = static_cast<float>(total);
  if (i < tab.pieces) load(i, v[0]);
  while (i < tab.pieces) {
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      if (i >= tab.pieces) break;
      if (i + gridDim.x < tab.pieces) load(i + gridDim.x, v[1 - turn]);
      int64_t piece;
      const Tensor& t = tensor(i, piece);
      if (t.dtype == MCB_F32) clip_piece<float>(t, piece, f, v[turn]);
      else clip_piece<__nv_bfloat16>(t, piece, f, v[turn]);
      i += gridDim.x;
    }
  }
}

// tensors [base, base + up to 512) as a table; empty ones are left out
int make_table(Table& tab, const mcb_grad_tensor* tensors, int n, const char* who) {
  tab.count = 0;
  int64_t pieces = 0;
  for (int i = 0; i < n; ++i) {
    const mcb_grad_tensor& t = tensors[i];
    if (t.n == 0) continue;
    Tensor& d = tab.t[tab.count++];
    d.g = t.g; d.out = t.out != nullptr ? t.out : const_cast<void*>(t.g); d.n = t.n; d.dtype = t.dtype;
    d.first = static_cast<uint32_t>(pieces);
    pieces += (t.n + kPiece - 1) / kPiece;
    if (pieces > 0x7fffffffll) return fail(MCB_ERR_SHAPE, "%s: more than 2^43 elements", who);
  }
  tab.pieces = static_cast<uint32_t>(pieces);
  return MCB_OK;
}

int check(const mcb_grad_tensor* tensors, int n, const char* who) {
  if (n <= 0) return fail(MCB_ERR_SHAPE, "%s: n_tensors=%d", who, n);
  if (!tensors) return fail(MCB_ERR_NULL, "%s: tensors is null", who);
  for (int i = 0; i < n; ++i) {
    const mcb_grad_tensor& t = tensors[i];
    if (t.n < 0) return fail(MCB_ERR_SHAPE, "%s: tensor %d has n=%lld", who, i, (long long)t.n);
    if (t.n > 0 && !t.g) return fail(MCB_ERR_NULL, "%s: tensor %d is null", who, i);
    if (t.dtype != MCB_F32 && t.dtype != MCB_BF16) return fail(MCB_ERR_UNSUPPORTED, "%s: tensor %d has dtype %d", who, i, t.dtype);
    const uintptr_t mis = reinterpret_cast<uintptr_t>(t.g) | reinterpret_cast<uintptr_t>(t.out);
    if ((mis & (t.dtype == MCB_F32 ? 3u : 1u)) != 0) return fail(MCB_ERR_ALIGN, "%s: tensor %d is not aligned to its elements", who, i);
  }
  return MCB_OK;
}

// Whether some output overlaps another tensor's gradient or output, or its own gradient in part: what one block writes another would read.
bool outputs_collide(const mcb_grad_tensor* tensors, int n) {
  struct Range {
    uintptr_t begin, end;
    int owner;
    bool written;
  };
  std::vector<Range> r;
  r.reserve(2 * static_cast<size_t>(n));
  for (int i = 0; i < n; ++i) {
    const mcb_grad_tensor& t = tensors[i];
    if (t.n == 0) continue;
    const uintptr_t bytes = static_cast<uintptr_t>(t.n) * (t.dtype == MCB_F32 ? 4 : 2), g = reinterpret_cast<uintptr_t>(t.g);
    const uintptr_t o = t.out != nullptr ? reinterpret_cast<uintptr_t>(t.out) : g;
    r.push_back({o, o + bytes, i, true});
    if (o != g) r.push_back({g, g + bytes, i, false});
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t any_end = 0, written_end = 0;   // of the ranges so far
  for (const Range& x : r) {
    if (x.begin < written_end || (x.written && x.begin < any_end)) return true;
    if (x.end > any_end) any_end = x.end;
    if (x.written && x.end > written_end) written_end = x.end;
  }
  return false;
}

constexpr int kMaxBlocks = 2048;
int blocks_for(uint32_t pieces, int sms) {
  const uint32_t most = static_cast<uint32_t>(sms * 8 < kMaxBlocks ? sms * 8 : kMaxBlocks);
  return static_cast<int>(pieces < most ? pieces : most);
}

}  // namespace

size_t workspace_bytes(int n) {
  const int64_t launches = n <= 0 ? 1 : (static_cast<int64_t>(n) + kMaxTensors - 1) / kMaxTensors;
  return static_cast<size_t>(launches) * kMaxBlocks * sizeof(double);
}

int launch_squares(const mcb_grad_tensor* tensors, int n, double* part, int* parts, const DeviceState* ds, cudaStream_t st, const char* who) {
  *parts = 0;
  for (int base = 0; base < n; base += kMaxTensors) {
    Table tab;
    if (int rc = make_table(tab, tensors + base, n - base < kMaxTensors ? n - base : kMaxTensors, who)) return rc;
    if (tab.pieces == 0) continue;
    const int blocks = blocks_for(tab.pieces, ds->sm_count);
    MCB_CHECK_CUDA(launch_kernel(squares_kernel, dim3(blocks), dim3(kThreads), 0, st, chained_launch(), tab, part + *parts));
    MCB_CHECK_LAUNCH("squares_kernel");
    *parts += blocks;
  }
  return MCB_OK;
}

}  // namespace gnorm
}  // namespace mcb

using namespace mcb;

extern "C" size_t mcb_grad_norm_workspace_bytes(int n_tensors) { return gnorm::workspace_bytes(n_tensors); }

extern "C" int mcb_grad_norm(const mcb_grad_tensor* tensors, int n_tensors, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_grad_norm");
  if (int rc = gnorm::check(tensors, n_tensors, "grad_norm")) return rc;
  if (!norm) return fail(MCB_ERR_NULL, "grad_norm: norm is null");
  if (!on_boundary(4, norm)) return fail(MCB_ERR_ALIGN, "grad_norm: norm is not aligned to its elements");
  if (!workspace || workspace_bytes < gnorm::workspace_bytes(n_tensors) || !aligned16(workspace))
    return fail(MCB_ERR_WORKSPACE, "grad_norm: workspace of %zu bytes, 16-byte aligned, needed", gnorm::workspace_bytes(n_tensors));
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  int parts = 0;
  if (int rc = gnorm::launch_squares(tensors, n_tensors, part, &parts, ds, st, "grad_norm")) return rc;
  MCB_CHECK_CUDA(launch_kernel(gnorm::norm_kernel, dim3(1), dim3(gnorm::kThreads), 0, st, chained_launch(), static_cast<const double*>(part), parts, norm));
  MCB_CHECK_LAUNCH("norm_kernel");
  return MCB_OK;
}

extern "C" int mcb_clip_grad_norm(const mcb_grad_tensor* tensors, int n_tensors, float max_norm, float* norm, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_clip_grad_norm");
  if (int rc = gnorm::check(tensors, n_tensors, "clip_grad_norm")) return rc;
  if (!(max_norm >= 0.0f)) return fail(MCB_ERR_SHAPE, "clip_grad_norm: max_norm must not be negative, got %g", max_norm);
  if (!on_boundary(4, norm)) return fail(MCB_ERR_ALIGN, "clip_grad_norm: norm is not aligned to its elements");
  if (!workspace || workspace_bytes < gnorm::workspace_bytes(n_tensors) || !aligned16(workspace))
    return fail(MCB_ERR_WORKSPACE, "clip_grad_norm: workspace of %zu bytes, 16-byte aligned, needed", gnorm::workspace_bytes(n_tensors));
  try {
    if (gnorm::outputs_collide(tensors, n_tensors))
      return fail(MCB_ERR_SHAPE, "clip_grad_norm: an output overlaps another tensor (or a tensor is given twice)");
  } catch (...) {
    return fail(MCB_ERR_SHAPE, "clip_grad_norm: no host memory for %d tensors", n_tensors);
  }
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  int parts = 0;
  if (int rc = gnorm::launch_squares(tensors, n_tensors, part, &parts, ds, st, "clip_grad_norm")) return rc;
  if (parts == 0) {   // nothing but empty tensors
    if (norm) {
      MCB_CHECK_CUDA(launch_kernel(gnorm::norm_kernel, dim3(1), dim3(gnorm::kThreads), 0, st, chained_launch(), static_cast<const double*>(part), 0, norm));
      MCB_CHECK_LAUNCH("norm_kernel");
    }
    return MCB_OK;
  }
  bool first = true;
  for (int base = 0; base < n_tensors; base += gnorm::kMaxTensors) {
    gnorm::Table tab;
    const int cnt = n_tensors - base < gnorm::kMaxTensors ? n_tensors - base : gnorm::kMaxTensors;
    if (int rc = gnorm::make_table(tab, tensors + base, cnt, "clip_grad_norm")) return rc;
    if (tab.pieces == 0) continue;
    MCB_CHECK_CUDA(launch_kernel(gnorm::clip_kernel, dim3(gnorm::blocks_for(tab.pieces, ds->sm_count)), dim3(gnorm::kThreads), 0, st, chained_launch(), tab,
                                 static_cast<const double*>(part), parts, max_norm, first ? norm : nullptr));
    MCB_CHECK_LAUNCH("clip_kernel");
    first = false;
  }
  return MCB_OK;
}

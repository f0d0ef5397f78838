// Counter-based dropout, and the backward pass of the GEMM epilogue
// y = residual + drop(act(z)), z = ga gb A B^T + bias (rb_nvfp4_gemm_epilogue).
//
// Both are bound by HBM traffic: dropout reads x (and the residual) once and writes y once; the
// backward reads dy and z once and writes dz once, and takes the global scale that dz's quantizer
// needs (max |dz| / 2688, quantize.py:205-213) and the bias gradient (dz.sum(0), linear.py:146) from
// the values in registers instead of from two more passes.
#include "epilogue.cuh"

#include <type_traits>

namespace rb {

// ---------------------------------------------------------------------------------------------
// Dropout: y = residual + drop(x), flat over n elements
// ---------------------------------------------------------------------------------------------
// kVec: every pointer is 16-byte aligned, and a thread takes a group of eight elements (one generator call) a
// turn, the next group's loads on their way while it computes.  Otherwise, and for the last n % 8 elements,
// elements go one by one.
// 16384 x 2048 bf16: 29 us (134 MB; a copy takes 23), with a residual 34 (201 MB, 5.9 TB/s); fp32 with a
// residual 68 (5.9 TB/s).  Without a residual the generator's wide multiplies and xors bound it (the heavy half
// of the FMA pipe 62% busy, the ALU 51%); more loads in flight (two or four groups a thread) cost occupancy
// and time, 35 and 42 us.
constexpr int kDropoutBlocksPerSm = 5;

// Eight elements as loaded.  Coherent loads, not the read-only path: the output may be the input itself.  Dropout of
// bf16, where a warp reads whole lines, passes L1 by (kL2: 16384 x 2048 with a residual 33.9 us against 34.8, 16384 x
// 5632 72.4 against 75.5); fp32's two vectors a thread (73.5 us against 69.6) and the epilogue's backward (without an
// activation 64.5 us against 63.1) take it.
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
  template <bool kL2 = false>
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
      const uint4* at = reinterpret_cast<const uint4*>(p) + i;
      if constexpr (kL2) q[i] = __ldcg(at);
      else q[i] = *at;
    }
  }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) v[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
      else v[j] = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    }
  }
};

template <typename T, bool kVec, bool kResidual>
__global__ void __launch_bounds__(256, kDropoutBlocksPerSm) dropout_kernel(const T* x, const T* residual, T* y, int64_t n,
                                                      const DropoutArgs d) {
  const PhiloxKeys key = philox_keys(d.seed);
  const int64_t step = (int64_t)gridDim.x * blockDim.x, first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t groups = kVec ? n / 8 : 0;
  if (kVec && first < groups) {
    constexpr bool kL2 = sizeof(T) == 2;
    Raw8<T> xn, rn;
    xn.template load<kL2>(x + 8 * first);
    if constexpr (kResidual) rn.template load<kL2>(residual + 8 * first);
    for (int64_t g = first; g < groups; g += step) {
      const Raw8<T> xc = xn, rc = rn;
      if (g + step < groups) {
        xn.template load<kL2>(x + 8 * (g + step));
        if constexpr (kResidual) rn.template load<kL2>(residual + 8 * (g + step));
      }
      float2 v[4];
      xc.get(v);
      if (d.seed != nullptr) dropout8(v, (uint64_t)g, key, d.below, d.scale);
      if constexpr (kResidual) {
        float2 r[4];
        rc.get(r);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __fadd2_rn(v[j], r[j]);
      }
      Io<T>::store8(y + 8 * g, v);
    }
  }
  for (int64_t i = 8 * groups + first; i < n; i += step) {
    float u = Io<T>::load(x + i);
    if (d.seed != nullptr) u = dropout1(u, (uint64_t)i, key, d.below, d.scale);
    Io<T>::store(y + i, kResidual ? u + Io<T>::load(residual + i) : u);
  }
}

// ---------------------------------------------------------------------------------------------
// Epilogue backward: dz = drop(dy) * act'(z), max |dz|, column sums of dz
// ---------------------------------------------------------------------------------------------
struct EpilogueBwdArgs {
  const void* dy;
  const void* z;  // nullptr: no activation
  void* dz;
  int64_t rows, cols, ldg, ldz, ldo;
  int64_t rows_per_block;
  DropoutArgs drop;
  uint32_t* pmax;   // one per block: bits of max |dz|
  float* partial;   // [gridDim.y][cols] column sums, or nullptr
};

constexpr int kBwdLanes = 32;  // threads along a row, 8 columns each: a block covers 256 columns
constexpr int kBwdRows = 8;    // rows a block reads at once
constexpr int kBwdBlocksPerSm = 3;

// Rows of a thread in flight: three of bf16, two of fp32 (a few registers of fp32 are spilled as it is).
template <typename T>
constexpr int kBwdBatchOf = sizeof(T) == 2 ? 3 : 2;

// 16384 x 5632 bf16 with the bias gradient: without an activation 63 us, relu^2 91, silu 91, GELU 104, against 57 and
// 86 for the bytes at the copy's rate.  Four blocks to an SM with a row or two in flight: 69 to 77, 90 to 96, 97
// to 100, 104 to 108; two blocks with four rows: 66, 89, 97, 108.
template <typename T, int kAct, bool kVec>
__global__ void __launch_bounds__(kBwdLanes* kBwdRows, kBwdBlocksPerSm) epilogue_backward_kernel(const EpilogueBwdArgs a) {
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * kBwdLanes + lane) * 8;
  const int64_t r0 = (int64_t)blockIdx.y * a.rows_per_block, r1 = min(a.rows, r0 + a.rows_per_block);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  const T* z = reinterpret_cast<const T*>(a.z);
  T* dz = reinterpret_cast<T*>(a.dz);
  float2 sum[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = both(0.0f);
  uint32_t m = 0;
  if (c < a.cols) {
    const PhiloxKeys key = philox_keys(a.drop.seed);
    if constexpr (kVec) {
      constexpr int kBwdBatch = kBwdBatchOf<T>;
      for (int64_t rb = r0 + ty; rb < r1; rb += kBwdBatch * kBwdRows) {
        Raw8<T> graw[kBwdBatch], zraw[kBwdBatch];
#pragma unroll
        for (int u = 0; u < kBwdBatch; ++u) {
          const int64_t r = rb + u * kBwdRows;
          if (r < r1) {
            graw[u].load(dy + r * a.ldg + c);
            if constexpr (kAct != RB_ACT_NONE) zraw[u].load(z + r * a.ldz + c);
          }
        }
#pragma unroll
        for (int u = 0; u < kBwdBatch; ++u) {
          const int64_t r = rb + u * kBwdRows;
          if (r >= r1) break;
          float2 g[4], zv[4];
          graw[u].get(g);
          if (a.drop.seed != nullptr) dropout8(g, (uint64_t)(r * a.cols + c) >> 3, key, a.drop.below, a.drop.scale);
          if constexpr (kAct != RB_ACT_NONE) zraw[u].get(zv);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kAct != RB_ACT_NONE) g[j] = __fmul2_rn(g[j], act_derivative2<kAct, sizeof(T) == 4>(zv[j]));
            sum[j] = __fadd2_rn(sum[j], g[j]);
          }
          m = max(m, Io<T>::store8(dz + r * a.ldo + c, g));
        }
      }
    } else {
      for (int64_t r = r0 + ty; r < r1; r += kBwdRows) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c + j >= a.cols) break;
          float v = Io<T>::load(dy + r * a.ldg + c + j);
          if (a.drop.seed != nullptr)
            v = dropout1(v, (uint64_t)(r * a.cols + c + j), key, a.drop.below, a.drop.scale);
          if constexpr (kAct != RB_ACT_NONE) v *= act_derivative2<kAct, sizeof(T) == 4>(both(Io<T>::load(z + r * a.ldz + c + j))).x;
          if (j & 1) sum[j / 2].y += v;
          else sum[j / 2].x += v;
          m = max(m, Io<T>::store(dz + r * a.ldo + c + j, v));
        }
      }
    }
  }
  // The eight row lanes' sums, added in order; the block's maximum.
  __shared__ float red[kBwdRows][kBwdLanes * 8 + 8];
  __shared__ uint32_t wmax[kBwdRows];
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if (lane == 0) wmax[ty] = m;
  if (a.partial != nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) red[ty][j * 32 + lane] = (j & 1) ? sum[j / 2].y : sum[j / 2].x;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBwdRows; ++w) m = max(m, wmax[w]);
    a.pmax[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = m;
  }
  if (a.partial != nullptr) {
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col < a.cols) {
      const int at = (threadIdx.x & 7) * 32 + (threadIdx.x >> 3);
      float s = red[0][at];
#pragma unroll
      for (int w = 1; w < kBwdRows; ++w) s += red[w][at];
      a.partial[(int64_t)blockIdx.y * a.cols + col] = s;
    }
  }
}

// The blocks' maxima into the global scale (block 0) and their column sums into the bias gradient
// (32 columns to a block; eight threads share a column's `parts` partial sums, in a fixed order).
__global__ void __launch_bounds__(256) epilogue_backward_finish_kernel(const uint32_t* pmax, int64_t blocks,
                                                                       const float* partial, int64_t parts,
                                                                       int64_t cols, float* gs, float* colsum) {
  __shared__ float red[8][32];
  __shared__ uint32_t wmax[8];
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  if (blockIdx.x == 0) {
    uint32_t m = 0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < blocks; i += 256) m = max(m, pmax[i]);
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (lane == 0) wmax[ty] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) m = max(m, wmax[w]);
      const float s = __fdiv_rn(__uint_as_float(m), 2688.0f);  // amax / (6 * 448), one IEEE divide
      *gs = (s < 1e-12f) ? 1e-12f : s;
    }
    return;
  }
  const int64_t col = (int64_t)(blockIdx.x - 1) * 32 + lane;
  float s = 0.0f;
  if (col < cols) {
#pragma unroll 8
    for (int64_t p = ty; p < parts; p += 8) s += partial[p * cols + col];
  }
  red[ty][lane] = s;
  __syncthreads();
  if (ty == 0 && col < cols) {
    for (int w = 1; w < 8; ++w) s += red[w][lane];
    colsum[col] = s;
  }
}

template <typename T, bool kVec>
static void launch_epilogue_backward(int act, dim3 grid, cudaStream_t st, const EpilogueBwdArgs& a) {
  const int threads = kBwdLanes * kBwdRows;
  switch (act) {
    case RB_ACT_RELU: epilogue_backward_kernel<T, RB_ACT_RELU, kVec><<<grid, threads, 0, st>>>(a); break;
    case RB_ACT_RELU2: epilogue_backward_kernel<T, RB_ACT_RELU2, kVec><<<grid, threads, 0, st>>>(a); break;
    case RB_ACT_SILU: epilogue_backward_kernel<T, RB_ACT_SILU, kVec><<<grid, threads, 0, st>>>(a); break;
    case RB_ACT_GELU: epilogue_backward_kernel<T, RB_ACT_GELU, kVec><<<grid, threads, 0, st>>>(a); break;
    case RB_ACT_GELU_TANH: epilogue_backward_kernel<T, RB_ACT_GELU_TANH, kVec><<<grid, threads, 0, st>>>(a); break;
    default: epilogue_backward_kernel<T, RB_ACT_NONE, kVec><<<grid, threads, 0, st>>>(a); break;
  }
}

}  // namespace rb

namespace {

bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

bool on_sm100(const char* what) { return rb_host::sm100(rb_host::current_device(), what); }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return RB_OK;
  rb_host::set_error("%s launch failed: %s", what, cudaGetErrorString(e));
  return RB_ERR_CUDA;
}

// dtype, probability and seed, shared by the entry points below.
int check_common(const char* what, int dtype, double p, const int64_t* seed) {
  if (dtype != RB_DTYPE_BF16 && dtype != RB_DTYPE_F32) {
    rb_host::set_error("%s: unsupported dtype %d", what, dtype);
    return RB_ERR_ARG;
  }
  if (!(p >= 0.0 && p <= 1.0)) {
    rb_host::set_error("%s: the dropout probability must be in [0, 1], got %g", what, p);
    return RB_ERR_ARG;
  }
  if (p > 0.0 && (seed == nullptr || (reinterpret_cast<uintptr_t>(seed) & 7) != 0)) {
    rb_host::set_error("%s: dropout needs an 8-byte aligned device seed", what);
    return RB_ERR_ARG;
  }
  return RB_OK;
}

// Row splits of the backward kernel: one wave of the blocks that an SM holds at once (one block
// more than that and the last ones run alone), each with at least 16 rows.
int64_t backward_parts(int64_t rows, int64_t gx, int sms) {
  const int64_t want = (int64_t)rb::kBwdBlocksPerSm * sms / gx;
  const int64_t most = (rows + 15) / 16;
  int64_t parts = want < most ? want : most;
  if (parts > 65535) parts = 65535;
  return parts < 1 ? 1 : parts;
}

size_t backward_scratch(int64_t parts, int64_t cols, int64_t gx) { return (size_t)(parts * cols + parts * gx) * 4; }

}  // namespace

extern "C" {

int rb_nvfp4_dropout(const void* x, const void* residual, int dtype, int64_t n, double p, const int64_t* seed, void* y,
                     void* stream) {
  const char* what = "nvfp4 dropout";
  if (const int rc = check_common(what, dtype, p, seed)) return rc;
  if (n < 0) {
    rb_host::set_error("%s: negative element count %lld", what, (long long)n);
    return RB_ERR_SHAPE;
  }
  if (n == 0) return RB_OK;
  if (x == nullptr || y == nullptr) {
    rb_host::set_error("%s: null pointer argument", what);
    return RB_ERR_ARG;
  }
  if (!on_sm100(what)) return RB_ERR_DEVICE;
  const rb::DropoutArgs d = rb_host::dropout_args(p, seed);
  const bool vec = !misaligned16(x) && !misaligned16(y) && !misaligned16(residual);
  const int64_t blocks = ((n + 7) / 8 + 255) / 256;
  const int64_t most = (int64_t)rb::kDropoutBlocksPerSm * rb_host::sm_budget(rb_host::current_device());
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto launch = [&](auto t, auto v) {
    using T = decltype(t);
    constexpr bool kVec = decltype(v)::value;
    const T *px = reinterpret_cast<const T*>(x), *pr = reinterpret_cast<const T*>(residual);
    if (pr != nullptr) rb::dropout_kernel<T, kVec, true><<<grid, 256, 0, st>>>(px, pr, reinterpret_cast<T*>(y), n, d);
    else rb::dropout_kernel<T, kVec, false><<<grid, 256, 0, st>>>(px, pr, reinterpret_cast<T*>(y), n, d);
  };
  if (dtype == RB_DTYPE_BF16) {
    if (vec) launch(__nv_bfloat16(), std::true_type());
    else launch(__nv_bfloat16(), std::false_type());
  } else {
    if (vec) launch(float(), std::true_type());
    else launch(float(), std::false_type());
  }
  return launched(what);
}

size_t rb_nvfp4_epilogue_backward_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // Enough for every SM budget (another thread may change it before the call): the splits grow with the SMs.
  const int64_t gx = (cols + 255) / 256;
  return backward_scratch(backward_parts(rows, gx, rb_host::num_sms(rb_host::current_device())), cols, gx);
}

int rb_nvfp4_epilogue_backward(const void* grad_y, int64_t ldg, const void* preact, int64_t ldz, int dtype,
                               int64_t rows, int64_t cols, int activation, double p, const int64_t* seed, void* grad_z,
                               int64_t ldo, float* gs_out, float* colsum_out, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const char* what = "nvfp4 epilogue_backward";
  if (const int rc = check_common(what, dtype, p, seed)) return rc;
  if (activation < RB_ACT_NONE || activation > RB_ACT_GELU_TANH) {
    rb_host::set_error("%s: unknown activation %d", what, activation);
    return RB_ERR_ARG;
  }
  const bool act = activation != RB_ACT_NONE;
  if (rows <= 0 || cols <= 0 || ldg < cols || ldo < cols || (act && ldz < cols)) {
    rb_host::set_error("%s: needs rows > 0, cols > 0 and row strides of at least cols, got rows=%lld cols=%lld", what,
                       (long long)rows, (long long)cols);
    return RB_ERR_SHAPE;
  }
  if (grad_y == nullptr || grad_z == nullptr || gs_out == nullptr || workspace == nullptr ||
      (act && preact == nullptr) || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0) {
    rb_host::set_error("%s: null pointer argument or misaligned workspace", what);
    return RB_ERR_ARG;
  }
  if (!on_sm100(what)) return RB_ERR_DEVICE;
  const int64_t gx = (cols + 255) / 256;
  int64_t parts = backward_parts(rows, gx, rb_host::sm_budget(rb_host::current_device()));
  if (workspace_bytes < backward_scratch(parts, cols, gx)) {
    rb_host::set_error("%s: a workspace of %zu bytes is too small", what, workspace_bytes);
    return RB_ERR_ARG;
  }
  rb::EpilogueBwdArgs a = {};
  a.dy = grad_y;
  a.z = act ? preact : nullptr;
  a.dz = grad_z;
  a.rows = rows;
  a.cols = cols;
  a.ldg = ldg;
  a.ldz = ldz;
  a.ldo = ldo;
  a.drop = rb_host::dropout_args(p, seed);
  if (gx > 0x7FFFFFFF) {
    rb_host::set_error("%s: tensor too wide", what);
    return RB_ERR_SHAPE;
  }
  a.rows_per_block = (rows + parts - 1) / parts;
  parts = (rows + a.rows_per_block - 1) / a.rows_per_block;
  float* ws = reinterpret_cast<float*>(workspace);
  a.pmax = reinterpret_cast<uint32_t*>(ws);
  a.partial = colsum_out != nullptr ? ws + parts * gx : nullptr;
  const int lanes = dtype == RB_DTYPE_BF16 ? 8 : 4;  // elements per 16 bytes
  const bool vec = cols % 8 == 0 && !misaligned16(grad_y) && !misaligned16(grad_z) && ldg % lanes == 0 &&
                   ldo % lanes == 0 && (!act || (!misaligned16(preact) && ldz % lanes == 0));
  const dim3 grid((unsigned)gx, (unsigned)parts);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == RB_DTYPE_BF16) {
    if (vec) rb::launch_epilogue_backward<__nv_bfloat16, true>(activation, grid, st, a);
    else rb::launch_epilogue_backward<__nv_bfloat16, false>(activation, grid, st, a);
  } else {
    if (vec) rb::launch_epilogue_backward<float, true>(activation, grid, st, a);
    else rb::launch_epilogue_backward<float, false>(activation, grid, st, a);
  }
  const unsigned finish = 1u + (colsum_out != nullptr ? (unsigned)((cols + 31) / 32) : 0u);
  rb::epilogue_backward_finish_kernel<<<finish, 256, 0, st>>>(a.pmax, parts * gx, a.partial, parts, cols, gs_out,
                                                              colsum_out);
  return launched(what);
}

}  // extern "C"

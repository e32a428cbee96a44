// Root-mean-square norm over the last dimension, with the residual's addition:
//   h = x + r (rounded to its type: it is the residual stream that the next layer adds to),
//   y = h rstd w,  rstd = 1 / sqrt(mean h^2 + eps)
// 8-bit output: q = rint(127 y / max|y|), scale = max|y| / 127 for each row.
// Backward, with g = dy w:  dx = dr = rstd (g - h rstd^2 mean(g h)) + dh,  dw = sum_rows dy h rstd.
//
// Bound by memory: a row is read once into registers (16-byte loads, EPT elements a thread), reduced
// over the TPR threads that share it, and written.  TPR grows with the row (rule in rms_dispatch) so
// that a thread holds 8 or 16 elements; groups walk the rows and keep the weight in registers.
// 34224 x 256 bf16 with residual: forward 17 us, backward 17 us (4.1 TB/s each) and 4 us for dw; 16384 x 4096
// to 8 bits with residual: 112 us (4.2 TB/s; a plain copy reaches 4.76).
#include "common.h"
#include "launchers.h"

namespace rms_detail {

template <typename T> struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  T v[N];
};

// N elements from p (any alignment), of which `left` exist
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int left, float* f) {
  constexpr int N = Vec<T>::N;
  if (left >= N) {
    Vec<T> t;
    __builtin_memcpy(&t, p, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)t.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, int left, const float* f) {
  constexpr int N = Vec<T>::N;
  if (left >= N) {
    Vec<T> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = (T)f[i];
    __builtin_memcpy(p, &t, 16);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (T)f[i];
  }
}

// sum / maximum of unsigned bits over the TPR threads of a row group (result in all of them)
template <int TPR>
__device__ __forceinline__ float group_sum(float v, float* sh) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += sh[i];
    __syncthreads();
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* sh) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v = max(v, sh[i]);
    __syncthreads();
  }
  return v;
}

template <typename T, int TPR, int EPT>
struct Rows {
  static constexpr int N = Vec<T>::N, NV = EPT / N, NT = TPR < 256 ? 256 : TPR, PER = NT / TPR;
  // element of this thread's vector v
  __device__ static __forceinline__ int at(int v) { return (v * TPR + (int)(threadIdx.x % TPR)) * N; }
  __device__ static __forceinline__ void weight(const RmsArgs& a, float* w) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (a.w_f32) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[v * N + i] = at(v) + i < a.C ? reinterpret_cast<const float*>(a.w)[at(v) + i] : 0.f;
      } else {
        load_vec(reinterpret_cast<const T*>(a.w) + at(v), a.C - at(v), w + v * N);
      }
    }
  }
  __device__ static __forceinline__ void load(const void* p, int64_t row, int C, float* f) {
#pragma unroll
    for (int v = 0; v < NV; ++v) load_vec(reinterpret_cast<const T*>(p) + row * C + at(v), C - at(v), f + v * N);
  }
  __device__ static __forceinline__ void store(void* p, int64_t row, int C, const float* f) {
#pragma unroll
    for (int v = 0; v < NV; ++v) store_vec(reinterpret_cast<T*>(p) + row * C + at(v), C - at(v), f + v * N);
  }
};

template <typename T, int TPR, int EPT, bool Q8>
__global__ __launch_bounds__((Rows<T, TPR, EPT>::NT)) void rms_fwd_kernel(RmsArgs a) {
  using R = Rows<T, TPR, EPT>;
  __shared__ float sh[16];
  float w[EPT];
  R::weight(a, w);
  for (int64_t r0 = (int64_t)blockIdx.x * R::PER; r0 < a.rows; r0 += (int64_t)gridDim.x * R::PER) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool ok = row < a.rows;  // (a group past the last row still takes part in the barriers)
    const int C = ok ? a.C : 0;
    float h[EPT], s = 0.f;
    R::load(a.x, ok ? row : 0, C, h);
    if (a.r) {
      float r[EPT];
      R::load(a.r, ok ? row : 0, C, r);
#pragma unroll
      for (int i = 0; i < EPT; ++i) h[i] = (float)(T)(h[i] + r[i]);
      R::store(a.h, row, C, h);
    }
#pragma unroll
    for (int i = 0; i < EPT; ++i) s = fmaf(h[i], h[i], s);
    const float rstd = rsqrtf(group_sum<TPR>(s, sh) / (float)a.C + a.eps);
#pragma unroll
    for (int i = 0; i < EPT; ++i) h[i] = h[i] * rstd * w[i];
    if constexpr (!Q8) {
      R::store(a.y, row, C, h);
      if (a.rstd && ok && threadIdx.x % TPR == 0) a.rstd[row] = rstd;
    } else {
      uint32_t top = 0;  // the bits of |y| are ordered like the values, with NaN above all
#pragma unroll
      for (int i = 0; i < EPT; ++i) top = max(top, __float_as_uint(h[i]) & 0x7fffffffu);
      const float m = __uint_as_float(group_max<TPR>(top, reinterpret_cast<uint32_t*>(sh)));
      // (127 / m passes fp32's range under m = 2^-121: such rows are raised by 2^64 first, exactly)
      const float up = m < 0x1p-100f ? 0x1p64f : 1.f, inv = m == 0.f ? 0.f : 127.f / (m * up);
#pragma unroll
      for (int v = 0; v < R::NV; ++v) {
        const int e = R::at(v);
        struct { int8_t b[R::N]; } q;
#pragma unroll
        for (int i = 0; i < R::N; ++i)
          q.b[i] = (int8_t)(int)rintf(fminf(fmaxf(h[v * R::N + i] * up * inv, -127.f), 127.f));
        int8_t* p = reinterpret_cast<int8_t*>(a.y) + row * a.C + e;
        if (C - e >= R::N) __builtin_memcpy(p, &q, R::N);
        else
#pragma unroll
          for (int i = 0; i < R::N; ++i)
            if (i < C - e) p[i] = q.b[i];
      }
      if (ok && threadIdx.x % TPR == 0) a.rstd[row] = m / 127.f;
    }
  }
}

// dx, and the block's rows' part of dw in part[block][C]
template <typename T, int TPR, int EPT>
__global__ __launch_bounds__((Rows<T, TPR, EPT>::NT)) void rms_bwd_kernel(RmsArgs a) {
  using R = Rows<T, TPR, EPT>;
  __shared__ float sh[16];
  __shared__ float join[R::PER > 1 ? R::PER * TPR * EPT : 1];
  float w[EPT], dw[EPT];
  R::weight(a, w);
#pragma unroll
  for (int i = 0; i < EPT; ++i) dw[i] = 0.f;
  for (int64_t r0 = (int64_t)blockIdx.x * R::PER; r0 < a.rows; r0 += (int64_t)gridDim.x * R::PER) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool ok = row < a.rows;
    const int C = ok ? a.C : 0;
    float h[EPT], g[EPT], s = 0.f;
    R::load(a.h, ok ? row : 0, C, h);
    R::load(a.dy, ok ? row : 0, C, g);
    const float rstd = ok ? a.rstd[row] : 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      dw[i] = fmaf(g[i] * rstd, h[i], dw[i]);
      g[i] *= w[i];
      s = fmaf(g[i], h[i], s);
    }
    const float c = group_sum<TPR>(s, sh) / (float)a.C * rstd * rstd;
    if (a.dh) {
      float d[EPT];
      R::load(a.dh, ok ? row : 0, C, d);
#pragma unroll
      for (int i = 0; i < EPT; ++i) g[i] = fmaf(rstd, g[i] - h[i] * c, d[i]);
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i) g[i] = rstd * (g[i] - h[i] * c);
    }
    R::store(a.dx, row, C, g);
  }
  if constexpr (R::PER > 1) {
#pragma unroll
    for (int v = 0; v < R::NV; ++v)
#pragma unroll
      for (int i = 0; i < R::N; ++i) join[threadIdx.x / TPR * TPR * EPT + R::at(v) + i] = dw[v * R::N + i];
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += R::NT) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < R::PER; ++k) t += join[k * TPR * EPT + c];
      a.part[(int64_t)blockIdx.x * a.C + c] = t;
    }
  } else {
#pragma unroll
    for (int v = 0; v < R::NV; ++v)
#pragma unroll
      for (int i = 0; i < R::N; ++i)
        if (R::at(v) + i < a.C) a.part[(int64_t)blockIdx.x * a.C + R::at(v) + i] = dw[v * R::N + i];
  }
}

// dw = sum of the blocks' parts in a fixed order: 32 columns x 32 slices of the parts
template <typename T>
__global__ __launch_bounds__(1024) void rms_dw_kernel(RmsArgs a) {
  __shared__ float sh[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  float s = 0.f;
  if (c < a.C)
#pragma unroll 8
    for (int p = k; p < a.parts; p += 32) s += a.part[(int64_t)p * a.C + c];
  sh[k][threadIdx.x & 31] = s;
  __syncthreads();
  if (k == 0 && c < a.C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sh[i][threadIdx.x];
    if (a.w_f32) reinterpret_cast<float*>(a.dw)[c] = s;
    else reinterpret_cast<T*>(a.dw)[c] = (T)s;
  }
}

template <typename T, int TPR, int EPT>
void rms_launch(const RmsArgs& a, int what, hipStream_t s) {
  using R = Rows<T, TPR, EPT>;
  if (what == 2) {
    rms_bwd_kernel<T, TPR, EPT><<<a.parts, R::NT, 0, s>>>(a);
    rms_dw_kernel<T><<<raft_cdiv(a.C, 32), 1024, 0, s>>>(a);
    return;
  }
  const unsigned grid = (unsigned)std::min<int64_t>((a.rows + R::PER - 1) / R::PER, 256 * 2048 / R::NT);
  if (what == 0) rms_fwd_kernel<T, TPR, EPT, false><<<grid, R::NT, 0, s>>>(a);
  else rms_fwd_kernel<T, TPR, EPT, true><<<grid, R::NT, 0, s>>>(a);
}

template <typename T>
void rms_dispatch(const RmsArgs& a, int what, hipStream_t s) {
  // threads of a row: enough for 8 (or 16) elements each
  if (a.C <= 128) rms_launch<T, 16, 8>(a, what, s);
  else if (a.C <= 256) rms_launch<T, 32, 8>(a, what, s);
  else if (a.C <= 512) rms_launch<T, 64, 8>(a, what, s);
  else if (a.C <= 1024) rms_launch<T, 64, 16>(a, what, s);
  else if (a.C <= 2048) rms_launch<T, 256, 8>(a, what, s);
  else if (a.C <= 4096) rms_launch<T, 256, 16>(a, what, s);
  else if (a.C <= 8192) rms_launch<T, 1024, 8>(a, what, s);
  else rms_launch<T, 1024, 16>(a, what, s);
}

void rms_any(const RmsArgs& a, int what, hipStream_t s) {
  if (a.dtype == 0) rms_dispatch<__bf16>(a, what, s);
  else if (a.dtype == 1) rms_dispatch<_Float16>(a, what, s);
  else rms_dispatch<float>(a, what, s);
}

}  // namespace rms_detail

int rms_parts(int64_t rows, int C) {
  // blocks of the backward: the partial dw of a block (C floats) stays small against its rows
  const int per = C <= 128 ? 16 : C <= 256 ? 8 : C <= 1024 ? 4 : 1;
  const int nt = C <= 4096 ? 256 : 1024;
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 4 * per - 1) / (4 * per), 256 * 1024 / nt));
}
void launch_rms_fwd(const RmsArgs& a, hipStream_t s) { rms_detail::rms_any(a, 0, s); }
void launch_rms_int8(const RmsArgs& a, hipStream_t s) { rms_detail::rms_any(a, 1, s); }
void launch_rms_bwd(const RmsArgs& a, hipStream_t s) { rms_detail::rms_any(a, 2, s); }

// 8-bit integer product with a scale for each token (row of x) and each channel (row of w):
//   out[m][n] = xs[m] ws[n] sum_k x[m][k] w[n][k]  (+ bias[n])
// The sum is exact in int32 (K <= 131071: 128 * 128 * K < 2^31); one rounding at the end.
//
// Both operands lie with k innermost, which is what v_mfma_i32_32x32x32_i8 wants of A and B (16
// consecutive k per lane).  w is the A operand and x the B operand, so a lane's accumulator holds 4
// consecutive channels of one token: vector stores, one token scale per lane.
#include "common.h"
#include "launchers.h"

namespace int8_detail {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr uint32_t kOob = 0x80000000u;

__device__ __forceinline__ rsrc_t rsrc_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// 16 bytes of row p at byte k, zeros from K on, any alignment
__device__ __forceinline__ i32x4 load16(const int8_t* p, int k, int K) {
  i32x4 r = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&r, p + k, 16);
  } else if (k < K) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) r[i >> 2] |= (int)((uint32_t)(uint8_t)p[k + i] << (8 * (i & 3)));
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store4(const Int8Args& a, int m, int n, i32x4 acc, float xs) {
  T* o = reinterpret_cast<T*>(a.out) + (int64_t)m * a.N + n;
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v = 0.f;
    if (n + i < a.N) {
      v = (float)acc[i] * xs * a.ws[n + i];
      if (a.bias) v += a.bias[n + i];
    }
    r[i] = (T)v;
  }
  if (n + 4 <= a.N) {
    __builtin_memcpy(o, &r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = r[i];
  }
}

// ---- tiles: BM tokens x BN channels, BK bytes of k a step, double-buffered LDS filled by LDS-DMA
// (rows on 16 bytes) or through registers (any K).  A 16-byte chunk c of row r lies in slot
// c ^ ((r >> 1) & 7): 16 rows of one chunk then cover all banks.
template <int BM, int BN, int WVM, bool ALIGNED, typename T>
__global__ __launch_bounds__(256, (BM * BN <= 128 * 128 ? 2 : 1)) void int8_tile_kernel(Int8Args a) {
  constexpr int BK = 128, WVN = 4 / WVM, WM = BM / WVM, WN = BN / WVN, TM = WM / 32, TN = WN / 32;
  constexpr int STAGE = (BM + BN) * BK;
  constexpr int PER = (BM + BN) * 8 / 256;
  __shared__ __attribute__((aligned(16))) uint8_t sm[2][STAGE];

  const int mt = (a.M + BM - 1) / BM, nt = (a.N + BN - 1) / BN;
  const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (id >= mt * nt) return;
  // groups of 8 token tiles walk the channel tiles together: the working set of an XCD's L2 is a
  // square of tiles, not a strip
  const int per = 8 * nt, grp = id / per, first = grp * 8, wide = min(8, mt - first);
  const int m0 = (first + (id % per) % wide) * BM, n0 = (id % per) / wide * BN;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WVM * WM, wn = wave / WVM * WN;

  const int8_t* x = a.x + (int64_t)m0 * a.K;
  const int8_t* w = a.w + (int64_t)n0 * a.K;
  const int mrows = min(BM, a.M - m0), nrows = min(BN, a.N - n0);
  const rsrc_t rx = rsrc_of(x, (uint32_t)mrows * (uint32_t)a.K), rw = rsrc_of(w, (uint32_t)nrows * (uint32_t)a.K);
  const uint32_t lds = raft_lds_addr(&sm[0][0]) + wave * 1024;

  // x rows first, then w rows
  auto issue = [&](int k0, int buf) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = j * 256 + tid, row = e >> 3, c = (e & 7) ^ ((row >> 1) & 7), k = k0 + c * 16;
      const bool isx = j * 256 < BM * 8;
      const int r = isx ? row : row - BM;
      if constexpr (ALIGNED) {
        const bool ok = k < a.K && r < (isx ? mrows : nrows);
        raft_dma16(isx ? rx : rw, lds + buf * STAGE + j * 4096, ok ? (uint32_t)r * (uint32_t)a.K + k : kOob);
      } else {
        i32x4 v = {0, 0, 0, 0};
        if (r < (isx ? mrows : nrows)) v = load16((isx ? x : w) + (int64_t)r * a.K, k, a.K);
        *reinterpret_cast<i32x4*>(&sm[buf][e * 16]) = v;
      }
    }
  };
  auto frag = [&](const uint8_t* base, int row, int kk) {
    return *reinterpret_cast<const i32x4*>(base + row * BK + (((2 * kk + hi) ^ ((row >> 1) & 7)) << 4));
  };

  i32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  const int steps = (a.K + BK - 1) / BK;
  issue(0, 0);
  for (int t = 0; t < steps; ++t) {
    const int buf = t & 1;
    raft_wait_vmcnt<0>();
    __syncthreads();
    if (t + 1 < steps) issue((t + 1) * BK, buf ^ 1);
    const uint8_t* xt = &sm[buf][0];
    const uint8_t* wt = &sm[buf][BM * BK];
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      i32x4 fx[TM], fw[TN];
#pragma unroll
      for (int j = 0; j < TM; ++j) fx[j] = frag(xt, wm + 32 * j + (lane & 31), kk);
#pragma unroll
      for (int i = 0; i < TN; ++i) fw[i] = frag(wt, wn + 32 * i + (lane & 31), kk);
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = m0 + wm + 32 * j + (lane & 31);
    if (m >= a.M) continue;
    const float xs = a.xs[m];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + wn + 32 * i + 8 * g + 4 * hi;
        if (n < a.N) store4<T>(a, m, n, i32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]}, xs);
      }
  }
}

// ---- few tokens (M <= 64): bound by reading w once.  A workgroup takes 16 channels, its 8 waves
// split k in steps of 64 bytes (16x16x64: lane = channel row, 16 bytes at k (lane >> 4) * 16), all
// straight from memory to registers; the waves' int32 sums meet in LDS.
template <int MT, typename T>
__global__ __launch_bounds__(512) void int8_few_kernel(Int8Args a) {
  __shared__ i32x4 sh[8][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 16, row = lane & 15, kq = (lane >> 4) * 16;
  const int8_t* w = a.w + (int64_t)min(n0 + row, a.N - 1) * a.K;
  const int8_t* x[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) x[j] = a.x + (int64_t)min(16 * j + row, a.M - 1) * a.K;
  i32x4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) acc[j] = i32x4{0, 0, 0, 0};
  for (int k0 = wave * 64; k0 < a.K; k0 += 2048) {
    i32x4 fw[4], fx[4][MT];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      fw[u] = load16(w, k0 + u * 512 + kq, a.K);
#pragma unroll
      for (int j = 0; j < MT; ++j) fx[u][j] = load16(x[j], k0 + u * 512 + kq, a.K);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], fx[u][j], acc[j], 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) sh[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave < MT) {
    i32x4 s = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sh[i][wave][lane];
    const int m = 16 * wave + (lane & 15), n = n0 + 4 * (lane >> 4);
    if (m < a.M && n < a.N) store4<T>(a, m, n, s, a.xs[m]);
  }
}

template <int BM, int BN, int WVM, typename T>
void tile_launch(const Int8Args& a, hipStream_t s) {
  const unsigned grid = raft_cdiv((int64_t)raft_cdiv(a.M, BM) * raft_cdiv(a.N, BN), 8) * 8;
  const bool aligned = a.K % 16 == 0 && (((uintptr_t)a.x | (uintptr_t)a.w) & 15) == 0;
  if (aligned) int8_tile_kernel<BM, BN, WVM, true, T><<<grid, 256, 0, s>>>(a);
  else int8_tile_kernel<BM, BN, WVM, false, T><<<grid, 256, 0, s>>>(a);
}

template <typename T>
void mm(const Int8Args& a, hipStream_t s) {
  if (a.M <= 64) {
    const unsigned grid = raft_cdiv(a.N, 16);
    if (a.M <= 16) int8_few_kernel<1, T><<<grid, 512, 0, s>>>(a);
    else if (a.M <= 32) int8_few_kernel<2, T><<<grid, 512, 0, s>>>(a);
    else int8_few_kernel<4, T><<<grid, 512, 0, s>>>(a);
    return;
  }
  // the largest tile that still gives every CU one
  if ((int64_t)raft_cdiv(a.M, 256) * raft_cdiv(a.N, 256) >= 256) tile_launch<256, 256, 2, T>(a, s);
  else if ((int64_t)raft_cdiv(a.M, 128) * raft_cdiv(a.N, 128) >= 256) tile_launch<128, 128, 2, T>(a, s);
  else tile_launch<64, 64, 2, T>(a, s);
}

}  // namespace int8_detail

void launch_int8_mm(const Int8Args& a, hipStream_t s) {
  if (a.dtype == 0) int8_detail::mm<__bf16>(a, s);
  else if (a.dtype == 1) int8_detail::mm<_Float16>(a, s);
  else int8_detail::mm<float>(a, s);
}

// 8-bit integer product with a scale for each token (row of x) and each channel (row of w):
//   out[m][n] = xs[m] ws[n] sum_k x[m][k] w[n][k]  (+ bias[n])
// The sum is exact in int32 (K <= 131071: 128 * 128 * K < 2^31); one rounding at the end.
//
// Both operands lie with k innermost, which is what v_mfma_i32_32x32x32_i8 wants of A and B (16
// consecutive k per lane).  w is the A operand and x the B operand, so a lane's accumulator holds 4
// consecutive channels of one token: vector stores, one token scale per lane.
// 8192 x 8192 x 4096 to bf16: 283 us, 1.94 POP/s (the library's int32 product without scales: 2.02).
#include "common.h"
#include "launchers.h"

namespace int8_detail {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
template <bool V>
struct Bool {
  static constexpr bool value = V;
};
constexpr uint32_t kOob = 0x80000000u;

__device__ __forceinline__ rsrc_t rsrc_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// 16 bytes of row p at byte k, zeros from K on, any alignment.  The last piece of a row is the row's
// last 16 bytes, shifted.
__device__ __forceinline__ i32x4 load16(const int8_t* p, int k, int K) {
  i32x4 r = {0, 0, 0, 0};
  if (K >= 16) {
    if (k < K) __builtin_memcpy(&r, p + min(k, K - 16), 16);
    const int drop = max(0, min(k, K) + 16 - K);
    if (drop > 0) r = __builtin_bit_cast(i32x4, drop < 16 ? __builtin_bit_cast(unsigned __int128, r) >> (8 * drop) : (unsigned __int128)0);
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

// ---- tiles: BM tokens x BN channels, BK bytes of k a step, four LDS stages.  Stage t + 1 has landed
// when step t begins, so a step's last products run beside the reads of the next step's first
// fragments.  Rows on 16 bytes come by LDS-DMA (two steps in flight), any other through registers
// (loaded one step, written the next).  A 16-byte chunk c of row r lies in slot c ^ ((r >> 2) & 3):
// 16 rows of one chunk then cover all banks.
template <int BM, int BN, int WVM, bool ALIGNED, typename T>
__global__ __launch_bounds__(256, (BM * BN <= 128 * 128 ? 2 : 1)) void int8_tile_kernel(Int8Args a) {
  constexpr int BK = 64, NS = 4, WVN = 4 / WVM, WM = BM / WVM, WN = BN / WVN, TM = WM / 32, TN = WN / 32;
  constexpr int STAGE = (BM + BN) * BK;
  constexpr int PER = (BM + BN) * 4 / 256;
  __shared__ __attribute__((aligned(16))) uint8_t sm[NS][STAGE];

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

  // this thread's chunks: x rows first, then w rows (rows past the last read as zeros)
  uint32_t off[PER];
  int kc[PER];
  bool ok[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = j * 256 + tid, row = e >> 2, c = (e & 3) ^ ((row >> 2) & 3);
    const bool isx = j * 256 < BM * 4;
    const int r = isx ? row : row - BM;
    ok[j] = r < (isx ? mrows : nrows);
    kc[j] = c * 16;
    off[j] = ok[j] ? (uint32_t)r * (uint32_t)a.K + c * 16 : kOob;
  }
  auto issue = [&](int t, int j) {  // chunk j of stage t (past the last step: zeros that nobody reads)
    const uint32_t at = lds + (t & (NS - 1)) * STAGE + j * 4096;
    const int k0 = t * BK;
    raft_dma16(j * 256 < BM * 4 ? rx : rw, at, k0 + kc[j] < a.K ? off[j] + k0 : kOob);
  };
  auto issue_all = [&](int t) {
#pragma unroll
    for (int j = 0; j < PER; ++j) issue(t, j);
  };
  i32x4 hold[ALIGNED ? 1 : PER];
  auto fetch = [&](int t) {
    const int k0 = t * BK;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int8_t* p = (j * 256 < BM * 4 ? x : w) + (ok[j] ? off[j] : 0);
      if (k0 + BK <= a.K) __builtin_memcpy(&hold[j], p + k0, 16);
      else hold[j] = load16(p - kc[j] * (ok[j] ? 1 : 0), k0 + kc[j], a.K);
      if (!ok[j]) hold[j] = i32x4{0, 0, 0, 0};
    }
  };
  auto put = [&](int t) {
#pragma unroll
    for (int j = 0; j < PER; ++j) *reinterpret_cast<i32x4*>(&sm[t & (NS - 1)][(j * 256 + tid) * 16]) = hold[j];
  };

  // fragment addresses: row * 64 + ((2 kk + hi) ^ swizzle) * 16, kk by an xor of 32
  const int sw = (lane >> 2) & 3;
  const uint32_t fbase = raft_lds_addr(&sm[0][0]) + (lane & 31) * BK + ((hi ^ sw) << 4);
  const uint32_t xbase = fbase + wm * BK, wbase = fbase + (BM + wn) * BK;
  i32x4 fx[2][TM], fw[2][TN];
  auto frag = [&](int s, int t, int kk, int f) {  // fragment f: TM of x, then TN of w
    const uint32_t at = (t & (NS - 1)) * STAGE;
    typedef const __attribute__((address_space(3))) i32x4* lds_ptr;
    if (f < TM) fx[s][f] = *reinterpret_cast<lds_ptr>((xbase ^ (kk * 32)) + at + 32 * f * BK);
    else fw[s][f - TM] = *reinterpret_cast<lds_ptr>((wbase ^ (kk * 32)) + at + 32 * (f - TM) * BK);
  };

  i32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  // Half a step: the products of fragment set s with, spread between them, the reads of the other set
  // (stage tf, half kk) and, in the first half, the DMA of stage td.  A DMA in one piece at the top of the
  // step kept the matrix unit waiting (one wave per SIMD): 292 us at 8192 x 8192 x 4096, 283 spread.
  auto half = [&](auto dma, int s, int tf, int kk, int td) {
#pragma unroll
    for (int q = 0; q < TM * TN; ++q) {
      acc[q / TM][q % TM] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[s][q / TM], fx[s][q % TM], acc[q / TM][q % TM], 0, 0, 0);
#pragma unroll
      for (int f = q * (TM + TN) / (TM * TN); f < (q + 1) * (TM + TN) / (TM * TN); ++f) frag(s ^ 1, tf, kk, f);
      if constexpr (ALIGNED && decltype(dma)::value) {
#pragma unroll
        for (int j = q * PER / (TM * TN); j < (q + 1) * PER / (TM * TN); ++j) issue(td, j);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  const int steps = (a.K + BK - 1) / BK;
  if (steps > 0) {
    if constexpr (ALIGNED) {
      issue_all(0);
      issue_all(1);
      issue_all(2);
      raft_wait_vmcnt<2 * PER>();
    } else {
      fetch(0);
      put(0);
      if (1 < steps) fetch(1), put(1);
      if (2 < steps) fetch(2);
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < TM + TN; ++f) frag(0, 0, 0, f);
  }
  for (int t = 0; t < steps; ++t) {
    if constexpr (ALIGNED) raft_wait_vmcnt<PER>();
    __syncthreads();  // stage t + 1 has landed for all waves, and all have left stage t - 1
    if constexpr (!ALIGNED) {
      if (t + 2 < steps) put(t + 2);
      if (t + 3 < steps) fetch(t + 3);
    }
    half(Bool<true>{}, 0, t, 1, t + 3);
    half(Bool<false>{}, 1, t + 1, 0, 0);  // (past the last step: whatever the stage holds, unused)
  }
  // Results go out through LDS, 32 tokens of a wave at a time: a lane holds 4 channels of one token
  // (stores of 8 bytes in 32 rows took 146 us of the 401 us of 8192 x 8192 x 4096), a row of the buffer
  // is WN channels in a row.
  constexpr int ROW = WN * (int)sizeof(T) + 16, CH = 16 / (int)sizeof(T), LPR = WN / CH;  // bytes, channels a chunk, lanes a row
  static_assert(4 * 32 * ROW + 2 * BN * 4 <= NS * STAGE, "epilogue buffers");
  raft_wait_vmcnt<0>();  // (the stages past the last)
  __syncthreads();
  float* scales = reinterpret_cast<float*>(&sm[0][0]);
  uint8_t* buf = &sm[0][0] + 2 * BN * 4 + wave * 32 * ROW;
  for (int i = tid; i < BN; i += 256) {
    scales[i] = n0 + i < a.N ? a.ws[n0 + i] : 0.f;
    scales[BN + i] = a.bias && n0 + i < a.N ? a.bias[n0 + i] : 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int mb = m0 + wm + 32 * j;
    const float xs = a.xs[min(mb + (lane & 31), a.M - 1)];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * i + 8 * g + 4 * hi;
        const f32x4 ws = *reinterpret_cast<const f32x4*>(scales + wn + c), bi = *reinterpret_cast<const f32x4*>(scales + BN + wn + c);
        typedef T v4 __attribute__((ext_vector_type(4)));
        v4 r;
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = (T)fmaf((float)acc[i][j][4 * g + k] * xs, ws[k], bi[k]);
        *reinterpret_cast<v4*>(buf + (lane & 31) * ROW + c * (int)sizeof(T)) = r;
      }
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int q = 0; q < 32 * LPR / 64; ++q) {
      const int row = (q * 64 + lane) / LPR, c = (lane % LPR) * CH, m = mb + row, n = n0 + wn + c;
      const uint4 v = *reinterpret_cast<const uint4*>(buf + row * ROW + c * (int)sizeof(T));
      T* o = reinterpret_cast<T*>(a.out) + (int64_t)m * a.N + n;
      if (m < a.M) {
        if (n + CH <= a.N) {
          __builtin_memcpy(o, &v, 16);
        } else {
          T e[CH];
          __builtin_memcpy(e, &v, 16);
#pragma unroll
          for (int k = 0; k < CH; ++k)
            if (n + k < a.N) o[k] = e[k];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
}

// ---- few tokens (M <= 64): bound by reading w once.  A workgroup takes 16 channels, its 8 waves
// split k in steps of 64 bytes (16x16x64: lane = channel row, 16 bytes at k (lane >> 4) * 16), all
// straight from memory to registers; the waves' int32 sums meet in LDS.  5 x 4096 x 4096: 6 us (2.8 TB/s; one
// workgroup a CU with 64 KB in flight, so a chain of two memory latencies and the launch).
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

// x and w with rows of kp (a multiple of 16) bytes, zeros from K on, in `to` (16 bytes a thread)
__global__ __launch_bounds__(256) void int8_pack_kernel(const int8_t* x, const int8_t* w, int8_t* to, int64_t M, int64_t N, int K, int kp) {
  const int64_t chunks = (M + N) * (kp / 16);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / (kp / 16);
    const int k = (int)(i - row * (kp / 16)) * 16;
    const i32x4 v = load16(row < M ? x + row * K : w + (row - M) * K, k, K);
    *reinterpret_cast<i32x4*>(to + row * kp + k) = v;
  }
}

bool on16(const Int8Args& a) { return a.K % 16 == 0 && (((uintptr_t)a.x | (uintptr_t)a.w) & 15) == 0; }
bool whole_tiles(const Int8Args& a) { return a.M > 64 && (int64_t)raft_cdiv(a.M, 256) * raft_cdiv(a.N, 256) >= 256; }

template <int BM, int BN, int WVM, typename T>
void tile_launch(const Int8Args& a, hipStream_t s) {
  const unsigned grid = raft_cdiv((int64_t)raft_cdiv(a.M, BM) * raft_cdiv(a.N, BN), 8) * 8;
  if (on16(a)) int8_tile_kernel<BM, BN, WVM, true, T><<<grid, 256, 0, s>>>(a);
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
  if (whole_tiles(a)) {
    Int8Args p = a;
    if (a.packed) {
      p.K = (a.K + 15) / 16 * 16;
      p.x = a.packed;
      p.w = a.packed + (int64_t)a.M * p.K;
      int8_pack_kernel<<<(unsigned)std::min<int64_t>((((int64_t)a.M + a.N) * (p.K / 16) + 255) / 256, 2048), 256, 0, s>>>(a.x, a.w, a.packed, a.M, a.N, a.K, p.K);
    }
    int8_tile_kernel<256, 256, 2, true, T><<<raft_cdiv((int64_t)raft_cdiv(a.M, 256) * raft_cdiv(a.N, 256), 8) * 8, 256, 0, s>>>(p);
  } else if ((int64_t)raft_cdiv(a.M, 128) * raft_cdiv(a.N, 128) >= 256) {
    tile_launch<128, 128, 2, T>(a, s);
  } else {
    tile_launch<64, 64, 2, T>(a, s);
  }
}

}  // namespace int8_detail

int64_t int8_packed_bytes(const Int8Args& a) {
  // Products of 256 x 256 tiles read every operand row many times: one copy with rows on 16 bytes
  // costs less than loads through registers (8192 x 8192 x 4099: 333 us against 538).
  if (int8_detail::on16(a) || !int8_detail::whole_tiles(a)) return 0;
  return ((int64_t)a.M + a.N) * ((a.K + 15) / 16 * 16);
}
void launch_int8_mm(const Int8Args& a, hipStream_t s) {
  if (a.dtype == 0) int8_detail::mm<__bf16>(a, s);
  else if (a.dtype == 1) int8_detail::mm<_Float16>(a, s);
  else int8_detail::mm<float>(a, s);
}

// Softmax attention over tokens, backward, with the probabilities recomputed from the saved
// log-sum-exp:
//   P = exp(scale q.k - lse), delta_i = sum_d do_id o_id, dP = do v^T, dS = P (dP - delta),
//   dq = scale dS k, dk = scale dS^T q, dv = P^T do   (dk, dv summed over the heads of a group).
//
// Three kernels, none with atomics on the results (the same inputs give the same bits): row sums
// delta; dk / dv with a workgroup per key block, walking the rows; dq with a workgroup per row
// block, walking the keys.  Scores and dP are formed twice (7 products of L^2 D instead of 5): one
// kernel for all three would have to add dq across key blocks, in an order that changes the sums.
// In each kernel the score tile lies so that it is the B operand of the gradient products as it is
// (attn_common.h): dk / dv own keys as columns, dq owns rows as columns.
//
// fp16: dS is rounded to fp16 before its product, and products of small dout with P ~ 1 / L fall
// under fp16's range.  It is scaled by a power of two, exactly, so that its upper bound
// 2 max|dout_i| max|v_j| maps to 2^14 (attn_delta_kernel finds the norms); P by 2^14 likewise.
#include "attn_common.h"

namespace attn_detail {

constexpr float kP16 = 14.f;  // log2 of the fp16 scale of P

template <typename T, int DP>
struct BwdCfg {
  // rows (dk / dv) or keys (dq) of a tile, walked in blocks of 32
  static constexpr int BT = sizeof(T) == 4 ? 32 : 64;
  static constexpr int TILE = BT * DP * (int)sizeof(T);
};

// power of two that brings the bound of |dS| to at most 2^14 (fp16; 1 otherwise)
template <typename T>
__device__ __forceinline__ float ds_scale(const AttnArgs& a) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
    const float bound = 2.f * sqrtf(__uint_as_float(a.amax[0])) * sqrtf(__uint_as_float(a.amax[1]));
    if (!(bound > 0.f) || !(bound < INFINITY)) return 1.f;
    const int e = 14 - (int)ceilf(log2f(bound));
    return ldexpf(1.f, max(-100, min(100, e)));
  } else {
    return 1.f;
  }
}

// delta of every row; fp16: also the largest squared 2-norm of a dout row and of a v row, as float
// bits (ordered like the floats; a maximum does not depend on the order it is taken in).
// A wave per row.  Rows R of all (b, kv head) first, then (fp16) the v rows.
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(AttnArgs a) {
  constexpr bool F16 = sizeof(T) == 2 && !__is_same(T, __bf16);
  const int lane = threadIdx.x & 63;
  const int64_t R = (int64_t)a.G * a.Lq, nrow = R * a.B * a.Hkv, nv = F16 ? (int64_t)a.B * a.Hkv * a.Lk : 0;
  uint32_t best = 0;
  int which = -1;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w < nrow) {
    const int bh = (int)(w / R), row = (int)(w - (int64_t)bh * R);
    const int b = bh / a.Hkv, hk = bh - b * a.Hkv, qi = row / a.G, h = hk * a.G + row % a.G;
    const T* po = reinterpret_cast<const T*>(a.o) + (((int64_t)b * a.Lq + qi) * a.Hkv * a.G + h) * a.D;
    const T* pd = reinterpret_cast<const T*>(a.dout) + b * a.d_sb + qi * a.d_sl + h * a.d_sh;
    float s = 0.f, n = 0.f;
    for (int d = lane; d < a.D; d += 64) {
      const float x = (float)pd[d];
      s = fmaf(x, (float)po[d], s);
      n = fmaf(x, x, n);
    }
    s = wave_sum(s);
    if (lane == 0) a.delta[w] = s;
    if constexpr (F16) {
      best = __float_as_uint(wave_sum(n));
      which = 0;
    }
  } else if (w < nrow + nv) {
    const int64_t e = w - nrow;
    const int bh = (int)(e / a.Lk), j = (int)(e - (int64_t)bh * a.Lk), b = bh / a.Hkv;
    const T* pv = reinterpret_cast<const T*>(a.v) + b * a.v_sb + j * a.v_sl + (bh - b * a.Hkv) * a.v_sh;
    const bool see = j < item_len(a, b) && (a.mask_mode != 1 || a.mask[b * a.m_sb + j * a.m_sk]);
    float n = 0.f;
    for (int d = lane; see && d < a.D; d += 64) n = fmaf((float)pv[d], (float)pv[d], n);
    best = __float_as_uint(wave_sum(n));
    which = 1;
  }
  if constexpr (F16) {
    if (lane == 0 && which >= 0 && best > __atomic_load_n(&a.amax[which], __ATOMIC_RELAXED))
      atomicMax(&a.amax[which], best);
  }
}

__global__ void attn_amax_clear_kernel(uint32_t* amax) {
  if (threadIdx.x < 2) amax[threadIdx.x] = 0;
}

// ---------------------------------------------------------------- dk, dv: a wave per 32 keys
template <typename T, int DP, int MASK>
__global__ __launch_bounds__(256, 1) void attn_dkv_kernel(AttnArgs a) {
  using TL = Tile<T, DP>;
  using Frag = typename TL::Frag;
  constexpr int BT = BwdCfg<T, DP>::BT, TILE = BwdCfg<T, DP>::TILE, DB = DP / 32, DT = DP / 16;
  constexpr bool F16 = sizeof(T) == 2 && !__is_same(T, __bf16);
  __shared__ __attribute__((aligned(16))) uint8_t qd[2][2][TILE];
  __shared__ __attribute__((aligned(16))) float stat[2][2][BT];  // lse, delta of the tile's rows

  const int R = a.G * a.Lq;
  const int tiles = (a.Lk + 127) / 128;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= tiles * a.B * a.Hkv) return;
  const int tile = id % tiles, bh = id / tiles;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = item_len(a, b), off = item_off(a, b);
  const int key = tile * 128 + wave * 32 + (lane & 31);
  bool see = key < len;
  if constexpr (MASK == 1) see = see && a.mask[b * a.m_sb + (int64_t)min(key, a.Lk - 1) * a.m_sk] != 0;
  // first query that sees any key of the workgroup / that sees all keys of the wave
  const int q_first = a.causal ? max(0, tile * 128 - off) : 0;
  const int q_full = a.causal ? tile * 128 + wave * 32 + 31 - off : 0;
  const int64_t row_first = (int64_t)q_first * a.G;
  const int t1 = (R + BT - 1) / BT;
  const int t0 = tile * 128 < len ? (int)min(row_first / BT, (int64_t)t1) : t1;

  Frag kf[DT], vf[DT];
  {
    const T* pk = reinterpret_cast<const T*>(a.k) + b * a.k_sb + (int64_t)min(key, a.Lk - 1) * a.k_sl + hk * a.k_sh;
    const T* pv = reinterpret_cast<const T*>(a.v) + b * a.v_sb + (int64_t)min(key, a.Lk - 1) * a.v_sl + hk * a.v_sh;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int d = 16 * t + 8 * hi;
      Frag z;
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = (T)0.f;
      kf[t] = see && d < a.D ? *reinterpret_cast<const Frag*>(pk + d) : z;
      vf[t] = see && d < a.D ? *reinterpret_cast<const Frag*>(pv + d) : z;
    }
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) dk[i] = dv[i] = zero16();

  using L = Loader<T, DP, BT, 256>;
  const uint8_t* qb = reinterpret_cast<const uint8_t*>(a.q) + (b * a.q_sb + (int64_t)hk * a.G * a.q_sh) * TL::ES;
  const uint8_t* db = reinterpret_cast<const uint8_t*>(a.dout) + (b * a.d_sb + (int64_t)hk * a.G * a.d_sh) * TL::ES;
  const uint32_t lds = raft_lds_addr(&qd[0][0][0]) + wave * 1024;
  const float* lse = a.lse + (int64_t)bh * R;
  const float* dl = a.delta + (int64_t)bh * R;

  auto issue = [&](int t, int buf) {
    // rows of a tile lie at query r / G, head r % G: offsets from the tile's first query
    const int r0 = t * BT, q0 = r0 / a.G;
    const rsrc_t rq = rsrc_of(qb + (int64_t)q0 * a.q_sl * TL::ES, 0x7fffffffu);
    const rsrc_t rd = rsrc_of(db + (int64_t)q0 * a.d_sl * TL::ES, 0x7fffffffu);
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      const int r = r0 + L::row_of(tid, j), c = L::chunk_of(tid, j) * 16;
      const int qi = r / a.G, g = r - qi * a.G;
      const bool ok = r < R && c < a.D * TL::ES;
      const uint32_t oq = (uint32_t)(((qi - q0) * a.q_sl + g * a.q_sh) * TL::ES) + c;
      const uint32_t od = (uint32_t)(((qi - q0) * a.d_sl + g * a.d_sh) * TL::ES) + c;
      raft_dma16(rq, lds + (2 * buf) * TILE + j * 4096, ok ? oq : kOob);
      raft_dma16(rd, lds + (2 * buf + 1) * TILE + j * 4096, ok ? od : kOob);
    }
    if (tid < 2 * BT) {
      const int r = r0 + tid % BT;
      const float z = tid < BT ? INFINITY : 0.f;  // rows past the last: P = 0
      stat[buf][tid / BT][tid % BT] = r < R ? (tid < BT ? lse[r] : dl[r]) : z;
    }
  };

  const float ds_mul = ds_scale<T>(a) * (F16 ? exp2f(-kP16) : 1.f);
  if (t0 < t1) issue(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    raft_wait_vmcnt<0>();
    __syncthreads();
    if (t + 1 < t1) issue(t + 1, buf ^ 1);
    const uint8_t* qt = &qd[buf][0][0];
    const uint8_t* dt = &qd[buf][1][0];
    for (int hb = 0; hb < BT / 32; ++hb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        s = mma(TL::rows(qt, 32 * hb + (lane & 31), i, hi), kf[i], s);
        dp = mma(TL::rows(dt, 32 * hb + (lane & 31), i, hi), vf[i], dp);
      }
      const bool diag = a.causal && (t * BT + 32 * hb) / a.G < q_full;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(&stat[buf][0][32 * hb + r4 * 8 + hi * 4]);
        const f32x4 de = *reinterpret_cast<const f32x4*>(&stat[buf][1][32 * hb + r4 * 8 + hi * 4]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 4 * r4 + k, row = t * BT + 32 * hb + r4 * 8 + hi * 4 + k;
          bool on = see;
          if (diag) on = on && key <= off + row / a.G;
          if constexpr (MASK == 2) {
            const int rr = min(row, R - 1), qi = rr / a.G;
            on = on && a.mask[b * a.m_sb + (int64_t)(hk * a.G + rr - qi * a.G) * a.m_sh + (int64_t)qi * a.m_sq +
                              (int64_t)min(key, a.Lk - 1) * a.m_sk] != 0;
          }
          float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, (F16 ? kP16 : 0.f) - ls[k]));
          p = on ? p : 0.f;
          s[r] = p;
          dp[r] = on ? p * (dp[r] - de[k]) * ds_mul : 0.f;  // a hidden place adds nothing, whatever dout holds
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Frag pf = to_frag<T>(s, i), df = to_frag<T>(dp, i);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          dv[d] = mma(TL::cols(dt, 32 * hb + 16 * i, d, lane), pf, dv[d]);
          dk[d] = mma(TL::cols(qt, 32 * hb + 16 * i, d, lane), df, dk[d]);
        }
      }
    }
  }
  if (key >= a.Lk) return;
  const int64_t o = (((int64_t)b * a.Lk + key) * a.Hkv + hk) * a.D;
  const float fk = a.scale / ds_scale<T>(a), fv = F16 ? exp2f(-kP16) : 1.f;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + hi * 4;
      if (d < a.D) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        v4 x, y;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = (T)(dk[i][4 * g + k] * fk);
          y[k] = (T)(dv[i][4 * g + k] * fv);
        }
        *reinterpret_cast<v4*>(reinterpret_cast<T*>(a.dk) + o + d) = x;
        *reinterpret_cast<v4*>(reinterpret_cast<T*>(a.dv) + o + d) = y;
      }
    }
}

// ---------------------------------------------------------------- dq: a wave per 32 rows
template <typename T, int DP, int MASK>
__global__ __launch_bounds__(256, 1) void attn_dq_kernel(AttnArgs a) {
  using TL = Tile<T, DP>;
  using Frag = typename TL::Frag;
  constexpr int BK = BwdCfg<T, DP>::BT, TILE = BwdCfg<T, DP>::TILE, DB = DP / 32, DT = DP / 16;
  constexpr bool F16 = sizeof(T) == 2 && !__is_same(T, __bf16);
  __shared__ __attribute__((aligned(16))) uint8_t kv[2][2][TILE];
  __shared__ __attribute__((aligned(16))) float bias[2][BK];

  const int R = a.G * a.Lq;
  const int tiles = (R + 127) / 128;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= tiles * a.B * a.Hkv) return;
  const int tile = tiles - 1 - id % tiles, bh = id / tiles;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = tile * 128 + wave * 32, row = r0 + (lane & 31), rc = min(row, R - 1);
  const bool ok = row < R;
  const int qi = rc / a.G, h = hk * a.G + rc - qi * a.G;
  const int len = item_len(a, b), off = item_off(a, b);
  const int lim = a.causal ? max(0, min(len, off + qi + 1)) : len;
  const int wlim = !a.causal ? len : max(0, min(len, off + min(r0 + 31, R - 1) / a.G + 1));
  const int wmin = !a.causal ? len : max(0, min(len, off + min(r0, R - 1) / a.G + 1));
  const int blim = !a.causal ? len : max(0, min(len, off + (min(tile * 128 + 128, R) - 1) / a.G + 1));
  const int t1 = (blim + BK - 1) / BK;

  Frag qf[DT], df[DT];
  {
    const T* pq = reinterpret_cast<const T*>(a.q) + b * a.q_sb + (int64_t)qi * a.q_sl + h * a.q_sh;
    const T* pd = reinterpret_cast<const T*>(a.dout) + b * a.d_sb + (int64_t)qi * a.d_sl + h * a.d_sh;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int d = 16 * t + 8 * hi;
      Frag z;
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = (T)0.f;
      qf[t] = ok && d < a.D ? *reinterpret_cast<const Frag*>(pq + d) : z;
      df[t] = ok && d < a.D ? *reinterpret_cast<const Frag*>(pd + d) : z;
    }
  }
  const float lse = ok ? a.lse[(int64_t)bh * R + row] : INFINITY;
  const float de = ok ? a.delta[(int64_t)bh * R + row] : 0.f;
  const float sub = (F16 ? kP16 : 0.f) - lse;
  const float ds_mul = ds_scale<T>(a) * (F16 ? exp2f(-kP16) : 1.f);

  f32x16 dq[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) dq[i] = zero16();
  const uint32_t kp = (uint32_t)(a.k_sl * TL::ES), vp = (uint32_t)(a.v_sl * TL::ES);
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k) + (b * a.k_sb + hk * a.k_sh) * TL::ES;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.v) + (b * a.v_sb + hk * a.v_sh) * TL::ES;
  using L = Loader<T, DP, BK, 256>;
  L lk, lv;
  lk.init(tid, kp, a.D * TL::ES);
  lv.init(tid, vp, a.D * TL::ES);
  const uint32_t lds = raft_lds_addr(&kv[0][0][0]) + wave * 1024;
  const uint8_t* mk = MASK ? a.mask + b * a.m_sb + (MASK == 2 ? h * a.m_sh + (int64_t)qi * a.m_sq : 0) : nullptr;

  auto issue = [&](int t, int buf) {
    const int k0 = t * BK, n = min(BK, len - k0);
    const rsrc_t rk = rows_rsrc(kb + (int64_t)k0 * kp, n, kp, a.D * TL::ES);
    const rsrc_t rv = rows_rsrc(vb + (int64_t)k0 * vp, n, vp, a.D * TL::ES);
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      bool see = true;
      if constexpr (MASK == 1) {
        const int r = L::row_of(tid, j);
        see = r < n && mk[(int64_t)(k0 + min(r, n - 1)) * a.m_sk] != 0;
      }
      raft_dma16(rk, lds + (2 * buf) * TILE + j * 4096, see ? lk.off[j] : kOob);
      raft_dma16(rv, lds + (2 * buf + 1) * TILE + j * 4096, see ? lv.off[j] : kOob);
    }
    if constexpr (MASK == 1) {
      if (tid < BK) bias[buf][tid] = tid < n && mk[(int64_t)(k0 + min(tid, n - 1)) * a.m_sk] != 0 ? 0.f : -INFINITY;
    }
  };

  if (t1 > 0) issue(0, 0);
  for (int t = 0; t < t1; ++t) {
    const int buf = t & 1, k0 = t * BK;
    raft_wait_vmcnt<0>();
    __syncthreads();
    if (t + 1 < t1) issue(t + 1, buf ^ 1);
    if (k0 >= wlim) continue;
    const uint8_t* kt = &kv[buf][0][0];
    const uint8_t* vt = &kv[buf][1][0];
    for (int hb = 0; hb < BK / 32; ++hb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        s = mma(TL::rows(kt, 32 * hb + (lane & 31), i, hi), qf[i], s);
        dp = mma(TL::rows(vt, 32 * hb + (lane & 31), i, hi), df[i], dp);
      }
      const bool part = MASK || k0 + BK > wmin;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 32 * hb + (r >> 2) * 8 + hi * 4 + (r & 3);
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, sub));
        float d = p * (dp[r] - de) * ds_mul;
        if (part) {
          bool on = j < lim - k0;
          if constexpr (MASK == 1) on = on && bias[buf][j] == 0.f;
          if constexpr (MASK == 2) on = on && mk[(int64_t)min(k0 + j, a.Lk - 1) * a.m_sk] != 0;
          d = on ? d : 0.f;
        }
        s[r] = d;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Frag f = to_frag<T>(s, i);
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = mma(TL::cols(kt, 32 * hb + 16 * i, d, lane), f, dq[d]);
      }
    }
  }
  if (!ok) return;
  const int64_t o = (((int64_t)b * a.Lq + qi) * a.Hkv * a.G + h) * a.D;
  const float f = a.scale / ds_scale<T>(a);
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + hi * 4;
      if (d < a.D) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        v4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (T)(dq[i][4 * g + k] * f);
        *reinterpret_cast<v4*>(reinterpret_cast<T*>(a.dq) + o + d) = x;
      }
    }
}

template <typename T, int DP, int MASK>
void bwd_launch(const AttnArgs& a, hipStream_t s) {
  const int64_t R = (int64_t)a.G * a.Lq, heads = (int64_t)a.B * a.Hkv;
  constexpr bool F16 = sizeof(T) == 2 && !__is_same(T, __bf16);
  if (F16) attn_amax_clear_kernel<<<1, 64, 0, s>>>(a.amax);
  const int64_t rows = R * heads + (F16 ? heads * a.Lk : 0);
  attn_delta_kernel<T><<<raft_cdiv(rows, 4), 256, 0, s>>>(a);
  attn_dkv_kernel<T, DP, MASK><<<raft_cdiv((int64_t)raft_cdiv(a.Lk, 128) * heads, 8) * 8, 256, 0, s>>>(a);
  attn_dq_kernel<T, DP, MASK><<<raft_cdiv((int64_t)raft_cdiv(R, 128) * heads, 8) * 8, 256, 0, s>>>(a);
}
template <typename T, int DP>
void bwd_mask(const AttnArgs& a, hipStream_t s) {
  if (a.mask_mode == 0) bwd_launch<T, DP, 0>(a, s);
  else if (a.mask_mode == 1) bwd_launch<T, DP, 1>(a, s);
  else bwd_launch<T, DP, 2>(a, s);
}
template <typename T>
void bwd_dim(const AttnArgs& a, hipStream_t s) {
  if (a.DP == 32) bwd_mask<T, 32>(a, s);
  else if (a.DP == 64) bwd_mask<T, 64>(a, s);
  else if (a.DP == 96) bwd_mask<T, 96>(a, s);
  else bwd_mask<T, 128>(a, s);
}

}  // namespace attn_detail

void launch_attn_bwd(const AttnArgs& a, hipStream_t s) {
  if (a.dtype == 0) attn_detail::bwd_dim<__bf16>(a, s);
  else if (a.dtype == 1) attn_detail::bwd_dim<_Float16>(a, s);
  else attn_detail::bwd_dim<float>(a, s);
}

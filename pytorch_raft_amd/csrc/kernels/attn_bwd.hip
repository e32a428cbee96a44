// Softmax attention over tokens, backward, with the probabilities recomputed from the saved
// log-sum-exp:
//   P = exp(scale q.k - lse), delta_i = sum_d do_id o_id, dP = do v^T, dS = P (dP - delta),
//   dq = scale dS k, dk = scale dS^T q, dv = P^T do   (dk, dv summed over the heads of a group).
//
// No atomics on the results (the same inputs give the same bits).  attn_prep_kernel forms delta; then
// one launch holds two kinds of workgroups: for dk / dv, one per 128 keys walking the rows, and for dq,
// one per 128 rows walking the keys.  Scores and dP are formed twice (7 products of L^2 D instead of
// 5): one kind alone would have to add dq across key blocks, in an order that changes the sums.  The
// kinds share a launch because a workgroup fills its CU (one wave per SIMD: 32 keys of dk and dv are
// 128 accumulators): 12 x 2852 tokens make 276 workgroups of each kind for 256 CUs, and the dq ones
// fill the second round of the others.
// 12 x 2852 tokens, a head of 128, bf16: 240 us (730 TFLOP/s of the 7 products), 4 x 7040 x 4 heads 1560 us
// (910).  The matrix unit is busy 30 % of the first one's cycles, the LDS 17 %.  A CU holds a workgroup 78 % of
// the time: 552 of unlike length run in rounds of 256.  Of their time the waves wait 34 %: lse and delta of a
// tile are loaded behind its DMA, loads return in order, and so two of the four waves wait for both.
// In each kind the score tile lies so that it is the B operand of the gradient products as it is
// (attn_common.h): dk / dv own keys as columns, dq owns rows as columns.
//
// fp16: dS is rounded to fp16 before its product, and products of small dout with P ~ 1 / L fall
// under fp16's range.  It is scaled by a power of two, exactly, so that its upper bound
// 2 max|dout_i| max|v_j| maps to 2^14 (attn_prep_kernel finds the norms); P by 2^14 likewise.
#include "attn_common.h"

namespace attn_detail {

constexpr float kP16 = 14.f;  // log2 of the fp16 scale of P
constexpr int kPrepMax = 1024;  // most blocks of attn_prep_kernel (each leaves two norms)

template <typename T>
constexpr bool is_f16 = sizeof(T) == 2 && !__is_same(T, __bf16);

template <typename T, int DP>
struct BwdCfg {
  // rows (dk / dv) or keys (dq) of a tile, walked in blocks of 32
  static constexpr int BT = sizeof(T) == 4 ? 32 : 64;
  static constexpr int TILE = BT * DP * (int)sizeof(T);
};

// waves per SIMD that the registers allow
template <typename T, int DP>
constexpr int bwd_waves = DP * (int)sizeof(T) > 128 ? 1 : 2;

// power of two that brings the bound of |dS| to at most 2^14 (fp16; 1 otherwise): a wave reads the
// prep blocks' largest squared norms
template <typename T>
__device__ __forceinline__ float ds_scale(const AttnArgs& a) {
  if constexpr (is_f16<T>) {
    uint32_t m0 = 0, m1 = 0;
    for (int i = threadIdx.x & 63; i < a.nprep; i += 64) {
      m0 = max(m0, a.amax[2 * i]);
      m1 = max(m1, a.amax[2 * i + 1]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      m0 = max(m0, (uint32_t)__shfl_xor((int)m0, o, 64));
      m1 = max(m1, (uint32_t)__shfl_xor((int)m1, o, 64));
    }
    const float bound = 2.f * sqrtf(__uint_as_float(m0)) * sqrtf(__uint_as_float(m1));
    if (!(bound > 0.f)) return 1.f;  // (finite: squares of fp16 values)
    const int e = 14 - (int)ceilf(log2f(bound));
    return ldexpf(1.f, max(-100, min(100, e)));
  } else {
    return 1.f;
  }
}

// delta of every row, from the output as a pair of 16-bit values (rounded value and what the rounding
// took away): where one key takes nearly all of a row, dP - delta cancels, and a delta from the rounded
// output alone left errors in dq and dk of up to 2.5 times the rounding of the result.  fp16: also the
// largest squared 2-norm of a dout row and of a v row that this block met, as float bits (ordered like the
// floats); a row with an infinity or NaN is left out, so that it does not undo the scale of all others.
// 16 lanes of 8 channels a row.
template <typename T>
__global__ __launch_bounds__(256) void attn_prep_kernel(AttnArgs a) {
  constexpr bool F16 = is_f16<T>;
  typedef T v8 __attribute__((ext_vector_type(8)));
  const int sub = threadIdx.x & 15, d = sub * 8;
  const int64_t R = (int64_t)a.G * a.Lq, nrow = R * a.B * a.Hkv, nv = F16 ? (int64_t)a.B * a.Hkv * a.Lk : 0;
  uint32_t best[2] = {0, 0};
  for (int64_t w = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); w < nrow + nv; w += (int64_t)gridDim.x * 16) {
    float s = 0.f, n = 0.f;
    const float l = w < nrow ? a.lse[w] : 0.f;
    if (w < nrow) {
      const int bh = (int)(w / R), row = (int)(w - (int64_t)bh * R);
      const int b = bh / a.Hkv, hk = bh - b * a.Hkv, qi = row / a.G, h = hk * a.G + row % a.G;
      if (d < a.D) {
        const int64_t at = (((int64_t)b * a.Lq + qi) * a.Hkv * a.G + h) * a.D + d;
        const v8 o = *reinterpret_cast<const v8*>(reinterpret_cast<const T*>(a.o) + at);
        v8 lo;
#pragma unroll
        for (int i = 0; i < 8; ++i) lo[i] = (T)0.f;
        if (a.o_lo) lo = *reinterpret_cast<const v8*>(reinterpret_cast<const T*>(a.o_lo) + at);
        const v8 g = *reinterpret_cast<const v8*>(reinterpret_cast<const T*>(a.dout) + b * a.d_sb + qi * a.d_sl + h * a.d_sh + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s = fmaf((float)g[i], (float)o[i] + (float)lo[i], s);
          n = fmaf((float)g[i], (float)g[i], n);
        }
      }
    } else {
      const int64_t e = w - nrow;
      const int bh = (int)(e / a.Lk), j = (int)(e - (int64_t)bh * a.Lk), b = bh / a.Hkv;
      const bool see = j < item_len(a, b) && (a.mask_mode != 1 || a.mask[b * a.m_sb + j * a.m_sk]);
      if (see && d < a.D) {
        const v8 v = *reinterpret_cast<const v8*>(reinterpret_cast<const T*>(a.v) + b * a.v_sb + j * a.v_sl + (bh - b * a.Hkv) * a.v_sh + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) n = fmaf((float)v[i], (float)v[i], n);
      }
    }
    s = raft_row16_sum(s);
    // a row that sees no key has no part in the gradients, whatever dout holds there
    if (l == INFINITY) s = n = 0.f;
    if (w < nrow && sub == 0) a.delta[w] = s;
    if constexpr (F16) {
      n = raft_row16_sum(n);
      const int k = w < nrow ? 0 : 1;
      best[k] = max(best[k], n < INFINITY ? __float_as_uint(n) : 0u);
    }
  }
  if constexpr (F16) {
    __shared__ uint32_t sh[2][16];
    if (sub == 0) sh[0][threadIdx.x >> 4] = best[0], sh[1][threadIdx.x >> 4] = best[1];
    __syncthreads();
    if (threadIdx.x < 2) {
      uint32_t m = 0;
      for (int i = 0; i < 16; ++i) m = max(m, sh[threadIdx.x][i]);
      a.amax[2 * blockIdx.x + threadIdx.x] = m;
    }
  }
}

template <bool V>
struct Bool {
  static constexpr bool value = V;
};

// pins the schedule of a run of N matrix instructions: READS LDS reads after each.  (Pinning vector
// instructions between them as well measured slower: 253 us with 0, 267 with 4, 290 with 6 each on the
// backward of 12 x 2852 tokens with a head of 128, 274 without any pin.)
template <int N, int READS>
__device__ __forceinline__ void pin() {
  if constexpr (N > 0) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    pin<N - 1, READS>();
  }
}

// 4 consecutive channels per 4 accumulator registers: to the result, or (part) to fp32 partials
template <typename T, int DB>
__device__ __forceinline__ void put_grad(void* out, float* part, int64_t at, const f32x16 (&acc)[DB], float f, bool keep, int D, int hi) {
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + hi * 4;
      if (d < D) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        f32x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = keep ? acc[i][4 * g + k] * f : 0.f;
        if (part) {
          *reinterpret_cast<f32x4*>(part + at + d) = x;
        } else {
          v4 y;
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = (T)x[k];
          *reinterpret_cast<v4*>(reinterpret_cast<T*>(out) + at + d) = y;
        }
      }
    }
}

// ---------------------------------------------------------------- dk, dv: a wave per 32 keys
template <typename T, int DP, int MASK>
__device__ __forceinline__ void dkv_body(const AttnArgs& a, int bid, int grid, uint8_t* sm) {
  using TL = Tile<T, DP>;
  using Frag = typename TL::Frag;
  constexpr int BT = BwdCfg<T, DP>::BT, TILE = BwdCfg<T, DP>::TILE, DB = DP / 32, DT = DP / 16, NB = BT / 32;
  constexpr bool AHEAD = sizeof(T) == 2;  // fp32: the products take 16 times as long, and fragments twice the registers
  constexpr bool F16 = is_f16<T>;
  float* stat = reinterpret_cast<float*>(sm + 6 * TILE);  // [buffer][-lse, delta][row of the tile]

  const int R = a.G * a.Lq;
  int tile, split, bh;
  if (!place(a, bid, grid, (a.Lk + 127) / 128, a.nsplit_kv, false, tile, split, bh)) return;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = item_len(a, b), off = item_off(a, b);
  const int key = tile * 128 + wave * 32 + (lane & 31);
  bool see = key < len;
  if constexpr (MASK == 1) see = see && a.mask[b * a.m_sb + (int64_t)min(key, a.Lk - 1) * a.m_sk] != 0;
  // first row that sees this lane's key (a position times the heads passes 32 bits either way)
  const int row_min = a.causal ? (int)max(min((int64_t)(key - off) * a.G, (int64_t)INT32_MAX), (int64_t)INT32_MIN) : INT32_MIN;
  // first query that sees any key of the workgroup / that sees all of them
  const int q_first = a.causal ? max(0, tile * 128 - off) : 0;
  const int q_full = a.causal ? tile * 128 + 127 - off : 0;
  int t1 = (R + BT - 1) / BT;
  int t0 = tile * 128 < len ? (int)min((int64_t)q_first * a.G / BT, (int64_t)t1) : t1;
  if (a.nsplit_kv > 1) {
    const int per = (t1 - t0 + a.nsplit_kv - 1) / a.nsplit_kv;
    t0 = min(t1, t0 + split * per);
    t1 = min(t1, t0 + per);
  }

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
  const uint32_t lds = raft_lds_addr(sm) + wave * 1024;
  const uint32_t qrow = TL::rows_base(raft_lds_addr(sm), lane), qcol = TL::cols_base(raft_lds_addr(sm), lane);
  const float* lse = a.lse + (int64_t)bh * R;
  const float* dl = a.delta + (int64_t)bh * R;
  const float up = ds_scale<T>(a), ds_mul = up * (F16 ? exp2f(-kP16) : 1.f);

  // Rows of a tile lie at query r / G, head r % G: byte offsets from the tile's first query.  Where G
  // divides the tile (every G up to 64 but 3, 5, 6, 7, ...) they are the same for all tiles.
  const bool even = BT % a.G == 0;
  uint32_t oq[L::PER], od[L::PER];
  auto offsets = [&](int r0, int q0) {
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      const int r = r0 + L::row_of(tid, j), c = L::chunk_of(tid, j) * 16;
      const int qi = r / a.G, g = r - qi * a.G;
      oq[j] = c < a.D * TL::ES ? (uint32_t)(((qi - q0) * a.q_sl + g * a.q_sh) * TL::ES) + c : kOob;
      od[j] = c < a.D * TL::ES ? (uint32_t)(((qi - q0) * a.d_sl + g * a.d_sh) * TL::ES) + c : kOob;
    }
  };
  offsets(0, 0);
  // Rows that see no key come as zeros: their q and dout may hold anything, and P = 0 times an infinity is
  // NaN.  Without a mask those are the first ones under causal; under masks their lse says so (+inf), looked
  // up a tile ahead and turned into bits by a ballot.
  const int first = a.causal ? max(0, -off) * a.G : 0;
  float ahead = INFINITY;
  auto look = [&](int t) {
    if constexpr (MASK != 0) {
      const int r = t * BT + (lane & (BT - 1));
      ahead = r < R ? lse[r] : INFINITY;
    }
  };
  auto issue = [&](int t, uint32_t buf, int sbuf) {
    const int r0 = t * BT, q0 = r0 / a.G;
    const uint64_t rows = MASK != 0 ? __ballot(ahead != INFINITY) >> L::row_of(tid, 0) : 0;
    const rsrc_t rq = rsrc_of(qb + (int64_t)q0 * a.q_sl * TL::ES, 0x7fffffffu);
    const rsrc_t rd = rsrc_of(db + (int64_t)q0 * a.d_sl * TL::ES, 0x7fffffffu);
    if (!even) offsets(r0, q0);
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      const int r = r0 + L::row_of(tid, j);
      const bool ok = MASK != 0 ? rows >> j * (256 / TL::NC) & 1 : r >= first && r < R;
      raft_dma16(rq, lds + buf + j * 4096, ok ? oq[j] : kOob);
      raft_dma16(rd, lds + buf + TILE + j * 4096, ok ? od[j] : kOob);
    }
    if (tid < 2 * BT) {
      const int r = r0 + tid % BT;
      // rows past the last: P = 0
      stat[sbuf + tid] = tid < BT ? (r < R ? (F16 ? kP16 : 0.f) - lse[r] : -INFINITY) : (r < R ? dl[r] * ds_mul : 0.f);
    }
    if (t + 1 < t1) look(t + 1);
  };

  // A tile of two 32-row blocks (16-bit types): scores and dP of both, exponentials of the first beside
  // the products of the second, exponentials of the second beside the gradients of the first, gradients
  // of the second; the fragments of each phase are read during the one before.  The order is pinned:
  // left alone, the compiler puts an LDS read right before its product and waits for it there.
  Frag fq[DT], fd[DT], cd[2][DB], cq[2][DB];
  auto load_rows = [&](uint32_t at, int hb) {
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      fq[i] = TL::rows(qrow + at, hb, i);
      fd[i] = TL::rows(qrow + at + TILE, hb, i);
    }
  };
  auto load_cols = [&](uint32_t at, int hb) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        cd[i][d] = TL::cols(qcol + at + TILE, 32 * hb + 16 * i, d);
        cq[i][d] = TL::cols(qcol + at, 32 * hb + 16 * i, d);
      }
  };
  auto products = [&](f32x16& s, f32x16& dp, uint32_t at, int hb) {
    s = dp = zero16();
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      s = mma(AHEAD ? fq[i] : TL::rows(qrow + at, hb, i), kf[i], s);
      dp = mma(AHEAD ? fd[i] : TL::rows(qrow + at + TILE, hb, i), vf[i], dp);
    }
  };
  auto weights = [&](auto edge, f32x16& s, f32x16& dp, int row0, const float* st, uint32_t bits) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x4 ls = *reinterpret_cast<const f32x4*>(st + r4 * 8 + hi * 4);
      const f32x4 de = *reinterpret_cast<const f32x4*>(st + BT + r4 * 8 + hi * 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 4 * r4 + k;
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, ls[k]));
        s[r] = p;
        dp[r] = p * (F16 ? fmaf(dp[r], ds_mul, -de[k]) : dp[r] - de[k]);
      }
    }
    if constexpr (decltype(edge)::value) {
      // a hidden place has no P and no dS (a hidden key's column is dropped at the end)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = row0 + (r >> 2) * 8 + hi * 4 + (r & 3);
        bool on = row >= row_min;
        if constexpr (MASK == 2) on = on && (bits >> ((r >> 2) * 8 + hi * 4 + (r & 3)) & 1);
        s[r] = on ? s[r] : 0.f;
        dp[r] = on ? dp[r] : 0.f;
      }
    }
  };
  auto gradients = [&](const f32x16& s, const f32x16& dp, uint32_t at, int hb) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Frag pf = to_frag<T>(s, i), df = to_frag<T>(dp, i);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        dv[d] = mma(AHEAD ? cd[i][d] : TL::cols(qcol + at + TILE, 32 * hb + 16 * i, d), pf, dv[d]);
        dk[d] = mma(AHEAD ? cq[i][d] : TL::cols(qcol + at, 32 * hb + 16 * i, d), df, dk[d]);
      }
    }
  };
  auto walk = [&](auto edge, int row0, uint32_t at, const float* st, uint32_t at_next, uint64_t bits) {
    if constexpr (NB == 2) {
      f32x16 s0, p0, s1, p1;
      products(s0, p0, at, 0);
      load_rows(at, 1);
      pin<2 * DT, 1>();
      products(s1, p1, at, 1);
      load_cols(at, 0);
      weights(edge, s0, p0, row0, st, (uint32_t)bits);
      pin<2 * DT, 2>();
      gradients(s0, p0, at, 0);
      load_cols(at, 1);
      weights(edge, s1, p1, row0 + 32, st + 32, (uint32_t)(bits >> 32));
      pin<2 * DT, 2>();
      gradients(s1, p1, at, 1);
      load_rows(at_next, 0);
      pin<2 * DT, 1>();
    } else {
      f32x16 s, dp;
      products(s, dp, at, 0);
      weights(edge, s, dp, row0, st, (uint32_t)bits);
      gradients(s, dp, at, 0);
    }
  };
  // three buffers: tile t + 1 has landed when tile t begins, for the last block's look ahead
  uint32_t b0 = 0, b1 = 2 * TILE, b2 = 4 * TILE;
  int s0 = 0, s1 = 2 * BT, s2 = 4 * BT;
  // mask: this key's bits over the rows of a tile, looked up a tile ahead
  const uint64_t* mw = MASK == 2 ? key_bits(a, b, hk, min(key, a.Lk - 1)) : nullptr;
  uint64_t word = MASK == 2 && t0 < t1 ? mw[t0 * BT / 64] >> (t0 * BT % 64) : 0;
  auto turn = [&](auto edge, int t) {
    raft_wait_vmcnt<0>();
    __syncthreads();  // tile t + 1 has landed for all waves, and all have left tile t - 1
    if (t + 2 < t1) issue(t + 2, b2, s2);
    const uint64_t bits = word;
    if constexpr (MASK == 2) word = t + 1 < t1 ? mw[(t + 1) * BT / 64] >> ((t + 1) * BT % 64) : 0;
    walk(edge, t * BT, b0, stat + s0, b1, bits);
    const uint32_t x = b0;
    b0 = b1, b1 = b2, b2 = x;
    const int y = s0;
    s0 = s1, s1 = s2, s2 = y;
  };
  if (t0 < t1) {
    look(t0);
    issue(t0, b0, s0);
    if (t0 + 1 < t1) issue(t0 + 1, b1, s1);
    raft_wait_vmcnt<0>();
    __syncthreads();
    if constexpr (AHEAD) load_rows(b0, 0);
    int t = t0;
    // tiles with rows that miss some of the wave's keys come first
    const int te = MASK == 2 ? t1 : a.causal ? max(t0, min(t1, (int)(((int64_t)max(q_full, 0) * a.G + BT - 1) / BT))) : t0;
    for (; t < te; ++t) turn(Bool<true>{}, t);
    if constexpr (MASK != 2)
      for (; t < t1; ++t) turn(Bool<false>{}, t);
  }
  if (key >= a.Lk) return;
  const int64_t o = (((int64_t)b * a.Lk + key) * a.Hkv + hk) * a.D, n = (int64_t)a.B * a.Lk * a.Hkv * a.D;
  put_grad<T>(a.dk, a.nsplit_kv > 1 ? a.part + split * n : nullptr, o, dk, a.scale / up, see, a.D, hi);
  put_grad<T>(a.dv, a.nsplit_kv > 1 ? a.part + (a.nsplit_kv + split) * n : nullptr, o, dv, F16 ? exp2f(-kP16) : 1.f, see, a.D, hi);
}

// ---------------------------------------------------------------- dq: a wave per 32 rows
template <typename T, int DP, int MASK>
__device__ __forceinline__ void dq_body(const AttnArgs& a, int bid, int grid, uint8_t* sm) {
  using TL = Tile<T, DP>;
  using Frag = typename TL::Frag;
  constexpr int BK = BwdCfg<T, DP>::BT, TILE = BwdCfg<T, DP>::TILE, DB = DP / 32, DT = DP / 16, NB = BK / 32;
  constexpr bool AHEAD = sizeof(T) == 2;
  constexpr bool F16 = is_f16<T>;

  const int R = a.G * a.Lq;
  int tile, split, bh;
  if (!place(a, bid, grid, (R + 127) / 128, a.nsplit_q, true, tile, split, bh)) return;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = tile * 128 + wave * 32, row = r0 + (lane & 31), rc = min(row, R - 1);
  const bool ok = row < R;
  const int qi = rc / a.G, h = hk * a.G + rc - qi * a.G;
  const int len = item_len(a, b), off = item_off(a, b);
  const int lim = a.causal ? max(0, min(len, off + qi + 1)) : len;
  // keys that the last / first row of the workgroup sees
  const int blim = !a.causal ? len : max(0, min(len, off + (min(tile * 128 + 128, R) - 1) / a.G + 1));
  const int bmin = !a.causal ? len : max(0, min(len, off + min(tile * 128, R - 1) / a.G + 1));
  int t0 = 0, t1 = (blim + BK - 1) / BK;
  if (a.nsplit_q > 1) {
    const int per = (t1 + a.nsplit_q - 1) / a.nsplit_q;
    t0 = min(t1, split * per);
    t1 = min(t1, t0 + per);
  }

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
  const float up = ds_scale<T>(a), ds_mul = up * (F16 ? exp2f(-kP16) : 1.f);
  const float sub = ok ? (F16 ? kP16 : 0.f) - a.lse[(int64_t)bh * R + row] : -INFINITY;
  const float de = ok ? a.delta[(int64_t)bh * R + row] * ds_mul : 0.f;

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
  const uint32_t lds = raft_lds_addr(sm) + wave * 1024;
  const uint32_t krow = TL::rows_base(raft_lds_addr(sm), lane), kcol = TL::cols_base(raft_lds_addr(sm), lane);
  const uint8_t* mk = MASK == 1 ? a.mask + b * a.m_sb : nullptr;
  const uint64_t* mw = MASK == 2 ? row_bits(a, b, hk, rc) : nullptr;

  uint8_t byte = 0;  // masks: looked up a tile ahead; the bits of three tiles
  uint64_t word = 0, m0 = 0, m1 = 0, m2 = 0;
  auto look = [&](int t) {
    if constexpr (MASK == 2) word = mw[t * BK / 64] >> (t * BK % 64);
    if constexpr (MASK == 1) byte = (lane & (BK - 1)) < len - t * BK ? mk[(int64_t)(t * BK + (lane & (BK - 1))) * a.m_sk] : 0;
  };
  auto issue = [&](int t, uint32_t buf) {
    const int k0 = t * BK, n = min(BK, len - k0);
    const rsrc_t rk = rows_rsrc(kb + (int64_t)k0 * kp, n, kp, a.D * TL::ES);
    const rsrc_t rv = rows_rsrc(vb + (int64_t)k0 * vp, n, vp, a.D * TL::ES);
    const uint64_t m = MASK == 1 ? __ballot(byte != 0) : word;
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      const bool see = MASK != 1 || (m >> L::row_of(tid, j) & 1);
      raft_dma16(rk, lds + buf + j * 4096, see ? lk.off[j] : kOob);
      raft_dma16(rv, lds + buf + TILE + j * 4096, see ? lv.off[j] : kOob);
    }
    if (t + 1 < t1) look(t + 1);
    return m;
  };

  // (the dk / dv kind's pattern with keys and rows exchanged)
  Frag fk[DT], fv[DT], ck[2][DB];
  auto load_rows = [&](uint32_t at, int hb) {
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      fk[i] = TL::rows(krow + at, hb, i);
      fv[i] = TL::rows(krow + at + TILE, hb, i);
    }
  };
  auto load_cols = [&](uint32_t at, int hb) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < DB; ++d) ck[i][d] = TL::cols(kcol + at, 32 * hb + 16 * i, d);
  };
  auto products = [&](f32x16& s, f32x16& dp, uint32_t at, int hb) {
    s = dp = zero16();
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      s = mma(AHEAD ? fk[i] : TL::rows(krow + at, hb, i), qf[i], s);
      dp = mma(AHEAD ? fv[i] : TL::rows(krow + at + TILE, hb, i), df[i], dp);
    }
  };
  auto weights = [&](auto edge, f32x16& s, const f32x16& dp, int k0, uint32_t keys) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, sub));
      s[r] = p * (F16 ? fmaf(dp[r], ds_mul, -de) : dp[r] - de);
    }
    if constexpr (decltype(edge)::value) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = (r >> 2) * 8 + hi * 4 + (r & 3);
        bool on = k0 + j < lim;
        if constexpr (MASK != 0) on = on && (keys >> j & 1);
        s[r] = on ? s[r] : 0.f;
      }
    }
  };
  auto gradients = [&](const f32x16& s, uint32_t at, int hb) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Frag f = to_frag<T>(s, i);
#pragma unroll
      for (int d = 0; d < DB; ++d) dq[d] = mma(AHEAD ? ck[i][d] : TL::cols(kcol + at, 32 * hb + 16 * i, d), f, dq[d]);
    }
  };
  auto walk = [&](auto edge, int k0, uint32_t at, uint64_t keys, uint32_t at_next) {
    if constexpr (NB == 2) {
      f32x16 s0, p0, s1, p1;
      products(s0, p0, at, 0);
      load_rows(at, 1);
      pin<2 * DT, 1>();
      products(s1, p1, at, 1);
      load_cols(at, 0);
      weights(edge, s0, p0, k0, (uint32_t)keys);
      pin<2 * DT, 1>();
      gradients(s0, at, 0);
      load_cols(at, 1);
      weights(edge, s1, p1, k0 + 32, (uint32_t)(keys >> 32));
      pin<DT, 2>();
      gradients(s1, at, 1);
      load_rows(at_next, 0);
      pin<DT, 2>();
    } else {
      f32x16 s, dp;
      products(s, dp, at, 0);
      weights(edge, s, dp, k0, (uint32_t)keys);
      gradients(s, at, 0);
    }
  };
  uint32_t b0 = 0, b1 = 2 * TILE, b2 = 4 * TILE;
  auto turn = [&](auto edge, int t) {
    raft_wait_vmcnt<0>();
    __syncthreads();
    if (t + 2 < t1) m2 = issue(t + 2, b2);
    walk(edge, t * BK, b0, m0, b1);
    const uint32_t x = b0;
    b0 = b1, b1 = b2, b2 = x;
    m0 = m1, m1 = m2;
  };
  if (t0 < t1) {
    look(t0);
    m0 = issue(t0, b0);
    if (t0 + 1 < t1) m1 = issue(t0 + 1, b1);
    raft_wait_vmcnt<0>();
    __syncthreads();
    if constexpr (AHEAD) load_rows(b0, 0);
    int t = t0;
    if constexpr (MASK == 0)
      for (const int te = min(t1, bmin / BK); t < te; ++t) turn(Bool<false>{}, t);
    for (; t < t1; ++t) turn(Bool<true>{}, t);
  }
  if (!ok) return;
  const int64_t o = (((int64_t)b * a.Lq + qi) * a.Hkv * a.G + h) * a.D, n = (int64_t)a.B * a.Lq * a.Hkv * a.G * a.D;
  put_grad<T>(a.dq, a.nsplit_q > 1 ? a.part_q + split * n : nullptr, o, dq, a.scale / up, true, a.D, hi);
}

template <typename T, int DP, int MASK>
__global__ __launch_bounds__(256, (bwd_waves<T, DP>)) __attribute__((amdgpu_waves_per_eu(bwd_waves<T, DP>, bwd_waves<T, DP>))) void attn_bwd_kernel(AttnArgs a, int grid_kv, int grid_q) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[6 * BwdCfg<T, DP>::TILE + 6 * BwdCfg<T, DP>::BT * 4];
  if ((int)blockIdx.x < grid_kv) dkv_body<T, DP, MASK>(a, blockIdx.x, grid_kv, sm);
  else dq_body<T, DP, MASK>(a, blockIdx.x - grid_kv, grid_q, sm);
}

// sums of the split parts, in order: dk, dv (n_kv elements each) and dq (n_q)
template <typename T>
__global__ __launch_bounds__(256) void attn_grad_join_kernel(AttnArgs a, int64_t n_kv, int64_t n_q) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const float* part = a.part;
  void* out = a.dk;
  int64_t n = n_kv;
  int splits = a.nsplit_kv;
  if (a.nsplit_kv > 1 && i < 2 * n_kv) {
    if (i >= n_kv) part += splits * n_kv, out = a.dv, i -= n_kv;
  } else {
    if (a.nsplit_kv > 1) i -= 2 * n_kv;
    part = a.part_q, out = a.dq, n = n_q, splits = a.nsplit_q;
    if (a.nsplit_q <= 1 || i >= n_q) return;
  }
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(part + k * n + i);
  v4 y;
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = (T)s[k];
  *reinterpret_cast<v4*>(reinterpret_cast<T*>(out) + i) = y;
}

template <typename T, int DP, int MASK>
void bwd_launch(const AttnArgs& a, hipStream_t s) {
  const int64_t R = (int64_t)a.G * a.Lq, heads = (int64_t)a.B * a.Hkv;
  if (a.mask_mode == 2) launch_attn_pack(a, s);
  attn_prep_kernel<T><<<a.nprep, 256, 0, s>>>(a);
  const int gk = (int)raft_cdiv((int64_t)raft_cdiv(a.Lk, 128) * heads * a.nsplit_kv, 8) * 8;
  const int gq = (int)raft_cdiv((int64_t)raft_cdiv(R, 128) * heads * a.nsplit_q, 8) * 8;
  attn_bwd_kernel<T, DP, MASK><<<gk + gq, 256, 0, s>>>(a, gk, gq);
  const int64_t n_kv = (int64_t)a.B * a.Lk * a.Hkv * a.D, n_q = R * heads * a.D;
  const int64_t n = (a.nsplit_kv > 1 ? 2 * n_kv : 0) + (a.nsplit_q > 1 ? n_q : 0);
  if (n > 0) attn_grad_join_kernel<T><<<raft_cdiv(n, 1024), 256, 0, s>>>(a, n_kv, n_q);
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

void attn_bwd_plan(AttnArgs& a) {
  const int64_t R = (int64_t)a.G * a.Lq, heads = (int64_t)a.B * a.Hkv;
  const int64_t rows = R * heads + (a.dtype == 1 ? heads * a.Lk : 0);
  a.nprep = (int)std::max<int64_t>(1, std::min<int64_t>((rows + 31) / 32, attn_detail::kPrepMax));
  // few tiles over a long other side: the walk is split so that each kind has about a workgroup per
  // CU, with at least 4 tiles of 64 each
  const auto split = [](int64_t blocks, int64_t walk) {
    return (int)std::max<int64_t>(1, std::min<int64_t>({256 / std::max<int64_t>(blocks, 1), walk / 256, 32}));
  };
  a.nsplit_kv = split((int64_t)raft_cdiv(a.Lk, 128) * heads, R);
  a.nsplit_q = split((int64_t)raft_cdiv(R, 128) * heads, a.Lk);
}

void launch_attn_bwd(const AttnArgs& a, hipStream_t s) {
  if (a.dtype == 0) attn_detail::bwd_dim<__bf16>(a, s);
  else if (a.dtype == 1) attn_detail::bwd_dim<_Float16>(a, s);
  else attn_detail::bwd_dim<float>(a, s);
}

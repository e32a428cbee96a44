// Softmax attention over tokens, forward: o_i = sum_j softmax_j(scale q_i . k_j) v_j.
//
// One pass over the keys with a running maximum and sum.  A wave owns 32 rows (queries); the scores
// of a key block are computed transposed, S^T = K Q^T, so that a lane holds one query's scores:
// maximum and sum are register reductions plus one half-wave exchange, rescaling the output is one
// multiply per register, and the probabilities are the B operand of O^T = V^T P^T as they lie.
//
// Four waves share the K and V tiles (64 keys; 32 in fp32), double-buffered by LDS-DMA.  Registers and LDS
// let two workgroups stay on a CU with heads of 128, three with 96, four with 64 and five with 32 (16-bit
// types without a mask; one to two fewer with one).
// bf16, 8 x 7040 tokens, 2 heads of 64: 250 us, 810 TFLOP/s.  880 workgroups, all resident, three or four a
// CU: a CU holds a wave 83 % of the time.  The vector unit is busy 59 % of all cycles (some 800 a tile and
// wave: exponential, scaling, sum, maximum, conversion) and the matrix unit 37 % (512), and the waves spend
// 41 % of their time ready behind another's issue.  Forming the next tile's scores ahead (295 us), 32-key
// steps with three or four waves a SIMD (302, 281) and 64 rows a wave (289) measured slower.
// Heads of 128: 4 x 7040, 4 heads 420 us, 970 TFLOP/s; 12 x 2852, 1 head 79 us, 630 TFLOP/s: 276 workgroups
// of 512 that fit, so 20 CUs with two decide the time (a CU holds a wave 69 % of it).
#include "attn_common.h"

namespace attn_detail {

template <typename T, int DP>
struct FwdCfg {
  static constexpr int BK = sizeof(T) == 4 ? 32 : 64;  // keys per tile
  static constexpr int BM = 32 * 4;                    // rows of a workgroup: 32 for each of its waves
  static constexpr int TILE = BK * DP * (int)sizeof(T);
};

// Running softmax state of a wave's 32 rows (one per lane pair) and the output accumulators.
template <typename T, int DP>
struct RowState {
  using TL = Tile<T, DP>;
  using Frag = typename TL::Frag;
  static constexpr int DB = DP / 32, DT = DP / 16;
  Frag q[DT];
  f32x16 o[DB];
  float m, l;  // reference exponent (log2 units), this half-wave's part of the sum

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = zero16();
    m = -INFINITY;
    l = 0.f;
  }
  // query row from global memory (zeros past the last row and past D)
  __device__ __forceinline__ void load_q(const T* p, bool ok, int D, int hi) {
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int d = 16 * t + 8 * hi;
      Frag f;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (T)0.f;
      if (ok && d < D) f = *reinterpret_cast<const Frag*>(p + d);
      q[t] = f;
    }
  }
  // scores of NB blocks of 32 keys
  template <int NB>
  __device__ __forceinline__ void scores(uint32_t kt, f32x16 (&s)[NB]) const {  // kt: rows view
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = zero16();
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
        s[b] = mma(TL::rows(kt, b, t), q[t], s[b]);
  }
  // The running reference exponent moves (rescaling sum and output) only when a row's maximum has
  // outgrown it by 2^8: the result is the same, since both carry the same factor, and p <= 2^8 is far
  // from every type's limit.
  template <int NB>
  __device__ __forceinline__ void raise(const f32x16 (&s)[NB], float c) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    mx = fmaxf(mx, other_half(mx)) * c;
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= al;
    }
  }
  // scores -> probabilities relative to the reference
  template <int NB>
  __device__ __forceinline__ void probs(f32x16 (&s)[NB], float c) {
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], c, -ms));
        l += s[b][r];
      }
  }
  template <int NB>
  __device__ __forceinline__ void values(uint32_t vt, const f32x16 (&s)[NB]) {  // vt: columns view
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag p = to_frag<T>(s[b], t);
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = mma(TL::cols(vt, b * 32 + 16 * t, i), p, o[i]);
      }
  }
};

// keys from `left` on (this lane's row) and keys that the mask's bits for the tile leave out -> -inf
template <int NB, int MASK>
__device__ __forceinline__ void hide(f32x16 (&s)[NB], int left, int hi, uint64_t keys) {
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t bits = (uint32_t)(keys >> (32 * b)) >> (4 * hi);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      bool see = b * 32 + (r >> 2) * 8 + hi * 4 + (r & 3) < left;
      if constexpr (MASK != 0) see = see && (bits >> ((r >> 2) * 8 + (r & 3)) & 1);
      s[b][r] = see ? s[b][r] : -INFINITY;
    }
  }
}

// lane's output row (column of O^T): 4 consecutive channels per 4 registers.  lo (training): what the
// rounding took away, for the backward's row sums.
template <typename T, int DB>
__device__ __forceinline__ void store_row(T* p, T* lo, const f32x16 (&o)[DB], float f, int D, int hi) {
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + hi * 4;
      if (d < D) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        v4 w, x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k] = (T)(o[i][4 * g + k] * f);
          x[k] = (T)(o[i][4 * g + k] * f - (float)w[k]);
        }
        *reinterpret_cast<v4*>(p + d) = w;
        if (lo) *reinterpret_cast<v4*>(lo + d) = x;
      }
    }
}

template <typename T, int DP, int MASK>
__global__ __launch_bounds__(256, 2) __attribute__((amdgpu_waves_per_eu(2, 2))) void attn_fwd_kernel(AttnArgs a) {
  using C = FwdCfg<T, DP>;
  using TL = Tile<T, DP>;
  constexpr int BK = C::BK, NB = BK / 32;
  __shared__ __attribute__((aligned(16))) uint8_t kv[2][2][C::TILE];

  const int R = a.G * a.Lq;
  const int tiles = (R + C::BM - 1) / C::BM;
  int tile, split, bh;
  if (!place(a, blockIdx.x, gridDim.x, tiles, a.nsplit, true, tile, split, bh)) return;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = tile * C::BM + wave * 32, row = r0 + (lane & 31);
  const bool ok = row < R;
  const int qi = min(row, R - 1) / a.G, g = min(row, R - 1) - qi * a.G;
  const int h = hk * a.G + g;

  const int len = item_len(a, b), off = item_off(a, b);
  const int lim = a.causal ? max(0, min(len, off + qi + 1)) : len;     // keys this lane's row sees
  const int wlim = !a.causal ? len : max(0, min(len, off + (min(r0 + 31, R - 1)) / a.G + 1));
  const int wmin = !a.causal ? len : max(0, min(len, off + min(r0, R - 1) / a.G + 1));
  const int blim = !a.causal ? len : max(0, min(len, off + (min(tile * C::BM + C::BM, R) - 1) / a.G + 1));
  int t0 = 0, t1 = (blim + BK - 1) / BK;
  if (a.nsplit > 1) {
    const int per = ((a.Lk + BK - 1) / BK + a.nsplit - 1) / a.nsplit;
    t0 = min(t1, split * per);
    t1 = min(t1, t0 + per);
  }

  RowState<T, DP> st;
  st.init();
  st.load_q(reinterpret_cast<const T*>(a.q) + b * a.q_sb + (int64_t)qi * a.q_sl + h * a.q_sh, ok, a.D, hi);

  const uint32_t kp = (uint32_t)(a.k_sl * TL::ES), vp = (uint32_t)(a.v_sl * TL::ES);
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k) + (b * a.k_sb + hk * a.k_sh) * TL::ES;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.v) + (b * a.v_sb + hk * a.v_sh) * TL::ES;
  Loader<T, DP, BK, 256> lk, lv;
  lk.init(tid, kp, a.D * TL::ES);
  lv.init(tid, vp, a.D * TL::ES);
  const uint32_t lds = raft_lds_addr(&kv[0][0][0]) + wave * 1024;
  const uint8_t* mk = MASK == 1 ? a.mask + b * a.m_sb : nullptr;
  const uint64_t* mw = MASK == 2 ? row_bits(a, b, hk, min(row, R - 1)) : nullptr;

  // masks: looked up a tile ahead; a key mask's bytes become bits by a ballot
  uint8_t byte = 0;
  uint64_t word = 0, keys = 0;
  auto look = [&](int t) {
    if constexpr (MASK == 2) word = mw[t * BK / 64] >> (t * BK % 64);
    if constexpr (MASK == 1) byte = (lane & (BK - 1)) < len - t * BK ? mk[(int64_t)(t * BK + (lane & (BK - 1))) * a.m_sk] : 0;
  };
  auto issue = [&](int t, int buf) {
    const int k0 = t * BK, n = min(BK, len - k0);
    const rsrc_t rk = rows_rsrc(kb + (int64_t)k0 * kp, n, kp, a.D * TL::ES);
    const rsrc_t rv = rows_rsrc(vb + (int64_t)k0 * vp, n, vp, a.D * TL::ES);
    const uint64_t m = MASK == 1 ? __ballot(byte != 0) : word;
#pragma unroll
    for (int j = 0; j < Loader<T, DP, BK, 256>::PER; ++j) {
      // (a hidden key's row is not fetched at all, whatever it holds)
      const bool see = MASK != 1 || (m >> Loader<T, DP, BK, 256>::row_of(tid, j) & 1);
      raft_dma16(rk, lds + 2 * buf * C::TILE + j * 4096, see ? lk.off[j] : kOob);
      raft_dma16(rv, lds + (2 * buf + 1) * C::TILE + j * 4096, see ? lv.off[j] : kOob);
    }
    if (t + 1 < t1) look(t + 1);
    return m;
  };
  const uint32_t krow = TL::rows_base(raft_lds_addr(&kv[0][0][0]), lane), vcol = TL::cols_base(raft_lds_addr(&kv[0][1][0]), lane);
  const float c = a.scale_log2;
  // Two waves share a SIMD: issue priority for one's score products parts their phases.  Heads of 128:
  // 12 x 2852 tokens 85 us against 90, 4 x 7040 x 4 heads 420 / 430, causal 2 x 4096 x 16 142 / 151;
  // smaller heads, bound by the vector unit, and fp32 gain nothing (198 / 194 with heads of 32).
  constexpr bool FIRST = sizeof(T) == 2 && DP == 128;
  uint64_t next = 0;
  if (t0 < t1) {
    look(t0);
    next = issue(t0, 0);
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, k0 = t * BK;
    raft_wait_vmcnt<0>();
    __syncthreads();  // tile t has landed for all waves, and all have left tile t - 1's buffer
    keys = next;
    if (t + 1 < t1) next = issue(t + 1, buf ^ 1);
    if (k0 >= wlim) continue;
    // Padding hides whole tiles or none of one: those are left out, these need no selects.  4 x 2852 tokens,
    // 2 heads of 64, the last tenth hidden: 50 us against 65 with selects in every tile (a scattered mask,
    // whose tiles all need them: 78 / 65; rows' own masks, mode 2, gain nothing: 87 / 81).
    if (MASK == 1 && (BK == 64 ? keys == 0 : (uint32_t)keys == 0)) continue;
    const bool selects = MASK == 2 || (MASK == 1 && (BK == 64 ? keys != ~0ull : (uint32_t)keys != ~0u));
    f32x16 s[NB];
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
    st.scores(krow + buf * 2 * C::TILE, s);
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
    if (selects || k0 + BK > wmin)
      hide<NB, MASK>(s, lim - k0, hi, keys);
    st.raise(s, c);
    st.probs(s, c);
    st.values(vcol + buf * 2 * C::TILE, s);
  }

  const float l = st.l + other_half(st.l);
  if (!ok) return;
  if (a.nsplit > 1) {
    const int64_t p = ((int64_t)bh * a.nsplit + split) * R + row;
    store_row<float>(a.part + p * DP, nullptr, st.o, 1.f, DP, hi);
    if (hi == 0) {
      a.part_ml[2 * p] = st.m;
      a.part_ml[2 * p + 1] = l;
    }
    return;
  }
  const int64_t at = (((int64_t)b * a.Lq + qi) * a.Hkv * a.G + h) * a.D;
  store_row<T>(reinterpret_cast<T*>(a.o) + at, a.o_lo ? reinterpret_cast<T*>(a.o_lo) + at : nullptr, st.o,
               l > 0.f || l != l ? 1.f / l : 0.f, a.D, hi);
  if (a.lse && hi == 0) a.lse[(int64_t)bh * R + row] = l > 0.f || l != l ? st.m + log2f(l) : INFINITY;
}

// ---- few rows (R <= 32) over long keys: bound by reading K and V once.  The four waves of a
// workgroup take different 32-key blocks of the workgroup's key range, each through LDS buffers of
// its own (no barrier in the loop), and are joined in LDS at the end.  32 items with caches of 8192 to
// 16384 keys, 8 key heads of 128 in bf16: 1.63 GB in 304 us, 5.35 TB/s.
template <typename T, int DP, int MASK>
__global__ __launch_bounds__(256, 1) void attn_few_kernel(AttnArgs a) {
  using TL = Tile<T, DP>;
  constexpr int TILE = 32 * DP * (int)sizeof(T);
  constexpr int DB = DP / 32;
  // two buffers of K and V for each wave where they fit the 160 KB (fp32 heads over 64: one)
  constexpr int BUFS = 4 * 2 * 2 * TILE <= 128 * 1024 ? 2 : 1;
  constexpr int BUF = 4 * 2 * BUFS * TILE, JOIN = 4 * 32 * (DP + 4) * 4;
  __shared__ __attribute__((aligned(16))) uint8_t sm[BUF > JOIN ? BUF : JOIN];
  __shared__ float ml[4][32][2];

  const int R = a.G * a.Lq;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= a.nsplit * a.B * a.Hkv) return;
  const int split = id % a.nsplit, bh = id / a.nsplit;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 31;
  const bool ok = row < R;
  const int qi = min(row, R - 1) / a.G, g = min(row, R - 1) - qi * a.G, h = hk * a.G + g;
  const int len = item_len(a, b), off = item_off(a, b);
  const int lim = a.causal ? max(0, min(len, off + qi + 1)) : len;
  const int wmin = !a.causal ? len : max(0, min(len, off + 1));
  const int blim = !a.causal ? len : max(0, min(len, off + a.Lq));
  // the item's own blocks are dealt evenly over the splits
  const int blocks = (blim + 31) / 32;
  const int per = (blocks + a.nsplit - 1) / a.nsplit;
  const int t0 = min(blocks, split * per), t1 = min(blocks, t0 + per);

  RowState<T, DP> st;
  st.init();
  st.load_q(reinterpret_cast<const T*>(a.q) + b * a.q_sb + (int64_t)qi * a.q_sl + h * a.q_sh, ok, a.D, hi);
  const uint32_t kp = (uint32_t)(a.k_sl * TL::ES), vp = (uint32_t)(a.v_sl * TL::ES);
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k) + (b * a.k_sb + hk * a.k_sh) * TL::ES;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.v) + (b * a.v_sb + hk * a.v_sh) * TL::ES;
  using L = Loader<T, DP, 32, 64>;
  L lk, lv;
  lk.init(lane, kp, a.D * TL::ES);
  lv.init(lane, vp, a.D * TL::ES);
  const uint32_t lds = raft_lds_addr(sm) + wave * 2 * BUFS * TILE;
  const uint32_t krow = TL::rows_base(lds, lane), vcol = TL::cols_base(lds + TILE, lane);
  const uint8_t* mk = MASK == 1 ? a.mask + b * a.m_sb : nullptr;
  const uint64_t* mw = MASK == 2 ? row_bits(a, b, hk, min(row, R - 1)) : nullptr;

  uint8_t byte = 0;
  uint64_t word = 0, keys = 0, next = 0;
  auto look = [&](int t) {
    if constexpr (MASK == 2) word = mw[t / 2] >> (t % 2 * 32);
    if constexpr (MASK == 1) byte = row < len - t * 32 ? mk[(int64_t)(t * 32 + row) * a.m_sk] : 0;
  };
  auto issue = [&](int t, int buf) {
    const int k0 = t * 32, n = min(32, len - k0);
    const rsrc_t rk = rows_rsrc(kb + (int64_t)k0 * kp, n, kp, a.D * TL::ES);
    const rsrc_t rv = rows_rsrc(vb + (int64_t)k0 * vp, n, vp, a.D * TL::ES);
    const uint64_t m = MASK == 1 ? __ballot(byte != 0) : word;
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      const bool see = MASK != 1 || (m >> L::row_of(lane, j) & 1);
      raft_dma16(rk, lds + 2 * buf * TILE + j * 1024, see ? lk.off[j] : kOob);
      raft_dma16(rv, lds + (2 * buf + 1) * TILE + j * 1024, see ? lv.off[j] : kOob);
    }
    if (t + 4 < t1) look(t + 4);
    return m;
  };

  int t = t0 + wave;
  if (t < t1) look(t);
  if (BUFS == 2 && t < t1) next = issue(t, 0);
  for (int buf = 0; t < t1; t += 4, buf ^= BUFS - 1) {
    const int k0 = t * 32;
    // the next block's DMA overwrites the buffer read two blocks ago: those reads have returned
    // (their products were issued), and the wait below leaves only the next block in flight
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    keys = next;
    if (BUFS == 1) {
      keys = issue(t, 0);
      raft_wait_vmcnt<0>();
    } else if (MASK != 0) {
      raft_wait_vmcnt<0>();  // (the look ahead is counted too)
      if (t + 4 < t1) next = issue(t + 4, buf ^ 1);
    } else if (t + 4 < t1) {
      issue(t + 4, buf ^ 1);
      raft_wait_vmcnt<2 * L::PER>();
    } else {
      raft_wait_vmcnt<0>();
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
    f32x16 s[1];
    st.scores(krow + 2 * buf * TILE, s);
    if (MASK || k0 + 32 > wmin)
      hide<1, MASK>(s, lim - k0, hi, keys);
    st.raise(s, a.scale_log2);
    st.probs(s, a.scale_log2);
    st.values(vcol + 2 * buf * TILE, s);
    asm volatile("" ::: "memory");
  }

  // join the waves: common reference exponent, then sums over waves of the scaled outputs
  const float l = st.l + other_half(st.l);
  if (hi == 0) {
    ml[wave][row][0] = st.m;
    ml[wave][row][1] = l;
  }
  __syncthreads();  // also: every wave has left its tiles, which the outputs now overwrite
  float mt = -INFINITY, lt = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ml[w][row][0]);
  const float ms = mt == -INFINITY ? 0.f : mt;
#pragma unroll
  for (int w = 0; w < 4; ++w) lt += ml[w][row][1] * __builtin_amdgcn_exp2f(ml[w][row][0] - ms);
  const float f = __builtin_amdgcn_exp2f(st.m - ms);
  float* jo = reinterpret_cast<float*>(sm);
  store_row<float>(jo + (wave * 32 + row) * (DP + 4), nullptr, st.o, f, DP, hi);
  __syncthreads();
  const bool some = lt > 0.f || lt != lt;
  if (a.nsplit == 1 && a.lse && wave == 0 && hi == 0 && ok) a.lse[(int64_t)bh * R + row] = some ? mt + log2f(lt) : INFINITY;
  if (a.nsplit > 1 && wave == 0 && hi == 0 && ok) {
    const int64_t p = ((int64_t)bh * a.nsplit + split) * R + row;
    a.part_ml[2 * p] = mt;
    a.part_ml[2 * p + 1] = lt;
  }
  // thread -> (row, channel): rows of DP channels
  if (wave == 0 && hi == 0) ml[0][row][0] = some ? 1.f / lt : 0.f;  // read after the barrier below
  __syncthreads();
  for (int e = tid; e < R * DP; e += 256) {
    const int r = e / DP, d = e - r * DP;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v += jo[(w * 32 + r) * (DP + 4) + d];
    if (a.nsplit > 1) {
      a.part[(((int64_t)bh * a.nsplit + split) * R + r) * DP + d] = v;
    } else if (d < a.D) {
      const int q2 = r / a.G, g2 = r - q2 * a.G;
      const int64_t at = (((int64_t)b * a.Lq + q2) * a.Hkv * a.G + hk * a.G + g2) * a.D + d;
      const T w = (T)(v * ml[0][r][0]);
      reinterpret_cast<T*>(a.o)[at] = w;
      if (a.o_lo) reinterpret_cast<T*>(a.o_lo)[at] = (T)(v * ml[0][r][0] - (float)w);
    }
  }
}

// ---- joins the key ranges: one wave per row (lane = channels)
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  const int R = a.G * a.Lq;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)a.B * a.Hkv * R) return;
  const int lane = threadIdx.x & 63;
  const int bh = (int)(w / R), row = (int)(w - (int64_t)bh * R);
  const int64_t p0 = (int64_t)bh * a.nsplit * R + row;
  // lane s: the s-th range's maximum, sum and factor (at most 64 ranges).  The first ranges' outputs are
  // fetched beside them: the launch is a chain of memory latencies.
  constexpr int PL = (DP + 63) / 64, PRE = 16;
  const bool mine = lane < a.nsplit;
  const float m = mine ? a.part_ml[2 * (p0 + (int64_t)lane * R)] : -INFINITY;
  const float l = mine ? a.part_ml[2 * (p0 + (int64_t)lane * R) + 1] : 0.f;
  float o[PL], pre[PRE][PL];
#pragma unroll
  for (int s = 0; s < PRE; ++s)
#pragma unroll
    for (int k = 0; k < PL; ++k)
      pre[s][k] = s < a.nsplit && lane + 64 * k < DP ? a.part[(p0 + (int64_t)s * R) * DP + lane + 64 * k] : 0.f;
  float mt = m;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x, 64));
  const float fs = __builtin_amdgcn_exp2f(m - (mt == -INFINITY ? 0.f : mt));
  const float lt = wave_sum(mine ? l * fs : 0.f);
#pragma unroll
  for (int k = 0; k < PL; ++k) o[k] = 0.f;
#pragma unroll
  for (int s = 0; s < PRE; ++s) {
    const float f = __shfl(fs, s, 64);
#pragma unroll
    for (int k = 0; k < PL; ++k) o[k] += pre[s][k] * f;
  }
#pragma unroll 8
  for (int s = PRE; s < a.nsplit; ++s) {
    const float f = __shfl(fs, s, 64);
#pragma unroll
    for (int k = 0; k < PL; ++k)
      if (lane + 64 * k < DP) o[k] += a.part[(p0 + (int64_t)s * R) * DP + lane + 64 * k] * f;
  }
  const bool some = lt > 0.f || lt != lt;
  const float inv = some ? 1.f / lt : 0.f;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv, qi = row / a.G, g = row - qi * a.G;
  const int64_t at = (((int64_t)b * a.Lq + qi) * a.Hkv * a.G + hk * a.G + g) * a.D;
#pragma unroll
  for (int k = 0; k < PL; ++k)
    if (lane + 64 * k < a.D) {
      const T w = (T)(o[k] * inv);
      reinterpret_cast<T*>(a.o)[at + lane + 64 * k] = w;
      if (a.o_lo) reinterpret_cast<T*>(a.o_lo)[at + lane + 64 * k] = (T)(o[k] * inv - (float)w);
    }
  if (a.lse && lane == 0) a.lse[(int64_t)bh * R + row] = some ? mt + log2f(lt) : INFINITY;
}

// A wave per 64 rows x 64 keys: a lane gathers its row's 64 bytes into a word; ballots over the words
// turn the square for the keys' words.  (A grid of bounded size walks them: a broadcast mask has no
// memory of its own that would bound them.)
__global__ __launch_bounds__(256) void attn_pack_kernel(AttnArgs a) {
  const int R = a.G * a.Lq, nrt = (R + 63) / 64, nkt = (a.Lk + 63) / 64, nh = a.m_sh ? a.Hkv : 1, nb = a.m_sb ? a.B : 1;
  const int64_t words = (int64_t)nb * nh * nrt * nkt;
  for (int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); w < words; w += (int64_t)gridDim.x * 4) {
    const int lane = threadIdx.x & 63;
    const int kt = (int)(w % nkt), rt = (int)(w / nkt % nrt), hk = (int)(w / nkt / nrt % nh), b = (int)(w / nkt / nrt / nh);
    const int row = rt * 64 + lane, rc = min(row, R - 1), qi = rc / a.G, h = hk * a.G + rc - qi * a.G;
    const uint8_t* p = a.mask + b * a.m_sb + h * a.m_sh + (int64_t)qi * a.m_sq + (int64_t)kt * 64 * a.m_sk;
    const int n = min(64, a.Lk - kt * 64);
    uint64_t mine = 0;
    if (a.m_sk == 1 && n == 64) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 v;
        __builtin_memcpy(&v, p + 16 * c, 16);  // any alignment
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // bit 0 of each byte = any of its bits, then the four bits side by side
          uint32_t y = x[i] | x[i] >> 4;
          y |= y >> 2;
          y = (y | y >> 1) & 0x01010101u;
          mine |= (uint64_t)(y * 0x10204080u >> 28) << (16 * c + 4 * i);
        }
      }
    } else {
      for (int k = 0; k < n; ++k) mine |= (uint64_t)(p[(int64_t)k * a.m_sk] != 0) << k;
    }
    if (row >= R) mine = 0;
    const int64_t head = (int64_t)b * nh + hk;
    if (row < R) a.row_bits[(head * R + row) * nkt + kt] = mine;
    if (a.key_bits) {
      uint64_t col = 0;
#pragma unroll
      for (int k = 0; k < 64; ++k) {
        const uint64_t bits = __ballot(mine >> k & 1);
        if (lane == k) col = bits;
      }
      if (lane < n) a.key_bits[(head * a.Lk + kt * 64 + lane) * nrt + rt] = col;
    }
  }
}

template <typename T, int DP, int MASK>
void fwd_launch(const AttnArgs& a, hipStream_t s) {
  const int64_t R = (int64_t)a.G * a.Lq;
  const int64_t n = (R <= 32 ? 1 : (R + 127) / 128) * a.nsplit * a.B * a.Hkv;
  const unsigned grid = raft_cdiv(n, 8) * 8;
  if (R <= 32) attn_few_kernel<T, DP, MASK><<<grid, 256, 0, s>>>(a);
  else attn_fwd_kernel<T, DP, MASK><<<grid, 256, 0, s>>>(a);
  if (a.nsplit > 1) attn_join_kernel<T, DP><<<raft_cdiv((int64_t)a.B * a.Hkv * R, 4), 256, 0, s>>>(a);
}
template <typename T, int DP>
void fwd_mask(const AttnArgs& a, hipStream_t s) {
  if (a.mask_mode == 0) fwd_launch<T, DP, 0>(a, s);
  else if (a.mask_mode == 1) fwd_launch<T, DP, 1>(a, s);
  else fwd_launch<T, DP, 2>(a, s);
}
template <typename T>
void fwd_dim(const AttnArgs& a, hipStream_t s) {
  if (a.DP == 32) fwd_mask<T, 32>(a, s);
  else if (a.DP == 64) fwd_mask<T, 64>(a, s);
  else if (a.DP == 96) fwd_mask<T, 96>(a, s);
  else fwd_mask<T, 128>(a, s);
}

}  // namespace attn_detail

void attn_fwd_plan(AttnArgs& a) {
  const int64_t R = (int64_t)a.G * a.Lq, heads = (int64_t)a.B * a.Hkv;
  // Enough workgroups for the 256 CUs: key ranges are split (and joined by a second launch) when the
  // row tiles alone leave CUs idle; a range keeps at least 256 keys (64 in fp32, whose products take 16
  // times as long) so the join stays small.  Few rows: two workgroups a CU (32 caches of up to 16384
  // keys: 304 us; with four or eight 306 and 308).
  const int64_t n = (R <= 32 ? 1 : (R + 127) / 128) * heads;
  const int64_t want = R <= 32 ? 512 : 256, least = a.dtype == 2 ? 64 : 256;
  const int64_t s = std::min<int64_t>(want / std::max<int64_t>(n, 1), (a.Lk + least - 1) / least);
  a.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(s, 64));
}

int64_t attn_bit_words(const AttnArgs& a, bool keys) {
  if (a.mask_mode != 2) return 0;
  const int64_t R = (int64_t)a.G * a.Lq, heads = (int64_t)(a.m_sb ? a.B : 1) * (a.m_sh ? a.Hkv : 1);
  return heads * (keys ? a.Lk * ((R + 63) / 64) : R * ((a.Lk + 63) / 64));
}

void launch_attn_pack(const AttnArgs& a, hipStream_t s) {
  const int64_t R = (int64_t)a.G * a.Lq, heads = (int64_t)(a.m_sb ? a.B : 1) * (a.m_sh ? a.Hkv : 1);
  attn_detail::attn_pack_kernel<<<(unsigned)std::min<int64_t>((heads * ((R + 63) / 64) * ((a.Lk + 63) / 64) + 3) / 4, 2048), 256, 0, s>>>(a);
}

void launch_attn_fwd(const AttnArgs& a, hipStream_t s) {
  if (a.mask_mode == 2) launch_attn_pack(a, s);
  if (a.dtype == 0) attn_detail::fwd_dim<__bf16>(a, s);
  else if (a.dtype == 1) attn_detail::fwd_dim<_Float16>(a, s);
  else attn_detail::fwd_dim<float>(a, s);
}

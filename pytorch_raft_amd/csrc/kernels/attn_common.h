// Shared pieces of the token-attention kernels (attn_fwd.hip, attn_bwd.hip).
//
// Every product runs on 32x32 MFMA tiles with an 8-element fragment per lane and a 16-wide K step:
// one v_mfma_f32_32x32x16 for bf16 / fp16, eight v_mfma_f32_32x32x2_f32 for fp32 (same lane roles,
// so one kernel body serves the three types; fp32 runs at 1/16 of the 16-bit rate).
//   A: lane holds row (lane & 31), K elements hi * 8 + i   (hi = lane >> 5, i = 0..7)
//   B: lane holds column (lane & 31), the same K elements
//   C: lane holds column (lane & 31), rows (r / 4) * 8 + hi * 4 + r % 4   (r = 0..15)
// Any bijection of the K elements works as long as A and B agree, so a C tile (probabilities) is fed
// straight back as the next product's B operand: K step t takes accumulator registers 8 t .. 8 t + 7,
// i.e. C rows 16 t + (i / 4) * 8 + hi * 4 + i % 4.  The A operand of that product is read from a
// row-major LDS tile, transposed, in the same order: two ds_read_b64_tr_b16 (four rows each).
// No probability ever goes through LDS.
//
// "Rows" are the queries of all G heads that share a key head, position-major: row r is query
// r / G of head r % G of the group.
#pragma once
#include "common.h"
#include "launchers.h"

namespace attn_detail {

typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4bf lds_v4bf;
typedef __amdgpu_buffer_rsrc_t rsrc_t;

constexpr uint32_t kOob = 0x80000000u;  // a byte offset past every descriptor's range: reads as zeros

template <typename T> struct FragOf;
template <> struct FragOf<__bf16> { typedef v8bf type; };
template <> struct FragOf<_Float16> { typedef v8h type; };
template <> struct FragOf<float> { typedef f32x8_t type; };

__device__ __forceinline__ f32x16 mma(v8bf a, v8bf b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(v8h a, v8h b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8_t a, f32x8_t b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// the other half-wave's value combined with this one's (lane ^ 32)
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// A tile of rows of DP elements in LDS as 16-byte chunks; chunk c of row r lies in slot c ^ swz(r),
// so that neither the fragment reads (16 rows, one chunk) nor the transposed reads (4 rows, 64
// bytes) meet in a bank.  The DMA image is lane-linear, so the lane that fills a slot fetches that
// slot's logical chunk.
template <typename T, int DP>
struct Tile {
  static constexpr int ES = sizeof(T);
  static constexpr int RB = DP * ES;   // bytes of a row
  static constexpr int NC = RB / 16;   // chunks of a row
  __device__ static __forceinline__ int swz(int row) {
    if constexpr (RB % 256 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (RB == 128) return (((row >> 1) & 1) << 2) | (((row >> 2) & 1) << 1) | ((row >> 3) & 1);
    else if constexpr (RB % 128 == 0) return ((row & 1) << 2) | ((row >> 1) & 3);
    else return (row >> 2) & 3;
  }
  using Frag = typename FragOf<T>::type;

  // swz is linear over xor and uses row bits 0..3 only, and what depends on the lane and what is known
  // at compile time never share a bit of row or chunk.  So one register per view of a tile (rows_base,
  // cols_base: byte addresses in LDS) gives every address by an xor of a constant into the chunk bits
  // (MASK) and an immediate offset.
  static constexpr int MASK = RB % 256 == 0 ? 15 : RB % 128 == 0 ? 7 : 3;
  template <typename V>
  __device__ static __forceinline__ V at(uint32_t base, int c, int off) {
    return *reinterpret_cast<const __attribute__((address_space(3))) V*>((base ^ ((uint32_t)(c & MASK) << 4)) + (uint32_t)((c & ~MASK) * 16 + off));
  }

  // rows view: fragment t of row 32 * rb + (lane & 31) = its elements 16 t + hi * 8 .. + 7
  __device__ static __forceinline__ uint32_t rows_base(uint32_t lds, int lane) {
    const int row = lane & 31, hi = lane >> 5;
    return lds + row * RB + (((ES == 2 ? hi : 2 * hi) ^ swz(row)) << 4);
  }
  __device__ static __forceinline__ Frag rows(uint32_t base, int rb, int t) {
    if constexpr (ES == 2) {
      return at<Frag>(base, 2 * t, rb * 32 * RB);
    } else {
      const f32x4 a = at<f32x4>(base, 4 * t, rb * 32 * RB);
      const f32x4 b = at<f32x4>(base, 4 * t + 1, rb * 32 * RB);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // columns view: column 32 * cb + (lane & 31), rows r0 + hi * 4 + {0..3}, r0 + 8 + hi * 4 + {0..3}
  // (r0 a multiple of 16)
  __device__ static __forceinline__ uint32_t cols_base(uint32_t lds, int lane) {
    if constexpr (ES == 2) {
      const int row = (lane >> 5) * 4 + ((lane & 15) >> 2), col = ((lane >> 4) & 1) * 16 + 4 * (lane & 3);
      return lds + row * RB + (((col >> 3) ^ swz(row)) << 4) + (col & 7) * 2;
    } else {
      const int row = (lane >> 5) * 4, col = lane & 31;
      return lds + row * RB + (((col >> 2) ^ swz(row)) << 4) + (col & 3) * 4;
    }
  }
  __device__ static __forceinline__ Frag cols(uint32_t base, int r0, int cb) {
    if constexpr (ES == 2) {
      const int c0 = (4 * cb) ^ swz(0), c1 = (4 * cb) ^ swz(8);
      const v4bf lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
          (lds_v4bf*)(size_t)((base ^ ((uint32_t)(c0 & MASK) << 4)) + (uint32_t)((c0 & ~MASK) * 16 + r0 * RB)));
      const v4bf hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
          (lds_v4bf*)(size_t)((base ^ ((uint32_t)(c1 & MASK) << 4)) + (uint32_t)((c1 & ~MASK) * 16 + (r0 + 8) * RB)));
      return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      Frag f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = (i >> 2) * 8 + (i & 3);
        f[i] = at<float>(base, (8 * cb) ^ swz(row), (r0 + row) * RB);
      }
      return f;
    }
  }
};

// eight probabilities (accumulator registers 8 t .. 8 t + 7) as a B fragment, rounded to nearest: the operand
// type of the matrix instructions, 16 times the rate of fp32 ones.  This rounding (and that of dS) is seen in
// the results: outputs and gradients in bf16 are off by 0.0023-0.0024 of their norm where their own rounding
// alone makes 0.0017, in fp16 by 0.00024-0.00031 where it makes 0.0002.
template <typename T>
__device__ __forceinline__ typename FragOf<T>::type to_frag(const f32x16& s, int t) {
  typename FragOf<T>::type f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (T)s[8 * t + i];
  return f;
}

__device__ __forceinline__ rsrc_t rsrc_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// 1-D grids are padded to a multiple of 8: the dispatcher deals consecutive blocks to the 8 XCDs in
// turn, so logical order xcd * (n / 8) + slot keeps the blocks that share a key head on one XCD's L2.
__device__ __forceinline__ int xcd_order(int bid, int grid) { return (bid & 7) * (grid >> 3) + (bid >> 3); }

// workgroup -> (tile, split, batch x key head).  Without causal the blocks of a head stay on one XCD;
// causal tiles differ in length, so they are dealt over all CUs, longest first.
__device__ __forceinline__ bool place(const AttnArgs& a, int bid, int grid, int tiles, int nsplit, bool last_first, int& tile, int& split, int& bh) {
  const int heads = a.B * a.Hkv;
  const int id = a.causal ? bid : xcd_order(bid, grid);
  if (id >= tiles * nsplit * heads) return false;
  if (a.causal) {
    bh = id % heads;
    split = id / heads % nsplit;
    tile = id / heads / nsplit;
  } else {
    tile = id % tiles;
    split = id / tiles % nsplit;
    bh = id / tiles / nsplit;
  }
  if (last_first) tile = tiles - 1 - tile;
  return true;
}

// One thread's share of the LDS-DMA of ROWS rows (x DP) by NTHR threads: byte offsets from the
// tile's first row, fixed over the loop (row pitch `pitch` bytes); rows past the descriptor's end
// and channels past D read as zeros.
template <typename T, int DP, int ROWS, int NTHR>
struct Loader {
  using TL = Tile<T, DP>;
  static constexpr int PER = ROWS * TL::NC / NTHR;
  static_assert(ROWS * TL::NC % NTHR == 0, "whole instructions");
  uint32_t off[PER];
  __device__ __forceinline__ static int row_of(int tid, int j) { return (j * NTHR + tid) / TL::NC; }
  __device__ __forceinline__ static int chunk_of(int tid, int j) {
    const int e = j * NTHR + tid;
    return (e % TL::NC) ^ TL::swz(e / TL::NC);
  }
  __device__ __forceinline__ void init(int tid, uint32_t pitch, int dbytes) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int c = chunk_of(tid, j) * 16;
      off[j] = c < dbytes ? row_of(tid, j) * pitch + c : kOob;
    }
  }
};

// descriptor of `rows` rows from `base` on (rows <= 0: nothing is read)
__device__ __forceinline__ rsrc_t rows_rsrc(const uint8_t* base, int rows, uint32_t pitch, int dbytes) {
  return rsrc_of(base, rows > 0 ? (uint32_t)(rows - 1) * pitch + dbytes : 0u);
}

// number of keys that item b holds
__device__ __forceinline__ int item_len(const AttnArgs& a, int b) {
  return a.lengths ? max(0, min(a.lengths[b], a.Lk)) : a.Lk;
}
// position of item b's first query among the keys (clamped to where it stops to matter)
__device__ __forceinline__ int item_off(const AttnArgs& a, int b) {
  return a.q_offset ? max(-a.Lq, min(a.q_offset[b], a.Lk)) : a.Lk - a.Lq;
}

// A (query, key) mask comes as bits, packed once a call by attn_pack_kernel: for each row (packed order)
// words over 64 keys, and for the dk / dv kernel for each key words over 64 rows.  Masks shared by heads
// or items are packed once (bit_head).
__device__ __forceinline__ int64_t bit_head(const AttnArgs& a, int b, int hk) {
  return (a.m_sb ? (int64_t)b * (a.m_sh ? a.Hkv : 1) : 0) + (a.m_sh ? hk : 0);
}
__device__ __forceinline__ const uint64_t* row_bits(const AttnArgs& a, int b, int hk, int row) {
  return a.row_bits + (bit_head(a, b, hk) * a.G * a.Lq + row) * ((a.Lk + 63) / 64);
}
__device__ __forceinline__ const uint64_t* key_bits(const AttnArgs& a, int b, int hk, int key) {
  return a.key_bits + (bit_head(a, b, hk) * a.Lk + key) * ((a.G * a.Lq + 63) / 64);
}

}  // namespace attn_detail

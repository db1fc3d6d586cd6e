// What the store into and the attention over a paged key-value cache share: the cache's and the batch's description as
// the kernels take it, the sequences' geometry, and wave-level helpers.
//
// A batch is ragged: sequence b has rows query_start[b] .. query_start[b+1] of q (without query_start: row b alone) and
// seq_lens[b] keys, those rows' own among them; its i-th row stands at position seq_lens[b] - n + i.  Key j lies in row
// j % page_size of page block_table[b][j / page_size].
#pragma once
#include "common.hpp"

namespace fmsmo {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

constexpr int PROMPT_ROWS = 128, PROMPT_KEYS = 64;  // tiles of the prompt kernel

constexpr float LOG2E = 1.44269504088896340736f;

struct PagedArgs {
  const char* k;
  const char* v;
  const float* ks;  // e4m3 caches: one scale per key and head
  const float* vs;
  int64_t k_page, k_head, v_page, v_head;      // bytes
  int64_t ks_page, ks_head, vs_page, vs_head;  // elements; the keys of a page lie side by side
  int k_slot, v_slot;                          // bytes
  const int* table;
  int64_t table_stride;
  const int* lens;
  const int* starts;  // NULL: one row per sequence
  int cap;            // keys a row of the block table can name
  int seqs, rows;     // rows of q
  int page_shift, pages, kv_heads, group;
  const char* q;
  char* out;
  int64_t q_row, q_head, o_row, o_head;  // bytes
  float c;                               // scale * log2(e): the softmax runs on powers of two
  int window, sinks;                     // window 0: every key up to the row's own
  int zero_rest;                         // rows of no sequence become zero (else: are left as they are)
};

// The rows of no sequence: `n` 16-byte pieces per head, every block of the launch takes some of the rows.
__device__ __forceinline__ void zero_rest(const PagedArgs& a, int n) {
  const int from = a.starts[0], to = a.starts[a.seqs], heads = a.kv_heads * a.group;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    if (r >= from && r < to) {
      if (to >= a.rows) break;
      r += (to - 1 - r) / (int)gridDim.x * (int)gridDim.x;  // on to the last of this block's rows before `to`
      continue;
    }
    for (int i = threadIdx.x; i < heads * n; i += blockDim.x)
      *(v4i*)(a.out + r * a.o_row + i / n * a.o_head + i % n * 16) = v4i{0, 0, 0, 0};
  }
}

// One sequence of the batch.  Nothing here trusts the arrays: rows outside of q and keys outside of the table's row are
// not there, whatever they say.
struct Seq {
  int n, row0;    // rows of q
  int pos0;       // position of the first of them
  int len;        // keys the table can name
};
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int b) {
  Seq s;
  int r0 = b, r1 = b + 1;
  if (a.starts) {
    r0 = a.starts[b];
    r1 = a.starts[b + 1];
  }
  const int len = a.lens[b];
  int n = r1 > r0 && r0 >= 0 ? r1 - r0 : 0;
  n = n < a.rows ? n : a.rows;
  s.pos0 = (len < 0 ? 0 : len) - n;
  s.row0 = r0;
  s.n = r0 >= a.rows ? 0 : n < a.rows - r0 ? n : a.rows - r0;
  s.len = len < 0 ? 0 : len < a.cap ? len : a.cap;
  return s;
}

// The keys that some row at a position of p_lo .. p_hi sees, in tiles of TILE keys: those of the sinks, then from the first one
// inside p_lo's window up to p_hi.  Tile t starts at key (t < sink_tiles ? t : t + skip) * TILE.
struct Tiles {
  int count, sink_tiles, skip;
};
template <int TILE>
__device__ __forceinline__ Tiles tiles_of(const PagedArgs& a, int len, int p_lo, int p_hi) {
  Tiles t;
  int end = p_hi + 1 < len ? p_hi + 1 : len;
  if (end < 0) end = 0;
  const int all = (end + TILE - 1) / TILE;
  int lo = a.window ? (p_lo > 0 ? p_lo : 0) - a.window + 1 : 0;
  if (lo < 0) lo = 0;
  const int s = a.sinks < lo ? a.sinks : lo;
  t.sink_tiles = (s + TILE - 1) / TILE;
  if (t.sink_tiles > all) t.sink_tiles = all;
  t.skip = lo / TILE - t.sink_tiles;
  if (t.skip < 0) t.skip = 0;
  t.count = all - t.skip > t.sink_tiles ? all - t.skip : t.sink_tiles;
  return t;
}
// every row of positions p_lo .. p_hi sees every key of j0 .. j1
__device__ __forceinline__ bool sees_all(const PagedArgs& a, int p_lo, int p_hi, int j0, int j1) {
  return j1 <= p_lo && (a.window == 0 || j0 > p_hi - a.window || j1 < a.sinks);
}

// The keys that rows at positions p_lo .. p_hi may see (some of them, p_lo < p_hi), as bounds of their offsets from key `at`:
// offset <= hi and (offset > lo or offset < sink)
struct Bounds {
  int hi, lo, sink;
};
__device__ __forceinline__ Bounds bounds_of(const PagedArgs& a, int p_lo, int p_hi, int len, int at) {
  Bounds b;
  b.hi = (p_hi < len - 1 ? p_hi : len - 1) - at;
  // (a length beyond the table's keys may be any int, and so may a window: nothing here leaves 32 bits)
  const int lo = (p_lo > 0 ? p_lo : 0) - a.window;
  b.lo = a.window ? (lo > -1 ? lo : -1) - at : -(1 << 30);
  b.sink = a.sinks - at;
  return b;
}
__device__ __forceinline__ bool inside(const Bounds& b, int off) { return off <= b.hi && (off > b.lo || off < b.sink); }

// ------------------------------------------------------------------ work split over a sequence's keys
struct SplitArgs {
  PagedArgs p;
  float* ws;
  int cuts;                 // entries that tell the join of a head and rows that several blocks share
  int workers, unit_shift;  // split kernel: 1 << unit_shift tiles are never divided between blocks
  int row_shift;            // 16 << row_shift rows in a share; split kernel: 1 << row_shift waves of a block take the same keys
  int splits;               // the workspace is there
  int tiles, parts;         // prompt kernel: tiles of rows, blocks for each
};
// Shares first .. last of rows row0 .. of a key head's queries (counted as tokens x heads of the group)
struct Cut {
  int rows;         // 0: nothing to join
  int first, last;  // shares
  int pad;
  int row0;       // q row of the sequence
  int pair_row0;  // first row in it
  int head;       // key head
  int pad2;
};
// workspace: Cut[cuts], then shares of { o[rows][D], (m, l)[rows] }
template <int D>
__device__ __forceinline__ float* share_of(const SplitArgs& a, int share) {
  return (float*)((Cut*)a.ws + a.cuts) + (((int64_t)share * 16 * (D + 2)) << a.row_shift);
}

// ------------------------------------------------------------------ cross-lane
// a maximum (sum) over the lanes that differ in bit 5, and in bits 5 and 4: v_permlane*_swap, no LDS round trip
__device__ __forceinline__ float max_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// 16 bytes a lane from `at` + off into 1 KiB of shared memory, lane after lane
__device__ __forceinline__ void to_shared(const char* at, char* lds, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)at, 0, 0x7fffffff, 0x00020000), FMSMO_LPTR(lds), 16, off, 0, 0, 0);
}

// ------------------------------------------------------------------ 16-bit operands
// two fp32 values rounded to nearest even, packed
template <int T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  uint32_t u;
  if constexpr (T == FMSMO_F16) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = {(_Float16)x, (_Float16)y};
    __builtin_memcpy(&u, &h, 4);
  } else {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 h = {(__bf16)x, (__bf16)y};
    __builtin_memcpy(&u, &h, 4);
  }
  return u;
}
// four e4m3 values (exact in fp16 and in bf16) as two packed pairs
template <int T>
__device__ __forceinline__ void widen4(uint32_t u, uint32_t& lo, uint32_t& hi) {
  if constexpr (T == FMSMO_F16) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, true);
    __builtin_memcpy(&lo, &a, 4);
    __builtin_memcpy(&hi, &b, 4);
  } else {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, true);
    __builtin_memcpy(&lo, &a, 4);
    __builtin_memcpy(&hi, &b, 4);
  }
}
// Infinities and NaN among the values of keys that some rows see and others don't: 0 * inf is not 0, so they leave the product
// (finite_only), and are added to the rows that see them behind the loop over the keys (add_odd) -- to which they are all that matters.
template <int T>
__device__ __forceinline__ uint32_t finite_only(uint32_t u) {
  constexpr uint32_t E = T == FMSMO_F16 ? 0x7c00u : 0x7f80u;
  return ((u & E) == E ? 0u : u & 0xffffu) | ((u >> 16 & E) == E ? 0u : u & 0xffff0000u);
}
template <int T>
__device__ __forceinline__ float add_odd(float o, u16 h, bool seen) {
  constexpr u16 E = T == FMSMO_F16 ? 0x7c00 : 0x7f80;
  return seen && (h & E) == E ? o + (T == FMSMO_F16 ? f16_to_f32(h) : bf16_to_f32(h)) : o;
}

// D[16 x 16] += A[16 x 32] . B[32 x 16]: lane l holds row (column) l % 16 of A (B), elements 8 (l / 16) .. + 7 of the reduction;
// of D column l % 16, rows 4 (l / 16) .. + 3
template <int T>
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
  if constexpr (T == FMSMO_F16) {
    h8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  } else {
    b8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
}
// D[32 x 32] += A[32 x 16] . B[16 x 32]: lane l holds row (column) l % 32 of A (B), elements 8 (l / 32) .. + 7 of the reduction;
// of D column l % 32, in register 4 i + j row 8 i + 4 (l / 32) + j
template <int T>
__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
  if constexpr (T == FMSMO_F16) {
    h8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
  } else {
    b8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  }
}

// ------------------------------------------------------------------ softmax
// exp2(x - m) where m is a maximum that may still be -inf (nothing seen yet)
__device__ __forceinline__ float safe_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace fmsmo

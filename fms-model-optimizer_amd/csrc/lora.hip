// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + scale_s B_s (A_s x[t]), s the adapter of the request that
// row t belongs to.  Two launches.  The first makes v = A_s x in fp32, K cut into parts where there are few rows; the second adds the
// parts, takes v as the sum of two 16-bit numbers (so that the product B v is as exact as its operands B; with rank 16 the two halves fill one
// matrix instruction) and adds the product to y, rounded once.
//
// A tile is up to 16 MT rows of one adapter.  One row per request: the rows of the requests that share an adapter, sixteen at a time, found by
// counting; else 16 MT consecutive rows of a request.
#include "paged_kv.hpp"
#include "stream_loads.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace fmsmo {

struct LoraArgs {
  const char* x;
  const char* y;
  char* out;
  const char* a;       // [slots, rank, K]
  const char* b;       // [slots, N, rank]
  const int* adapters; // [seqs]
  const int* starts;   // [seqs + 1], NULL: one row per request
  const float* scales; // [slots] or NULL
  float* ws;           // [parts][tiles][16 MT][16 RT]
  int64_t ldx, ldy, ldo, a_slot, a_row, b_slot, b_row;  // bytes
  int rows, seqs, slots, rank, K, N;
  int parts, part_steps;  // steps of 64 elements a part
  int tiles, cols;        // cols: groups of 64 outputs a block of the second launch
};

// The rows of a tile: `n` of them, in `list` where they are not row0, row0 + 1, ..  slot < 0: no adapter.  n = 0: nothing to do.
struct LoraTile {
  int n, row0, slot;
};
template <int TR>
__device__ __forceinline__ LoraTile lora_tile(const LoraArgs& a, int tile, int* list) {
  const int lane = threadIdx.x & 63;
  LoraTile t{0, 0, -1};
  if (!a.starts) {
    // The adapters of the first 256 requests at once, the others 64 by 64. One load behind the other for the first too:
    // 256 requests of rank 16 8.9 + 8.3 us, 7.8 + 7.4 so.
    constexpr int Q = 4;
    int held[Q] = {a.adapters[min(lane, a.seqs - 1)], -1, -1, -1}, slot = 0;
    if (a.seqs > 64) {
#pragma unroll
      for (int q = 1; q < Q; ++q) held[q] = a.adapters[min(64 * q + lane, a.seqs - 1)];
    }
    if (tile >= 64 * Q) slot = a.adapters[tile];
#pragma unroll
    for (int q = 0; q < Q; ++q) slot = tile >> 6 == q ? __builtin_amdgcn_readlane(held[q], tile & 63) : slot;
    slot = uniform(slot);
    if ((unsigned)slot >= (unsigned)a.slots) {  // on its own: the copy of its row
      t.n = 1;
      t.row0 = tile;
      if (threadIdx.x == 0) list[0] = tile;
      return t;
    }
    // the requests of this adapter before this one; a tile starts at each TR-th of them
    int before = 0, mine = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) before += __popcll(__ballot(64 * q + lane < tile && held[q] == slot));
    for (int i = 64 * Q; i < tile; i += 64) before += __popcll(__ballot(i + lane < tile && a.adapters[i + lane] == slot));
    before = uniform(before);
    if (before % TR) return t;
    const auto take = [&](int i, int id) {
      const bool same = i + lane >= tile && i + lane < a.seqs && id == slot;
      const uint64_t m = __ballot(same);
      const int at = mine + __popcll(m & ((1ull << lane) - 1));
      if (same && at < TR && threadIdx.x < 64) list[at] = i + lane;
      mine += __popcll(m);
    };
#pragma unroll
    for (int q = 0; q < Q; ++q) take(64 * q, held[q]);
    for (int i = max(tile & ~63, 64 * Q); i < a.seqs && mine < TR; i += 64) take(i, a.adapters[min(i + lane, a.seqs - 1)]);
    mine = uniform(mine);
    t.n = mine < TR ? mine : TR;
    t.row0 = tile;
    t.slot = slot;
    return t;
  }
  // request -1: the rows before the first one, request `seqs`: those behind the last; neither has an adapter
  int seen = 0;
  for (int i = -1; i <= a.seqs; i += 64) {
    const int b = i + lane;
    int r0 = 0, r1 = 0, id = -1;
    if (b <= a.seqs) {
      r0 = b < 0 ? 0 : a.starts[b];
      r1 = b >= a.seqs ? a.rows : a.starts[b + 1];
      if (b >= 0 && b < a.seqs) id = a.adapters[b];
      r0 = r0 < 0 ? 0 : r0 < a.rows ? r0 : a.rows;
      r1 = r1 < 0 ? 0 : r1 < a.rows ? r1 : a.rows;
    }
    const int n = r1 > r0 ? r1 - r0 : 0, mine = (int)(((int64_t)n + TR - 1) / TR);
    int upto = mine;  // tiles of this lane's request and of those before it (starts that go up and down may name very many)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      upto = min(upto + (lane >= d ? o : 0), 1 << 29);
    }
    const int first = seen + upto - mine;
    const uint64_t hit = __ballot(tile >= first && tile < first + mine);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int at = (tile - __shfl(first, l)) * TR;
      const int rn = __shfl(n, l) - at;
      t.row0 = uniform(__shfl(r0, l) + at);
      t.n = uniform(rn < TR ? rn : TR);
      const int slot = uniform(__shfl(id, l));
      t.slot = (unsigned)slot < (unsigned)a.slots ? slot : -1;
      return t;
    }
    seen += uniform(__shfl(upto, 63));
    if (seen > tile) break;
  }
  return t;
}

constexpr int LORA_STEP = 64;  // elements of K a step: 128 bytes of a row

// v of a tile over a part of K.  Rows of A (16 RT) and of x (16 MT) meet as the two operands of 16 x 16 x 32; the side with more bytes comes
// through shared memory, eight rows of 128 bytes a load, the other one straight into the operands' layout, D steps of a wave on their way.  Rows past
// the rank and the tile's end are the last one again: what comes of them is not looked at.
// (From rank 33 on the sums stay in the registers that the products are made in: two waves a SIMD are asked for.  Rank 128, 4096 rows of 4096: 30 us
// without, 22 with; at rank 32 that leaves too few, 45 and 79 us.)
template <int T, int RT, int MT, int D>
__global__ __launch_bounds__(256, RT >= 4 ? 2 : 1) void lora_shrink_kernel(LoraArgs a) {
  constexpr bool X_STAGED = MT > 1;
  constexpr int S = X_STAGED ? MT : RT, O = X_STAGED ? RT : MT;  // tiles of 16 rows of the staged and the other side
  constexpr int SUMS = MT * 16 * (RT * 16 + 4) * 4;  // bytes of a wave's sums; they take the place of the staged rows
  __shared__ __attribute__((aligned(16))) char stage[S * 8192 > 2 * SUMS ? S * 8192 : 2 * SUMS];
  __shared__ int list[MT * 16];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const LoraTile t = lora_tile<16 * MT>(a, blockIdx.x, list);
  if (t.n == 0 || t.slot < 0) return;
  if (!a.starts) __syncthreads();
  const int r = lane & 15, g = lane >> 4, drow = lane >> 3, dpos = lane & 7;
  // rows of x are counted from the tile's first one (the host sees to it that offsets fit)
  const Buf A = buf_of(a.a + (int64_t)t.slot * a.a_slot), X = buf_of(a.x + (int64_t)t.row0 * a.ldx);
  const int s0 = blockIdx.y * a.part_steps, s1 = min(s0 + a.part_steps, (a.K + LORA_STEP - 1) / LORA_STEP);
  const auto a_off = [&](int q) { return (uint32_t)min(q, a.rank - 1) * (uint32_t)a.a_row; };
  const auto x_off = [&](int q) {
    q = min(q, t.n - 1);
    return (uint32_t)(a.starts ? q : list[q] - t.row0) * (uint32_t)a.ldx;
  };
  uint32_t so[2 * S], oo[O];
#pragma unroll
  for (int i = 0; i < 2 * S; ++i) so[i] = (X_STAGED ? x_off(8 * i + drow) : a_off(8 * i + drow)) + dpos * 16;
#pragma unroll
  for (int i = 0; i < O; ++i) oo[i] = (X_STAGED ? a_off(16 * i + r) : x_off(16 * i + r)) + g * 16;
  const Buf sp = X_STAGED ? X : A, op = X_STAGED ? A : X;
  v4f acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  char* st = stage + wave * (S * 2048);
  const int rr = r & 7;
  v4i sb[D][2 * S], ob[D][O][2];
  const auto fetch = [&](int s, int d) {  // (zeros past the part and past the row's end)
    const uint32_t k = s * 2 * LORA_STEP;
    const int left = s < s1 ? a.K - s * LORA_STEP : 0;
#pragma unroll
    for (int i = 0; i < 2 * S; ++i)
      sb[d][i] = X_STAGED ? buf_stream(sp, dpos * 8 < left ? so[i] : BUF_NONE, k) : buf_load(sp, dpos * 8 < left ? so[i] : BUF_NONE, k);
#pragma unroll
    for (int i = 0; i < O; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) ob[d][i][h] = buf_load(op, (4 * h + g) * 8 < left ? oo[i] + 64 * h : BUF_NONE, k);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(s0 + wave + 4 * d, d);
  for (int s = s0 + wave; s < s1; s += 4 * D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      // chunk c of row q lies at position c ^ (q % 8)
#pragma unroll
      for (int i = 0; i < 2 * S; ++i) *(v4i*)(st + (8 * i + drow) * 128 + ((dpos ^ drow) * 16)) = sb[d][i];
      __builtin_amdgcn_wave_barrier();  // (the rows go to other lanes of the wave)
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const v4i w = *(const v4i*)(st + (16 * i + r) * 128 + (((4 * h + g) ^ rr) * 16));
#pragma unroll
          for (int j = 0; j < O; ++j) {
            if constexpr (X_STAGED) acc[j][i] = mfma16<T>(ob[d][j][h], w, acc[j][i]);
            else acc[i][j] = mfma16<T>(w, ob[d][j][h], acc[i][j]);
          }
        }
      __builtin_amdgcn_wave_barrier();
      fetch(s + 4 * (D + d), d);
    }
  }
  // the waves' sums: (0 + 2) + (1 + 3)
  const auto put = [&](int at) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) *(v4f*)(stage + at * SUMS + ((16 * j + r) * (16 * RT + 4) + 16 * i + 4 * g) * 4) = acc[i][j];
  };
  const auto add = [&](int at) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] += *(const v4f*)(stage + at * SUMS + ((16 * j + r) * (16 * RT + 4) + 16 * i + 4 * g) * 4);
  };
  __syncthreads();
  if (wave >= 2) put(wave - 2);
  __syncthreads();
  if (wave < 2) add(wave);
  __syncthreads();
  if (wave == 1) put(0);
  __syncthreads();
  if (wave) return;
  add(0);
  float* to = a.ws + ((int64_t)blockIdx.y * a.tiles + blockIdx.x) * (256 * MT * RT);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *(v4f*)(to + (16 * j + r) * 16 * RT + 16 * i + 4 * g) = acc[i][j];
}

// out = y + B v for a tile and `cols` groups of 64 outputs, a group a wave at a time: 64 rows of B as operands in registers, then the tile's rows,
// sixteen by sixteen, whose products go through shared memory so that y is read and out is written in eight rows of 128 bytes.  The next group's y
// (and B, where the rank leaves registers) are on their way meanwhile.
template <int T, int RT, int MT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  constexpr int TR = 16 * MT, LD = 64 * RT + 16;  // bytes of a row of v: both halves of 16 RT numbers, and a step in banks
  constexpr int KB = RT == 1 ? 1 : RT / 2;        // products over the rank; up to 16 both halves of v fill one
  constexpr int NB = RT <= 4 ? 2 : 1;
  constexpr int LT = 68;                          // numbers of a row of products
  constexpr int GONE = 1 << 17;                   // no group: past any N
  __shared__ __attribute__((aligned(16))) char vs[TR][LD];
  __shared__ __attribute__((aligned(16))) float turn[4][16 * LT];
  __shared__ float lift[TR];
  __shared__ int list[TR];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const LoraTile t = lora_tile<TR>(a, blockIdx.x, list);
  if (t.n == 0) return;
  if (t.slot < 0 && a.y == a.out) return;
  if (!a.starts) __syncthreads();
  const int r = lane & 15, g = lane >> 4, drow = lane >> 3, dpos = lane & 7;
  const int c0 = blockIdx.y * a.cols + wave, c1 = min((int)(blockIdx.y + 1) * a.cols, (a.N + 63) / 64);
  const int R = a.rank;
  const Buf B = buf_of(a.b + (int64_t)(t.slot < 0 ? 0 : t.slot) * a.b_slot);
  const Buf Y = buf_of(a.y + (int64_t)t.row0 * a.ldy), O = buf_of(a.out + (int64_t)t.row0 * a.ldo);
  // row 8 q + drow of the tile, eight outputs a lane
  const auto row_of = [&](int q) { return a.starts ? q : list[q] - t.row0; };
  v4i yv[MT][2], bw[NB][KB][4];
  const auto fetch_y = [&](int c, int j) {
    const bool in = c * 64 + 8 * dpos < a.N;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int q = 16 * j + 8 * h + drow;
      yv[j][h] = buf_load(Y, in && q < t.n ? (uint32_t)row_of(q) * (uint32_t)a.ldy + dpos * 16 : BUF_NONE, (uint32_t)c * 128);
    }
  };
  const auto put = [&](int c, int j, int h, v4i o) {
    const int q = 16 * j + 8 * h + drow;
    buf_store(O, o, q < t.n && c * 64 + 8 * dpos < a.N ? (uint32_t)row_of(q) * (uint32_t)a.ldo + dpos * 16 + (uint32_t)c * 128 : BUF_NONE);
  };
  const auto fetch_b = [&](int c, v4i (&w)[KB][4]) {
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const int e = RT == 1 ? 8 * (g & 1) : 32 * k + 8 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = c * 64 + 16 * i + r;
        w[k][i] = buf_load(B, n < a.N && e < R ? (uint32_t)n * (uint32_t)a.b_row + 2 * e : BUF_NONE);
      }
    }
  };
  if (t.slot < 0) {  // the bits of y
    for (int c = c0; c < c1; c += 4)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        fetch_y(c, j);
        put(c, j, 0, yv[j][0]);
        put(c, j, 1, yv[j][1]);
      }
    return;
  }
  fetch_b(c0, bw[0]);
#pragma unroll
  for (int j = 0; j < MT; ++j) fetch_y(c0, j);
  {
    const float scale = a.scales ? a.scales[t.slot] : 1.0f;
    const float* from = a.ws + (int64_t)blockIdx.x * (256 * MT * RT);
    const int64_t part = (int64_t)a.tiles * (256 * MT * RT);
    // In quadruples of a row: v, brought to a maximum of 1 to 4 by a power of two (fp16 holds neither large numbers nor the lower halves of
    // small ones), its upper half at k, what that leaves 16 RT numbers behind.  Rows past the tile's end and numbers past the rank are zero.
    constexpr int QS = (TR * 4 * RT + 255) / 256;  // quadruples of a thread (of the first 64 or 128 threads alone, where there are few)
    v4f sum[QS];
#pragma unroll
    for (int q = 0; q < QS; ++q) sum[q] = v4f{0, 0, 0, 0};
    const int last = t.n * 4 * RT - 1;
    int p = 0;
    for (; p + 4 <= a.parts; p += 4) {  // (four loads on their way)
#pragma unroll
      for (int q = 0; q < QS; ++q) {
        const float* at = from + p * part + 4 * min((int)threadIdx.x + 256 * q, last);
        const v4f v0 = *(const v4f*)at, v1 = *(const v4f*)(at + part), v2 = *(const v4f*)(at + 2 * part), v3 = *(const v4f*)(at + 3 * part);
        sum[q] += (v0 + v1) + (v2 + v3);
      }
    }
    for (; p < a.parts; ++p)
#pragma unroll
      for (int q = 0; q < QS; ++q) sum[q] += *(const v4f*)(from + p * part + 4 * min((int)threadIdx.x + 256 * q, last));
#pragma unroll
    for (int q = 0; q < QS; ++q) {
      const int i = threadIdx.x + 256 * q, c = i / (4 * RT), k = i % (4 * RT) * 4;
      if (i >= TR * 4 * RT) break;  // (whole waves)
      const v4f v = c < t.n && k < R ? sum[q] * scale : v4f{0, 0, 0, 0};
      float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
      for (int d = 1; d < 4 * RT; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
      int e = (int)(__float_as_uint(m) >> 23);
      e = e < 1 ? 1 : e > 253 ? 253 : e;
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      if (k == 0) lift[c] = __uint_as_float((uint32_t)e << 23);
      float hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = v[j] * down;
        hi[j] = round_to<T>(s);
        lo[j] = fabsf(hi[j]) < 8.0f ? s - hi[j] : 0.0f;  // (infinities and NaN are in the upper half alone)
      }
      *(uint2*)(vs[c] + 2 * k) = make_uint2(pack2<T>(hi[0], hi[1]), pack2<T>(hi[2], hi[3]));
      *(uint2*)(vs[c] + 2 * (16 * RT + k)) = make_uint2(pack2<T>(lo[0], lo[1]), pack2<T>(lo[2], lo[3]));
    }
  }
  __syncthreads();
  float* tw = turn[wave];
  // (groups past the last one: zeros are loaded)
  const auto group = [&](int c, v4i (&w)[KB][4], v4i (&next)[KB][4]) {
    if constexpr (NB == 2) fetch_b(c + 4 < c1 ? c + 4 : GONE, next);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      v4f acc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const v4i hi = *(const v4i*)(vs[16 * j + r] + 64 * k + 16 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = mfma16<T>(w[k][i], hi, acc[i]);
        if constexpr (RT > 1) {
          const v4i lo = *(const v4i*)(vs[16 * j + r] + 32 * RT + 64 * k + 16 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = mfma16<T>(w[k][i], lo, acc[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) *(v4f*)(tw + r * LT + 16 * i + 4 * g) = acc[i];
      __builtin_amdgcn_wave_barrier();
      v4i o[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int q = 8 * h + drow;
        const float by = lift[16 * j + q];
        const v4f d0 = *(const v4f*)(tw + q * LT + 8 * dpos), d1 = *(const v4f*)(tw + q * LT + 8 * dpos + 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t u = (uint32_t)yv[j][h][k];
          const float lo = T == FMSMO_F16 ? f16_to_f32((u16)u) : bf16_to_f32((u16)u);
          const float hi = T == FMSMO_F16 ? f16_to_f32((u16)(u >> 16)) : bf16_to_f32((u16)(u >> 16));
          const v4f& d = k < 2 ? d0 : d1;
          o[h][k] = (int)pack2<T>(__fmaf_rn(d[k % 2 * 2], by, lo), __fmaf_rn(d[k % 2 * 2 + 1], by, hi));
        }
      }
      __builtin_amdgcn_wave_barrier();
      fetch_y(c + 4 < c1 ? c + 4 : GONE, j);  // (out may be y: other columns)
      put(c, j, 0, o[0]);
      put(c, j, 1, o[1]);
    }
    if constexpr (NB == 1) fetch_b(c + 4 < c1 ? c + 4 : GONE, w);
  };
  for (int c = c0; c < c1; c += 8) {
    group(c, bw[0], bw[NB - 1]);
    if (c + 4 < c1) group(c + 4, bw[NB - 1], bw[0]);
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();

// Steps on their way of a wave of the first launch on tiles of 64 rows: what the registers hold.
static constexpr int lora_depth(int rt) { return rt <= 2 ? 4 : rt == 4 ? 2 : 1; }
// What a call is cut into.  Rows: tiles of 64 where a request has 32 on average and they are so many that A and B, read for every tile, weigh, else
// of 16.  (Tiles of 128 rows read half of A and B and hold half as
// many waves' rows: rank 64, 6972 rows, 4096 -> 6144 79 us and 66.)
struct LoraPlan {
  int mt, rt, tiles, parts, part_steps, cols;
};
// Many rows: a compute unit takes in about 23 GB/s however many blocks it has once 128 KB are on their way, so that what counts is how evenly the
// blocks fall on the units (8192 rows of 14336, rank 32: 393 blocks with two steps a wave 63 us, 512 50, 256 with four steps 45 and with two 73),
// and what they read of A and B beside the rows.  A part's sums are read by every block of the second launch (4096 rows, rank 128, 4096 -> 4096:
// 94 us with 16 parts, 65 with those chosen here).
static void lora_many(LoraPlan& p, double rows, double seqs, int steps, int groups) {
  constexpr int R = 64;
  const double real = std::max(1.0, rows / R + 0.5 * (seqs - 1)), rate = 23e9;  // tiles with rows in them, about
  const double sums = R * 16 * p.rt * 4 / 40e9, way = 4.0 * lora_depth(p.rt) * (8 + 2 * p.rt) / 128;  // seconds; of what is on its way
  const double again = std::ceil(real * std::max(1.0, std::floor(256 / real)) / 256);
  double first = 1e30, second = 1e30;
  for (int n = 1; n <= 16; ++n) {
    const int each = div_up(div_up(steps, n), 4) * 4, parts = div_up(steps, each);
    const double rounds = std::ceil(real * parts / 256);
    const double cost = rounds * (each * (R + 16 * p.rt) * 128 / rate / std::min(1.0, rounds * way) + 1e-6) + parts * sums * again;
    if (cost < first) first = cost, p.part_steps = each;
  }
  const double before = div_up(steps, p.part_steps) * sums + 2e-6;
  for (int m = 1; m <= 16; ++m) {
    const double cost = std::ceil(real * div_up(groups, 4 * m) / 256) * (m * 4 * (256 * R + 2048 * p.rt) / rate + before);
    if (cost < second) second = cost, p.cols = 4 * m;
  }
}
static LoraPlan lora_plan(int64_t rows, int64_t seqs, bool ragged, int64_t slots, int rank, int64_t K, int64_t N) {
  LoraPlan p;
  p.rt = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  const int steps = div_up(K, LORA_STEP), groups = div_up(N, 64);
  // (Tiles of 64 rows and of 16: rank 128, 156 rows of 2088 -> 1280 26.4 us and 14.3; 4096 -> 4096 of rank 32, 100 rows 16.0 and 10.3, 3000 24.7
  // and 17.6, 8192 40.7 and 50.4; rank 64, 3000 31.2 and 26.2, 4096 31.1 and 32.6.  Rank 128 has less to gain from few rows, its A and B being
  // most of what they read: the sum of 15 calls, 4096 -> 4096 to 14336 -> 4096 for one to nine requests, 2048 rows 814 and 767, 2800 913 and 898, 3200 942
  // and 1018, 4095 1102 and 1257; but rank 72, padded to as many products, 2800 819 and 675, 3200 845 and 732, 4095 973 and 957.)
  if (!ragged || rows < 32 * seqs || rows < (rank >= 120 ? 3000 : 4096)) {
    // Few rows: parts of K for about 512 blocks, a step of 64 elements for each of their four waves at least (and 64 MB of sums at most), and of the
    // outputs for about 768.  Of requests of one row, those of an adapter are one tile (196 requests of 32 adapters, rank 64, 8872 -> 8376: 52 us
    // with the parts that as many tiles as requests would have, 33 so).
    p.mt = 1;
    // (Requests of one row 8192 at a time: each counts those before it, and 64 MB hold their sums.  64 -> 64 of rank 16, 65536 requests: 6.7 ms at
    // once, 0.92 so; of rank 128: 16.2 and 2.0.)
    p.tiles = (int)(ragged ? rows / 16 + seqs + 2 : std::min<int64_t>(seqs, 8192));
    const int real = (int)(ragged ? p.tiles : std::min(seqs, slots + seqs / 16 + 1));
    // What a block of the first launch takes in falls with the parts, what one of the second adds up grows with them: the sum is least at the root of
    // steps (2 rt + 2) KB / 23 GB/s over rt KB / 33 GB/s (one row, 14336 inputs, rank 16: 56 parts 8.2 + 3.8 us, 36 6.0 + 3.8; 72 rows of 4 adapters,
    // rank 128, 10592 -> 3352: 14.4 + 15.8 and 12.8 + 12.5).
    const int even = (int)std::sqrt(2.9 * steps * (p.rt + 1) / p.rt);
    const int parts = std::min({512 / real, div_up(steps, 4), even, (int)((64 << 10) / ((int64_t)p.tiles * p.rt))});
    p.part_steps = div_up(div_up(steps, std::max(parts, 1)), 4) * 4;
    const int blocks = std::max(1, std::min(768 / real, div_up(groups, 4)));
    p.cols = div_up(div_up(groups, blocks), 4) * 4;
  } else {
    p.mt = 4;
    lora_many(p, (double)rows, (double)seqs, steps, groups);
    p.tiles = (int)(rows / 64 + seqs + 2);
  }
  p.parts = div_up(steps, p.part_steps);
  return p;
}
static bool lora_sizes(int64_t rows, int64_t seqs, int rank, int64_t K) {
  return rows >= 0 && seqs >= 0 && rows < 1 << 30 && seqs < 1 << 29 && rank >= 8 && rank <= 128 && rank % 8 == 0 && K >= 8 && K <= 1 << 22;
}

extern "C" int64_t fmsmo_lora_workspace_bytes(int64_t rows, int64_t seqs, int ragged, int64_t slots, int rank, int64_t K) {
  if (!lora_sizes(rows, seqs, rank, K) || rows == 0 || slots < 0 || (!ragged && rows != seqs)) return 0;
  const LoraPlan p = lora_plan(rows, seqs, ragged != 0, std::min<int64_t>(slots, 1 << 29), rank, K, 64);
  return (int64_t)p.parts * p.tiles * (1024 * p.mt * p.rt);
}

template <int T, int RT, int MT>
static void run_lora(const LoraArgs& a, hipStream_t s) {
  constexpr int D = MT > 1 ? lora_depth(RT) : RT == 8 ? 1 : 2;  // (rank 128 and 16 rows: two steps leave the registers, 6.9 us and 5.5)
  hipLaunchKernelGGL((lora_shrink_kernel<T, RT, MT, D>), dim3((unsigned)a.tiles, (unsigned)a.parts), dim3(256), 0, s, a);
  hipLaunchKernelGGL((lora_expand_kernel<T, RT, MT>), dim3((unsigned)a.tiles, (unsigned)div_up(div_up(a.N, 64), a.cols)), dim3(256), 0, s, a);
}

extern "C" int fmsmo_lora_add(int dtype, const void* x, int64_t ldx, const void* y, int64_t ldy, void* out, int64_t ldo, const void* a,
                              int64_t a_slot, int64_t a_row, const void* b, int64_t b_slot, int64_t b_row, int64_t slots, int rank,
                              const int32_t* adapters, const int32_t* query_start, int64_t seqs, const float* scales, int64_t rows, int64_t N,
                              int64_t K, void* workspace, int64_t workspace_bytes, fmsmo_stream_t stream) {
  if (rows < 0 || seqs < 0 || N < 0 || K < 0 || slots < 0) return FMSMO_ERR_SHAPE;
  if (dtype != FMSMO_F16 && dtype != FMSMO_BF16) return FMSMO_ERR_UNSUPPORTED;
  if (rows == 0 || N == 0) return FMSMO_OK;
  if (!x || !y || !out || (slots && (!a || !b)) || (seqs && !adapters)) return FMSMO_ERR_NULL;
  if (!query_start && rows != seqs) return FMSMO_ERR_SHAPE;
  if (!lora_sizes(rows, seqs, rank, K) || N > 1 << 22 || slots > 0x7fffffff) return FMSMO_ERR_UNSUPPORTED;
  if ((rows > 1 && (ldx < K || ldy < N || ldo < N)) || a_row < K || b_row < rank || a_slot < 0 || b_slot < 0) return FMSMO_ERR_SHAPE;
  const auto off = [](const void* p) { return (((uintptr_t)p) & 15) != 0; };
  if (K % 8 || N % 8 || off(x) || off(y) || off(out) || off(a) || off(b) || (rows > 1 && (ldx % 8 || ldy % 8 || ldo % 8)) || a_slot % 8 ||
      a_row % 8 || b_slot % 8 || b_row % 8 || off(workspace))
    return FMSMO_ERR_ALIGN;
  // the kernels count 32 bits from a tile's first row, from an adapter and from its B
  constexpr int64_t MOST = 0x7f000000;
  if (64 * (2 * a_row) > MOST || 128 * (2 * a_row) > MOST || N * (2 * b_row) > MOST) return FMSMO_ERR_UNSUPPORTED;
  const int64_t widest = 2 * std::max(ldx, std::max(ldy, ldo));
  if (rows > 1 && 64 * widest + 2 * std::max(K, N) > MOST) return FMSMO_ERR_UNSUPPORTED;
  if (!workspace) return FMSMO_ERR_NULL;
  const LoraPlan p = lora_plan(rows, seqs, query_start != nullptr, std::min<int64_t>(slots, 1 << 29), rank, K, N);
  if (p.tiles >= 1 << 24) return FMSMO_ERR_UNSUPPORTED;  // (a launch has fewer than 2^32 threads)
  if (workspace_bytes < (int64_t)p.parts * p.tiles * (1024 * p.mt * p.rt)) return FMSMO_ERR_SCRATCH;
  // rows of one adapter may lie anywhere among the requests of one row: as many of them at a time as 32 bits reach
  const int64_t most = query_start || rows == 1 ? rows : std::min<int64_t>(p.tiles, (MOST - 2 * std::max(K, N)) / widest);
  for (int64_t from = 0; from < rows; from += most) {
    const int64_t some = std::min(most, rows - from);
    LoraArgs g{(const char*)x + 2 * from * ldx, (const char*)y + 2 * from * ldy, (char*)out + 2 * from * ldo, (const char*)a, (const char*)b,
               adapters + from, query_start, scales, (float*)workspace, 2 * ldx, 2 * ldy, 2 * ldo, 2 * a_slot, 2 * a_row, 2 * b_slot, 2 * b_row,
               (int)some, (int)(query_start ? seqs : some), (int)slots, rank, (int)K, (int)N, p.parts, p.part_steps, (int)(query_start ? p.tiles : some),
               p.cols};
    const auto go = [&](auto t, auto rt) {
      constexpr int T = decltype(t)::value, RT = decltype(rt)::value;
      if (p.mt == 4) run_lora<T, RT, 4>(g, (hipStream_t)stream);
      else run_lora<T, RT, 1>(g, (hipStream_t)stream);
    };
    const auto ranks = [&](auto t) {
      if (p.rt == 1) go(t, std::integral_constant<int, 1>{});
      else if (p.rt == 2) go(t, std::integral_constant<int, 2>{});
      else if (p.rt == 4) go(t, std::integral_constant<int, 4>{});
      else go(t, std::integral_constant<int, 8>{});
    };
    if (dtype == FMSMO_F16) ranks(std::integral_constant<int, FMSMO_F16>{});
    else ranks(std::integral_constant<int, FMSMO_BF16>{});
  }
  return fmsmo_check_launch();
}

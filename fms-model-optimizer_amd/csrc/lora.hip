// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + scale_s B_s (A_s x[t]), s the adapter of the request that
// row t belongs to.  Two launches.  The first makes v = A_s x in fp32, K cut into parts where there are few rows; the second adds the
// parts, takes v as the sum of two 16-bit numbers (so that the product B v is as exact as its operands B; with rank 16 the two halves fill one
// matrix instruction) and adds the product to y, rounded once.
//
// A tile is up to 16 MT rows of one adapter.  One row per request: the rows of the requests that share an adapter, sixteen at a time, found by
// counting; else 16 MT consecutive rows of a request.
#include "paged_kv.hpp"

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
    const int slot = a.adapters[tile];
    if ((unsigned)slot >= (unsigned)a.slots) {  // on its own: the copy of its row
      t.n = 1;
      t.row0 = tile;
      if (threadIdx.x == 0) list[0] = tile;
      return t;
    }
    // the requests of this adapter before this one; a tile starts at each TR-th of them
    int before = 0, mine = 0;
    for (int i = 0; i < tile; i += 64) before += __popcll(__ballot(i + lane < tile && a.adapters[i + lane] == slot));
    before = uniform(before);
    if (before % TR) return t;
    for (int i = tile & ~63; i < a.seqs && mine < TR; i += 64) {
      const bool same = i + lane >= tile && i + lane < a.seqs && a.adapters[i + lane] == slot;
      const uint64_t m = __ballot(same);
      const int at = mine + __popcll(m & ((1ull << lane) - 1));
      if (same && at < TR && threadIdx.x < 64) list[at] = i + lane;
      mine += __popcll(m);
    }
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
    int r0 = 0, r1 = 0;
    if (b <= a.seqs) {
      r0 = b < 0 ? 0 : a.starts[b];
      r1 = b >= a.seqs ? a.rows : a.starts[b + 1];
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
      const int at = (tile - __shfl(first, l)) * TR, req = i + l;
      const int rn = __shfl(n, l) - at;
      t.row0 = uniform(__shfl(r0, l) + at);
      t.n = uniform(rn < TR ? rn : TR);
      const int slot = req >= 0 && req < a.seqs ? a.adapters[req] : -1;
      t.slot = (unsigned)slot < (unsigned)a.slots ? slot : -1;
      return t;
    }
    seen += uniform(__shfl(upto, 63));
    if (seen > tile) break;
  }
  return t;
}

constexpr int LORA_STEP = 64;  // elements of K a step: 128 bytes of a row

// 16 bytes at `off` behind `base`, or zeros
__device__ __forceinline__ v4i load_or_zero(const char* base, int64_t off, bool there) {
  v4i v = {0, 0, 0, 0};
  if (there) v = *(const v4i*)(base + off);
  return v;
}

// v of a tile over a part of K.  Rows of A (16 RT) and of x (16 MT) meet as the two operands of 16 x 16 x 32; the side with more bytes comes
// through shared memory, eight rows of 128 bytes a load, the other one straight into the operands' layout.
template <int T, int RT, int MT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs a) {
  constexpr bool X_STAGED = MT > 1;
  constexpr int S = X_STAGED ? MT : RT, O = X_STAGED ? RT : MT;  // tiles of 16 rows of the staged and the other side
  constexpr int SUMS = MT * 16 * (RT * 16 + 4) * 4;  // bytes of a wave's sums; they take the place of the staged rows
  __shared__ __attribute__((aligned(16))) char stage[S * 8192 > 2 * SUMS ? S * 8192 : 2 * SUMS];
  __shared__ int list[MT * 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const LoraTile t = lora_tile<16 * MT>(a, blockIdx.x, list);
  if (t.n == 0 || t.slot < 0) return;
  __syncthreads();
  const char* A = a.a + (int64_t)t.slot * a.a_slot;
  const int s0 = blockIdx.y * a.part_steps, s1 = min(s0 + a.part_steps, (a.K + LORA_STEP - 1) / LORA_STEP);
  const int r = lane & 15, g = lane >> 4, drow = lane >> 3, dpos = lane & 7;
  const auto row_of = [&](int i) -> int64_t { return a.starts ? t.row0 + i : list[i]; };
  // the staged side: rows drow, drow + 8, .. of this lane
  const char* sp[2 * S];
  bool sv[2 * S];
#pragma unroll
  for (int i = 0; i < 2 * S; ++i) {
    const int q = 8 * i + drow;
    sv[i] = q < (X_STAGED ? t.n : a.rank);
    sp[i] = X_STAGED ? a.x + (sv[i] ? row_of(q) : 0) * a.ldx : A + (int64_t)(sv[i] ? q : 0) * a.a_row;
  }
  const char* op[O];
  bool ov[O];
#pragma unroll
  for (int i = 0; i < O; ++i) {
    const int q = 16 * i + r;
    ov[i] = q < (X_STAGED ? a.rank : t.n);
    op[i] = X_STAGED ? A + (int64_t)(ov[i] ? q : 0) * a.a_row : a.x + (ov[i] ? row_of(q) : 0) * a.ldx;
  }
  v4f acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  char* st = stage + wave * (S * 2048);
  const int rr = r & 7;
  v4i sb[2 * S], ob[O][2];
  const auto fetch_staged = [&](int s) {
    const int e = s * LORA_STEP + dpos * 8;
#pragma unroll
    for (int i = 0; i < 2 * S; ++i) sb[i] = load_or_zero(sp[i], 2 * e, sv[i] && e < a.K);
  };
  const auto fetch_other = [&](int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = s * LORA_STEP + (4 * h + g) * 8;
#pragma unroll
      for (int i = 0; i < O; ++i) ob[i][h] = load_or_zero(op[i], 2 * e, ov[i] && e < a.K);
    }
  };
  constexpr bool EARLY = O <= 2;  // the other side's next rows too are asked for ahead of the products (else: registers)
  int s = s0 + wave;
  if (s < s1) {
    fetch_staged(s);
    fetch_other(s);
  }
  for (; s < s1; s += 4) {
    // chunk c of row q lies at position c ^ (q % 8)
#pragma unroll
    for (int i = 0; i < 2 * S; ++i) *(v4i*)(st + (8 * i + drow) * 128 + ((dpos ^ drow) * 16)) = sb[i];
    __builtin_amdgcn_wave_barrier();  // (the rows go to other lanes of the wave)
    if (s + 4 < s1) fetch_staged(s + 4);
    v4i o[O][2];
#pragma unroll
    for (int i = 0; i < O; ++i) o[i][0] = ob[i][0], o[i][1] = ob[i][1];
    if (EARLY && s + 4 < s1) fetch_other(s + 4);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const v4i w = *(const v4i*)(st + (16 * i + r) * 128 + (((4 * h + g) ^ rr) * 16));
#pragma unroll
        for (int j = 0; j < O; ++j) {
          if constexpr (X_STAGED) acc[j][i] = mfma16<T>(o[j][h], w, acc[j][i]);
          else acc[i][j] = mfma16<T>(w, o[j][h], acc[i][j]);
        }
      }
    if (!EARLY && s + 4 < s1) fetch_other(s + 4);
    __builtin_amdgcn_wave_barrier();
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

// out = y + B v for a tile and `cols` groups of 64 outputs, one group a wave at a time
template <int T, int RT, int MT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  constexpr int TR = 16 * MT, LD = 64 * RT + 16;  // bytes of a row of v: both halves of 16 RT numbers, and a step in banks
  __shared__ __attribute__((aligned(16))) char vs[TR][LD];
  __shared__ float lift[TR];
  __shared__ int list[TR];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const LoraTile t = lora_tile<TR>(a, blockIdx.x, list);
  if (t.n == 0) return;
  if (t.slot < 0 && a.y == a.out) return;
  const int r = lane & 15, g = lane >> 4;
  const int c0 = blockIdx.y * a.cols, c1 = min(c0 + a.cols, (a.N + 63) / 64);
  const int R = a.rank;
  if (t.slot >= 0) {
    const float scale = a.scales ? a.scales[t.slot] : 1.0f;
    const float* from = a.ws + (int64_t)blockIdx.x * (256 * MT * RT);
    const int64_t part = (int64_t)a.tiles * (256 * MT * RT);
    // In quadruples of a row: v, brought to a maximum of 1 to 4 by a power of two (fp16 holds neither large numbers nor the lower halves of
    // small ones), its upper half at k, what that leaves at rank + k; zeros behind 2 rank.
    for (int i = threadIdx.x; i < TR * 4 * RT; i += 256) {
      const int c = i / (4 * RT), k = i % (4 * RT) * 4;
      v4f v = {0, 0, 0, 0};
      if (k < R && c < t.n) {
        for (int p = 0; p < a.parts; ++p) v += *(const v4f*)(from + p * part + c * 16 * RT + k);
        v *= scale;
      }
      float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
      for (int d = 1; d < 4 * RT; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
      int e = (int)(__float_as_uint(m) >> 23);
      e = e < 1 ? 1 : e > 253 ? 253 : e;
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      if (k == 0) lift[c] = __uint_as_float((uint32_t)e << 23);
      if (k < R) {
        float hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s = v[j] * down;
          hi[j] = round_to<T>(s);
          lo[j] = fabsf(hi[j]) < 8.0f ? s - hi[j] : 0.0f;  // (infinities and NaN are in the upper half alone)
        }
        *(uint2*)(vs[c] + 2 * k) = make_uint2(pack2<T>(hi[0], hi[1]), pack2<T>(hi[2], hi[3]));
        *(uint2*)(vs[c] + 2 * (R + k)) = make_uint2(pack2<T>(lo[0], lo[1]), pack2<T>(lo[2], lo[3]));
      } else {  // (16 RT - rank numbers a row, half as many as 2 rank is short of 32 RT)
        *(uint4*)(vs[c] + 2 * (2 * R + 2 * (k - R))) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  __syncthreads();
  const char* B = a.b + (int64_t)(t.slot < 0 ? 0 : t.slot) * a.b_slot;
  const auto row_of = [&](int i) -> int64_t { return a.starts ? t.row0 + i : list[i]; };
  for (int c = c0 + wave; c < c1; c += 4) {
    const int n0 = c * 64 + 16 * g;  // this lane's sixteen outputs
    v4i yv[MT][2];
    bool there[MT][2];
    int64_t row[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const bool mine = 16 * j + r < t.n;
      row[j] = mine ? row_of(16 * j + r) : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        there[j][h] = mine && n0 + 8 * h < a.N;
        yv[j][h] = load_or_zero(a.y + row[j] * a.ldy, 2 * (int64_t)(n0 + 8 * h), there[j][h]);
      }
    }
    if (t.slot >= 0) {
      // row 4 g' + j of part i of the product is output 16 g' + 4 i + j: a lane's results lie side by side
      v4f acc[4][MT];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
      const int nb = c * 64 + 16 * (r >> 2) + (r & 3);
      for (int k = 0; k < 2 * R; k += 32) {
        const int kk = k + 8 * g, e = kk < R ? kk : kk - R;
        v4i bw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) bw[i] = load_or_zero(B, (int64_t)(nb + 4 * i) * a.b_row + 2 * e, nb + 4 * i < a.N && kk < 2 * R);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const v4i vv = *(const v4i*)(vs[16 * j + r] + 2 * kk);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i][j] = mfma16<T>(bw[i], vv, acc[i][j]);
        }
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const float by = lift[16 * j + r];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v4i o;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w = (uint32_t)yv[j][h][q];
            const float lo = T == FMSMO_F16 ? f16_to_f32((u16)w) : bf16_to_f32((u16)w);
            const float hi = T == FMSMO_F16 ? f16_to_f32((u16)(w >> 16)) : bf16_to_f32((u16)(w >> 16));
            const v4f& d = acc[2 * h + q / 2][j];
            o[q] = (int)pack2<T>(__fmaf_rn(d[q % 2 * 2], by, lo), __fmaf_rn(d[q % 2 * 2 + 1], by, hi));
          }
          yv[j][h] = o;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (there[j][h]) *(v4i*)(a.out + row[j] * a.ldo + 2 * (int64_t)(n0 + 8 * h)) = yv[j][h];
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();

// What a call is cut into.  Rows: tiles of 64 where a request has 32 on average, else of 16.  K: parts for about 512 blocks, a step of 64
// elements for each of their four waves at least.  Outputs: blocks for about 1024.
struct LoraPlan {
  int mt, rt, tiles, parts, part_steps, cols;
};
static LoraPlan lora_plan(int64_t rows, int64_t seqs, bool ragged, int rank, int64_t K, int64_t N) {
  LoraPlan p;
  p.mt = ragged && rows >= 32 * seqs ? 4 : 1;
  p.rt = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  p.tiles = (int)(ragged ? rows / (16 * p.mt) + seqs + 2 : seqs);
  const int steps = div_up(K, LORA_STEP), groups = div_up(N, 64);
  int parts = 512 / p.tiles;
  parts = parts < 1 ? 1 : parts < div_up(steps, 4) ? parts : div_up(steps, 4);
  p.part_steps = div_up(div_up(steps, parts), 4) * 4;
  p.parts = div_up(steps, p.part_steps);
  int blocks = 1024 / p.tiles;
  blocks = blocks < 1 ? 1 : blocks < div_up(groups, 4) ? blocks : div_up(groups, 4);
  p.cols = div_up(div_up(groups, blocks), 4) * 4;
  return p;
}
static bool lora_sizes(int64_t rows, int64_t seqs, int rank, int64_t K) {
  return rows >= 0 && seqs >= 0 && rows < 1 << 30 && seqs < 1 << 29 && rank >= 8 && rank <= 128 && rank % 8 == 0 && K >= 8 && K < 1 << 28;
}

extern "C" int64_t fmsmo_lora_workspace_bytes(int64_t rows, int64_t seqs, int ragged, int rank, int64_t K) {
  if (!lora_sizes(rows, seqs, rank, K) || rows == 0) return 0;
  const LoraPlan p = lora_plan(rows, seqs, ragged != 0, rank, K, 64);
  return (int64_t)p.parts * p.tiles * (1024 * p.mt * p.rt);
}

template <int T, int RT, int MT>
static void run_lora(const LoraArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((lora_shrink_kernel<T, RT, MT>), dim3((unsigned)a.tiles, (unsigned)a.parts), dim3(256), 0, s, a);
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
  if (!lora_sizes(rows, seqs, rank, K) || N >= 1 << 28 || slots > 0x7fffffff) return FMSMO_ERR_UNSUPPORTED;
  if ((rows > 1 && (ldx < K || ldy < N || ldo < N)) || a_row < K || b_row < rank || a_slot < 0 || b_slot < 0) return FMSMO_ERR_SHAPE;
  const auto off = [](const void* p) { return (((uintptr_t)p) & 15) != 0; };
  if (K % 8 || N % 8 || off(x) || off(y) || off(out) || off(a) || off(b) || (rows > 1 && (ldx % 8 || ldy % 8 || ldo % 8)) || a_slot % 8 ||
      a_row % 8 || b_slot % 8 || b_row % 8 || off(workspace))
    return FMSMO_ERR_ALIGN;
  const LoraPlan p = lora_plan(rows, seqs, query_start != nullptr, rank, K, N);
  if (!workspace) return FMSMO_ERR_NULL;
  if (workspace_bytes < (int64_t)p.parts * p.tiles * (1024 * p.mt * p.rt)) return FMSMO_ERR_SCRATCH;
  LoraArgs g{(const char*)x, (const char*)y, (char*)out, (const char*)a, (const char*)b, adapters, query_start, scales, (float*)workspace,
             2 * ldx, 2 * ldy, 2 * ldo, 2 * a_slot, 2 * a_row, 2 * b_slot, 2 * b_row, (int)rows, (int)seqs, (int)slots, rank, (int)K, (int)N,
             p.parts, p.part_steps, p.tiles, p.cols};
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
  return fmsmo_check_launch();
}

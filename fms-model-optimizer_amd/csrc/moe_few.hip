// A mixture-of-experts block for a few tokens (up to 64), whose weights bound it: routing, gate and up products, gated silu in 8 bits, down
// products and the weighted sum.
//
//   p = softmax(logits[t]); S = the `top` experts of the largest logits (of equal ones the lower index); c_e = p_e / sum_S p, or p_e
//   g, u = (a[t] . w13[e]^T) a_scale[t] w13_scale[e]  (rows 0 .. I - 1 and I .. 2I - 1),  h = g / (1 + exp(-g)) u  in fp32
//   codes of h per token and expert: int8 s = max(max|h|, 1e-5) / 127, e4m3 s = max(max|h| / 448, 1e-12), as the per-token quantizers in fp32
//   y[t] = sum_S c_e s (codes . w2[e]^T) w2_scale[e]
//
// The chosen (token, expert) pairs are sorted by expert: a `position` each.  The weights stream past, once for a group of up to 8 to 64 tokens of an
// expert (by the plan; mostly all of them), and are turned into matrix operands in shared memory; a group's tokens are the columns of the product.
#include "paged_kv.hpp"
#include "stream_loads.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace fmsmo {

constexpr int MOE_TOKENS = 64, MOE_EXPERTS = 512, MOE_TOP = 16;
// Tokens up to which every block of the gate and up products routes for itself (16 tokens over 128 experts: 80 us so, 72 with a launch of its own).
// The number of tokens alone decides, though over few experts ten tokens would gain yet (small ones, of 8: 15.2 us so, 16.2 with the launch).
constexpr int MOE_ROUTED = 8;

struct MoeArgs {
  const uint8_t* a;     // [T, K] codes
  const float* a_scale; // [T] or [1]
  const void* logits;
  const uint8_t* w13;
  const float* s13;
  const uint8_t* w2;
  const float* s2;
  void* y;
  int64_t lda, ldl, ldy;
  int a_stride, logits_dtype, y_dtype;
  int T, E, top, K, I, renorm;
  int down_group;   // tokens of a group of the down product, at most
  // workspace
  int* ids;         // [T top] experts of a token, -1: a share of zero
  float* share;     // [T top]
  int* count;       // entries
  uint32_t* entry;  // [MOE_ENTRIES]
  int* token;       // [T top] of a position
  float* weight;    // [T top] its share
  float* hs;        // [T top]
  float* h;         // [T top][I]
  uint8_t* hq;      // [T top][I]
  float* parts;     // [splits][T][K] of the down product, where blocks share outputs
  uint32_t* tops;   // [T top][I / 8] largest |h| of eight, as integers; NULL: not wanted
};
// A group of tokens of one expert: expert, tokens and first position in one number.
constexpr int MOE_ENTRIES = MOE_EXPERTS + MOE_TOKENS * MOE_TOP / 8;
__device__ __forceinline__ uint32_t entry_of(int e, int cnt, int off) { return (uint32_t)e | (uint32_t)cnt << 9 | (uint32_t)off << 16; }
struct MoeGroup {
  int e, cnt, off;
};
__device__ __forceinline__ MoeGroup group_of(uint32_t x) { return MoeGroup{(int)(x & 511u), (int)(x >> 9 & 127u), (int)(x >> 16)}; }

// an order of floats as unsigned integers (both zeros are one number); 0 is none of them
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  const uint32_t k = u >> 31 ? ~u : u | 0x80000000u;
  return k ? k : 1u;
}

// The choices of token t by one wave, V logits a lane, the largest by the largest: lane s returns the s-th expert and its share.
template <int V>
__device__ __forceinline__ void choose(const MoeArgs& a, int t, int& id, float& share) {
  const int lane = threadIdx.x & 63;
  uint32_t key[V];
  float val[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 64 * i;
    val[i] = scalar_f32(a.logits, a.logits_dtype, t * a.ldl + (e < a.E ? e : 0));
    key[i] = e < a.E ? order_of(val[i]) : 0u;
  }
  float mine = 0.0f;  // lane s keeps the s-th choice
  id = -1;
  for (int s = 0; s < a.top; ++s) {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = m > key[i] ? m : key[i];
    m = wave_max_u32(m);
    int e = 0;
    float v = 0.0f;
    bool found = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint64_t at = __ballot(key[i] == m);
      if (!found && at) {
        found = true;
        const int l = __ffsll((unsigned long long)at) - 1;
        e = l + 64 * i;
        v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(val[i]), l));
        if (lane == l) key[i] = 0;
      }
    }
    if (lane == s) {
      id = e;
      mine = v;
    }
  }
  const float first = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), 0));
  const bool some = first != -__builtin_inff();
  const float p = lane < a.top && some ? expf(mine - first) : 0.0f;
  float sum = p;
  if (!a.renorm) {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane + 64 * i < a.E && some) sum += expf(val[i] - first);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  share = p == 0.0f ? 0.0f : p / sum;
  if (share == 0.0f) id = -1;  // (the expert is not run)
}
__device__ __forceinline__ void choose_any(const MoeArgs& a, int t, int& id, float& share) {
  if (a.E <= 64) choose<1>(a, t, id, share);
  else if (a.E <= 128) choose<2>(a, t, id, share);
  else choose<MOE_EXPERTS / 64>(a, t, id, share);
}

// a wave per token
__global__ __launch_bounds__(256) void moe_route_kernel(MoeArgs a) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= a.T) return;
  int id;
  float share;
  choose_any(a, t, id, share);
  if (lane < a.top) {
    a.ids[t * a.top + lane] = id;
    a.share[t * a.top + lane] = share;
  }
}

// The choices sorted by expert, made by every block for itself: groups of up to 16 MT tokens and the tokens of the positions.
struct MoeLists {
  unsigned long long mask[MOE_EXPERTS];  // tokens of an expert
  uint32_t entry[MOE_ENTRIES];
  short off[MOE_EXPERTS], id[MOE_TOKENS * MOE_TOP];
  uint8_t token[MOE_TOKENS * MOE_TOP];
  int count;
};
// ROUTE: from the logits; else from what the routing kernel left.  Block 0 leaves all of it for the kernels behind.
template <int NT, int MT, bool ROUTE>
__device__ __forceinline__ void make_lists(const MoeArgs& a, MoeLists& l) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pairs = a.T * a.top;
  if (ROUTE && a.T == 1) {  // a group per choice, in the order of the experts
    if (wave == 0) {
      int id, at = 0;
      float share;
      choose_any(a, 0, id, share);
      for (int s = 0; s < a.top; ++s) {
        const int o = __builtin_amdgcn_readlane(id, s);
        at += o >= 0 && o < id;
      }
      if (lane < a.top) l.token[lane] = 0;
      const int n = __popcll(__ballot(lane < a.top && id >= 0));
      if (lane == 0) l.count = n;
      if (lane < a.top && id >= 0) {
        l.entry[at] = entry_of(id, 1, at);
        if (blockIdx.x == 0) {
          a.entry[at] = entry_of(id, 1, at);
          a.token[at] = 0;
          a.weight[at] = share;
        }
      }
      if (blockIdx.x == 0 && lane == 0) a.count[0] = n;
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < a.E; e += NT) l.mask[e] = 0;
  __syncthreads();
  if constexpr (ROUTE) {
    for (int t = wave; t < a.T; t += NT / 64) {
      int id;
      float share;
      choose_any(a, t, id, share);
      if (lane < a.top) {
        l.id[t * a.top + lane] = (short)id;
        if (id >= 0) atomicOr(&l.mask[id], 1ull << t);
        if (blockIdx.x == 0) a.share[t * a.top + lane] = share;
      }
    }
  } else {
    for (int i = threadIdx.x; i < pairs; i += NT) {
      const int id = a.ids[i];
      l.id[i] = (short)id;
      if (id >= 0) atomicOr(&l.mask[id], 1ull << (i / a.top));
    }
  }
  __syncthreads();
  // groups and positions, by one wave; those of the down product by another one of block 0
  const int size = wave == 0 ? 16 * MT : a.down_group;
  if (wave == 0 || (wave == 1 && blockIdx.x == 0)) {
    int pos = 0, groups = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + lane, cnt = e < a.E ? __popcll(l.mask[e]) : 0, mine = (cnt + size - 1) / size;
      int both = cnt | mine << 16;  // both sums at once (up to 1024 and 640)
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(both, d);
        both += lane >= d ? o : 0;
      }
      const int off = pos + (both & 0xffff) - cnt, at = groups + (both >> 16) - mine;
      if (wave == 0 && e < a.E) l.off[e] = (short)off;
      for (int i = 0; i < mine; ++i) (wave ? a.entry : l.entry)[at + i] = entry_of(e, min(cnt - size * i, size), off + size * i);
      const int total = __builtin_amdgcn_readlane(both, 63);
      pos += total & 0xffff;
      groups += total >> 16;
    }
    if (lane == 0) (wave ? a.count[0] : l.count) = groups;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += NT) {
    const int id = l.id[i], t = i / a.top;
    if (id < 0) continue;
    const int pos = l.off[id] + __popcll(l.mask[id] & ((1ull << t) - 1));
    l.token[pos] = (uint8_t)t;
    if (blockIdx.x == 0) {
      a.token[pos] = t;
      a.weight[pos] = a.share[i];
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------ streaming weights
template <int OP>
struct MoeAcc {
  typedef typename std::conditional<OP == FMSMO_OP_I8, v4i, v4f>::type type;
};
template <int OP>
__device__ __forceinline__ void moe_mfma(typename MoeAcc<OP>::type& c, v4i w0, v4i w1, v4i x0, v4i x1) {
  if constexpr (OP == FMSMO_OP_I8) {
    c = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, x0, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, x1, c, 0, 0, 0);
  } else {
    // e4m3 codes as the fp16 numbers that they are: exact products, sums in fp32.  (The scaled instruction drops what lies 2^-13 below the
    // largest of the 128 products it adds at a time, which moves codes of h.)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v4i& w = i < 2 ? w0 : w1;
      const v4i& x = i < 2 ? x0 : x1;
      v4i wh, xh;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t lo, hi;
        widen4<FMSMO_F16>((uint32_t)w[2 * (i & 1) + k], lo, hi);
        wh[2 * k] = (int)lo, wh[2 * k + 1] = (int)hi;
        widen4<FMSMO_F16>((uint32_t)x[2 * (i & 1) + k], lo, hi);
        xh[2 * k] = (int)lo, xh[2 * k + 1] = (int)hi;
      }
      c = mfma16<FMSMO_F16>(wh, xh, c);
    }
  }
}
// Weights are loaded as 16 rows of 256 bytes, four rows a load.  Where rows are no multiples of 128 bytes, the lines at the ends of a piece are
// its neighbours' too, and weights stay in the caches (KEEP: 16 tokens over 8 experts of 4112 x 14352 gate and up 194 us, 203 streamed; 47 over 32 of
// 656 x 3264 48 and 53); else they are read past them (64 tokens over 128 experts of 2048 x 768 67 us, 77 kept).
constexpr int MOE_STEP = 256;
template <bool KEEP>
__device__ __forceinline__ v4i moe_weights(Buf b, uint32_t off, uint32_t uniform_off) {
  return KEEP ? buf_load(b, off, uniform_off) : buf_stream(b, off, uniform_off);
}
// Four loads into shared memory, the first 128 bytes of the 16 rows and then the others, chunk c of row q at position c ^ (q % 8)
__device__ __forceinline__ void moe_stage(uint8_t* st, const v4i (&w)[4]) {
  const int lane = threadIdx.x & 63, row = lane >> 4, c = lane & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = 4 * i + row;
    *(v4i*)(st + (c >> 3) * 2048 + q * 128 + (((c ^ q) & 7) * 16)) = w[i];
  }
  __builtin_amdgcn_wave_barrier();  // (the rows go to other lanes of the wave)
}

// h of the positions.  A unit: 8 RW gate rows and the up rows that belong to them, for one group of tokens: RW products' 16 rows, each eight
// gate rows and their up rows.  D steps of 256 bytes a row are on their way, those of the next unit among them.  SHARE: the four waves of a block
// share a unit's K, every fourth step each; their sums meet in shared memory, one barrier a unit, and a wave in turn finishes it.  Else each wave
// has units of its own.
template <int OP, int MT, int RW, int D, bool ROUTE, bool SHARE, bool KEEP>
__global__ __launch_bounds__(256, RW * D >= 2 ? 2 : MT == 1 ? 4 : 3) void moe_up_kernel(MoeArgs a) {
  typedef typename MoeAcc<OP>::type Acc;
  __shared__ MoeLists lists;
  __shared__ __attribute__((aligned(16))) uint8_t stage[4][4096 * RW];
  __shared__ __attribute__((aligned(16))) Acc part[SHARE ? 2 : 1][SHARE ? 4 : 1][RW * MT][64];
  make_lists<256, MT, ROUTE>(a, lists);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;  // operands: row or column r, 16-byte pieces g and 4 + g; loads: rows g, 4 + g, .., piece r
  const int groups = a.I / (8 * RW), units = lists.count * groups;
  constexpr int KS = SHARE ? 4 : 1;
  const int steps = ((a.K + MOE_STEP * KS - 1) / (MOE_STEP * KS) + D - 1) / D * D;  // of a wave
  uint8_t* st = stage[wave];
  const int rr = r & 7;
  struct Unit {
    Buf w;             // of the expert
    uint32_t wo;       // the lane's gate row
    uint32_t xo[MT];   // and tokens
    MoeGroup m;
    int gi;
  };
  const Buf xb_of = buf_of(a.a);
  const auto unit_of = [&](int u) {  // (past the last one: nothing is loaded)
    Unit q;
    const bool there = u < units;
    const int en = there ? u / groups : 0;
    q.gi = there ? u - en * groups : 0;
    q.m = group_of(uniform((int)lists.entry[en]));
    q.w = buf_of(a.w13 + (int64_t)q.m.e * 2 * a.I * a.K);
    q.wo = there ? (uint32_t)(q.gi * 8 * RW + g) * (uint32_t)a.K + r * 16 : BUF_NONE;
#pragma unroll
    for (int j = 0; j < MT; ++j)
      q.xo[j] = there && 16 * j + r < q.m.cnt ? lists.token[q.m.off + 16 * j + r] * (uint32_t)a.lda + g * 16 : BUF_NONE;
    return q;
  };
  const uint32_t up = (uint32_t)a.I * (uint32_t)a.K;
  v4i wb[D][RW][4], xb[D][MT][4];
  const auto fetch = [&](const Unit& q, int s, int d) {
    const uint32_t k = (SHARE ? s * 4 + wave : s) * MOE_STEP;
    const int left = a.K - (int)k;
    const uint32_t wo = r * 16 < left ? q.wo : BUF_NONE;
#pragma unroll
    for (int w = 0; w < RW; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) wb[d][w][i] = moe_weights<KEEP>(q.w, wo, k + (2 * w + (i & 1)) * 4 * a.K + (i >> 1) * up);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      if (MT > 1 && 16 * j >= q.m.cnt) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) xb[d][j][i] = buf_load(xb_of, g * 16 + 64 * i < left ? q.xo[j] : BUF_NONE, k + 64 * i);
    }
  };
  const int first = SHARE ? blockIdx.x : blockIdx.x * 4 + wave, stride = SHARE ? gridDim.x : gridDim.x * 4;
  if (first >= units) return;
  Unit cur = unit_of(first);
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(cur, d, d);
  int turn = 0;
  for (int u = first; u < units; u += stride, ++turn) {
    const Unit next = unit_of(u + stride);
    const bool finish = !SHARE || (turn & 3) == wave;
    float sg[RW][4], su[RW][4], as[MT];
    if (finish) {  // asked for ahead of the products
      const float* sc = a.s13 + (int64_t)cur.m.e * 2 * a.I + cur.gi * 8 * RW + 4 * (g & 1);
#pragma unroll
      for (int w = 0; w < RW; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sg[w][i] = sc[8 * w + i];
          su[w][i] = sc[a.I + 8 * w + i];
        }
#pragma unroll
      for (int j = 0; j < MT; ++j) as[j] = a.a_scale[16 * j + r < cur.m.cnt ? (int)lists.token[cur.m.off + 16 * j + r] * a.a_stride : 0];
    }
    Acc acc[RW][MT];
#pragma unroll
    for (int w = 0; w < RW; ++w)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[w][j] = Acc{0, 0, 0, 0};
    for (int s = 0; s < steps; s += D) {
      const bool last = s + D >= steps;
#pragma unroll
      for (int d = 0; d < D; ++d) {
#pragma unroll
        for (int w = 0; w < RW; ++w) moe_stage(st + w * 4096, wb[d][w]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v4i wv[RW][2];
#pragma unroll
          for (int w = 0; w < RW; ++w)
#pragma unroll
            for (int i = 0; i < 2; ++i) wv[w][i] = *(const v4i*)(st + w * 4096 + h * 2048 + r * 128 + (((4 * i + g) ^ rr) * 16));
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            if (MT > 1 && 16 * j >= cur.m.cnt) break;
#pragma unroll
            for (int w = 0; w < RW; ++w) moe_mfma<OP>(acc[w][j], wv[w][0], wv[w][1], xb[d][j][2 * h], xb[d][j][2 * h + 1]);
          }
        }
        __builtin_amdgcn_wave_barrier();
        fetch(last ? next : cur, last ? d : s + D + d, d);
      }
    }
    Acc(*mine)[RW * MT][64] = part[SHARE ? turn & 1 : 0];
    if constexpr (SHARE) {
#pragma unroll
      for (int w = 0; w < RW; ++w)
#pragma unroll
        for (int j = 0; j < MT; ++j) mine[wave][w * MT + j][lane] = acc[w][j];
      __syncthreads();
    }
    if (finish) {
      // lane (r, g): column r, rows 4 g .. + 3: gate rows in the lower half of the wave, their up rows 32 lanes on
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (16 * j >= cur.m.cnt) break;
        const int pos = cur.m.off + 16 * j + r;
        const bool there = 16 * j + r < cur.m.cnt;
#pragma unroll
        for (int w = 0; w < RW; ++w) {
          Acc sum = acc[w][j];
          if constexpr (SHARE) sum = (mine[0][w * MT + j][lane] + mine[1][w * MT + j][lane]) + (mine[2][w * MT + j][lane] + mine[3][w * MT + j][lane]);
          v4f h;
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float own = (float)sum[i];
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(own), __float_as_uint(own), false, false);
            const float gate = __uint_as_float(both[0]) * (as[j] * sg[w][i]), upv = __uint_as_float(both[1]) * (as[j] * su[w][i]);
            h[i] = gate / (1.0f + expf(-gate)) * upv;
            const uint32_t m = __float_as_uint(h[i]) & 0x7fffffffu;  // (as integers: a NaN is larger than everything)
            top = top > m ? top : m;
          }
          const int at = cur.gi * RW + w;
          if (there && g < 2) *(v4f*)(a.h + (int64_t)pos * a.I + at * 8 + 4 * g) = h;
          if (a.tops) {
            const auto o = __builtin_amdgcn_permlane16_swap(top, top, false, false);
            top = o[0] > o[1] ? o[0] : o[1];
            if (there && g == 0) a.tops[(int64_t)pos * (a.I / 8) + at] = top;
          }
        }
      }
    }
    cur = next;
  }
}

template <int OP>
__device__ __forceinline__ float moe_scale(uint32_t top) {
  const float m = __uint_as_float(top);
  if constexpr (OP == FMSMO_OP_E4M3) {
    const float s = m / 448.0f;
    return s < 1e-12f ? 1e-12f : s;  // (a NaN stays)
  } else {
    return (m < 1e-5f ? 1e-5f : m) / 127.0f;
  }
}
template <int OP>
__device__ __forceinline__ uint32_t moe_codes(v4f h, float s) {
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = h[i] / s;
  if constexpr (OP == FMSMO_OP_E4M3) {
    int o = 0;
    o = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], o, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], o, true);
  } else {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(q[i] + 12582912.0f);  // rint in the low mantissa bits (1.5 * 2^23)
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u), __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), 0x05040100u);
  }
}
// 1024 elements of a position a block
constexpr int MOE_QUANT = 1024;
template <int OP>
__global__ __launch_bounds__(256) void moe_quant_kernel(MoeArgs a) {
  __shared__ uint32_t tops[4];
  const int pos = blockIdx.x, groups = a.I / 8, i = blockIdx.y * (MOE_QUANT / 4) + threadIdx.x;
  const bool in = 4 * i < a.I;
  const v4f v = in ? ((const v4f*)(a.h + (int64_t)pos * a.I))[i] : v4f{0, 0, 0, 0};
  uint32_t top = 0;
  for (int k = threadIdx.x; k < groups; k += 256) {
    const uint32_t u = a.tops[(int64_t)pos * groups + k];
    top = top > u ? top : u;
  }
  top = wave_max_u32(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) top = top > tops[w] ? top : tops[w];
  const float s = moe_scale<OP>(top);
  if (threadIdx.x == 0 && blockIdx.y == 0) a.hs[pos] = s;
  if (in) ((uint32_t*)(a.hq + (int64_t)pos * a.I))[i] = moe_codes<OP>(v, s);
}

__device__ __forceinline__ void moe_put(const MoeArgs& a, int tok, int n, float v) {
  const int64_t at = tok * a.ldy + n;
  if (a.y_dtype == FMSMO_F16) ((u16*)a.y)[at] = f32_to_f16(v);
  else if (a.y_dtype == FMSMO_BF16) ((u16*)a.y)[at] = f32_to_bf16(v);
  else ((float*)a.y)[at] = v;
}
// y.  A block owns ROWS outputs and goes through all groups of tokens: their steps of 256 bytes one behind the other, cut into equal parts
// for the waves, D steps on their way; at the end of a group a wave adds its products, with their scales and shares, to sums of its own, and the
// waves' sums are added in their order.  Where few outputs leave units without a block, several blocks share the steps of the same outputs
// and a kernel behind adds what they leave.  ROWS = 8, groups of up to eight tokens: a product takes two steps, the first with its upper eight
// rows and left eight columns, the second with the others, and the two blocks on its diagonal are added.  ROWS = 32, groups of more than 16 tokens:
// two products, so that tokens are read half as often (64 tokens, two of 8 experts of 4096 x 14336 90 us and 5 of the join, 116 with 16 rows; two of
// 4 of 4096 x 8192 37 + 5 and 50).  QUANT: few positions, whose codes every block makes for itself in shared memory.  Up to TM tokens.
constexpr int MOE_QUANT_MOST = 16384;
template <int OP, int MT, int ROWS, int NW, int D, int TM, bool QUANT, bool KEEP>
__global__ __launch_bounds__(NW * 64) void moe_down_kernel(MoeArgs a) {
  typedef typename MoeAcc<OP>::type Acc;
  constexpr int NT = NW * 64;
  constexpr bool PAIR = ROWS == 8;  // two steps a product
  static_assert(!PAIR || MT == 1, "");
  constexpr int WL = PAIR ? 2 : 4, RW = PAIR ? 1 : ROWS / 16;  // loads of a step for a product's rows, products beside each other
  __shared__ __attribute__((aligned(16))) uint8_t stage[NW][1024 * WL * RW];
  __shared__ uint32_t entry[MOE_ENTRIES];
  __shared__ uint8_t token[MOE_TOKENS * MOE_TOP];
  __shared__ float share[MOE_TOKENS * MOE_TOP];
  __shared__ __attribute__((aligned(16))) float sums[NW * TM * ROWS];
  __shared__ __attribute__((aligned(16))) uint8_t codes[QUANT ? MOE_QUANT_MOST : 16];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * ROWS, steps = (a.I + MOE_STEP - 1) / MOE_STEP, pairs = a.T * a.top;
  const int count = a.count[0], all = count * steps;
  for (int i = threadIdx.x; i < min(a.E, pairs) + pairs / 8; i += NT) entry[i] = a.entry[i];  // (as many as there may be: not after the count)
  // (positions that no pair took hold what was there before: they are not in any group)
  for (int i = threadIdx.x; i < pairs; i += NT) {
    token[i] = (uint8_t)a.token[i];
    share[i] = a.weight[i];
    if (!QUANT) share[i] *= a.hs[i];
  }
  for (int i = threadIdx.x; i < NW * a.T * ROWS; i += NT) sums[i] = 0.0f;
  __syncthreads();
  const int part = blockIdx.y * NW + wave, parts = gridDim.y * NW;
  const int from = (int)((int64_t)part * all / parts), to = (int)((int64_t)(part + 1) * all / parts);
  uint8_t* st = stage[wave];
  const int rr = r & 7;
  int le = steps ? from / steps : 0, ls = from - le * steps, ce = le, cs = ls;  // what is loaded and what is multiplied next: group and step
  MoeGroup lm = group_of(entry[0]), cm = lm;
  // column r of a product: token col of tile j, and in a pair the step's half
  const int col = PAIR ? rr : r, half = PAIR ? 128 * (r >> 3) : 0;
  Buf w = buf_of(a.w2);
  const Buf xb_of = buf_of(a.hq);
  uint32_t wo[RW], xo[MT];
  const auto load_from = [&] {
    lm = group_of(uniform((int)entry[le]));
    w = buf_of(a.w2 + (int64_t)lm.e * a.K * a.I);
#pragma unroll
    for (int w = 0; w < RW; ++w) wo[w] = RW == 1 || n0 + 16 * w < a.K ? (uint32_t)(n0 + 16 * w + g) * (uint32_t)a.I + r * 16 : BUF_NONE;
#pragma unroll
    for (int j = 0; j < MT; ++j) xo[j] = 16 * j + col < lm.cnt ? (uint32_t)(lm.off + 16 * j + col) * (uint32_t)a.I + half + g * 16 : BUF_NONE;
  };
  constexpr int XL = PAIR ? 2 : 4;
  v4i wb[D][RW][WL], xb[QUANT ? 1 : D][MT][XL];
  int loads = to - from;  // steps that are not on their way yet; behind the last one zeros are loaded
  const auto fetch = [&](int d) {
    const uint32_t k = ls * MOE_STEP;
    const int left = loads > 0 ? a.I - (int)k : 0;
#pragma unroll
    for (int v = 0; v < RW; ++v)
#pragma unroll
      for (int i = 0; i < WL; ++i) wb[d][v][i] = moe_weights<KEEP>(w, r * 16 < left ? wo[v] : BUF_NONE, k + i * 4 * a.I);
    if constexpr (!QUANT) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (MT > 1 && 16 * j >= lm.cnt) break;
#pragma unroll
        for (int i = 0; i < XL; ++i) xb[d][j][i] = buf_load(xb_of, half + g * 16 + 64 * i < left ? xo[j] : BUF_NONE, k + 64 * i);
      }
    }
    --loads;
    if (++ls == steps) {
      ls = 0;
      ++le;
      if (le < count) load_from();
    }
  };
  Acc acc[RW][MT];
  const int ng = PAIR ? g & 1 : g;  // the four outputs of this lane
  v4f sc[RW], sn[RW];  // scales of the group that is multiplied, and of the next one
  const auto ahead = [&](int i) {
    const float* of = a.s2 + (int64_t)group_of(uniform((int)entry[i])).e * a.K + n0 + 4 * ng;
#pragma unroll
    for (int w = 0; w < RW; ++w) sn[w] = *(const v4f*)(of + (n0 + 16 * w < a.K ? 16 * w : 0));
  };
  const auto begin = [&] {
    cm = group_of(uniform((int)entry[ce]));
#pragma unroll
    for (int w = 0; w < RW; ++w) sc[w] = sn[w];
    if (ce + 1 < count) ahead(ce + 1);
#pragma unroll
    for (int w = 0; w < RW; ++w)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[w][j] = Acc{0, 0, 0, 0};
  };
  const auto end = [&] {
    if constexpr (PAIR) {  // rows 8 .. 15 of columns 8 .. 15 belong to rows 0 .. 7 of columns 0 .. 7: 32 + 8 lanes on
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][0][i] += __shfl(acc[0][0][i], (lane + 40) & 63);
      if (lane >= 32) return;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      if (16 * j + r >= cm.cnt) break;
      const int pos = cm.off + 16 * j + r;
      const float c = share[pos];
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        v4f* sum = (v4f*)(sums + (wave * a.T + token[pos]) * ROWS + 16 * w + 4 * ng);
        v4f v = *sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fmaf_rn((float)acc[w][j][i], c * sc[w][i], v[i]);
        *sum = v;
      }
    }
  };
  if (from < to) {  // the first weights, ahead of the codes
    load_from();
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(d);
    ahead(ce);
  }
  if constexpr (QUANT) {
    const MoeGroup m = count ? group_of(entry[count - 1]) : MoeGroup{0, 0, 0};
    for (int pos = wave; pos < m.off + m.cnt; pos += NW) {
      const v4f* h = (const v4f*)(a.h + (int64_t)pos * a.I);
      const auto max4 = [](v4f v, uint32_t top) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t u = __float_as_uint(v[k]) & 0x7fffffffu;
          top = top > u ? top : u;
        }
        return top;
      };
      constexpr int HELD = 4;  // 1024 elements of a row stay in registers, the others are read again
      v4f v[HELD];
      uint32_t top = 0;
#pragma unroll
      for (int q = 0; q < HELD; ++q) v[q] = h[min(lane + 64 * q, a.I / 4 - 1)];
#pragma unroll
      for (int q = 0; q < HELD; ++q) top = max4(v[q], top);
      for (int i = lane + 64 * HELD; i < a.I / 4; i += 64) top = max4(h[i], top);
      const float s = moe_scale<OP>(wave_max_u32(top));
      if (lane == 0) share[pos] *= s;
      uint32_t* to = (uint32_t*)(codes + pos * a.I);
#pragma unroll
      for (int q = 0; q < HELD; ++q)
        if (lane + 64 * q < a.I / 4) to[lane + 64 * q] = moe_codes<OP>(v[q], s);
      for (int i = lane + 64 * HELD; i < a.I / 4; i += 64) to[i] = moe_codes<OP>(h[i], s);
    }
    __syncthreads();
  }
  if (from < to) {
    begin();
    for (int f = from; f < to; f += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if constexpr (PAIR) {  // rows 0 .. 7 of the product: the first 128 bytes of the eight rows, rows 8 .. 15: the others
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int q = 4 * i + g;
            *(v4i*)(st + (r >> 3) * 1024 + q * 128 + (((r ^ q) & 7) * 16)) = wb[d][0][i];
          }
          __builtin_amdgcn_wave_barrier();
        } else {
#pragma unroll
          for (int w = 0; w < RW; ++w) moe_stage(st + 4096 * w, wb[d][w]);
        }
#pragma unroll
        for (int h = 0; h < WL / 2; ++h) {
          v4i wv[RW][2];
#pragma unroll
          for (int w = 0; w < RW; ++w)
#pragma unroll
            for (int i = 0; i < 2; ++i) wv[w][i] = *(const v4i*)(st + w * 4096 + h * 2048 + r * 128 + (((4 * i + g) ^ rr) * 16));
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            if (MT > 1 && 16 * j >= cm.cnt) break;
            v4i x0, x1;
            if constexpr (QUANT) {
              const int k = cs * MOE_STEP + 128 * h + half + g * 16;
              const bool v = 16 * j + col < cm.cnt;
              x0 = x1 = v4i{0, 0, 0, 0};
              if (v && k < a.I) x0 = *(const v4i*)(codes + (cm.off + 16 * j + col) * a.I + k);
              if (v && k + 64 < a.I) x1 = *(const v4i*)(codes + (cm.off + 16 * j + col) * a.I + k + 64);
            } else {
              x0 = xb[d][j][2 * h];
              x1 = xb[d][j][2 * h + 1];
            }
#pragma unroll
            for (int w = 0; w < RW; ++w) moe_mfma<OP>(acc[w][j], wv[w][0], wv[w][1], x0, x1);
          }
        }
        __builtin_amdgcn_wave_barrier();
        fetch(d);
        if (f + d < to && (++cs == steps || f + d + 1 == to)) {
          end();
          cs = 0;
          ++ce;
          if (f + d + 1 < to) begin();
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * ROWS; i += NT) {
    float v = sums[i];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += sums[w * a.T * ROWS + i];
    const int tok = i / ROWS, n = n0 + i % ROWS;
    if (n >= a.K) continue;
    if (gridDim.y > 1) a.parts[((int64_t)blockIdx.y * a.T + tok) * a.K + n] = v;
    else moe_put(a, tok, n, v);
  }
}
__global__ __launch_bounds__(256) void moe_join_kernel(MoeArgs a, int splits) {
  const int n = blockIdx.x * 256 + threadIdx.x, tok = blockIdx.y;
  if (n >= a.K) return;
  float v = 0.0f;
  for (int s = 0; s < splits; ++s) v += a.parts[((int64_t)s * a.T + tok) * a.K + n];
  moe_put(a, tok, n, v);
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();

static bool moe_sizes(int64_t T, int64_t E, int top, int64_t K, int64_t I) {
  return T >= 0 && T <= MOE_TOKENS && E >= 1 && E <= MOE_EXPERTS && top >= 1 && top <= MOE_TOP && top <= E && K >= 16 && I >= 16 && K % 16 == 0 &&
         I % 16 == 0 && K < 1 << 17 && I < 1 << 17 && 2 * I * K <= 0x7f000000;  // (sums of products, and offsets into an expert's weights, in 32 bits)
}
// What a call is cut into.
struct MoePlan {
  int mt;       // tiles of 16 tokens of a group
  bool narrow;  // the down product's blocks have eight outputs
  bool quant;   // and make the codes of h themselves
  bool share;   // the waves of a block share a unit of the gate and up products
  bool deep;    // four steps on their way there
  bool wide;    // two products' rows a unit there
  int splits;   // blocks for the same outputs
};
static MoePlan moe_plan(int64_t T, int64_t E, int top, int64_t K, int64_t I) {
  MoePlan p;
  // Groups of 16 tokens, 32 or 64: experts with more stream their weights again.  With up to six tokens an expert on average few have more than 16,
  // with up to twenty few have more than 32 (one product's rows a unit: 64 tokens, two of 8 experts of 4096 x 14336: gate and up 219 us in groups of 32, 252 of 64;
  // 40, four of 16: 21 and 28; 64, two of 4: 180 and 157).
  p.mt = T <= 16 || T * top <= 6 * E ? 1 : T <= 32 || T * top <= 20 * E ? 2 : 4;
  const int64_t used = std::min(E, T * top);
  // Waves with units of their own where rows are short and units many (13 tokens over 32 experts of 1024 x 14080: 160 us, 176 shared; 16 over 8 of
  // 4096 x 14336: 159 and 151; one token over 128 of 2048 x 768: 12.4 and 9.5).  Four steps on their way where a wave has a multiple of four for a
  // unit (K = 4096: 151 us, 177 with one).
  p.share = K >= 2048 || used * (I / 8) < 4096;
  p.deep = p.mt == 1 && p.share && div_up(K, 1024) % 4 == 0;
  // Two products' rows a unit, so that tokens are read half as often (a compute unit takes in about 33 GB/s of both), where it leaves enough of them
  // and tokens weigh: 64 tokens, two of 8 experts of 4096 x 14336 197 us, 222 with one; two of 4 of 4096 x 8192 80 and 110; 64 over 128 experts 64
  // and 68; but 27, all of 4 experts of 2784 x 352, 9.2 and 7.6, 32 over 64 experts of 2048 x 1408 58 and 57.
  p.wide = p.mt > 1 ? used * (I / 8) >= 1024 : p.share && !p.deep && T * top >= 4 * used && used * (I / 8) >= 4096;
  // The down product: a compute unit takes in 23 GB/s, a little less on eight rows, so that what counts is how evenly the blocks fall on the units
  // (8 experts, 14336 -> 4096 columns, 256 blocks: 71 us, 4112 columns, 257 blocks: 137); a split is a launch more.  On eight rows an expert's
  // tokens are groups of eight, and its weights stream past for each of them: m tokens an expert on average are about m / 8 + 0.5 groups.
  // Sixteen rows and eight, the whole block: 16 tokens, all of 2 experts of 2048 x 16384 58 us and 67, all of 8 of 2048 x 7168 90 and 103; 12, six of 8 of
  // 2048 x 5632 63 and 71; 64, six of 64 of 2048 x 1408 108 and 114; but 32, four of 32 of 2048 x 2048 79 and 77.
  const double bytes = (double)used * K * I;
  const double again = std::min(std::max((double)(T * top) / (8.0 * used) + 0.5, 1.0), (double)div_up(T, 8));
  double best = 1e30;
  p.narrow = false;
  p.splits = 1;
  for (int narrow = p.mt == 1; narrow >= 0; --narrow)
    for (int n = 1; n <= 8; ++n) {
      const double blocks = (double)n * (double)(p.mt > 1 ? div_up(K, 32) : K / (narrow ? 8 : 16));
      const double cost = std::ceil(blocks / 256) * bytes * (narrow ? again : 1.0) / blocks / (narrow ? 21e9 : 23e9) + (n > 1 ? 4e-6 : 0.0);
      if (cost < best * 0.98) best = cost, p.narrow = narrow, p.splits = n;
    }
  // (a launch or so many rows for every block: 2 tokens, eight of 128 experts of 2048 x 768 23.4 us and 24.3, 4 tokens 34.9 and 31.9)
  p.quant = p.mt == 1 && T * top <= 16 && T * top * I <= MOE_QUANT_MOST;
  return p;
}
// bytes up to each piece of the workspace
struct MoeSpace {
  int64_t ids, share, entry, token, weight, hs, h, hq, tops, parts, all;
};
static MoeSpace moe_space(int64_t T, int64_t E, int top, int64_t K, int64_t I) {
  const int64_t P = T * top, p16 = (P + 3) / 4 * 16;
  MoeSpace s;
  s.ids = 16;
  s.share = s.ids + p16;
  s.entry = s.share + p16;
  s.token = s.entry + 4 * MOE_ENTRIES;
  s.weight = s.token + p16;
  s.hs = s.weight + p16;
  s.h = s.hs + p16;
  s.hq = s.h + 4 * P * I;
  s.tops = s.hq + P * I;
  s.parts = s.tops + P * I / 2;
  const int splits = moe_plan(T, E, top, K, I).splits;
  s.all = s.parts + (splits > 1 ? 4 * splits * T * K : 0);
  return s;
}

extern "C" int64_t fmsmo_moe_few_workspace_bytes(int64_t T, int64_t E, int top, int64_t K, int64_t I) {
  return moe_sizes(T, E, top, K, I) && T ? moe_space(T, E, top, K, I).all : 0;
}

template <int OP, int MT, int ROWS, bool QUANT, bool KEEP>
static void run_down(const MoeArgs& a, int splits, hipStream_t s) {
  // waves and steps on their way: eight rows want more waves (64 tokens over 128 experts: 41 us with 16 and 2, 50 with 8 and 4, 54 with 16 and 4,
  // whose registers do not suffice), sixteen are indifferent
  constexpr int NW = ROWS == 8 ? 16 : 8, D = MT == 4 ? 1 : 2;
  const dim3 grid((unsigned)div_up(a.K, ROWS), (unsigned)splits), block(NW * 64);
  if constexpr (MT == 1) {
    if (QUANT || a.T <= 16) {  // (up to 16 positions where QUANT, so no more tokens)
      hipLaunchKernelGGL((moe_down_kernel<OP, 1, ROWS, NW, D, 16, QUANT, KEEP>), grid, block, 0, s, a);
      return;
    }
  }
  if constexpr (!QUANT) hipLaunchKernelGGL((moe_down_kernel<OP, MT, ROWS, NW, D, 64, false, KEEP>), grid, block, 0, s, a);
}
template <int OP, int MT, int RW, int D, bool SHARE, bool KEEP>
static void run_up(const MoeArgs& a, hipStream_t s) {
  // groups of tokens, at most
  const int64_t units = (int64_t)std::min(a.E + a.T * a.top / (16 * MT), a.T * a.top) * (a.I / (8 * RW));
  const dim3 grid((unsigned)std::min<int64_t>(SHARE ? units : div_up(units, 4), RW * D > 1 ? 512 : MT > 1 ? 768 : 1024)), block(256);
  if constexpr (MT == 1) {
    if (a.T <= MOE_ROUTED) {
      hipLaunchKernelGGL((moe_up_kernel<OP, 1, RW, D, true, SHARE, KEEP>), grid, block, 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((moe_up_kernel<OP, MT, RW, D, false, SHARE, KEEP>), grid, block, 0, s, a);
}
template <int OP, int MT>
static void run_moe(MoeArgs a, const MoePlan& p, hipStream_t s) {
  if (p.quant) a.tops = nullptr;
  a.down_group = p.narrow ? 8 : 16 * MT;
  if (a.T > MOE_ROUTED) hipLaunchKernelGGL(moe_route_kernel, dim3((unsigned)div_up(a.T, 4)), dim3(256), 0, s, a);
  const auto up = [&](auto keep) {
    constexpr bool KEEP = decltype(keep)::value;
    if constexpr (MT == 1) {
      if (!p.share) return run_up<OP, 1, 1, 1, false, KEEP>(a, s);
      if (p.deep) return run_up<OP, 1, 1, 4, true, KEEP>(a, s);
    } else {
      if (!p.share) return run_up<OP, MT, 2, 1, false, KEEP>(a, s);  // (so many units that it is the wide form)
    }
    p.wide ? run_up<OP, MT, 2, 1, true, KEEP>(a, s) : run_up<OP, MT, 1, 1, true, KEEP>(a, s);
  };
  const auto down = [&](auto keep) {
    constexpr bool KEEP = decltype(keep)::value;
    if constexpr (MT == 1) {
      if (p.narrow) return p.quant ? run_down<OP, 1, 8, true, KEEP>(a, p.splits, s) : run_down<OP, 1, 8, false, KEEP>(a, p.splits, s);
      if (p.quant) return run_down<OP, 1, 16, true, KEEP>(a, p.splits, s);
    }
    run_down<OP, MT, (MT > 1 ? 32 : 16), false, KEEP>(a, p.splits, s);
  };
  if (a.K % 128) up(std::true_type{});
  else up(std::false_type{});
  if (!p.quant) hipLaunchKernelGGL((moe_quant_kernel<OP>), dim3((unsigned)(a.T * a.top), (unsigned)div_up(a.I, MOE_QUANT)), dim3(256), 0, s, a);
  if (a.I % 128) down(std::true_type{});
  else down(std::false_type{});
  if (p.splits > 1) hipLaunchKernelGGL(moe_join_kernel, dim3((unsigned)div_up(a.K, 256), (unsigned)a.T), dim3(256), 0, s, a, p.splits);
}

extern "C" int fmsmo_moe_few_tokens(int codes, const void* a, int64_t lda, const float* a_scale, int64_t a_scale_n, const void* logits,
                                    int logits_dtype, int64_t ldl, const void* w13, const float* w13_scale, const void* w2,
                                    const float* w2_scale, int64_t T, int64_t E, int top, int renormalize, void* y, int y_dtype, int64_t ldy,
                                    int64_t K, int64_t I, void* workspace, int64_t workspace_bytes, fmsmo_stream_t stream) {
  if (T < 0 || E < 0 || K < 0 || I < 0) return FMSMO_ERR_SHAPE;
  if (codes != FMSMO_OP_I8 && codes != FMSMO_OP_E4M3) return FMSMO_ERR_UNSUPPORTED;
  if (logits_dtype < FMSMO_F16 || logits_dtype > FMSMO_F32 || y_dtype < FMSMO_F16 || y_dtype > FMSMO_F32) return FMSMO_ERR_UNSUPPORTED;
  if (!moe_sizes(T, E, top, K, I)) return FMSMO_ERR_UNSUPPORTED;
  if (T == 0) return FMSMO_OK;
  if (!a || !a_scale || !logits || !w13 || !w13_scale || !w2 || !w2_scale || !y || !workspace) return FMSMO_ERR_NULL;
  if ((a_scale_n != 1 && a_scale_n != T) || (T > 1 && (lda < K || ldl < E || ldy < K))) return FMSMO_ERR_SHAPE;
  const auto off = [](const void* p) { return (((uintptr_t)p) & 15) != 0; };
  if (T > 1 && lda > 1 << 24) return FMSMO_ERR_UNSUPPORTED;
  if (off(a) || off(w13) || off(w2) || off(w2_scale) || off(workspace) || (T > 1 && lda % 16)) return FMSMO_ERR_ALIGN;
  const MoeSpace sp = moe_space(T, E, top, K, I);
  if (workspace_bytes < sp.all) return FMSMO_ERR_SCRATCH;
  char* ws = (char*)workspace;
  MoeArgs g{(const uint8_t*)a, a_scale, logits, (const uint8_t*)w13, w13_scale, (const uint8_t*)w2, w2_scale, y, lda, ldl, ldy,
            a_scale_n == 1 ? 0 : 1, logits_dtype, y_dtype, (int)T, (int)E, top, (int)K, (int)I, renormalize != 0, 0,
            (int*)(ws + sp.ids), (float*)(ws + sp.share), (int*)ws, (uint32_t*)(ws + sp.entry), (int*)(ws + sp.token), (float*)(ws + sp.weight),
            (float*)(ws + sp.hs), (float*)(ws + sp.h), (uint8_t*)(ws + sp.hq), (float*)(ws + sp.parts), (uint32_t*)(ws + sp.tops)};
  const MoePlan p = moe_plan(T, E, top, K, I);
  const auto tiles = [&](auto op) {
    constexpr int OP = decltype(op)::value;
    if (p.mt == 1) run_moe<OP, 1>(g, p, (hipStream_t)stream);
    else if (p.mt == 2) run_moe<OP, 2>(g, p, (hipStream_t)stream);
    else run_moe<OP, 4>(g, p, (hipStream_t)stream);
  };
  if (codes == FMSMO_OP_I8) tiles(std::integral_constant<int, FMSMO_OP_I8>{});
  else tiles(std::integral_constant<int, FMSMO_OP_E4M3>{});
  return fmsmo_check_launch();
}

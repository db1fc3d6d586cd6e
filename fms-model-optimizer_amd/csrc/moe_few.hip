// A mixture-of-experts block for a few tokens (up to 64), whose weights are read once and bound it: routing, gate and up products, gated
// silu in 8 bits, down products and the weighted sum.
//
//   p = softmax(logits[t]); S = the `top` experts of the largest logits (of equal ones the lower index); c_e = p_e / sum_S p, or p_e
//   g, u = (a[t] . w13[e]^T) a_scale[t] w13_scale[e]  (rows 0 .. I - 1 and I .. 2I - 1),  h = g / (1 + exp(-g)) u  in fp32
//   codes of h per token and expert: int8 s = max(max|h|, 1e-5) / 127, e4m3 s = max(max|h| / 448, 1e-12), as the per-token quantizers in fp32
//   y[t] = sum_S c_e s (codes . w2[e]^T) w2_scale[e]
//
// The chosen (token, expert) pairs are sorted by expert: a `position` each.  The weights stream past once, eight rows of 128 bytes a load,
// and are turned into matrix operands in shared memory; an expert's tokens are the columns of the product.
#include "paged_kv.hpp"

#include <type_traits>

namespace fmsmo {

constexpr int MOE_TOKENS = 64, MOE_EXPERTS = 512, MOE_TOP = 16;

struct MoeEntry {  // an expert that some token chose
  int e, off, cnt, pad;
};
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
  // workspace
  int* count;       // [0]: entries, [1]: positions
  MoeEntry* entry;  // [E]
  int* token;       // [T top]: of a position
  float* weight;
  float* h;         // [T top][I]
  float* hs;        // [T top]
  uint8_t* hq;      // [T top][I]
};

// an order of floats as unsigned integers (both zeros are one number); 0 is none of them
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  const uint32_t k = u >> 31 ? ~u : u | 0x80000000u;
  return k ? k : 1u;
}

// One block.  A wave finds a token's experts, eight logits a lane, the largest by the largest; the rest is counting.
__global__ __launch_bounds__(1024) void moe_route_kernel(MoeArgs a) {
  constexpr int V = MOE_EXPERTS / 64;
  __shared__ unsigned long long mask[MOE_EXPERTS];  // tokens of an expert
  __shared__ int off[MOE_EXPERTS];
  __shared__ short ids[MOE_TOKENS][MOE_TOP];
  __shared__ float share[MOE_TOKENS][MOE_TOP];
  __shared__ int wave_cnt[16], wave_act[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = threadIdx.x; e < a.E; e += 1024) mask[e] = 0;
  __syncthreads();
  for (int t = wave; t < a.T; t += 16) {
    uint32_t key[V];
    float val[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 64 * i;
      const bool in = e < a.E;
      val[i] = in ? scalar_f32(a.logits, a.logits_dtype, t * a.ldl + e) : 0.0f;
      key[i] = in ? order_of(val[i]) : 0u;
    }
    float first = 0.0f, sum = 0.0f, mine = 0.0f;
    int id = -1;  // lane s keeps the s-th choice
    for (int s = 0; s < a.top; ++s) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) m = m > key[i] ? m : key[i];
      m = wave_max_u32(m);
      int e = 0;
      bool found = false;
      float v = 0.0f;
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
      if (s == 0) first = v;
      const float p = first == -__builtin_inff() ? 0.0f : expf(v - first);
      sum += p;
      if (lane == s) {
        id = e;
        mine = p;
      }
    }
    if (!a.renorm) {
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane + 64 * i < a.E && first != -__builtin_inff()) sum += expf(val[i] - first);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    }
    if (lane < a.top) {
      const float c = mine == 0.0f ? 0.0f : mine / sum;  // (a share of zero: the expert is not run)
      share[t][lane] = c;
      ids[t][lane] = (short)(c == 0.0f ? -1 : id);
      if (c != 0.0f) atomicOr(&mask[id], 1ull << t);
    }
  }
  __syncthreads();
  const int e = threadIdx.x;
  const int cnt = e < a.E ? __popcll(mask[e]) : 0;
  int upto = cnt;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    upto += lane >= d ? o : 0;
  }
  const uint64_t act = __ballot(cnt > 0);
  if (lane == 63) {
    wave_cnt[wave] = upto;
    wave_act[wave] = __popcll(act);
  }
  __syncthreads();
  int before = 0, rank = __popcll(act & ((1ull << lane) - 1));
  for (int w = 0; w < wave; ++w) {
    before += wave_cnt[w];
    rank += wave_act[w];
  }
  if (e < a.E) off[e] = before + upto - cnt;
  if (cnt > 0) a.entry[rank] = MoeEntry{e, before + upto - cnt, cnt, 0};
  if (threadIdx.x == 1023) {
    a.count[0] = rank + (cnt > 0);
    a.count[1] = before + upto;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * a.top; i += 1024) {
    const int t = i / a.top, s = i % a.top, id = ids[t][s];
    if (id < 0) continue;
    const int pos = off[id] + __popcll(mask[id] & ((1ull << t) - 1));
    a.token[pos] = t;
    a.weight[pos] = share[t][s];
  }
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
__device__ __forceinline__ v4i stream16(const uint8_t* p, int64_t off, bool there) {
  v4i v = {0, 0, 0, 0};
  if (there) v = __builtin_nontemporal_load((const v4i*)(p + off));
  return v;
}

// h of the positions.  A unit: eight gate rows and the eight up rows that belong to them, over all of K, for one expert: the 16 rows of the
// product.  KS = 1: each wave takes units of its own, one behind the other, D steps of 128 bytes a row on their way; KS = 4: the
// four waves of a block share a unit's K.
template <int OP, int MT, int KS, int D>
__global__ __launch_bounds__(256) void moe_up_kernel(MoeArgs a) {
  typedef typename MoeAcc<OP>::type Acc;
  __shared__ __attribute__((aligned(16))) uint8_t stage[4][2048];
  __shared__ __attribute__((aligned(16))) Acc part[KS > 1 ? 3 : 1][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4, drow = lane >> 3, dpos = lane & 7;
  const int groups = a.I / 8, units = a.count[0] * groups, steps = (a.K + 127) / 128;
  const int stride = KS == 1 ? gridDim.x * 4 : gridDim.x, first = KS == 1 ? wave * gridDim.x + blockIdx.x : blockIdx.x;
  const int s0 = KS == 1 ? 0 : wave, ds = KS == 1 ? 1 : 4;
  uint8_t* st = stage[wave];
  const int rr = r & 7;
  for (int u = first; u < units; u += stride) {
    const int en = u / groups, gi = u - en * groups;
    const MoeEntry x = a.entry[en];
    const int e = uniform(x.e), off = uniform(x.off), cnt = uniform(x.cnt);
    const uint8_t* wg = a.w13 + ((int64_t)e * 2 * a.I + gi * 8 + drow) * a.K;
    const uint8_t* wu = wg + (int64_t)a.I * a.K;
    const uint8_t* xp[MT];
    bool xv[MT];
    int tok[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      xv[j] = 16 * j + r < cnt;
      tok[j] = xv[j] ? a.token[off + 16 * j + r] : 0;
      xp[j] = a.a + tok[j] * a.lda;
    }
    v4i wb[D][2], xb[D][MT][2];
    const auto fetch = [&](int s, int d) {
      const int k = s * 128;
      const bool in = k + dpos * 16 < a.K;
      wb[d][0] = stream16(wg, k + dpos * 16, in);
      wb[d][1] = stream16(wu, k + dpos * 16, in);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (16 * j >= cnt) break;
        xb[d][j][0] = xv[j] && k + g * 16 < a.K ? *(const v4i*)(xp[j] + k + g * 16) : v4i{0, 0, 0, 0};
        xb[d][j][1] = xv[j] && k + 64 + g * 16 < a.K ? *(const v4i*)(xp[j] + k + 64 + g * 16) : v4i{0, 0, 0, 0};
      }
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (s0 + d * ds < steps) fetch(s0 + d * ds, d);
    Acc acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = Acc{0, 0, 0, 0};
    for (int s = s0; s < steps; s += D * ds) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int at = s + d * ds;
        if (at >= steps) break;
        *(v4i*)(st + drow * 128 + ((dpos ^ drow) * 16)) = wb[d][0];
        *(v4i*)(st + (8 + drow) * 128 + ((dpos ^ drow) * 16)) = wb[d][1];
        __builtin_amdgcn_wave_barrier();
        const v4i w0 = *(const v4i*)(st + r * 128 + ((g ^ rr) * 16));
        const v4i w1 = *(const v4i*)(st + r * 128 + (((4 + g) ^ rr) * 16));
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          if (16 * j >= cnt) break;
          moe_mfma<OP>(acc[j], w0, w1, xb[d][j][0], xb[d][j][1]);
        }
        if (at + D * ds < steps) fetch(at + D * ds, d);
      }
    }
    if constexpr (KS > 1) {
      if (wave) {
#pragma unroll
        for (int j = 0; j < MT; ++j) part[wave - 1][j][lane] = acc[j];
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int w = 0; w < 3; ++w) acc[j] += part[w][j][lane];
      }
      __syncthreads();
      if (wave) continue;
    }
    // lane (r, g): column r, rows 4 g .. + 3: gate rows in the lower half of the wave, their up rows 32 lanes on
    const float* sc = a.s13 + (int64_t)e * 2 * a.I + gi * 8 + 4 * (g & 1);
    float sg[4], su[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sg[i] = sc[i];
      su[i] = sc[a.I + i];
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      if (16 * j >= cnt) break;
      const float as = a.a_scale[tok[j] * a.a_stride];
      v4f h;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float own = (float)acc[j][i];
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(own), __float_as_uint(own), false, false);
        const float gate = __uint_as_float(both[0]) * (as * sg[i]), up = __uint_as_float(both[1]) * (as * su[i]);
        h[i] = gate / (1.0f + expf(-gate)) * up;
      }
      if (xv[j] && g < 2) *(v4f*)(a.h + (int64_t)(off + 16 * j + r) * a.I + gi * 8 + 4 * g) = h;
    }
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
// a block per position
template <int OP>
__global__ __launch_bounds__(256) void moe_quant_kernel(MoeArgs a) {
  __shared__ uint32_t tops[4];
  const int pos = blockIdx.x;
  if (pos >= a.count[1]) return;
  const v4f* h = (const v4f*)(a.h + (int64_t)pos * a.I);
  uint32_t top = 0;
  for (int i = threadIdx.x; i < a.I / 4; i += 256) {
    const v4f v = h[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t u = __float_as_uint(v[k]) & 0x7fffffffu;  // (as integers: a NaN is larger than everything)
      top = top > u ? top : u;
    }
  }
  top = wave_max_u32(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) top = top > tops[w] ? top : tops[w];
  const float s = moe_scale<OP>(top);
  if (threadIdx.x == 0) a.hs[pos] = s;
  for (int i = threadIdx.x; i < a.I / 4; i += 256) ((uint32_t*)(a.hq + (int64_t)pos * a.I))[i] = moe_codes<OP>(h[i], s);
}

// y.  A block owns ROWS outputs and goes through all chosen experts: their steps of 128 bytes in a row, cut into equal parts for the waves;
// at the end of an expert a wave adds its products, with their scales and shares, to sums of its own, and the waves' sums are added in their order.
template <int OP, int MT, int ROWS, int D>
__global__ __launch_bounds__(512) void moe_down_kernel(MoeArgs a) {
  typedef typename MoeAcc<OP>::type Acc;
  constexpr int NW = 8, L = ROWS / 8;
  __shared__ __attribute__((aligned(16))) uint8_t stage[NW][ROWS * 128];
  __shared__ __attribute__((aligned(16))) float sums[NW][16 * MT][ROWS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4, drow = lane >> 3, dpos = lane & 7;
  const int n0 = blockIdx.x * ROWS, steps = (a.I + 127) / 128, all = a.count[0] * steps;
  for (int i = threadIdx.x; i < NW * 16 * MT * ROWS; i += 512) (&sums[0][0][0])[i] = 0.0f;
  __syncthreads();
  const int from = (int)((int64_t)wave * all / NW), to = (int)((int64_t)(wave + 1) * all / NW);
  uint8_t* st = stage[wave];
  const int rr = r & 7;
  int at = from;
  while (at < to) {
    const int en = at / steps, s_lo = at - en * steps, s_hi = min(steps, s_lo + to - at);
    const MoeEntry x = a.entry[en];
    const int e = uniform(x.e), off = uniform(x.off), cnt = uniform(x.cnt);
    const uint8_t* wp = a.w2 + ((int64_t)e * a.K + n0 + drow) * a.I;
    const uint8_t* xp = a.hq + (int64_t)(off + r) * a.I;
    v4i wb[D][L], xb[D][MT][2];
    const auto fetch = [&](int s, int d) {
      const int k = s * 128;
#pragma unroll
      for (int l = 0; l < L; ++l) wb[d][l] = stream16(wp + (int64_t)l * 8 * a.I, k + dpos * 16, k + dpos * 16 < a.I);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (16 * j >= cnt) break;
        const bool v = 16 * j + r < cnt;
        xb[d][j][0] = v && k + g * 16 < a.I ? *(const v4i*)(xp + (int64_t)16 * j * a.I + k + g * 16) : v4i{0, 0, 0, 0};
        xb[d][j][1] = v && k + 64 + g * 16 < a.I ? *(const v4i*)(xp + (int64_t)16 * j * a.I + k + 64 + g * 16) : v4i{0, 0, 0, 0};
      }
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (s_lo + d < s_hi) fetch(s_lo + d, d);
    Acc acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = Acc{0, 0, 0, 0};
    for (int s = s_lo; s < s_hi; s += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (s + d >= s_hi) break;
#pragma unroll
        for (int l = 0; l < L; ++l) *(v4i*)(st + (8 * l + drow) * 128 + ((dpos ^ drow) * 16)) = wb[d][l];
        __builtin_amdgcn_wave_barrier();
        const int row = ROWS == 16 ? r : rr;  // (eight rows: twice)
        const v4i w0 = *(const v4i*)(st + row * 128 + ((g ^ rr) * 16));
        const v4i w1 = *(const v4i*)(st + row * 128 + (((4 + g) ^ rr) * 16));
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          if (16 * j >= cnt) break;
          moe_mfma<OP>(acc[j], w0, w1, xb[d][j][0], xb[d][j][1]);
        }
        if (s + d + D < s_hi) fetch(s + d + D, d);
      }
    }
    if (ROWS == 16 || g < 2) {
      const v4f sc = *(const v4f*)(a.s2 + (int64_t)e * a.K + n0 + 4 * g);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (16 * j + r >= cnt) break;
        const int pos = off + 16 * j + r;
        const float c = a.weight[pos] * a.hs[pos];
        v4f* sum = (v4f*)&sums[wave][a.token[pos]][4 * g];
        v4f v = *sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fmaf_rn((float)acc[j][i], c * sc[i], v[i]);
        *sum = v;
      }
    }
    at += s_hi - s_lo;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * ROWS; i += 512) {
    const int t = i / ROWS, n = i % ROWS;
    float v = sums[0][t][n];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += sums[w][t][n];
    const int64_t to_at = t * a.ldy + n0 + n;
    if (a.y_dtype == FMSMO_F16) ((u16*)a.y)[to_at] = f32_to_f16(v);
    else if (a.y_dtype == FMSMO_BF16) ((u16*)a.y)[to_at] = f32_to_bf16(v);
    else ((float*)a.y)[to_at] = v;
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();

static bool moe_sizes(int64_t T, int64_t E, int top, int64_t K, int64_t I) {
  return T >= 0 && T <= MOE_TOKENS && E >= 1 && E <= MOE_EXPERTS && top >= 1 && top <= MOE_TOP && top <= E && K >= 16 && I >= 16 && K % 16 == 0 &&
         I % 16 == 0 && K < 1 << 20 && I < 1 << 20;
}
// bytes up to each piece of the workspace: counts, entries, tokens, shares, scales, h, codes
struct MoeSpace {
  int64_t entry, token, weight, hs, h, hq, all;
};
static MoeSpace moe_space(int64_t T, int64_t E, int top, int64_t I) {
  const int64_t P = T * top, p16 = (P + 3) / 4 * 16;
  MoeSpace s;
  s.entry = 16;
  s.token = s.entry + 16 * E;
  s.weight = s.token + p16;
  s.hs = s.weight + p16;
  s.h = s.hs + p16;
  s.hq = s.h + 4 * P * I;
  s.all = s.hq + P * I;
  return s;
}

extern "C" int64_t fmsmo_moe_few_workspace_bytes(int64_t T, int64_t E, int top, int64_t K, int64_t I) {
  return moe_sizes(T, E, top, K, I) && T ? moe_space(T, E, top, I).all : 0;
}

template <int OP, int MT>
static void run_moe(const MoeArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(moe_route_kernel, dim3(1), dim3(1024), 0, s, a);
  // experts that may be chosen, at most; a wave to a unit where that gives every SIMD two of them
  const int64_t units = (int64_t)std::min(a.E, a.T * a.top) * (a.I / 8);
  if (units >= 2048) hipLaunchKernelGGL((moe_up_kernel<OP, MT, 1, 4>), dim3(512), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((moe_up_kernel<OP, MT, 4, 4>), dim3((unsigned)std::min<int64_t>(units, 1024)), dim3(256), 0, s, a);
  hipLaunchKernelGGL((moe_quant_kernel<OP>), dim3((unsigned)(a.T * a.top)), dim3(256), 0, s, a);
  if (a.K / 16 >= 256) hipLaunchKernelGGL((moe_down_kernel<OP, MT, 16, 4>), dim3((unsigned)(a.K / 16)), dim3(512), 0, s, a);
  else hipLaunchKernelGGL((moe_down_kernel<OP, MT, 8, 4>), dim3((unsigned)(a.K / 8)), dim3(512), 0, s, a);
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
  if (off(a) || off(w13) || off(w2) || off(w2_scale) || off(workspace) || (T > 1 && lda % 16)) return FMSMO_ERR_ALIGN;
  const MoeSpace sp = moe_space(T, E, top, I);
  if (workspace_bytes < sp.all) return FMSMO_ERR_SCRATCH;
  char* ws = (char*)workspace;
  MoeArgs g{(const uint8_t*)a, a_scale, logits, (const uint8_t*)w13, w13_scale, (const uint8_t*)w2, w2_scale, y, lda, ldl, ldy,
            a_scale_n == 1 ? 0 : 1, logits_dtype, y_dtype, (int)T, (int)E, top, (int)K, (int)I, renormalize != 0,
            (int*)ws, (MoeEntry*)(ws + sp.entry), (int*)(ws + sp.token), (float*)(ws + sp.weight), (float*)(ws + sp.h), (float*)(ws + sp.hs),
            (uint8_t*)(ws + sp.hq)};
  const auto tiles = [&](auto op) {
    constexpr int OP = decltype(op)::value;
    if (T <= 16) run_moe<OP, 1>(g, (hipStream_t)stream);
    else if (T <= 32) run_moe<OP, 2>(g, (hipStream_t)stream);
    else run_moe<OP, 4>(g, (hipStream_t)stream);
  };
  if (codes == FMSMO_OP_I8) tiles(std::integral_constant<int, FMSMO_OP_I8>{});
  else tiles(std::integral_constant<int, FMSMO_OP_E4M3>{});
  return fmsmo_check_launch();
}

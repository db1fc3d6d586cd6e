// Norm, rotation and store of new tokens: q and k normalized per head and rotated by their position in one pass, q written
// beside the input, k and v into the pages of the cache -- in its 16-bit type, or as e4m3 codes with a scale per token and head.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (heads with a norm weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)   (the first `rotary` elements, in pairs (i, i + rotary / 2) or (2i, 2i + 1))
//   16 bit: rounded once.   e4m3: s = max(max|y| / 448, 1e-12), code = e4m3(clamp(y / s, +-448)) of the fp32 y.
//
// Everything is fp32 between the load and the one rounding.  The scale and the quotient are those of IEEE divisions: the recipe of
// the linears' dynamic per-token quantizer.
#include "paged_kv.hpp"

#include <type_traits>

namespace fmsmo {

struct StoreArgs {
  PagedArgs p;  // q: the input queries, out: the rotated ones; k, v: the cache
  const char* xk;
  const char* xv;
  int64_t xk_row, xk_head, xv_row, xv_head;  // bytes
  const void* qw;
  const void* kw;
  float eps;
  const float* cos;
  const float* sin;
  int table_rows, half;  // rotary / 2
  int heads;             // of q
};

// eight elements of 16 bits
template <int T>
__device__ __forceinline__ void widen8(v4i u, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = T == FMSMO_F16 ? f16_to_f32((u16)u[i]) : __uint_as_float((uint32_t)u[i] << 16);
    x[2 * i + 1] = T == FMSMO_F16 ? f16_to_f32((u16)((uint32_t)u[i] >> 16)) : __uint_as_float((uint32_t)u[i] & 0xffff0000u);
  }
}
template <int WT>
__device__ __forceinline__ void load_weight(const void* w, int piece, float* x) {
  if constexpr (WT == FMSMO_F32) {
    const v4f a = ((const v4f*)w)[2 * piece], b = ((const v4f*)w)[2 * piece + 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    widen8<WT>(((const v4i*)w)[piece], x);
  }
}

// over the LG lanes that hold a row, the same result in all of them: moves inside rows of 16 lanes, then one between rows
#define FMSMO_DPP(v, ctrl) __builtin_amdgcn_update_dpp((int)(v), (int)(v), ctrl, 0xf, 0xf, false)
template <int LG>
__device__ __forceinline__ float sum_lanes(float v) {
  v += __int_as_float(FMSMO_DPP(__float_as_int(v), 0xb1));   // quad_perm [1,0,3,2]
  v += __int_as_float(FMSMO_DPP(__float_as_int(v), 0x4e));   // quad_perm [2,3,0,1]
  v += __int_as_float(FMSMO_DPP(__float_as_int(v), 0x141));  // row_half_mirror
  if constexpr (LG >= 16) v += __int_as_float(FMSMO_DPP(__float_as_int(v), 0x140));  // row_mirror
  if constexpr (LG >= 32) v = sum_x16(v);
  return v;
}
template <int LG>
__device__ __forceinline__ uint32_t max_lanes(uint32_t v) {
  const auto max2 = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = max2(v, (uint32_t)FMSMO_DPP(v, 0xb1));
  v = max2(v, (uint32_t)FMSMO_DPP(v, 0x4e));
  v = max2(v, (uint32_t)FMSMO_DPP(v, 0x141));
  if constexpr (LG >= 16) v = max2(v, (uint32_t)FMSMO_DPP(v, 0x140));
  if constexpr (LG >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max2(r[0], r[1]);
  }
  return v;
}
#undef FMSMO_DPP

// One block per token and `per` groups of heads, one lane per eight elements of a row: the token, its position, its angles and its
// page are the same for the whole block, and a row's sums stay inside a wave.  The other half of a pair is loaded again (it is
// in the cache lines that the row's lanes just fetched) instead of being passed between lanes.  Bound by the latency of a token's
// chain of loads (sequence, length, page, row), so where tokens are many a block goes through all of its heads, the next group's rows on
// their way meanwhile: 4 uneven prompts of up to 4095 tokens, 32 + 8 + 8 heads of 128, e4m3: 79 us, 105 with a block per group of heads.
// It pays from about 768 tokens on: 512 tokens 6.9 us so and 6.6 with a block per group, 1024 tokens 9.7 and 11.1.  With the quotients and
// the norm below (IEEE divisions before) the prompts take 75 us: 262 MB in and out, 3.5 TB/s, a large copy reaches 4.9.  A few tokens are
// the launch: 3 us on the device for one.  Tried without gain: the first rows asked for before the sequence is looked up (79), weights and
// angles multiplied once for all heads of a kind and places counted on from head to head (104: more registers, longer before the first
// row), the blocks' part of the places by the scalar unit (81: 78 registers, six waves per SIMD instead of seven), eight waves (111: spills).
template <int T, bool E4M3, int D, int WT, bool INTERLEAVED>
__global__ __launch_bounds__(256) void kv_store_kernel(StoreArgs a, int per) {
  constexpr int LG = D / 8, ROWS = 256 / LG;
  const PagedArgs& p = a.p;
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  // the token's sequence: as many as start at or before it
  int b = t;
  const int h0 = blockIdx.y * per * ROWS + threadIdx.x / LG, c = threadIdx.x % LG;
  const int kv = p.kv_heads, all = a.heads + 2 * kv;
  const auto none = [&] {  // a row of no sequence
    if (!p.zero_rest) return;
    for (int h = h0; h < h0 + per * ROWS && h < a.heads; h += ROWS) *(v4i*)(p.out + t * p.o_row + h * p.o_head + c * 16) = v4i{0, 0, 0, 0};
  };
  if (p.starts) {
    int before = 0;
    for (int i = 0; i < p.seqs; i += 64) {
      const bool yes = i + lane < p.seqs && p.starts[i + lane] <= t;
      before += __popcll(__ballot(yes));
    }
    b = uniform(before) - 1;
    if (b < 0) return none();
  }
  const Seq s = seq_of(p, b);
  if ((unsigned)t - (unsigned)s.row0 >= (unsigned)s.n) return none();  // (before the first one, too: descending starts)
  const int pos = s.pos0 + (t - s.row0);
  int page = pos >= 0 && pos < p.cap ? p.table[b * p.table_stride + (pos >> p.page_shift)] : -1;
  if ((unsigned)page >= (unsigned)p.pages) page = -1;
  const int64_t slot = pos & ((1 << p.page_shift) - 1);

  const bool paired = a.cos && 8 * c < 2 * a.half;  // this lane's piece is turned
  const bool far = paired && pos >= a.table_rows;   // by a position that the tables don't hold
  const bool first = 8 * c < a.half;
  const int other = first ? c + a.half / 8 : c - a.half / 8;
  // angles: of eight pairs across the halves, or of four neighbours
  constexpr int PAIRS = INTERLEAVED ? 4 : 8;
  float cs[PAIRS], sn[PAIRS];
  if (paired) {
    const int64_t at = (int64_t)(far || pos < 0 ? 0 : pos) * a.half + (INTERLEAVED ? 4 * c : first ? 8 * c : 8 * c - a.half);
#pragma unroll
    for (int i = 0; i < PAIRS; i += 4) {
      const v4f u = *(const v4f*)(a.cos + at + i), v = *(const v4f*)(a.sin + at + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        cs[i + k] = u[k];
        sn[i + k] = INTERLEAVED || !first ? v[k] : -v[k];
      }
    }
  }
  v4i own = {0, 0, 0, 0}, far_half = {0, 0, 0, 0};
  const auto fetch = [&](int h) {
    if (h >= all) return;
    const char* src = h < a.heads        ? p.q + t * p.q_row + h * p.q_head
                      : h < a.heads + kv ? a.xk + t * a.xk_row + (h - a.heads) * a.xk_head
                                         : a.xv + t * a.xv_row + (h - a.heads - kv) * a.xv_head;
    own = *(const v4i*)(src + c * 16);
    if (!INTERLEAVED && paired && h < a.heads + kv) far_half = *(const v4i*)(src + other * 16);
  };
  fetch(h0);
  for (int i = 0; i < per; ++i) {
    const int h = h0 + i * ROWS;
    if (h >= all) break;  // (whole lane groups: the others of a wave go on)
    const int kind = h < a.heads ? 0 : h < a.heads + kv ? 1 : 2;
    const int hh = kind == 0 ? h : kind == 1 ? h - a.heads : h - a.heads - kv;
    const void* w = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
    const bool turn = kind < 2 && paired;
    float x[8], y[8];
    widen8<T>(own, x);
    if (!INTERLEAVED) widen8<T>(far_half, y);
    // (before any of this row's is written: q_out may be q)
    if (i + 1 < per) fetch(h + ROWS);
    float r = 1.0f;  // (multiplied in at the end, once for a pair)
    if (w) {
      float ss = 0.0f, g[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = __fmaf_rn(x[k], x[k], ss);
      r = rsqrtf(sum_lanes<LG>(ss) * (1.0f / D) + a.eps);
      load_weight<WT>(w, c, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= g[k];
      if (!INTERLEAVED && turn) {
        load_weight<WT>(w, other, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] *= g[k];
      }
    }
    if (turn) {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = x[2 * k], o = x[2 * k + 1];
          x[2 * k] = e * cs[k] - o * sn[k];
          x[2 * k + 1] = o * cs[k] + e * sn[k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __fmaf_rn(x[k], cs[k], y[k] * sn[k]);
      }
      if (far) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __builtin_nanf("");
      }
    }
    if (w) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= r;
    }
    if (kind == 0) {
      v4i o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = pos < 0 ? 0 : (int)pack2<T>(x[2 * k], x[2 * k + 1]);
      *(v4i*)(p.out + t * p.o_row + hh * p.o_head + c * 16) = o;
      continue;
    }
    float scale = 1.0f;
    if constexpr (E4M3) {
      uint32_t m = 0;  // (as integers: a NaN is larger than everything)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t u = __float_as_uint(x[k]) & 0x7fffffffu;
        m = m > u ? m : u;
      }
      scale = __uint_as_float(max_lanes<LG>(m)) / 448.0f;
      scale = scale < 1e-12f ? 1e-12f : scale;
    }
    if (page < 0) continue;
    char* to = kind == 1 ? (char*)p.k + page * p.k_page + hh * p.k_head + slot * p.k_slot
                         : (char*)p.v + page * p.v_page + hh * p.v_head + slot * p.v_slot;
    if constexpr (E4M3) {
      // x / scale as IEEE division has it: the reciprocal's product and two corrections, each with an exact remainder; zeros, infinities
      // and NaN by the fixup.  No clamp: of a finite row no quotient leaves 448 by more than a rounding.
      const float inverse = 1.0f / scale;
      int lo = 0, hi = 0;
      float q[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        q[k] = x[k] * inverse;
        q[k] = __fmaf_rn(__fmaf_rn(-q[k], scale, x[k]), inverse, q[k]);
        q[k] = __fmaf_rn(__fmaf_rn(-q[k], scale, x[k]), inverse, q[k]);
        q[k] = __builtin_amdgcn_div_fixupf(q[k], scale, x[k]);
      }
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
      *(int2*)(to + c * 8) = make_int2(lo, hi);
      if (c == 0) {
        if (kind == 1) ((float*)p.ks)[page * p.ks_page + hh * p.ks_head + slot] = scale;
        else ((float*)p.vs)[page * p.vs_page + hh * p.vs_head + slot] = scale;
      }
    } else {
      v4i o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = (int)pack2<T>(x[2 * k], x[2 * k + 1]);
      *(v4i*)(to + c * 16) = o;
    }
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();
int fmsmo_paged_args(const fmsmo_kv_cache_t* cache, const fmsmo_kv_batch_t* batch, const void* q, int64_t q_row, int64_t q_head,
                     int q_heads, int dtype, void* out, int64_t o_row, int64_t o_head, int64_t rows, PagedArgs* to);

template <int T, bool E4M3, int D, int WT>
static void run_store(const StoreArgs& a, bool interleaved, int64_t rows, hipStream_t s) {
  // groups of 2048 elements; a block takes all of them where there are blocks enough without (figures at the kernel)
  const int groups = div_up(a.heads + 2 * a.p.kv_heads, 2048 / D), per = rows >= 768 ? (groups < 8 ? groups : 8) : 1;
  const dim3 grid((unsigned)rows, (unsigned)div_up(groups, per));
  if (interleaved) hipLaunchKernelGGL((kv_store_kernel<T, E4M3, D, WT, true>), grid, dim3(256), 0, s, a, per);
  else hipLaunchKernelGGL((kv_store_kernel<T, E4M3, D, WT, false>), grid, dim3(256), 0, s, a, per);
}

extern "C" int fmsmo_kv_store(const fmsmo_kv_cache_t* cache, const fmsmo_kv_batch_t* batch, int dtype, int64_t rows, int q_heads,
                              const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                              const void* v, int64_t v_row, int64_t v_head, void* q_out, int64_t o_row, int64_t o_head,
                              const void* q_weight, const void* k_weight, int weight_dtype, float eps, const float* cos,
                              const float* sin, int64_t table_rows, int rotary, int interleaved, int zero_rest,
                              fmsmo_stream_t stream) {
  StoreArgs a{};
  const int rc = fmsmo_paged_args(cache, batch, q, q_row, q_head, q_heads, dtype, q_out, o_row, o_head, rows, &a.p);
  if (rc) return rc;
  if (!k || !v) return FMSMO_ERR_NULL;
  if (rotary < 0 || rotary > cache->dim || table_rows < 0 || table_rows > 0x7fffffff) return FMSMO_ERR_SHAPE;
  if (rotary && (!cos || !sin)) return FMSMO_ERR_NULL;
  if (rotary && table_rows < 1) return FMSMO_ERR_SHAPE;
  if (rotary % 16) return FMSMO_ERR_UNSUPPORTED;
  if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != FMSMO_F32) return FMSMO_ERR_UNSUPPORTED;
  const auto off = [](const void* x) { return (((uintptr_t)x) & 15) != 0; };
  if (off(k) || off(v) || off(cos) || off(sin) || off(q_weight) || off(k_weight) || k_row % 8 || k_head % 8 || v_row % 8 || v_head % 8)
    return FMSMO_ERR_ALIGN;
  if (k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0) return FMSMO_ERR_SHAPE;
  if (q_heads + 2 * cache->heads > 65535) return FMSMO_ERR_UNSUPPORTED;
  if (rows == 0 || batch->seqs == 0) return FMSMO_OK;
  a.xk = (const char*)k;
  a.xv = (const char*)v;
  a.xk_row = 2 * k_row;
  a.xk_head = 2 * k_head;
  a.xv_row = 2 * v_row;
  a.xv_head = 2 * v_head;
  a.qw = q_weight;
  a.kw = k_weight;
  a.eps = eps;
  a.cos = rotary ? cos : nullptr;
  a.sin = sin;
  a.table_rows = (int)table_rows;
  a.half = rotary / 2;
  a.heads = q_heads;
  a.p.zero_rest = zero_rest && batch->query_start;
  const bool f32w = (q_weight || k_weight) && weight_dtype == FMSMO_F32;
  const auto go = [&](auto t, auto e, auto d) {
    constexpr int T = decltype(t)::value, D = decltype(d)::value;
    constexpr bool E = decltype(e)::value;
    if (f32w) run_store<T, E, D, FMSMO_F32>(a, interleaved != 0, rows, (hipStream_t)stream);
    else run_store<T, E, D, T>(a, interleaved != 0, rows, (hipStream_t)stream);
  };
  const auto dims = [&](auto t, auto e) {
    if (cache->dim == 64) go(t, e, std::integral_constant<int, 64>{});
    else if (cache->dim == 128) go(t, e, std::integral_constant<int, 128>{});
    else go(t, e, std::integral_constant<int, 256>{});
  };
  const auto types = [&](auto t) {
    if (cache->dtype == FMSMO_KV_E4M3) dims(t, std::true_type{});
    else dims(t, std::false_type{});
  };
  if (dtype == FMSMO_F16) types(std::integral_constant<int, FMSMO_F16>{});
  else types(std::integral_constant<int, FMSMO_BF16>{});
  return fmsmo_check_launch();
}

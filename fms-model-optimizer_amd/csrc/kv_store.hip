// Norm, rotation and store of new tokens: q and k normalized per head and rotated by their position in one pass, q written
// beside the input, k and v into the pages of the cache -- in its 16-bit type, or as e4m3 codes with a scale per token and head.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (heads with a norm weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)   (the first `rotary` elements, in pairs (i, i + rotary / 2) or (2i, 2i + 1))
//   16 bit: rounded once.   e4m3: s = max(max|y| / 448, 1e-12), code = e4m3(clamp(y / s, +-448)) of the fp32 y.
//
// Everything is fp32 between the load and the one rounding.  The scale and the quotient are IEEE divisions: the recipe of
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

__device__ __forceinline__ void load8(const char* p, int dt, float* x) {
  const v4i u = *(const v4i*)p;
  if (dt == FMSMO_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = f16_to_f32((u16)u[i]);
      x[2 * i + 1] = f16_to_f32((u16)((uint32_t)u[i] >> 16));
    }
  } else if (dt == FMSMO_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float((uint32_t)u[i] << 16);
      x[2 * i + 1] = __uint_as_float((uint32_t)u[i] & 0xffff0000u);
    }
  } else {
    const v4i w = *(const v4i*)(p + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __int_as_float(u[i]);
      x[4 + i] = __int_as_float(w[i]);
    }
  }
}

// over the LG lanes that hold a row
template <int LG>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = 1; o < LG; o *= 2) v += __shfl_xor(v, o);
  return v;
}
template <int LG>
__device__ __forceinline__ uint32_t max_lanes(uint32_t v) {
#pragma unroll
  for (int o = 1; o < LG; o *= 2) {
    const uint32_t w = __shfl_xor(v, o);
    v = v > w ? v : w;
  }
  return v;
}

// One block per token and group of heads, one lane per eight elements of a row: the token, its position and its page are
// the same for the whole block, and a row's sums stay inside a wave.  The other half of a pair is loaded again (it is
// in the cache lines that the row's lanes just fetched) instead of being passed between lanes.
template <int T, bool E4M3, int D, int WT, bool INTERLEAVED>
__global__ __launch_bounds__(256) void kv_store_kernel(StoreArgs a) {
  constexpr int LG = D / 8, ROWS = 256 / LG;
  const PagedArgs& p = a.p;
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  // the token's sequence: as many as start at or before it
  int b = t;
  const int h = blockIdx.y * ROWS + threadIdx.x / LG, c = threadIdx.x % LG;
  const auto none = [&] {  // a row of no sequence
    if (p.zero_rest && h < a.heads) *(v4i*)(p.out + t * p.o_row + h * p.o_head + c * 16) = v4i{0, 0, 0, 0};
  };
  if (p.starts) {
    int before = 0;
    for (int c = 0; c < p.seqs; c += 64) {
      const bool yes = c + lane < p.seqs && p.starts[c + lane] <= t;
      before += __popcll(__ballot(yes));
    }
    b = uniform(before) - 1;
    if (b < 0) return none();
  }
  const Seq s = seq_of(p, b);
  if (t >= s.row0 + s.n) return none();
  const int pos = s.pos0 + (t - s.row0);

  const int kv = p.kv_heads;
  if (h >= a.heads + 2 * kv) return;  // (whole lane groups: the others of a wave go on)
  const int kind = h < a.heads ? 0 : h < a.heads + kv ? 1 : 2;
  const int hh = kind == 0 ? h : kind == 1 ? h - a.heads : h - a.heads - kv;
  const char* src = kind == 0 ? p.q + t * p.q_row + hh * p.q_head
                  : kind == 1 ? a.xk + t * a.xk_row + hh * a.xk_head
                              : a.xv + t * a.xv_row + hh * a.xv_head;
  const void* w = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
  float x[8];
  load8(src + c * 16, T, x);
  const bool turn = kind < 2 && a.cos && 8 * c < 2 * a.half;
  const bool far = turn && pos >= a.table_rows;  // a position that the tables don't hold
  const int other = 8 * c < a.half ? c + a.half / 8 : c - a.half / 8;
  float y[8];
  if (!INTERLEAVED && turn) load8(src + other * 16, T, y);
  if (w) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
    const float r = 1.0f / sqrtf(sum_lanes<LG>(ss) * (1.0f / D) + a.eps);
    constexpr int WB = WT == FMSMO_F32 ? 4 : 2;
    float g[8];
    load8((const char*)w + c * 8 * WB, WT, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * g[i];
    if (!INTERLEAVED && turn) {
      load8((const char*)w + other * 8 * WB, WT, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * r * g[i];
    }
  }
  if (turn) {
    const int at = far || pos < 0 ? 0 : pos;
    const float* cs = a.cos + (int64_t)at * a.half;
    const float* sn = a.sin + (int64_t)at * a.half;
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = cs[4 * c + i], v = sn[4 * c + i], e = x[2 * i], o = x[2 * i + 1];
        x[2 * i] = e * u - o * v;
        x[2 * i + 1] = o * u + e * v;
      }
    } else {
      const bool first = 8 * c < a.half;
      const int i0 = first ? 8 * c : 8 * c - a.half;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = cs[i0 + i], v = sn[i0 + i];
        x[i] = first ? x[i] * u - y[i] * v : x[i] * u + y[i] * v;
      }
    }
  }
  if (far) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
  }
  if (kind == 0) {
    v4i o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pos < 0 ? 0 : (int)pack2<T>(x[2 * i], x[2 * i + 1]);
    *(v4i*)(p.out + t * p.o_row + hh * p.o_head + c * 16) = o;
    return;
  }
  float scale = 1.0f;
  if constexpr (E4M3) {
    uint32_t m = 0;  // (as integers: a NaN is larger than everything)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
      m = m > u ? m : u;
    }
    scale = __uint_as_float(max_lanes<LG>(m)) / 448.0f;
    scale = scale < 1e-12f ? 1e-12f : scale;
  }
  if (pos < 0 || pos >= p.cap) return;
  const int page = p.table[b * p.table_stride + (pos >> p.page_shift)], slot = pos & ((1 << p.page_shift) - 1);
  if ((unsigned)page >= (unsigned)p.pages) return;
  char* to = kind == 1 ? (char*)p.k + page * p.k_page + hh * p.k_head + (int64_t)slot * p.k_slot
                       : (char*)p.v + page * p.v_page + hh * p.v_head + (int64_t)slot * p.v_slot;
  if constexpr (E4M3) {
    int lo = 0, hi = 0;
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[i] = x[i] / scale;
      q[i] = q[i] != q[i] ? q[i] : fminf(fmaxf(q[i], -448.0f), 448.0f);
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
    for (int i = 0; i < 4; ++i) o[i] = (int)pack2<T>(x[2 * i], x[2 * i + 1]);
    *(v4i*)(to + c * 16) = o;
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();
int fmsmo_paged_args(const fmsmo_kv_cache_t* cache, const fmsmo_kv_batch_t* batch, const void* q, int64_t q_row, int64_t q_head,
                     int q_heads, int dtype, void* out, int64_t o_row, int64_t o_head, int64_t rows, PagedArgs* to);

template <int T, bool E4M3, int D, int WT>
static void run_store(const StoreArgs& a, bool interleaved, int64_t rows, hipStream_t s) {
  const dim3 grid((unsigned)rows, (unsigned)div_up(a.heads + 2 * a.p.kv_heads, 2048 / D));
  if (interleaved) hipLaunchKernelGGL((kv_store_kernel<T, E4M3, D, WT, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv_store_kernel<T, E4M3, D, WT, false>), grid, dim3(256), 0, s, a);
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

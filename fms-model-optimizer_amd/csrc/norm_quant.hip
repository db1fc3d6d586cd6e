// Residual addition, RMS norm and 8-bit codes of a hidden row in one pass: what stands in front of every 8-bit product of a layer.
//
//   h = x + residual                              (fp32; residual_out = h rounded once)
//   n = h / sqrt(mean(h^2) + eps) * weight        (fp32; normed = n rounded once, where it is wanted)
//   int8: s = max(max|n|, 1e-5) / 127, q = rint(n / s)          e4m3: s = max(max|n| / 448, 1e-12), q = e4m3(n / s)
//   with a scale that is given: q of clamp(n / s) to +-127 or +-448
//
// The recipes are those of the per-token quantizers in fp32, so a product takes these codes as it takes theirs.
#include "quant_math.hpp"

#include <algorithm>
#include <type_traits>

namespace fmsmo {

struct NormArgs {
  const u16* x;
  const u16* residual;  // or NULL
  const void* weight;
  u16* residual_out;    // or NULL
  u16* normed;          // or NULL
  uint8_t* q;
  float* scale;
  int64_t ldx, ldr, ldo, ldn, ldq;
  int64_t rows;
  int K;
  float eps, inv_k;
  int given;  // scale is read
};

__device__ __forceinline__ float wave_sum(float v) {
#define FMSMO_DPP_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, false));
  FMSMO_DPP_ADD(0xb1)   // quad_perm [1,0,3,2]
  FMSMO_DPP_ADD(0x4e)   // quad_perm [2,3,0,1]
  FMSMO_DPP_ADD(0x141)  // row_half_mirror
  FMSMO_DPP_ADD(0x140)  // row_mirror
#undef FMSMO_DPP_ADD
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// eight elements as they lie in memory, and widened
template <int T>
struct Raw {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* p, size_t piece) {
    if constexpr (T == FMSMO_F32) {
      a = ((const uint4*)p)[2 * piece];
      b = ((const uint4*)p)[2 * piece + 1];
    } else {
      a = ((const uint4*)p)[piece];
    }
  }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
    if constexpr (T == FMSMO_F32) {
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = __uint_as_float(u[i]);
        v[4 + i] = __uint_as_float(w[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = cvt16<T>((u16)(u[i] & 0xffff));
        v[2 * i + 1] = cvt16<T>((u16)(u[i] >> 16));
      }
    }
  }
};
// h of eight elements
template <int T>
__device__ __forceinline__ void sum_h(const NormArgs& a, const Raw<T>& x, const Raw<T>& r, float (&h)[8]) {
  x.widen(h);
  if (a.residual) {
    float v[8];
    r.widen(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] += v[i];
  }
}
template <int T>
__device__ __forceinline__ void load_h(const NormArgs& a, int64_t row, int c, float (&h)[8]) {
  Raw<T> x, r;
  x.load(a.x + row * a.ldx, c);
  if (a.residual) r.load(a.residual + row * a.ldr, c);
  sum_h<T>(a, x, r, h);
}
template <int T>
__device__ __forceinline__ void put16(u16* at, const float (&v)[8]) {
  *(uint4*)at = make_uint4(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]), pack16<T>(v[6], v[7]));
}
template <int WT>
__device__ __forceinline__ void times_weight(const Raw<WT>& weight, float r, float (&h)[8]) {
  float w[8];
  weight.widen(w);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = __fmul_rn(__fmul_rn(h[i], r), w[i]);
}
__device__ __forceinline__ uint32_t max8(const float (&n)[8], uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(n[i]) & 0x7fffffffu;  // (as integers: a NaN is larger than everything)
    m = m > u ? m : u;
  }
  return m;
}
// n / s as IEEE division has it, for s that is normal: the reciprocal's product and two corrections, each with an exact remainder
__device__ __forceinline__ float quotient(float n, float s, float inverse) {
  float q = n * inverse;
  q = __fmaf_rn(__fmaf_rn(-q, s, n), inverse, q);
  q = __fmaf_rn(__fmaf_rn(-q, s, n), inverse, q);
  return __builtin_amdgcn_div_fixupf(q, s, n);
}
template <bool E4M3>
__device__ __forceinline__ uint2 codes8(const float (&n)[8], float s, float inverse, bool given) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = given ? n[i] / s : quotient(n[i], s, inverse);  // (a given scale may have no reciprocal; 8192 tokens of 4096, int8: 40.9 us, 39.2 else)
    if (given) {
      constexpr float MOST = E4M3 ? 448.0f : 127.0f;
      q[i] = q[i] > MOST ? MOST : q[i] < -MOST ? -MOST : q[i];  // (a NaN stays)
    }
  }
  uint2 o;
  if constexpr (E4M3) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    o.x = (uint32_t)lo;
    o.y = (uint32_t)hi;
  } else {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(q[i] + 12582912.0f);  // rint in the low mantissa bits (1.5 * 2^23)
    o.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u), __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), 0x05040100u);
    o.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[7], c[6], 0x0c0c0400u), __builtin_amdgcn_perm(c[5], c[4], 0x0c0c0400u), 0x05040100u);
  }
  return o;
}
template <bool E4M3>
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float m = __uint_as_float(top);
  if constexpr (E4M3) {
    const float s = m / 448.0f;
    return s < 1e-12f ? 1e-12f : s;  // (a NaN stays)
  } else {
    return (m < 1e-5f ? 1e-5f : m) / 127.0f;
  }
}

// NW waves a row, CH pieces of eight elements a lane, held in registers between the sum and the codes; a block of one-wave rows takes four.
// CH = 0: rows longer than that, read three times, twice with a scale that is given (4096 tokens of 16392 118 us and 104, floor 96; of 16384 87).
template <int T, int WT, bool E4M3, int NW, int CH>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void norm_quant_kernel(NormArgs a) {
  constexpr int NT = NW * 64, HELD = CH ? CH : 1;
  __shared__ float sums[NW];
  __shared__ uint32_t tops[NW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
  if (NW == 1 && row >= a.rows) return;  // (no barrier follows in this form)
  const int at = NW == 1 ? lane : (int)threadIdx.x, pieces = a.K / AQ_VEC;
  float h[HELD][8];
  float ss = 0.0f;
  Raw<WT> w[HELD];
  const auto add_squares = [&](const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = __fmaf_rn(v[k], v[k], ss);
  };
  if constexpr (CH > 0) {
    // all loads at once, the weight's too; a lane past the row's end loads the last piece again (a branch around a load makes the
    // others wait for it: one token of 4096 3.6 us so, 2.5 with one piece a lane and no branch taken)
    Raw<T> x[CH], res[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) x[i].load(a.x + row * a.ldx, min(at + i * NT, pieces - 1));
    if (a.residual) {
#pragma unroll
      for (int i = 0; i < CH; ++i) res[i].load(a.residual + row * a.ldr, min(at + i * NT, pieces - 1));
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) w[i].load(a.weight, min(at + i * NT, pieces - 1));
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      sum_h<T>(a, x[i], res[i], h[i]);
      if (at + i * NT >= pieces) {
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i][k] = 0.0f;
      }
      add_squares(h[i]);
    }
  } else {
    for (int c = at; c < pieces; c += NT) {
      load_h<T>(a, row, c, h[0]);
      add_squares(h[0]);
    }
  }
  ss = wave_sum(ss);
  if constexpr (NW > 1) {
    if (lane == 0) sums[wave] = ss;
    __syncthreads();
    ss = sums[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) ss += sums[w];
  }
  const float r = rsqrtf(__fmaf_rn(ss, a.inv_k, a.eps));
  uint32_t top = 0;
  if constexpr (CH > 0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = at + i * NT;
      const bool in = c < pieces;
      if (a.residual_out && in) put16<T>(a.residual_out + row * a.ldo + (size_t)c * AQ_VEC, h[i]);
      times_weight<WT>(w[i], r, h[i]);
      if (a.normed && in) put16<T>(a.normed + row * a.ldn + (size_t)c * AQ_VEC, h[i]);
      if (in) top = max8(h[i], top);
    }
  } else if (!a.given) {
    for (int c = at; c < pieces; c += NT) {
      w[0].load(a.weight, c);
      load_h<T>(a, row, c, h[0]);
      times_weight<WT>(w[0], r, h[0]);
      top = max8(h[0], top);
    }
  }
  float s;
  if (a.given) {
    s = a.scale[0];
  } else {
    top = wave_max_u32(top);
    if constexpr (NW > 1) {
      if (lane == 0) tops[wave] = top;
      __syncthreads();
      top = tops[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = top > tops[w] ? top : tops[w];
    }
    s = scale_of<E4M3>(top);
    if (at == 0) a.scale[row] = s;
  }
  const float inverse = 1.0f / s;
  const bool given = a.given != 0;
  uint8_t* q = a.q + row * a.ldq;
  if constexpr (CH > 0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = at + i * NT;
      if (c < pieces) *(uint2*)(q + (size_t)c * AQ_VEC) = codes8<E4M3>(h[i], s, inverse, given);
    }
  } else {
    for (int c = at; c < pieces; c += NT) {  // (each piece is read by the thread that writes it: residual_out may be x or residual)
      w[0].load(a.weight, c);
      load_h<T>(a, row, c, h[0]);
      if (a.residual_out) put16<T>(a.residual_out + row * a.ldo + (size_t)c * AQ_VEC, h[0]);
      times_weight<WT>(w[0], r, h[0]);
      if (a.normed) put16<T>(a.normed + row * a.ldn + (size_t)c * AQ_VEC, h[0]);
      *(uint2*)(q + (size_t)c * AQ_VEC) = codes8<E4M3>(h[0], s, inverse, given);
    }
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();

template <int T, int WT, bool E4M3>
static void run_norm(const NormArgs& a, hipStream_t s) {
  const auto go = [&](auto nw, auto ch) {
    constexpr int NW = decltype(nw)::value, CH = decltype(ch)::value;
    const dim3 grid((unsigned)(NW == 1 ? div_up(a.rows, 4) : a.rows)), block(NW == 1 ? 256 : NW * 64);
    hipLaunchKernelGGL((norm_quant_kernel<T, WT, E4M3, NW, CH>), grid, block, 0, s, a);
  };
#define GO(nw, ch) go(std::integral_constant<int, nw>{}, std::integral_constant<int, ch>{})
  // Few rows: a piece a lane, which is the shortest way through a row (one token of 4096: 2.4 us, 3.2 with two pieces, 4.3 with four; 64 tokens
  // 3.9, 4.6, 5.8).  Many: two, with which more rows are on their way (8192 tokens 39.5, 37.6, 38.4; 1777 of 12800: 19.8 with two, 18.2 with four).
  const bool many = a.rows >= 1024;
  if (a.K <= 512) GO(1, 1);
  else if (a.K <= 1024) GO(2, 1);
  else if (a.K <= 2048) GO(4, 1);
  else if (a.K <= 4096) {
    if (many) GO(4, 2);
    else GO(8, 1);
  } else if (a.K <= 8192) {
    if (many) GO(8, 2);
    else GO(16, 1);
  } else if (a.K <= 16384) {
    if (many) GO(8, 4);
    else GO(16, 2);
  } else {
    GO(16, 0);
  }
#undef GO
}

extern "C" int fmsmo_add_rms_norm_quant(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                        int weight_dtype, float eps, int codes, int static_scale, void* q, int64_t ldq, float* scale,
                                        void* residual_out, int64_t ldo, void* normed, int64_t ldn, int64_t M, int64_t K,
                                        fmsmo_stream_t stream) {
  if (M < 0 || K < 0) return FMSMO_ERR_SHAPE;
  if (dtype != FMSMO_F16 && dtype != FMSMO_BF16) return FMSMO_ERR_UNSUPPORTED;
  if (weight_dtype != dtype && weight_dtype != FMSMO_F32) return FMSMO_ERR_UNSUPPORTED;
  if (codes != FMSMO_OP_I8 && codes != FMSMO_OP_E4M3) return FMSMO_ERR_UNSUPPORTED;
  if (M == 0 || K == 0) return FMSMO_OK;
  if (!x || !weight || !q || !scale || (residual_out && !residual)) return FMSMO_ERR_NULL;
  if (M > 0x7fffffff || K > 0x7ffffff0) return FMSMO_ERR_UNSUPPORTED;
  const auto row = [&](const void* p, int64_t ld) { return p && M > 1 && ld < K; };
  if (row(x, ldx) || row(residual, ldr) || row(residual_out, ldo) || row(normed, ldn) || row(q, ldq)) return FMSMO_ERR_SHAPE;
  const auto off = [&](const void* p, int64_t ld) { return p && (((uintptr_t)p & 15) || (M > 1 && ld % 8)); };
  if (K % 8 || off(x, ldx) || off(residual, ldr) || off(residual_out, ldo) || off(normed, ldn) || ((uintptr_t)weight & 15) ||
      ((uintptr_t)q & 7) || (M > 1 && ldq % 8) || ((uintptr_t)scale & 3))
    return FMSMO_ERR_ALIGN;
  const auto types = [&](auto t, const NormArgs& a) {
    constexpr int T = decltype(t)::value;
    if (weight_dtype == FMSMO_F32) {
      if (codes == FMSMO_OP_E4M3) run_norm<T, FMSMO_F32, true>(a, (hipStream_t)stream);
      else run_norm<T, FMSMO_F32, false>(a, (hipStream_t)stream);
    } else {
      if (codes == FMSMO_OP_E4M3) run_norm<T, T, true>(a, (hipStream_t)stream);
      else run_norm<T, T, false>(a, (hipStream_t)stream);
    }
  };
  // A launch has fewer than 2^32 threads, and a row up to 1024 of them.
  constexpr int64_t MOST = 1 << 21;
  for (int64_t from = 0; from < M; from += MOST) {
    const NormArgs a{(const u16*)x + from * ldx, residual ? (const u16*)residual + from * ldr : nullptr, weight,
                     residual_out ? (u16*)residual_out + from * ldo : nullptr, normed ? (u16*)normed + from * ldn : nullptr, (uint8_t*)q + from * ldq,
                     static_scale ? scale : scale + from, ldx, ldr, ldo, ldn, ldq, std::min(MOST, M - from), (int)K, eps, 1.0f / (float)K,
                     static_scale != 0};
    if (dtype == FMSMO_F16) types(std::integral_constant<int, FMSMO_F16>{}, a);
    else types(std::integral_constant<int, FMSMO_BF16>{}, a);
  }
  return fmsmo_check_launch();
}

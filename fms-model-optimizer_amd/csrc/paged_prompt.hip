// Attention of many new rows per sequence (prompts, chunks of prompts) over a paged key-value cache.
//
// One block takes 128 rows (tokens x the query heads that share a key head, in that order, so that the keys in shared memory
// serve all of those heads) through the keys that they see, 64 at a time; its four waves hold 32 rows each.
//   S^T = K Q^T   32 x 32 x 16: a lane holds one row's scores for half of the keys in its registers, so the softmax needs one exchange
//                 (lane l with l + 32) for the maximum and none for anything else,
//   O^T = V^T P^T the scores as they stand are the second operand (the reduction's order is free), and what rescales O is a
//                 number per lane.  V^T comes out of row-major shared memory by ds_read_b64_tr_b16.
// Keys and values go through registers into the other of two buffers while the present one is used: the pages are looked up on
// the way, e4m3 codes become 16-bit numbers once per block, and what nobody may see becomes zero.
#include "paged_kv.hpp"

#include <algorithm>
#include <type_traits>

namespace fmsmo {

constexpr int BM = 128, BN = 64;

template <int QT, bool E4M3, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_prompt_kernel(PagedArgs a, int tiles_x) {
  constexpr int PT = E4M3 ? FMSMO_BF16 : QT;  // (see the split kernel: e4m3 scales are multiplied in before the rounding)
  constexpr bool TWO = E4M3 && QT == FMSMO_F16;
  constexpr int QS = D / 16, NV = D / 32;
  // Strides in 16-bit elements.  Keys are read 16 bytes a lane from 32 rows, values four rows by 64 bytes an instruction: 16 and 64
  // bytes more than a row spread both over all banks.
  constexpr int KLD = D + 8, VLD = D + 32;
  constexpr int CH = D * (E4M3 ? 1 : 2) / 16;  // 16-byte chunks of a row
  constexpr int NJ = BN * CH / 256;            // of them per thread
  __shared__ __attribute__((aligned(16))) u16 kl[2][BN * KLD];
  __shared__ __attribute__((aligned(16))) u16 vl[2][BN * VLD];
  __shared__ __attribute__((aligned(16))) float sc[2][2][E4M3 ? BN : 4];
  __shared__ int odd;  // values of a tile that some rows see in part held infinities or NaN
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c32 = lane & 31, hl = lane >> 5;

  if (a.zero_rest) zero_rest(a, D / 8);
  // the tile of rows: sequence b's start at tile query_start[b] group / BM + b, which leaves room for all of them
  const int hk = blockIdx.x % a.kv_heads, x = tiles_x - 1 - blockIdx.x / a.kv_heads;
  int before = 0;
  for (int c = 0; c < a.seqs; c += 64) {
    bool yes = false;
    if (c + lane < a.seqs) {
      const int r0 = a.starts ? a.starts[c + lane] : c + lane;
      yes = r0 >= 0 && r0 <= a.rows && (int64_t)r0 * a.group / BM + c + lane <= x;
    }
    before += __popcll(__ballot(yes));
  }
  const int b = uniform(before) - 1;
  if (b < 0) return;
  const Seq s = seq_of(a, b);
  const int r0 = (x - (int)((int64_t)s.row0 * a.group / BM) - b) * BM;
  if (s.n == 0 || r0 < 0 || r0 >= s.n * a.group) return;
  const int nrows = s.n * a.group - r0 < BM ? s.n * a.group - r0 : BM;
  const int p_lo = s.pos0 + r0 / a.group, p_hi = s.pos0 + (r0 + nrows - 1) / a.group;
  const Tiles t = tiles_of<BN>(a, s.len, p_lo, p_hi);
  // this wave's rows
  const int wr = wave * 32, wn = nrows - wr < 32 ? nrows - wr : 32;
  const bool mine = wr + c32 < nrows;
  const int row = r0 + wr + c32, tok = mine ? row / a.group : 0, head = hk * a.group + (mine ? row - tok * a.group : 0);
  const int pos = mine ? s.pos0 + tok : -1;
  const int w_lo = s.pos0 + (r0 + wr) / a.group, w_hi = wn > 0 ? s.pos0 + (r0 + wr + wn - 1) / a.group : w_lo;
  v4i q[QS];
  {
    const char* src = a.q + (s.row0 + tok) * a.q_row + head * a.q_head;
#pragma unroll
    for (int k = 0; k < QS; ++k) q[k] = mine ? *(const v4i*)(src + (k * 16 + hl * 8) * 2) : v4i{0, 0, 0, 0};
  }
  v16f o[NV];
#pragma unroll
  for (int d = 0; d < NV; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m = -__builtin_inff(), l = 0.0f;

  const auto key_of = [&](int tile) { return (tile < t.sink_tiles ? tile : tile + t.skip) * BN; };
  const int in_page = (1 << a.page_shift) - 1;
  const int* table = a.table + b * a.table_stride;
  // lane i holds the page of the tile's i-th 16 keys; -1: not there
  const auto pages_of = [&](int tile) {
    const int k = key_of(tile) + 16 * (lane & 3);
    int pg = tile < t.count && k < s.len ? table[k >> a.page_shift] : -1;
    return (unsigned)pg < (unsigned)a.pages ? pg : -1;
  };
  v4i kr[NJ], vr[NJ];
  float sr = 0.0f;
  const auto load = [&](int tile, int pgs) {
    const int k0 = key_of(tile);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int at = threadIdx.x + 256 * j, r = at / CH, ch = at % CH;
      const int sub = uniform(r >> 4), page = __builtin_amdgcn_readlane(pgs, sub);
      kr[j] = vr[j] = v4i{0, 0, 0, 0};
      if (page >= 0 && k0 + r < s.len) {  // (anything else has to read as zero: 0 * NaN is not 0)
        const int64_t slot = (k0 + r) & in_page;
        kr[j] = *(const v4i*)(a.k + page * a.k_page + hk * a.k_head + slot * a.k_slot + ch * 16);
        vr[j] = *(const v4i*)(a.v + page * a.v_page + hk * a.v_head + slot * a.v_slot + ch * 16);
      }
    }
    if constexpr (E4M3) {
      if (wave < 2) {  // one lane per key: wave 0 the scales of the keys, wave 1 those of the values
        const int page = __shfl(pgs, lane >> 4), slot = (k0 + lane) & in_page;
        sr = 0.0f;
        if (page >= 0 && k0 + lane < s.len)
          sr = wave == 0 ? a.ks[page * a.ks_page + hk * a.ks_head + slot] * a.c : a.vs[page * a.vs_page + hk * a.vs_head + slot];
      }
    }
  };
  const auto put = [&](int buf, bool look) {
    uint32_t fine = 0x80008000u;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int at = threadIdx.x + 256 * j, r = at / CH, ch = at % CH;
      if constexpr (E4M3) {
        uint32_t y[8], z[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          widen4<QT>((uint32_t)kr[j][i], y[2 * i], y[2 * i + 1]);
          widen4<PT>((uint32_t)vr[j][i], z[2 * i], z[2 * i + 1]);
        }
        __builtin_memcpy(&kl[buf][r * KLD + ch * 16], y, 32);
        __builtin_memcpy(&vl[buf][r * VLD + ch * 16], z, 32);
        if (look) {
#pragma unroll
          for (int i = 0; i < 8; ++i) fine &= finite2<PT>(z[i]);
        }
      } else {
        *(v4i*)&kl[buf][r * KLD + ch * 8] = kr[j];
        *(v4i*)&vl[buf][r * VLD + ch * 8] = vr[j];
        if (look) {
#pragma unroll
          for (int i = 0; i < 4; ++i) fine &= finite2<PT>((uint32_t)vr[j][i]);
        }
      }
    }
    if constexpr (E4M3) {
      if (wave < 2) sc[buf][wave][lane] = sr;
    }
    if (look && __any(fine != 0x80008000u) && lane == 0) odd = 1;
  };
  // a tile that some rows see in part
  const auto partial = [&](int tile) {
    const int k0 = key_of(tile);
    return !(k0 + BN <= s.len && sees_all(a, p_lo, p_hi, k0, k0 + BN - 1));
  };

  if (threadIdx.x == 0) odd = 0;
  __syncthreads();
  int pgs = pages_of(0), pgs_next = pages_of(1);
  uint64_t there = 0;
  if (t.count > 0) {
    load(0, pgs);
    put(0, partial(0));
  }
  there = __ballot(pgs >= 0) & 15;
  __syncthreads();
  for (int tile = 0; tile < t.count; ++tile) {
    const int buf = tile & 1, k0 = key_of(tile);
    const bool whole = there == 15 && k0 + BN <= s.len && sees_all(a, w_lo, w_hi, k0, k0 + BN - 1);
    const uint64_t there_now = there;
    const bool more = tile + 1 < t.count;
    if (more) {
      pgs = pgs_next;
      there = __ballot(pgs >= 0) & 15;
      load(tile + 1, pgs);
      pgs_next = pages_of(tile + 2);
    }
    // S^T
    v16f st[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kt][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < QS; ++k)
        st[kt] = mfma32<QT>(*(const v4i*)&kl[buf][(kt * 32 + c32) * KLD + k * 16 + hl * 8], q[k], st[kt]);
    }
    // register 4 i + j of st[kt]: key kt * 32 + 8 i + 4 hl + j
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (E4M3) {
          const v4f ks = *(const v4f*)&sc[buf][0][kt * 32 + 8 * i + 4 * hl];
#pragma unroll
          for (int j = 0; j < 4; ++j) st[kt][4 * i + j] *= ks[j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) st[kt][4 * i + j] *= a.c;
        }
      }
    if (!whole) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = kt * 32 + 8 * (i / 4) + 4 * hl + i % 4, key = k0 + at;
          const bool in = (there_now >> (at >> 4) & 1) && key < s.len && sees(a, pos, key);
          st[kt][i] = in ? st[kt][i] : -__builtin_inff();
        }
    }
    float top = st[0][0];
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(st[0][i], st[1][i]));
    top = max_x32(top);
    const float m_new = fmaxf(m, top), ms = safe_max(m_new), f = exp2_hw(m - ms);
    if (__any(m_new > m)) {
#pragma unroll
      for (int d = 0; d < NV; ++d) o[d] *= f;
    }
    l *= f;
    m = m_new;
    v4i pb[4], pl[4];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float pr[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pr[j] = exp2_hw(st[kt][4 * i + j] - ms);
          l += pr[j];
        }
        if constexpr (E4M3) {
          const v4f vs = *(const v4f*)&sc[buf][1][kt * 32 + 8 * i + 4 * hl];
#pragma unroll
          for (int j = 0; j < 4; ++j) pr[j] = whole || st[kt][4 * i + j] != -__builtin_inff() ? pr[j] * vs[j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t hi = pack2<PT>(pr[2 * j], pr[2 * j + 1]);
          pb[kt * 2 + i / 2][i % 2 * 2 + j] = (int)hi;
          if constexpr (TWO)
            pl[kt * 2 + i / 2][i % 2 * 2 + j] = (int)pack2<PT>(pr[2 * j] - __uint_as_float(hi << 16), pr[2 * j + 1] - __uint_as_float(hi & 0xffff0000u));
        }
      }
    // O^T: step k of the reduction has keys 16 k + 4 hl + (0..3) and those + 8, as the scores lie
    const auto values = [&](int d, int k) {
      const int l16 = lane & 15, r = 16 * k + 4 * hl + l16 / 4, col = d * 32 + (lane >> 4 & 1) * 16 + l16 % 4 * 4;
      const s4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)&vl[buf][r * VLD + col]);
      const s4v w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)&vl[buf][(r + 8) * VLD + col]);
      v4i f;
      __builtin_memcpy(&f, &u, 8);
      __builtin_memcpy((char*)&f + 8, &w, 8);
      return f;
    };
    if (whole || !uniform(odd)) {
#pragma unroll
      for (int d = 0; d < NV; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const v4i f = values(d, k);
          o[d] = mfma32<PT>(f, pb[k], o[d]);
          if constexpr (TWO) o[d] = mfma32<PT>(f, pl[k], o[d]);
        }
    } else {
      // infinities or NaN among the values: one row at a time, with the values it sees (0 * inf is not 0)
      for (int r = 0; r < wn; ++r) {
        const int p = s.pos0 + (r0 + wr + r) / a.group;
        for (int d = 0; d < NV; ++d) {
          v16f acc = o[0];
#pragma unroll
          for (int e = 1; e < NV; ++e)
            if (e == d) acc = o[e];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v4i f = values(d, k);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = k0 + 16 * k + 4 * hl + (i / 2) * 8 + (i % 2) * 2;
              const uint32_t keep = (sees(a, p, key) ? 0xffffu : 0u) | (sees(a, p, key + 1) ? 0xffff0000u : 0u);
              f[i] = (int)((uint32_t)f[i] & keep);
            }
            acc = mfma32<PT>(f, pb[k], acc);
            if constexpr (TWO) acc = mfma32<PT>(f, pl[k], acc);
          }
#pragma unroll
          for (int e = 0; e < NV; ++e)
            if (e == d && c32 == r) o[e] = acc;
        }
      }
    }
    if (more) put(buf ^ 1, partial(tile + 1));
    __syncthreads();
  }

  l = sum_x32(l);
  if (!mine) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  char* to = a.out + (s.row0 + tok) * a.o_row + head * a.o_head;
#pragma unroll
  for (int d = 0; d < NV; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t y[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        y[j] = l == 0.0f ? 0u : pack2<QT>(o[d][4 * i + 2 * j] * inv, o[d][4 * i + 2 * j + 1] * inv);
      __builtin_memcpy(to + (d * 32 + 8 * i + 4 * hl) * 2, y, 8);
    }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();

int fmsmo_paged_prompt(const PagedArgs& a, int dtype, bool e4m3, int dim, fmsmo_stream_t stream) {
  const int64_t tiles = (int64_t)a.rows * a.group / BM + a.seqs;
  if (tiles * a.kv_heads > 0x7fffffffll / 256) return FMSMO_ERR_UNSUPPORTED;
  const auto go = [&](auto t, auto e, auto d) {
    hipLaunchKernelGGL((paged_prompt_kernel<decltype(t)::value, decltype(e)::value, decltype(d)::value>),
                       dim3((unsigned)(tiles * a.kv_heads)), dim3(256), 0, (hipStream_t)stream, a, (int)tiles);
  };
  const auto dims = [&](auto t, auto e) {
    if (dim == 64) go(t, e, std::integral_constant<int, 64>{});
    else if (dim == 128) go(t, e, std::integral_constant<int, 128>{});
    else go(t, e, std::integral_constant<int, 256>{});
  };
  const auto types = [&](auto t) {
    if (e4m3) dims(t, std::true_type{});
    else dims(t, std::false_type{});
  };
  if (dtype == FMSMO_F16) types(std::integral_constant<int, FMSMO_F16>{});
  else types(std::integral_constant<int, FMSMO_BF16>{});
  return fmsmo_check_launch();
}

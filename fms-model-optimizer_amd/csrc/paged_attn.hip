// Attention of a few new rows per sequence over a paged key-value cache: the work split over the cache's length and joined.
//
//   S = scale * q . k (k = code * k_scale for e4m3 caches),  o = sum_j exp(S_j - m) v_j / sum_j exp(S_j - m)
// over the keys that a row sees, with the running maximum m and sum l of each wave's share; shares are joined as
//   m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), o likewise (everything in powers of two, fp32).
//
// What bounds it is reading the cache once.  Up to 16 RT rows (tokens x the query heads that share a key head) are the columns of
// one matrix instruction, so the arithmetic is 1 / 10 of what the units could do in that time; the kernel is made of loads
// in flight: every wave owns tiles of 32 keys, from memory straight into the operands' registers -- no shared memory, no barrier --
// and asks for the keys of its next tile before the softmax of the present one, for its values after them.
//   S^T = K Q^T   16 x 16 x 32: lane l has key l % 16, and 16 bytes of it; the scores of row l % 16 for keys 4 (l / 16) .. + 3
//   O^T = V^T P^T the same instruction over 32 keys: the scores are the second operand as they stand (the reduction's order is
//                 free: element 4 t + i of lane group g is key 16 t + 4 g + i), and lane c reads elements ND c .. of those eight keys,
//                 from which v_perm makes columns ND c + n of V^T for the ND instructions n.
//
// Shares: all tiles of all sequences and heads in a row, cut into `workers` equal parts on the device from seq_lens, so a batch of
// uneven lengths keeps every block busy for the same time and nothing about the lengths has to be known on the host.
#include "paged_kv.hpp"

#include <algorithm>
#include <type_traits>

namespace fmsmo {

constexpr int TILE = 32, WAVES = 4;

struct SplitArgs {
  PagedArgs p;
  float* ws;
  int workers, unit;  // unit: tiles that are never divided between blocks (a multiple of WAVES)
};

// A sequence's share of the work: (heads x groups of rows) x units
struct Share {
  int groups, units, pairs;
};
template <int ROWS>
__device__ __forceinline__ Share share_of(const PagedArgs& a, const Seq& s, int unit) {
  Share w{0, 0, 0};
  if (s.n > 0) {
    const Tiles t = tiles_of<TILE>(a, s.len, s.pos0, s.pos0 + s.n - 1);
    w.groups = (s.n * a.group + ROWS - 1) / ROWS;
    w.units = t.count > unit ? (t.count + unit - 1) / unit : 1;  // (no keys: one that writes zeros)
    w.pairs = a.kv_heads * w.groups;
  }
  return w;
}
__device__ __forceinline__ int scan_lanes(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  return v;
}
// sum over the sequences of f(its share)
template <int ROWS, class F>
__device__ __forceinline__ int total_of(const PagedArgs& a, int unit, int lane, F f) {
  int sum = 0;
  for (int c = 0; c < a.seqs; c += 64) {
    int v = 0;
    if (c + lane < a.seqs) v = f(share_of<ROWS>(a, seq_of(a, c + lane), unit));
    sum += __shfl(scan_lanes(v, lane), 63);
  }
  return uniform(sum);
}
// the sequence in which the at-th of all f(share)'s lies (at < their sum); base: the sums before it; also_base: those of g
template <int ROWS, class F, class G>
__device__ __forceinline__ int find_of(const PagedArgs& a, int unit, int lane, int at, F f, G g, int& base, int& also_base) {
  int sum = 0, also = 0;
  for (int c = 0; c < a.seqs; c += 64) {
    int v = 0, w = 0;
    if (c + lane < a.seqs) {
      const Share s = share_of<ROWS>(a, seq_of(a, c + lane), unit);
      v = f(s);
      w = g(s);
    }
    const int iv = scan_lanes(v, lane), iw = scan_lanes(w, lane);
    const uint64_t m = __ballot(sum + iv > at);
    if (m) {
      const int l = __ffsll((unsigned long long)m) - 1;
      base = uniform(sum + __shfl(iv - v, l));
      also_base = uniform(also + __shfl(iw - w, l));
      return c + l;
    }
    sum += __shfl(iv, 63);
    also += __shfl(iw, 63);
  }
  base = also_base = 0;
  return -1;
}

// ws: [2 workers] x { o[ROWS][D], (m, l)[ROWS] }, slot 0 of a worker its first share, slot 1 its last
template <int ROWS, int D>
__device__ __forceinline__ float* slot_of(float* ws, int worker, int slot) {
  return ws + (int64_t)(2 * worker + slot) * (ROWS * (D + 2));
}

template <int QT, bool E4M3, int D, int RT>
__global__ __launch_bounds__(256, 2) void paged_split_kernel(SplitArgs sa) {
  constexpr int ROWS = 16 * RT, ND = D / 16;
  // Type of the probabilities and the values in the product.  e4m3 caches: the probabilities are multiplied by the values'
  // scales before they are rounded, which takes the exponents of bf16; for an fp16 output, of which bf16 would lose three bits, they
  // are the sum of two bf16 numbers, and the product is made twice.
  constexpr int PT = E4M3 ? FMSMO_BF16 : QT;
  constexpr bool TWO = E4M3 && QT == FMSMO_F16;
  constexpr int KW = E4M3 ? D / 64 : D / 32;           // 16-byte loads per key and lane group
  constexpr int QS = D / 32;                           // steps of the reduction over D
  constexpr int VW = E4M3 ? ND / 4 : ND / 2;           // words of a lane's values per key
  __shared__ float join[2][(RT * ND * 4 + 2 * RT) * 64];
  const PagedArgs& a = sa.p;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;

  if (a.zero_rest) zero_rest(a, D / 8);
  const auto work = [](const Share& s) { return s.pairs * s.units; };
  const auto none = [](const Share&) { return 0; };
  const int total = total_of<ROWS>(a, sa.unit, lane, work);
  int u = (int)((int64_t)blockIdx.x * total / sa.workers);
  const int u_end = (int)((int64_t)(blockIdx.x + 1) * total / sa.workers);
  for (bool first = true; u < u_end; first = false) {
    int base, unused;
    const int b = find_of<ROWS>(a, sa.unit, lane, u, work, none, base, unused);
    if (b < 0) return;
    const Seq s = seq_of(a, b);
    const Share w = share_of<ROWS>(a, s, sa.unit);
    const Tiles t = tiles_of<TILE>(a, s.len, s.pos0, s.pos0 + s.n - 1);
    const int pair = (u - base) / w.units, u0 = (u - base) % w.units;
    const int u1 = w.units - u0 < u_end - u ? w.units : u0 + (u_end - u);
    const int hk = pair / w.groups, r0 = pair % w.groups * ROWS;
    const int nrows = s.n * a.group - r0 < ROWS ? s.n * a.group - r0 : ROWS;
    const int p_lo = s.pos0 + r0 / a.group, p_hi = s.pos0 + (r0 + nrows - 1) / a.group;

    // the rows: operand of the scores, and each lane's position
    v4i q[RT][QS];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = r0 + rt * 16 + c16;
      const bool in = rt * 16 + c16 < nrows;
      const int i = in ? r / a.group : 0, h = in ? r - i * a.group : 0;
      pos[rt] = in ? s.pos0 + i : -1;
      const char* src = a.q + (s.row0 + i) * a.q_row + (hk * a.group + h) * a.q_head;
#pragma unroll
      for (int x = 0; x < QS; ++x) {
        // element order of the reduction: that in which the keys come (e4m3: 16 bytes are two steps)
        const int at = E4M3 ? (x / 2) * 64 + g * 16 + (x % 2) * 8 : x * 32 + g * 8;
        q[rt][x] = in ? *(const v4i*)(src + at * 2) : v4i{0, 0, 0, 0};
      }
    }
    v4f o[RT][ND];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -__builtin_inff();
      l[rt] = 0.0f;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[rt][n] = v4f{0, 0, 0, 0};
    }

    const int end = u1 * sa.unit < t.count ? u1 * sa.unit : t.count;
    const int in_page = (1 << a.page_shift) - 1;
    const int* row = a.table + b * a.table_stride;
    const auto key_of = [&](int tile) { return (tile < t.sink_tiles ? tile : tile + t.skip) * TILE; };
    // page numbers of a tile's two halves; -1: no such page, or behind the sequence
    const auto pages_of = [&](int tile, int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + 16 * h;
        pg[h] = tile < end && k < s.len ? row[k >> a.page_shift] : -1;
        if ((unsigned)pg[h] >= (unsigned)a.pages) pg[h] = -1;
      }
    };
    v4i kr[2][KW];
    uint32_t vr[8][VW];
    v4f ksr[2], vsr[2];
    const int k_lane = c16 * a.k_slot + g * 16, v_lane = 4 * g * a.v_slot + c16 * (VW * 4);
    const auto load_k = [&](int tile, const int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = uniform(pg[h] < 0 ? 0 : pg[h]), slot = (k0 + 16 * h) & in_page;
        const char* at = a.k + page * a.k_page + hk * a.k_head + (int64_t)slot * a.k_slot;
#pragma unroll
        for (int x = 0; x < KW; ++x) kr[h][x] = *(const v4i*)(at + k_lane + x * 64);
        if constexpr (E4M3) {
          ksr[h] = *(const v4f*)(a.ks + page * a.ks_page + hk * a.ks_head + slot + 4 * g);
          vsr[h] = *(const v4f*)(a.vs + page * a.vs_page + hk * a.vs_head + slot + 4 * g);
        }
      }
    };
    const auto load_v = [&](int tile, const int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = uniform(pg[h] < 0 ? 0 : pg[h]), slot = (k0 + 16 * h) & in_page;
        const char* at = a.v + page * a.v_page + hk * a.v_head + (int64_t)slot * a.v_slot;
#pragma unroll
        for (int j = 0; j < 4; ++j) __builtin_memcpy(vr[4 * h + j], at + v_lane + j * a.v_slot, VW * 4);
      }
    };

    int tile = u0 * sa.unit + wave;
    int pg[2], pg_next[2];
    if (tile < end) {
      pages_of(tile, pg);
      load_k(tile, pg);
      load_v(tile, pg);
      pages_of(tile + WAVES, pg_next);
    }
    for (; tile < end; tile += WAVES) {
      const int k0 = key_of(tile);
      // S^T
      v4f st[RT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) st[rt][h] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < QS; ++x) {
          v4i kx;
          if constexpr (E4M3) {
            const v4i src = kr[h][x / 2];
            uint32_t y[4];
            widen4<QT>((uint32_t)src[x % 2 * 2], y[0], y[1]);
            widen4<QT>((uint32_t)src[x % 2 * 2 + 1], y[2], y[3]);
            __builtin_memcpy(&kx, y, 16);
          } else {
            kx = kr[h][x];
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) st[rt][h] = mfma16<QT>(kx, q[rt][x], st[rt][h]);
        }
      }
      v4f ks[2], vs[2];
      if constexpr (E4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ks[h] = ksr[h] * a.c;
          vs[h] = vsr[h];
        }
      }
      const bool there0 = pg[0] >= 0, there1 = pg[1] >= 0;
      const bool whole = there0 && there1 && k0 + TILE <= s.len && sees_all(a, p_lo, p_hi, k0, k0 + TILE - 1);
      const int more = tile + WAVES;
      pg[0] = pg_next[0];
      pg[1] = pg_next[1];
      if (more < end) {
        load_k(more, pg);
        pages_of(more + WAVES, pg_next);
      }
      // the keys a lane holds scores of: 16 h + 4 g + i
      const auto there = [&](int h, int i) { return (h ? there1 : there0) && k0 + 16 * h + 4 * g + i < s.len; };
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[rt][h][i] *= E4M3 ? ks[h][i] : a.c;
      if (!whole) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool in = there(h, i);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              st[rt][h][i] = in && sees(a, pos[rt], k0 + 16 * h + 4 * g + i) ? st[rt][h][i] : -__builtin_inff();
          }
      }
      v4i pb[RT], pl[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float top = fmaxf(fmaxf(fmaxf(st[rt][0][0], st[rt][0][1]), fmaxf(st[rt][0][2], st[rt][0][3])),
                          fmaxf(fmaxf(st[rt][1][0], st[rt][1][1]), fmaxf(st[rt][1][2], st[rt][1][3])));
        top = max_x32(max_x16(top));
        const float m_new = fmaxf(m[rt], top), ms = safe_max(m_new);
        const float f = exp2_hw(m[rt] - ms);
        if (__any(m_new > m[rt])) {
#pragma unroll
          for (int n = 0; n < ND; ++n) o[rt][n] *= f;
        }
        l[rt] *= f;
        m[rt] = m_new;
        float pr[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = exp2_hw(st[rt][h][i] - ms);
            l[rt] += x;
            // (a key that the row does not see counts nothing, whatever its scale holds)
            pr[4 * h + i] = E4M3 ? (whole || st[rt][h][i] != -__builtin_inff() ? x * vs[h][i] : 0.0f) : x;
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t hi = pack2<PT>(pr[2 * i], pr[2 * i + 1]);
          pb[rt][i] = (int)hi;
          if constexpr (TWO)
            pl[rt][i] = (int)pack2<PT>(pr[2 * i] - __uint_as_float(hi << 16), pr[2 * i + 1] - __uint_as_float(hi & 0xffff0000u));
        }
      }
      // O^T
      uint32_t vw[8][ND / 2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (E4M3) {
#pragma unroll
          for (int x = 0; x < VW; ++x) widen4<PT>(vr[j][x], vw[j][2 * x], vw[j][2 * x + 1]);
        } else {
#pragma unroll
          for (int x = 0; x < VW; ++x) vw[j][x] = vr[j][x];
        }
      }
      bool apart = false;
      if (!whole) {
        // what no row sees may hold anything, and 0 * inf is not 0: such values count as zero.  Where rows see different keys, a
        // value that is not finite goes to those only that see it (below).
        uint32_t fine = 0x80008000u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = there(j / 4, j % 4) && sees_one(a, p_lo, p_hi, k0 + 16 * (j / 4) + 4 * g + j % 4);
#pragma unroll
          for (int x = 0; x < ND / 2; ++x) {
            vw[j][x] = in ? vw[j][x] : 0u;
            fine &= finite2<PT>(vw[j][x]);
          }
        }
        apart = p_lo != p_hi && __any(fine != 0x80008000u);
      }
      const auto column = [&](int n) {
        const uint32_t sel = n % 2 ? 0x07060302u : 0x05040100u;
        v4i f;
#pragma unroll
        for (int x = 0; x < 4; ++x) f[x] = (int)__builtin_amdgcn_perm(vw[2 * x + 1][n / 2], vw[2 * x][n / 2], sel);
        return f;
      };
      if (!apart) {
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const v4i f = column(n);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            o[rt][n] = mfma16<PT>(f, pb[rt], o[rt][n]);
            if constexpr (TWO) o[rt][n] = mfma16<PT>(f, pl[rt], o[rt][n]);
          }
        }
      } else {
        for (int r = 0; r < nrows; ++r) {  // one row at a time, with the values it sees
          const int p = s.pos0 + (r0 + r) / a.group;
          uint32_t keep[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) keep[j] = sees(a, p, k0 + 16 * (j / 4) + 4 * g + j % 4) ? ~0u : 0u;
#pragma unroll
          for (int n = 0; n < ND; ++n) {
            const uint32_t sel = n % 2 ? 0x07060302u : 0x05040100u;
            v4i f;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              f[x] = (int)__builtin_amdgcn_perm(vw[2 * x + 1][n / 2] & keep[2 * x + 1], vw[2 * x][n / 2] & keep[2 * x], sel);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              v4f d = mfma16<PT>(f, pb[rt], o[rt][n]);
              if constexpr (TWO) d = mfma16<PT>(f, pl[rt], d);
              if (rt * 16 + c16 == r) o[rt][n] = d;
            }
          }
        }
      }
      if (more < end) load_v(more, pg);
    }

    // the four waves' shares: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = sum_x32(sum_x16(l[rt]));
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
      if (wave >= half && wave < 2 * half) {
        float* to = join[wave - half] + lane;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[((rt * ND + n) * 4 + i) * 64] = o[rt][n][i];
          to[(RT * ND * 4 + 2 * rt) * 64] = m[rt];
          to[(RT * ND * 4 + 2 * rt + 1) * 64] = l[rt];
        }
      }
      __syncthreads();
      if (wave < half) {
        const float* from = join[wave] + lane;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float m2 = from[(RT * ND * 4 + 2 * rt) * 64], l2 = from[(RT * ND * 4 + 2 * rt + 1) * 64];
          const float mx = fmaxf(m[rt], m2), ms = safe_max(mx);
          const float f1 = exp2_hw(m[rt] - ms), f2 = exp2_hw(m2 - ms);
          m[rt] = mx;
          l[rt] = l[rt] * f1 + l2 * f2;
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[rt][n][i] = o[rt][n][i] * f1 + from[((rt * ND + n) * 4 + i) * 64] * f2;
        }
      }
      __syncthreads();
    }
    if (wave == 0) {
      const bool complete = u0 == 0 && u1 == w.units;
      float* part = slot_of<ROWS, D>(sa.ws, blockIdx.x, first ? 0 : 1);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = rt * 16 + c16;
        if (r >= nrows) continue;
        if (complete) {
          const int i = (r0 + r) / a.group, h = r0 + r - i * a.group;
          char* to = a.out + (s.row0 + i) * a.o_row + (hk * a.group + h) * a.o_head;
          const float inv = l[rt] == 0.0f ? 0.0f : 1.0f / l[rt];
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            uint32_t y[ND / 2];
#pragma unroll
            for (int n = 0; n < ND; n += 2)
              y[n / 2] = l[rt] == 0.0f ? 0u : pack2<QT>(o[rt][n][i4] * inv, o[rt][n + 1][i4] * inv);
            __builtin_memcpy(to + (4 * g + i4) * ND * 2, y, ND * 2);
          }
        } else {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            float y[ND];
#pragma unroll
            for (int n = 0; n < ND; ++n) y[n] = o[rt][n][i4];
            __builtin_memcpy(part + r * D + (4 * g + i4) * ND, y, ND * 4);
          }
          if (g == 0) {
            part[ROWS * D + 2 * r] = m[rt];
            part[ROWS * D + 2 * r + 1] = l[rt];
          }
        }
      }
    }
    u += u1 - u0;
  }
}

// Joins the shares of the heads and groups of rows that were cut: one block per row, its waves take every fourth share.
template <int QT, int D, int ROWS>
__global__ __launch_bounds__(256) void paged_join_kernel(SplitArgs sa) {
  constexpr int W = D / 64;
  __shared__ float om[WAVES][D + 2];
  const PagedArgs& a = sa.p;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const auto work = [](const Share& s) { return s.pairs * s.units; };
  const auto rows = [](const Share& s) { return s.pairs * ROWS; };
  const int total = total_of<ROWS>(a, sa.unit, lane, work), jobs = total_of<ROWS>(a, sa.unit, lane, rows);
  for (int job = blockIdx.x; job < jobs; job += gridDim.x) {
    int base, unit_base;
    const int b = find_of<ROWS>(a, sa.unit, lane, job, rows, work, base, unit_base);
    if (b < 0) return;
    const Seq s = seq_of(a, b);
    const Share w = share_of<ROWS>(a, s, sa.unit);
    const int pair = (job - base) / ROWS, r = (job - base) % ROWS;
    const int row = pair % w.groups * ROWS + r;
    if (row >= s.n * a.group) continue;
    const int64_t u0 = unit_base + pair * w.units, u1 = u0 + w.units;
    // the workers of the first and the last unit
    const int w0 = (int)(((u0 + 1) * sa.workers - 1) / total), w1 = (int)((u1 * sa.workers - 1) / total);
    if (w0 == w1) continue;  // whole: written by its block
    float m = -__builtin_inff(), l = 0.0f, o[W];
#pragma unroll
    for (int x = 0; x < W; ++x) o[x] = 0.0f;
    for (int k = w0 + wave; k <= w1; k += WAVES) {
      const int64_t start = (int64_t)k * total / sa.workers, stop = (int64_t)(k + 1) * total / sa.workers;
      if (start == stop) continue;  // a worker without work
      const float* part = slot_of<ROWS, D>(sa.ws, k, u0 <= start ? 0 : 1);
      const float m2 = part[ROWS * D + 2 * r], l2 = part[ROWS * D + 2 * r + 1];
      const float mx = fmaxf(m, m2), ms = safe_max(mx), f1 = exp2_hw(m - ms), f2 = exp2_hw(m2 - ms);
      m = mx;
      l = l * f1 + l2 * f2;
#pragma unroll
      for (int x = 0; x < W; ++x) o[x] = o[x] * f1 + part[r * D + lane * W + x] * f2;
    }
#pragma unroll
    for (int x = 0; x < W; ++x) om[wave][lane * W + x] = o[x];
    if (lane == 0) {
      om[wave][D] = m;
      om[wave][D + 1] = l;
    }
    __syncthreads();
    if (wave == 0) {
      float mx = om[0][D];
#pragma unroll
      for (int k = 1; k < WAVES; ++k) mx = fmaxf(mx, om[k][D]);
      const float ms = safe_max(mx);
      l = 0.0f;
#pragma unroll
      for (int x = 0; x < W; ++x) o[x] = 0.0f;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) {
        const float f = exp2_hw(om[k][D] - ms);
        l += om[k][D + 1] * f;
#pragma unroll
        for (int x = 0; x < W; ++x) o[x] += om[k][lane * W + x] * f;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int i = row / a.group, h = row - i * a.group;
      u16* to = (u16*)(a.out + (s.row0 + i) * a.o_row + (pair / w.groups * a.group + h) * a.o_head) + lane * W;
#pragma unroll
      for (int x = 0; x < W; ++x) store_from_f32<QT>(to, x, l == 0.0f ? 0.0f : o[x] * inv);
    }
    __syncthreads();
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();
int fmsmo_paged_prompt(const PagedArgs& a, int dtype, bool e4m3, int dim, fmsmo_stream_t stream);

// Checks a call's arguments and puts them into the kernels' form.
int fmsmo_paged_args(const fmsmo_kv_cache_t* cache, const fmsmo_kv_batch_t* batch, const void* q, int64_t q_row, int64_t q_head,
                     int q_heads, int dtype, void* out, int64_t o_row, int64_t o_head, int64_t rows, PagedArgs* to) {
  if (!cache || !batch || !cache->k || !cache->v || !batch->block_table || !batch->seq_lens || !q || !out) return FMSMO_ERR_NULL;
  const bool e4m3 = cache->dtype == FMSMO_KV_E4M3;
  if (e4m3 && (!cache->k_scale || !cache->v_scale)) return FMSMO_ERR_NULL;
  if (dtype != FMSMO_F16 && dtype != FMSMO_BF16) return FMSMO_ERR_UNSUPPORTED;
  if (!e4m3 && cache->dtype != dtype) return FMSMO_ERR_UNSUPPORTED;
  if (cache->dim != 64 && cache->dim != 128 && cache->dim != 256) return FMSMO_ERR_UNSUPPORTED;
  const int size = cache->page_size;
  if (size < 16 || size > 65536 || (size & (size - 1))) return FMSMO_ERR_UNSUPPORTED;
  if (rows < 0 || rows > 0x7fffffff || batch->seqs < 0 || cache->pages < 1 || cache->heads < 1 || q_heads < 1 || q_heads % cache->heads || batch->table_width < 1 ||
      batch->table_stride < 0 || q_row < 0 || q_head < 0 || o_row < 0 || o_head < 0)
    return FMSMO_ERR_SHAPE;
  if (!batch->query_start && rows != batch->seqs) return FMSMO_ERR_SHAPE;
  if (rows * q_heads > 0x7fffffff / 2 || batch->seqs > (1 << 20) || cache->pages > 0x7fffffff || q_heads > 4096 ||
      batch->table_width > ((1ll << 30) / size))
    return FMSMO_ERR_UNSUPPORTED;
  const int64_t* strides[] = {cache->k_strides, cache->v_strides};
  for (const int64_t* s : strides) {
    if (s[0] < 0 || s[1] < 0 || s[2] < cache->dim) return FMSMO_ERR_SHAPE;
    const int unit = e4m3 ? 16 : 8;  // 16 bytes
    if (s[0] % unit || s[1] % unit || s[2] % unit) return FMSMO_ERR_ALIGN;
    if (s[2] * size * 2 > 0x7fffffff) return FMSMO_ERR_UNSUPPORTED;
  }
  const int64_t* scales[] = {cache->k_scale_strides, cache->v_scale_strides};
  for (const int64_t* s : scales) {
    if (!e4m3) break;
    if (s[0] < 0 || s[1] < 0) return FMSMO_ERR_SHAPE;
    if (s[0] % 4 || s[1] % 4) return FMSMO_ERR_ALIGN;
  }
  const auto off = [](const void* p, int by) { return ((uintptr_t)p) % by != 0; };
  if (off(cache->k, 16) || off(cache->v, 16) || off(q, 16) || off(out, 16) || off(batch->block_table, 4) || off(batch->seq_lens, 4) ||
      off(batch->query_start, 4) || (e4m3 && (off(cache->k_scale, 16) || off(cache->v_scale, 16))))
    return FMSMO_ERR_ALIGN;
  if (q_row % 8 || q_head % 8 || o_row % 8 || o_head % 8) return FMSMO_ERR_ALIGN;
  const int by = e4m3 ? 1 : 2;
  PagedArgs& a = *to;
  a.k = (const char*)cache->k;
  a.v = (const char*)cache->v;
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.k_page = cache->k_strides[0] * by;
  a.k_head = cache->k_strides[1] * by;
  a.k_slot = (int)cache->k_strides[2] * by;
  a.v_page = cache->v_strides[0] * by;
  a.v_head = cache->v_strides[1] * by;
  a.v_slot = (int)cache->v_strides[2] * by;
  a.ks_page = cache->k_scale_strides[0];
  a.ks_head = cache->k_scale_strides[1];
  a.vs_page = cache->v_scale_strides[0];
  a.vs_head = cache->v_scale_strides[1];
  a.table = batch->block_table;
  a.table_stride = batch->table_stride;
  a.lens = batch->seq_lens;
  a.starts = batch->query_start;
  a.cap = (int)batch->table_width * size;
  a.seqs = (int)batch->seqs;
  a.rows = (int)rows;
  a.page_shift = __builtin_ctz(size);
  a.pages = (int)cache->pages;
  a.kv_heads = cache->heads;
  a.group = q_heads / cache->heads;
  a.q = (const char*)q;
  a.out = (char*)out;
  a.q_row = q_row * 2;
  a.q_head = q_head * 2;
  a.o_row = o_row * 2;
  a.o_head = o_head * 2;
  return FMSMO_OK;
}

// How a call is run, from what the host knows of it: bounds of the new rows and of the keys of a sequence.
struct Plan {
  bool prompt;   // the kernel of many rows
  int row_tiles; // of the split kernel
  int workers, unit;
};
static Plan plan_of(int group, int kv_heads, int dim, int64_t seqs, int64_t rows, int64_t max_rows, int64_t max_keys) {
  Plan p{};
  const int64_t most = max_rows * group;
  p.prompt = most > 64;
  p.row_tiles = most <= 16 ? 1 : 2;
  const int64_t tiles = std::max<int64_t>(1, (max_keys + TILE - 1) / TILE);
  const int64_t pairs = std::max<int64_t>(1, std::min(seqs, rows)) * kv_heads * ((most + 16 * p.row_tiles - 1) / (16 * p.row_tiles));
  p.unit = WAVES;
  if (tiles <= 2 * WAVES) p.unit = 1 << 24;  // nothing to split: one launch
  const int64_t units = pairs * ((tiles + p.unit - 1) / p.unit);
  p.workers = (int)std::min<int64_t>(p.unit > WAVES ? 65536 : 512, units);
  return p;
}
static int64_t plan_bytes(const Plan& p, int dim) {
  return p.prompt || p.unit > WAVES ? 0 : (int64_t)p.workers * 2 * 16 * p.row_tiles * (dim + 2) * 4;
}
static void bounds(int64_t& max_rows, int64_t& max_keys, int64_t rows, int64_t cap, bool ragged) {
  if (!ragged) max_rows = 1;
  if (max_rows < 1 || max_rows > rows) max_rows = std::max<int64_t>(1, rows);
  if (max_keys < 1 || max_keys > cap) max_keys = std::max<int64_t>(1, cap);
}

extern "C" int64_t fmsmo_paged_attn_workspace_bytes(int q_heads, int kv_heads, int dim, int64_t seqs, int64_t rows, int64_t max_rows,
                                                    int64_t max_keys) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || rows < 1 || seqs < 1) return 0;
  bounds(max_rows, max_keys, rows, 1ll << 30, true);
  return plan_bytes(plan_of(q_heads / kv_heads, kv_heads, dim, seqs, rows, max_rows, max_keys), dim);
}

extern "C" int fmsmo_paged_attn(const fmsmo_kv_cache_t* cache, const fmsmo_kv_batch_t* batch, int dtype, int64_t rows, int q_heads,
                                const void* q, int64_t q_row, int64_t q_head, void* out, int64_t o_row, int64_t o_head, float scale,
                                int64_t window, int64_t sinks, int64_t max_rows, int64_t max_keys, int zero_rest, void* workspace,
                                int64_t workspace_bytes, fmsmo_stream_t stream) {
  SplitArgs sa{};
  PagedArgs& a = sa.p;
  const int rc = fmsmo_paged_args(cache, batch, q, q_row, q_head, q_heads, dtype, out, o_row, o_head, rows, &a);
  if (rc) return rc;
  if (window < 0 || sinks < 0 || workspace_bytes < 0) return FMSMO_ERR_SHAPE;
  if (rows == 0 || batch->seqs == 0) return FMSMO_OK;
  a.c = scale * LOG2E;
  a.window = (int)std::min<int64_t>(window, 1 << 30);
  a.sinks = (int)std::min<int64_t>(sinks, 1 << 30);
  a.zero_rest = zero_rest && batch->query_start;
  bounds(max_rows, max_keys, rows, a.cap, batch->query_start != nullptr);
  const bool e4m3 = cache->dtype == FMSMO_KV_E4M3;
  const Plan p = plan_of(a.group, a.kv_heads, cache->dim, a.seqs, rows, max_rows, max_keys);
  if (p.prompt) return fmsmo_paged_prompt(a, dtype, e4m3, cache->dim, stream);
  const int64_t need = plan_bytes(p, cache->dim);
  if (need > workspace_bytes || (need && !workspace)) return FMSMO_ERR_SCRATCH;
  if (((uintptr_t)workspace) & 15) return FMSMO_ERR_ALIGN;
  // (units are counted in 31 bits: heads x groups of rows x units of a sequence, summed)
  const int64_t pairs = (rows * a.group / (16 * p.row_tiles) + a.seqs) * a.kv_heads;
  if (pairs > 0x7fffffffll / 32 || pairs * (a.cap / TILE / p.unit + 2) > 0x7fffffffll) return FMSMO_ERR_UNSUPPORTED;
  sa.ws = (float*)workspace;
  sa.workers = p.workers;
  sa.unit = p.unit;
  const auto go = [&](auto t, auto e, auto d, auto r) {
    constexpr int T = decltype(t)::value, D = decltype(d)::value, RT = decltype(r)::value;
    hipLaunchKernelGGL((paged_split_kernel<T, decltype(e)::value, D, RT>), dim3(p.workers), dim3(256), 0, (hipStream_t)stream, sa);
    if (need) {
      const int64_t jobs = (rows * a.group + (int64_t)a.seqs * 16 * RT) * a.kv_heads;
      hipLaunchKernelGGL((paged_join_kernel<T, D, 16 * RT>), dim3((unsigned)std::min<int64_t>(jobs, 2048)), dim3(256), 0,
                         (hipStream_t)stream, sa);
    }
  };
  const auto tiles = [&](auto t, auto e, auto d) {
    if (p.row_tiles == 1) go(t, e, d, std::integral_constant<int, 1>{});
    else go(t, e, d, std::integral_constant<int, 2>{});
  };
  const auto dims = [&](auto t, auto e) {
    if (cache->dim == 64) tiles(t, e, std::integral_constant<int, 64>{});
    else if (cache->dim == 128) tiles(t, e, std::integral_constant<int, 128>{});
    else tiles(t, e, std::integral_constant<int, 256>{});
  };
  const auto types = [&](auto t) {
    if (e4m3) dims(t, std::true_type{});
    else dims(t, std::false_type{});
  };
  if (dtype == FMSMO_F16) types(std::integral_constant<int, FMSMO_F16>{});
  else types(std::integral_constant<int, FMSMO_BF16>{});
  return fmsmo_check_launch();
}

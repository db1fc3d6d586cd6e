// Attention of a few new rows per sequence over a paged key-value cache: the work split over the cache's length and joined.
//
//   S = scale * q . k (k = code * k_scale for e4m3 caches),  o = sum_j exp(S_j - m) v_j / sum_j exp(S_j - m)
// over the keys that a row sees, with the running maximum m and sum l of each wave's share; shares are joined as
//   m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), o likewise (everything in powers of two, fp32).
//
// What bounds it is reading the cache once.  Up to 16 rows (tokens x the query heads that share a key head) are the columns of
// one matrix instruction, so the arithmetic is 1 / 10 of what the units could do in that time; the kernel is made of loads
// in flight: every wave owns tiles of 32 keys, from memory straight into the operands' registers -- no shared memory and no barrier
// before the waves' shares are joined -- and asks for the keys of its next tile before the softmax of the present one, for its values after them.
//   S^T = K Q^T   16 x 16 x 32: lane l has key l % 16, and 16 bytes of it; the scores of row l % 16 for keys 4 (l / 16) .. + 3
//   O^T = V^T P^T the same instruction over 32 keys: the scores are the second operand as they stand (the reduction's order is
//                 free: element 4 t + i of lane group g is key 16 t + 4 g + i), and lane c reads elements ND c .. of those eight keys,
//                 from which v_perm makes columns ND c + n of V^T for the ND instructions n.
//
// 64 sequences of up to 8000 keys, 32 + 8 heads of 128, bf16: 180 us, 6.1 TB/s, where a launch that only reads reaches 6.9.  Tried without
// gain: tiles asked for two ahead, three waves per SIMD, eight waves a block, more blocks.  (All of it at 128 elements; 64 leave registers for
// three or four blocks per compute unit, which have not been measured.)
//
// Work: all tiles of all sequences and heads in a row, cut into `workers` equal parts on the device from seq_lens, so a batch of
// uneven lengths keeps every block busy for the same time and nothing about the lengths has to be known on the host.
#include "paged_kv.hpp"

#include <algorithm>
#include <type_traits>

namespace fmsmo {

constexpr int TILE = 32, WAVES = 4;
constexpr int MAX_WORKERS = 512;  // two blocks per compute unit

// A sequence's part of the work: (heads x groups of rows) x units
struct Part {
  int groups, units, pairs;
};
__device__ __forceinline__ Part part_of(const PagedArgs& a, const Seq& s, int unit_shift, int row_shift) {
  Part w{0, 0, 0};
  if (s.n > 0) {
    const Tiles t = tiles_of<TILE>(a, s.len, s.pos0, s.pos0 + s.n - 1);
    w.groups = (s.n * a.group + (16 << row_shift) - 1) >> (4 + row_shift);
    const int units = (t.count + (1 << unit_shift) - 1) >> unit_shift;
    w.units = units > 1 ? units : 1;  // (no keys: one that writes zeros)
    w.pairs = a.kv_heads * w.groups;
  }
  return w;
}
// inclusive sums over the lanes of the wave (HELD: that stop at 2^31 - 1): within rows of 16, then the rows before
template <bool HELD = false>
__device__ __forceinline__ int scan_lanes(int v) {
  const auto add = [](int x, int y) { return HELD ? __builtin_elementwise_add_sat(x, y) : x + y; };
#define FMSMO_DPP_ADD(ctrl, rows) v = add(v, __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, true))
  FMSMO_DPP_ADD(0x111, 0xf);  // row_shr 1, 2, 4, 8
  FMSMO_DPP_ADD(0x112, 0xf);
  FMSMO_DPP_ADD(0x114, 0xf);
  FMSMO_DPP_ADD(0x118, 0xf);
  FMSMO_DPP_ADD(0x142, 0xa);  // row_bcast15 into rows 1 and 3
  FMSMO_DPP_ADD(0x143, 0xc);  // row_bcast31 into rows 2 and 3
#undef FMSMO_DPP_ADD
  return v;
}

// The units of each worker: `each` of them, one more for the first `more`
struct Deal {
  unsigned each, more;
  __device__ __forceinline__ int first(unsigned w) const { return (int)(w * each + (w < more ? w : more)); }
  __device__ __forceinline__ int worker(unsigned u) const {
    const unsigned big = more * (each + 1);
    return (int)(u < big ? u / (each + 1) : more + (u - big) / each);
  }
};

// MULTI: rows of a group may stand at different positions.  SHARED: row_shift > 0
template <int QT, bool E4M3, int D, bool MULTI, bool SHARED>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void paged_split_kernel(SplitArgs sa) {
  constexpr int ND = D / 16;
  // Type of the probabilities and the values in the product.  e4m3 caches: the probabilities are multiplied by the values' scales before
  // they are rounded, which takes the exponents of bf16.  A probability of 16 bits has lost as much as the rounded result may, so it
  // enters as the sum of two such numbers and the product is made twice: the matrix units have nothing else to do.
  constexpr int PT = E4M3 ? FMSMO_BF16 : QT;
  // fp16 ends at 2^-24, and where one key stands out the many small probabilities beside it are what the result is made of: powers go
  // up to 2^14, in the sums as well (it cancels in o / l and in the joins), so that what is lost of one is below 2^-39.
  constexpr float LIFT = PT == FMSMO_F16 ? 14.0f : 0.0f;
  constexpr int KW = E4M3 ? D / 64 : D / 32;  // 16-byte loads per key and lane group
  constexpr int QS = D / 32;                  // steps of the reduction over D
  constexpr int VW = E4M3 ? ND / 4 : ND / 2;  // words of a lane's values per key
  __shared__ float join[2][(ND * 4 + 2) * 64];
  const PagedArgs& a = sa.p;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int row_shift = SHARED ? sa.row_shift : 0, rows = 16 << row_shift;
  const int waves = WAVES >> row_shift, sub = wave & (waves - 1), row_tile = SHARED ? wave / waves : 0;  // of a row tile
  if (MULTI && a.zero_rest) zero_rest(a, D / 8);

  // The sequences, one per lane, 64 at a time: the last 64 stay in registers (all of them, as a rule).
  Seq seq{};
  Part part{};
  int scan = 0, kept = 0;
  const auto look = [&](int c) {
    seq = Seq{};
    if (c + lane < a.seqs) seq = seq_of(a, c + lane);
    part = part_of(a, seq, sa.unit_shift, row_shift);
    scan = scan_lanes(part.pairs * part.units);
    kept = c;
  };
  int total = 0, given = 0;
  for (int c = 0; c < a.seqs; c += 64) {
    look(c);
    total += __builtin_amdgcn_readlane(scan, 63);
    if constexpr (MULTI) given = __builtin_elementwise_add_sat(given, __builtin_amdgcn_readlane(scan_lanes<true>(seq.n), 63));
  }
  // (starts that go up and down name rows again and again: more units than 31 bits hold, or than anybody waits for)
  if (MULTI && given > a.rows) total = 0;
  const int workers = sa.workers < total ? sa.workers : total;  // (so that no worker is without work)
  const bool idle = (int)blockIdx.x >= workers;
  Cut* cut = (Cut*)sa.ws + blockIdx.x;
  if (idle) {
    if (threadIdx.x == 0 && sa.splits) cut->rows = 0;
    return;
  }
  Deal deal;
  deal.each = (unsigned)total / (unsigned)workers;
  deal.more = (unsigned)total - deal.each * (unsigned)workers;
  int u = deal.first(blockIdx.x);
  const int u_end = deal.first(blockIdx.x + 1);
  for (bool first = true; u < u_end; first = false) {
    // the sequence, head and group of rows that unit u belongs to
    int base = 0, at = 0;
    if (a.seqs > 64) {
      for (int c = 0; c < a.seqs; c += 64) {
        look(c);
        const int sum = __builtin_amdgcn_readlane(scan, 63);
        if (base + sum > u) break;
        base += sum;
      }
    }
    const uint64_t behind = __ballot(base + scan > u);
    at = behind ? __ffsll((unsigned long long)behind) - 1 : 0;
    const auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
    const int b = kept + at;
    Seq s;
    s.n = pick(seq.n);
    s.row0 = pick(seq.row0);
    s.pos0 = pick(seq.pos0);
    s.len = pick(seq.len);
    const int units = pick(part.units), groups = pick(part.groups);
    base += pick(scan) - units * pick(part.pairs);
    const Tiles t = tiles_of<TILE>(a, s.len, s.pos0, s.pos0 + s.n - 1);
    const int pair = (int)((unsigned)(u - base) / (unsigned)units), u0 = u - base - pair * units;
    const int u1 = units - u0 < u_end - u ? units : u0 + (u_end - u);
    const int hk = groups == 1 ? pair : pair / groups, g0 = groups == 1 ? 0 : pair % groups * rows;
    const int grows = s.n * a.group - g0 < rows ? s.n * a.group - g0 : rows;  // rows of the group, and of them this wave's
    const int r0 = g0 + 16 * row_tile, nrows = grows - 16 * row_tile < 16 ? grows - 16 * row_tile : 16;
    const int p_lo = MULTI ? s.pos0 + r0 / a.group : s.pos0, p_hi = MULTI ? s.pos0 + (r0 + nrows - 1) / a.group : s.pos0;
    const int end = SHARED && nrows <= 0 ? 0 : u1 << sa.unit_shift < t.count ? u1 << sa.unit_shift : t.count;
    const int in_page = (1 << a.page_shift) - 1;
    const auto row = (const __attribute__((address_space(4))) int*)(uintptr_t)(a.table + b * a.table_stride);
    const auto key_of = [&](int tile) { return (tile < t.sink_tiles ? tile : tile + t.skip) * TILE; };
    // page numbers of a tile's two halves as the table has them, asked for an iteration before they are looked at
    const auto pages_of = [&](int tile, int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + 16 * h;
        pg[h] = row[((unsigned)k < (unsigned)s.len ? k : 0) >> a.page_shift];
      }
    };
    // -1: no such page, or behind the sequence
    const auto check = [&](int tile, const int* from, int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        pg[h] = tile < end && k0 + 16 * h < s.len && (unsigned)from[h] < (unsigned)a.pages ? from[h] : -1;
    };
    int tile = (u0 << sa.unit_shift) + sub;
    int pg[2], pg_next[2];
    pages_of(tile, pg_next);
    // the rows: operand of the scores, and each lane's position
    v4i q[QS];
    const bool valid = c16 < nrows;
    int pos;
    {
      const int r = r0 + c16, i = MULTI && valid ? r / a.group : 0, h = valid ? r - i * a.group : 0;
      pos = valid ? s.pos0 + i : -1;
      const char* src = a.q + (s.row0 + i) * a.q_row + (hk * a.group + h) * a.q_head;
#pragma unroll
      for (int x = 0; x < QS; ++x) {
        // element order of the reduction: that in which the keys come (e4m3: 16 bytes are two steps)
        const int el = E4M3 ? (x / 2) * 64 + g * 16 + (x % 2) * 8 : x * 32 + g * 8;
        q[x] = *(const v4i*)(src + el * 2);
        q[x] = valid ? q[x] : v4i{0, 0, 0, 0};
      }
    }
    v4f o[ND];
    float m = -__builtin_inff(), l = 0.0f;
    bool odd = false;  // (MULTI) infinities or NaN among the values of keys that some rows see
#pragma unroll
    for (int n = 0; n < ND; ++n) o[n] = v4f{0, 0, 0, 0};

    // Every iteration makes the same loads, so that the wait for one of them never waits for those after it; of a half that is
    // not there (behind the end, too) they come back as zeros without a request: a buffer of no bytes.
    const auto buffer = [&](const char* at, bool there) {
      return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, there ? 0x7fffffff : 0, 0x00020000);
    };
    v4i kr[2][KW];
    uint32_t vr[8][VW];
    v4f ksr[2], vsr[2];
    const int k_lane = c16 * a.k_slot + g * 16;
    int v_lane[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v_lane[j] = (4 * g + j) * a.v_slot + c16 * (VW * 4);
    // (NT: read once, kept from pushing other things out of the caches.  64 sequences of up to 8000 keys 197 us without, 182 with)
    constexpr int NT = SHARED ? 0 : 2;
    const auto load_k = [&](int tile, const int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t page = pg[h] < 0 ? 0 : pg[h], slot = (k0 + 16 * h) & in_page;
        const auto src = buffer(a.k + page * a.k_page + hk * a.k_head + slot * a.k_slot, pg[h] >= 0);
#pragma unroll
        for (int x = 0; x < KW; ++x) kr[h][x] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(src, k_lane + x * 64, 0, NT));
        if constexpr (E4M3) {
          const auto ks = buffer((const char*)(a.ks + page * a.ks_page + hk * a.ks_head + slot), pg[h] >= 0);
          const auto vs = buffer((const char*)(a.vs + page * a.vs_page + hk * a.vs_head + slot), pg[h] >= 0);
          ksr[h] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(ks, 16 * g, 0, NT));
          vsr[h] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(vs, 16 * g, 0, NT));
        }
      }
    };
    const auto load_v = [&](int tile, const int* pg) {
      const int k0 = key_of(tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t page = pg[h] < 0 ? 0 : pg[h], slot = (k0 + 16 * h) & in_page;
        const auto src = buffer(a.v + page * a.v_page + hk * a.v_head + slot * a.v_slot, pg[h] >= 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t* to = vr[4 * h + j];
          if constexpr (VW == 1) to[0] = __builtin_amdgcn_raw_buffer_load_b32(src, v_lane[j], 0, NT);
          else if constexpr (VW == 2) {
            const auto u = __builtin_amdgcn_raw_buffer_load_b64(src, v_lane[j], 0, NT);
            __builtin_memcpy(to, &u, 8);
          } else {
#pragma unroll
            for (int x = 0; x < VW / 4; ++x) {
              const auto u = __builtin_amdgcn_raw_buffer_load_b128(src, v_lane[j] + 16 * x, 0, NT);
              __builtin_memcpy(to + 4 * x, &u, 16);
            }
          }
        }
      }
    };

    if (tile < end) {
      check(tile, pg_next, pg);
      load_k(tile, pg);
      load_v(tile, pg);
      pages_of(tile + waves, pg_next);
    }
    if (first && sa.splits && threadIdx.x == 0) {
      Cut d{};
      if (u0 > 0) {
        const int from = u - u0;
        const int worker = deal.worker(from);
        d.first = 2 * worker + (from <= deal.first(worker) ? 0 : 1);
        d.last = 2 * deal.worker(from + units - 1);
        d.rows = worker == (int)blockIdx.x - 1 ? grows : 0;
        d.row0 = s.row0;
        d.pair_row0 = g0;
        d.head = hk;
      }
      *cut = d;
    }
    for (; tile < end; tile += waves) {
      const int k0 = key_of(tile);
      // S^T
      v4f st[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        st[h] = v4f{0, 0, 0, 0};
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
          st[h] = mfma16<QT>(kx, q[x], st[h]);
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
      const int more = tile + waves;
      check(more, pg_next, pg);
      load_k(more, pg);
      pages_of(more + waves, pg_next);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[h][i] *= E4M3 ? ks[h][i] : a.c;
      if (!whole) {
        const Bounds bd = bounds_of(a, pos, pos, s.len, k0 + 4 * g);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[h][i] = (h ? there1 : there0) && inside(bd, 16 * h + i) ? st[h][i] : -__builtin_inff();
      }
      float top = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                        fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
      top = max_x32(max_x16(top));
      const float m_new = fmaxf(m, top), ms = safe_max(m_new);
      if (__any(m_new > m)) {
        const float f = exp2_hw(m - ms);
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] *= f;
        l *= f;
        m = m_new;
      }
      float pr[8];
      const float ml = ms - LIFT;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = exp2_hw(st[h][i] - ml);
          l += x;
          // (a key that the row does not see counts nothing, whatever its scale holds)
          pr[4 * h + i] = E4M3 ? (whole || st[h][i] != -__builtin_inff() ? x * vs[h][i] : 0.0f) : x;
        }
      v4i pb, pl;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t hi = pack2<PT>(pr[2 * i], pr[2 * i + 1]);
        pb[i] = (int)hi;
        if constexpr (PT == FMSMO_F16) pl[i] = (int)pack2<PT>(pr[2 * i] - f16_to_f32((u16)hi), pr[2 * i + 1] - f16_to_f32((u16)(hi >> 16)));
        else pl[i] = (int)pack2<PT>(pr[2 * i] - __uint_as_float(hi << 16), pr[2 * i + 1] - __uint_as_float(hi & 0xffff0000u));
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
      if (!whole) {
        // what no row sees may hold anything
        const Bounds bd = bounds_of(a, p_lo, p_hi, s.len, k0 + 4 * g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = (j / 4 ? there1 : there0) && inside(bd, 16 * (j / 4) + j % 4);
#pragma unroll
          for (int x = 0; x < ND / 2; ++x) {
            vw[j][x] = in ? vw[j][x] : 0u;
            if constexpr (MULTI) {
              const uint32_t u = finite_only<PT>(vw[j][x]);
              odd = odd || u != vw[j][x];
              vw[j][x] = u;
            }
          }
        }
      }
      const auto column = [&](int n, int x) {  // words x of column n: keys 2 x and 2 x + 1 of the lane's eight
        return (int)__builtin_amdgcn_perm(vw[2 * x + 1][n / 2], vw[2 * x][n / 2], n % 2 ? 0x07060302u : 0x05040100u);
      };
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const v4i f = {column(n, 0), column(n, 1), column(n, 2), column(n, 3)};
        o[n] = mfma16<PT>(f, pb, o[n]);
        o[n] = mfma16<PT>(f, pl, o[n]);
      }
      load_v(more, pg);
    }
    if (MULTI && __any(odd)) {
#pragma unroll 1
      for (int again = (u0 << sa.unit_shift) + sub; again < end; again += waves) {
        const int k0 = key_of(again);
        int pages[2];
        pages_of(again, pages);
        check(again, pages, pages);
        if (pages[0] >= 0 && pages[1] >= 0 && k0 + TILE <= s.len && sees_all(a, p_lo, p_hi, k0, k0 + TILE - 1)) continue;
#pragma unroll 1
        for (int i = 0; i < TILE; ++i) {
          const int key = k0 + i, page = i < 16 ? pages[0] : pages[1];
          if (page < 0 || key >= s.len) continue;
          const bool seen = valid && inside(bounds_of(a, pos, pos, s.len, key), 0);
          const char* src = a.v + page * a.v_page + hk * a.v_head + (int64_t)(key & in_page) * a.v_slot;
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            uint32_t u[ND / 2];
            if constexpr (E4M3) {
#pragma unroll
              for (int x = 0; x < ND / 4; ++x) widen4<PT>(*(const uint32_t*)(src + (4 * g + i4) * ND + 4 * x), u[2 * x], u[2 * x + 1]);
            } else {
              __builtin_memcpy(u, src + (4 * g + i4) * ND * 2, ND * 2);
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) o[n][i4] = add_odd<PT>(o[n][i4], (u16)(u[n / 2] >> 16 * (n % 2)), seen);
          }
        }
      }
    }

    // the shares of the waves of a row tile: the upper half into the lower one, until one is left
    l = sum_x32(sum_x16(l));
    for (int half = waves / 2; half >= 1; half /= 2) {
      if (sub >= half && sub < 2 * half) {
        float* to = join[row_tile * half + sub - half] + lane;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) to[(n * 4 + i) * 64] = o[n][i];
        to[ND * 4 * 64] = m;
        to[(ND * 4 + 1) * 64] = l;
      }
      __syncthreads();
      if (sub < half) {
        const float* from = join[row_tile * half + sub] + lane;
        const float m2 = from[ND * 4 * 64], l2 = from[(ND * 4 + 1) * 64];
        const float mx = fmaxf(m, m2), ms = safe_max(mx);
        const float f1 = exp2_hw(m - ms), f2 = exp2_hw(m2 - ms);
        m = mx;
        l = l * f1 + l2 * f2;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][i] = o[n][i] * f1 + from[(n * 4 + i) * 64] * f2;
      }
      __syncthreads();
    }
    if (sub == 0 && valid) {
      if (u0 == 0 && u1 == units) {
        const int r = r0 + c16, i = MULTI ? r / a.group : 0, h = r - i * a.group;
        char* to = a.out + (s.row0 + i) * a.o_row + (hk * a.group + h) * a.o_head;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          uint32_t y[ND / 2];
#pragma unroll
          for (int n = 0; n < ND; n += 2) y[n / 2] = l == 0.0f ? 0u : pack2<QT>(o[n][i4] * inv, o[n + 1][i4] * inv);
          __builtin_memcpy(to + (4 * g + i4) * ND * 2, y, ND * 2);
        }
      } else {
        const int r = 16 * row_tile + c16;
        float* share = share_of<D>(sa, 2 * blockIdx.x + (first ? 0 : 1));
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          float y[ND];
#pragma unroll
          for (int n = 0; n < ND; ++n) y[n] = o[n][i4];
          __builtin_memcpy(share + r * D + (4 * g + i4) * ND, y, ND * 4);
        }
        if (g == 0) {
          share[rows * D + 2 * r] = m;
          share[rows * D + 2 * r + 1] = l;
        }
      }
    }
    u += u1 - u0;
  }
}

// Joins the shares of the pairs that were cut: a block per cut and row, rows side by side, since neighbouring blocks go to different parts
// of the chip and cuts may come in steps of eight (with the cuts side by side 32 pairs of 32 rows in 16 shares took 23 us, not 8).  The
// weights of all shares first (a share per thread), then every group of D / 4 threads adds up every (1024 / D)-th share: loads that wait
// for nothing but the weights.  Bound by those two dependent rounds of loads, and with hundreds of shares by one block reading all of a
// row's: a few shares of 128 elements 4 us, 64 of them 6.5 (131072 keys, 8 key heads), 512 of them 22 (one key head; 13 at 64 elements).
template <int QT, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(SplitArgs sa) {
  constexpr int LG = D / 4, GROUPS = 256 / LG;
  __shared__ float2 weight[MAX_WORKERS];
  __shared__ float red[8];
  __shared__ __attribute__((aligned(16))) float sum[GROUPS][D];
  const PagedArgs& a = sa.p;
  const Cut d = ((const Cut*)sa.ws)[blockIdx.y];
  // split kernel: every worker has two shares, and but for the first one it is its first part that belongs here
  const int step = sa.parts ? 1 : 2, shares = sa.parts ? sa.parts : d.last / 2 - d.first / 2 + 1;
  const int rows = 16 << sa.row_shift, tid = threadIdx.x, wave = tid >> 6;
  for (int r = blockIdx.x; r < d.rows; r += gridDim.x) {
    const auto share = [&](int k) { return share_of<D>(sa, k == 0 ? d.first : (d.first / step + k) * step); };
    float top = -__builtin_inff();
    for (int k = tid; k < shares; k += 256) {
      weight[k] = *(const float2*)(share(k) + rows * D + 2 * r);
      top = fmaxf(top, weight[k].x);
    }
    top = wave_max(top);
    if ((tid & 63) == 0) red[wave] = top;
    __syncthreads();
    const float ms = safe_max(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    float l = 0.0f;
    for (int k = tid; k < shares; k += 256) {
      const float f = exp2_hw(weight[k].x - ms);
      weight[k].x = f;
      l += weight[k].y * f;
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) l += __shfl_xor(l, o);
    if ((tid & 63) == 0) red[4 + wave] = l;
    __syncthreads();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    const int c = tid % LG;
    v4f o = {0, 0, 0, 0};
#pragma unroll 4
    for (int k = tid / LG; k < shares; k += GROUPS) {
      const v4f x = *(const v4f*)(share(k) + r * D + 4 * c);
      const float f = weight[k].x;
      o += f == 0.0f && weight[k].y == 0.0f ? v4f{0, 0, 0, 0} : x * f;  // (a share without keys holds no sums)
    }
    *(v4f*)&sum[tid / LG][4 * c] = o;
    __syncthreads();
    if (tid < LG) {
#pragma unroll
      for (int k = 1; k < GROUPS; ++k) o += *(const v4f*)&sum[k][4 * c];
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int row = d.pair_row0 + r, i = row / a.group, h = row - i * a.group;
      char* to = a.out + (d.row0 + i) * a.o_row + (d.head * a.group + h) * a.o_head;
      uint32_t y[2] = {0, 0};
      if (l != 0.0f) {
        y[0] = pack2<QT>(o[0] * inv, o[1] * inv);
        y[1] = pack2<QT>(o[2] * inv, o[3] * inv);
      }
      __builtin_memcpy(to + 8 * c, y, 8);
    }
    __syncthreads();
  }
}

}  // namespace fmsmo

using namespace fmsmo;

int fmsmo_check_launch();
int fmsmo_paged_prompt(const SplitArgs& a, int dtype, bool e4m3, int dim, fmsmo_stream_t stream);

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
  if (rows < 0 || rows > 0x7fffffff || batch->seqs < 0 || cache->pages < 1 || cache->heads < 1 || q_heads < 1 || q_heads % cache->heads ||
      batch->table_width < 1 || batch->table_stride < 0 || q_row < 0 || q_head < 0 || o_row < 0 || o_head < 0)
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
  bool prompt;  // the kernel of many rows
  int row_shift, unit_shift, workers;
  bool splits;
  int tiles, parts;  // prompt kernel
  int64_t cuts, shares;
};
static Plan plan_of(int group, int kv_heads, int dim, bool e4m3, int64_t seqs, int64_t rows, int64_t max_rows, int64_t max_keys) {
  Plan p{};
  const int64_t most = max_rows * group, tokens = std::max<int64_t>(1, std::min(seqs, rows));
  // Up to 16 rows are one tile of the split kernel; up to 32 rows of an e4m3 cache, whose codes it widens on the way to the products,
  // two waves take the same keys.  5 tokens x 4 heads, 16 sequences of 16000 keys: 16 bits 229 us so and 221 by the prompt kernel,
  // e4m3 157 and 260.  (One wave taking both tiles of rows through its keys, codes widened once, has half as many waves to wait with: 8
  // sequences of 4000 keys 29 us instead of 26, 32 of 16000 124 instead of 134.)
  p.prompt = most > (e4m3 ? 32 : 16);
  if (p.prompt) {
    p.row_shift = 3;
    p.tiles = (int)(rows * group / PROMPT_ROWS + seqs);
    // Few tiles of rows: several blocks for each, as many as leave every one eight tiles of keys, up to two for a compute unit
    // where rows fill their tiles.  (Many sequences of fewer rows than a tile get more, which evens them out: 64 single tokens, 20 heads on a key
    // head, 16000 keys 125 us so, 138 with a tile counted for each; up to 16000 keys 68 and 73.)
    const int64_t blocks = std::max<int64_t>(rows * group / PROMPT_ROWS, 1) * kv_heads, key_tiles = (max_keys + PROMPT_KEYS - 1) / PROMPT_KEYS;
    p.cuts = (int64_t)p.tiles * kv_heads;  // (counted with the room between sequences: at most 2048 shares, 64 KiB each at 128 elements)
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({(dim > 128 ? 256 : 512) / blocks, key_tiles / 8, 2048 / p.cuts, 64}));
    p.splits = p.parts > 1;
    p.shares = p.cuts * p.parts;
    return p;
  }
  p.row_shift = most <= 16 ? 0 : 1;
  const int64_t tiles = std::max<int64_t>(1, (max_keys + TILE - 1) / TILE), waves = WAVES >> p.row_shift;
  const int64_t pairs = tokens * kv_heads;
  // One launch where a block per pair is through as early as the second launch would be: it takes 4 us, an iteration of
  // all waves 1.5 to 2 us while memory is not busy.  Single tokens, 8 key heads of 128 elements, one launch / two: 1 sequence of 400 keys
  // 11.6 / 9.6 us, 8 of them 13.1 / 10.9, 32 of them 13.3 / 18.6.
  p.splits = tiles > waves && !(pairs >= 192 && tiles <= 4 * waves);
  p.unit_shift = p.splits ? 2 - p.row_shift : 26;
  const int64_t units = pairs * (((tiles - 1) >> p.unit_shift) + 1);
  // One block per compute unit, and a second one where all of them have two units to do (8 sequences of 1000 keys: 15.3 us with two, 13.8
  // so); the registers of 256 elements leave room for one.
  const int64_t most_workers = dim > 128 ? MAX_WORKERS / 2 : MAX_WORKERS;
  p.workers = (int)(p.splits ? std::min(most_workers, std::max(std::min<int64_t>(units, MAX_WORKERS / 2), units / 2)) : std::min<int64_t>(65536, units));
  p.cuts = p.workers;
  p.shares = 2 * p.workers;
  return p;
}
static int64_t plan_bytes(const Plan& p, int dim) {
  return p.splits ? p.cuts * (int64_t)sizeof(Cut) + (p.shares * 16 * (dim + 2) * 4 << p.row_shift) : 0;
}
static void bounds(int64_t& max_rows, int64_t& max_keys, int64_t rows, int64_t cap, bool ragged) {
  if (!ragged) max_rows = 1;
  if (max_rows < 1 || max_rows > rows) max_rows = std::max<int64_t>(1, rows);
  if (max_keys < 1 || max_keys > cap) max_keys = std::max<int64_t>(1, cap);
}
// the keys that a tile of rows (one token at least) goes through
static int64_t visited(int64_t max_rows, int64_t max_keys, int64_t window, int64_t sinks) {
  return window ? std::min(max_keys, window + sinks + std::min<int64_t>(max_rows, PROMPT_ROWS)) : max_keys;
}

extern "C" int64_t fmsmo_paged_attn_workspace_bytes(int q_heads, int kv_heads, int dim, int cache_dtype, int64_t seqs, int64_t rows, int64_t max_rows,
                                                    int64_t max_keys) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || rows < 1 || seqs < 1) return 0;
  bounds(max_rows, max_keys, rows, 1ll << 30, true);
  return plan_bytes(plan_of(q_heads / kv_heads, kv_heads, dim, cache_dtype == FMSMO_KV_E4M3, seqs, rows, max_rows, max_keys), dim);
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
  a.window = (int)std::min<int64_t>(window, 0x7fffffff);
  a.sinks = (int)std::min<int64_t>(sinks, 1 << 30);
  a.zero_rest = zero_rest && batch->query_start;
  bounds(max_rows, max_keys, rows, a.cap, batch->query_start != nullptr);
  const bool e4m3 = cache->dtype == FMSMO_KV_E4M3;
  const Plan p = plan_of(a.group, a.kv_heads, cache->dim, e4m3, a.seqs, rows, max_rows, visited(max_rows, max_keys, a.window, a.sinks));
  const int64_t need = plan_bytes(p, cache->dim);
  if (need > workspace_bytes || (need && !workspace)) return FMSMO_ERR_SCRATCH;
  if (((uintptr_t)workspace) & 15) return FMSMO_ERR_ALIGN;
  sa.ws = (float*)workspace;
  sa.cuts = (int)p.cuts;
  sa.splits = p.splits;
  sa.row_shift = p.row_shift;
  sa.tiles = p.tiles;
  sa.parts = p.parts;
  const hipStream_t s = (hipStream_t)stream;
  const auto join = [&](auto t, auto d) {
    if (!p.splits) return;
    // rows of a pair, as a rule; of a prompt's a block takes every 32nd
    const unsigned per = (unsigned)std::min<int64_t>(max_rows * a.group, p.prompt ? 32 : 16 << p.row_shift);
    hipLaunchKernelGGL((paged_join_kernel<decltype(t)::value, decltype(d)::value>), dim3(per, (unsigned)p.cuts), dim3(256), 0, s, sa);
  };
  if (p.prompt) {
    if (p.cuts * p.parts > 0x7fffffffll / 256) return FMSMO_ERR_UNSUPPORTED;
    const int done = fmsmo_paged_prompt(sa, dtype, e4m3, cache->dim, stream);
    if (done) return done;
  }
  // (units are counted in 31 bits: heads x groups of rows x units of a sequence, summed)
  const int64_t pairs = ((rows * a.group >> (4 + p.row_shift)) + a.seqs) * a.kv_heads;
  if (!p.prompt && pairs * ((a.cap / TILE >> p.unit_shift) + 2) > 0x7fffffffll) return FMSMO_ERR_UNSUPPORTED;
  sa.workers = p.workers;
  sa.unit_shift = p.unit_shift;
  const auto go = [&](auto t, auto e, auto d) {
    constexpr int T = decltype(t)::value, D = decltype(d)::value;
    constexpr bool E = decltype(e)::value;
    const dim3 grid(p.workers), threads(64 * WAVES);
    if (p.prompt) return join(t, d);
    if constexpr (E) {
      if (p.row_shift) {
        if (a.starts) hipLaunchKernelGGL((paged_split_kernel<T, E, D, true, true>), grid, threads, 0, s, sa);
        else hipLaunchKernelGGL((paged_split_kernel<T, E, D, false, true>), grid, threads, 0, s, sa);
        return join(t, d);
      }
    }
    if (a.starts) hipLaunchKernelGGL((paged_split_kernel<T, E, D, true, false>), grid, threads, 0, s, sa);
    else hipLaunchKernelGGL((paged_split_kernel<T, E, D, false, false>), grid, threads, 0, s, sa);
    join(t, d);
  };
  const auto dims = [&](auto t, auto e) {
    if (cache->dim == 64) go(t, e, std::integral_constant<int, 64>{});
    else if (cache->dim == 128) go(t, e, std::integral_constant<int, 128>{});
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

// Attention of many new rows per sequence (prompts, chunks of prompts) over a paged key-value cache.
//
// One block takes 128 rows (tokens x the query heads that share a key head, in that order, so that the keys in shared memory
// serve all of those heads) through the keys that they see, 64 at a time; its four waves hold 32 rows each.
//   S^T = K Q^T   32 x 32 x 16: a lane holds one row's scores for half of the keys in its registers, so the softmax needs one exchange
//                 (lane l with l + 32) for the maximum and none for anything else,
//   O^T = V^T P^T the scores as they stand are the second operand (the reduction's order is free), and what rescales O is a
//                 number per lane.  V^T comes out of row-major shared memory by ds_read_b64_tr_b16.
// Each wave brings 16 of a tile's keys, one page, straight from memory into the other of two buffers while the present one is used;
// e4m3 codes become 16-bit numbers there, once per block.
//
// What bounds it: the matrix instructions and the softmax of two blocks share a compute unit, 51 % of the first's cycles in use at the
// 1.8 GHz that the power limit leaves; one prompt of 8192 tokens, 32 + 8 heads of 128, bf16: 545 us, 1010 TFLOP/s, where a large library
// product reaches 1409.  e4m3 has 290 vector instructions for a tile and wave instead of 210, codes widened and scales multiplied in:
// 2 x 2048 tokens behind 30000 keys 2415 us, 860 TFLOP/s.  Tried and slower, the one prompt (560 us then): the scores of the next tile
// beside the softmax of this one (649; a third of the registers more and no better order), the values' reads ahead of their products
// (621), s_setprio around the products (571), sums of the probabilities by dot products (587).
//
// Probabilities over 16-bit caches enter the second product once rounded to the cache's type: a second term would make half as many
// matrix instructions again.  Error against 64 bits, in units of the result's size: bf16, 8192 tokens, 0.0021, where probabilities of fp32 leave
// 0.0016; fp16 in a window 0.00026 and 0.00020; e4m3 with bf16 results 0.0023 and 0.0017.
#include "paged_kv.hpp"

#include <algorithm>
#include <type_traits>

namespace fmsmo {

constexpr int BM = PROMPT_ROWS, BN = PROMPT_KEYS;

template <int QT, bool E4M3, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 ? 2 : E4M3 ? 3 : 4) void paged_prompt_kernel(SplitArgs sa) {
  const PagedArgs& a = sa.p;
  // e4m3 caches: the values' scales are multiplied in before the probabilities are rounded, which takes the exponents of bf16; for
  // an fp16 result, of which bf16 would lose three bits, they are the sum of two bf16 numbers
  constexpr int PT = E4M3 ? FMSMO_BF16 : QT;
  constexpr bool TWO = E4M3 && QT == FMSMO_F16;
  // The maximum is held back by up to HOLD, and powers are LIFT larger than it leaves them, in the sums as well.  fp16 ends at 2^-24
  // and 2^16, and where one key stands out the many small probabilities beside it are what the result is made of: powers up to 2^15, of which
  // less than 2^-36 of the largest one's share is lost.  bf16 has fp32's exponents.  (fp16, powers up to 2^8 that end at 2^-24: 6 prompts of
  // up to 6001 tokens in a window of 1024 425 us, 430 so; 32768 keys at 2^-26 beside one without a value came out as zeros.)
  constexpr bool HALF = PT == FMSMO_F16;
  constexpr float HOLD = HALF ? 4.0f : 8.0f, LIFT = HALF ? 11.0f : 0.0f;
  constexpr int QS = D / 16, NV = D / 32;
  // Shared memory holds rows as they are in memory, D elements; 16-byte piece c of row r lies at place c ^ f(r), by which neither the keys
  // (16 bytes of 32 rows per instruction) nor the values (64 bytes of 8 rows) ask a bank for two things at once.
  constexpr int ROW = 2 * D, WRAP = ROW < 256 ? 256 / ROW : 1;  // bytes of a row; rows in a turn of the banks
  const auto key_place = [](int r) { return r / WRAP % (D == 64 ? 8 : 16); };
  // (by turns of the bits: any four rows that follow each other, and any eight of which 32 bytes are read, lie apart)
  const auto value_place = [](int r) { return ((r & 1) << 3 | (r & 2) << 1 | (r & 4) >> 1) & (D == 64 ? 7 : 15); };
  constexpr int LOADS = 16 * ROW / 1024;              // of 1 KiB for 16 rows of 16-bit numbers
  constexpr int CODES = 16 * D / 1024;                // of e4m3
  __shared__ __attribute__((aligned(1024))) char kl[2][BN * ROW];
  __shared__ __attribute__((aligned(1024))) char vl[2][BN * ROW];
  __shared__ __attribute__((aligned(16))) float sc[2][2][E4M3 ? BN : 4];
  __shared__ int odd;  // values of a tile that some rows see in part held infinities or NaN
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c32 = lane & 31, hl = lane >> 5;
  if (a.zero_rest) zero_rest(a, D / 8);

  // the tile of rows: sequence b's start at tile query_start[b] group / BM + b, which leaves room for all of them
  const int hk = blockIdx.x % a.kv_heads, y = blockIdx.x / a.kv_heads, part_no = sa.splits ? y % sa.parts : 0;
  const int x = sa.tiles - 1 - (sa.splits ? y / sa.parts : y), pair = x * a.kv_heads + hk;
  const auto nothing = [&] {
    if (sa.splits && part_no == 0 && threadIdx.x == 0) ((Cut*)sa.ws)[pair].rows = 0;
  };
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
  if (b < 0) return nothing();
  Seq s = seq_of(a, b);
  s.n = uniform(s.n);
  s.row0 = uniform(s.row0);
  s.pos0 = uniform(s.pos0);
  s.len = uniform(s.len);
  const int r0 = (x - (int)((int64_t)s.row0 * a.group / BM) - b) * BM;
  if (s.n == 0 || r0 < 0 || r0 >= s.n * a.group) return nothing();
  const int nrows = s.n * a.group - r0 < BM ? s.n * a.group - r0 : BM;
  const int p_lo = s.pos0 + r0 / a.group, p_hi = s.pos0 + (r0 + nrows - 1) / a.group;
  const Tiles t = tiles_of<BN>(a, s.len, p_lo, p_hi);
  // this block's tiles of keys
  const int begin = sa.splits ? t.count * part_no / sa.parts : 0, end = sa.splits ? t.count * (part_no + 1) / sa.parts : t.count;
  // this wave's rows
  const int wr = wave * 32, wn = nrows - wr < 32 ? nrows - wr : 32;
  const bool mine = wr + c32 < nrows;
  const int row = r0 + wr + c32, tok = mine ? row / a.group : 0, head = hk * a.group + (mine ? row - tok * a.group : 0);
  const int pos = mine ? s.pos0 + tok : -1;
  const int w_lo = s.pos0 + (r0 + wr) / a.group, w_hi = wn > 0 ? s.pos0 + (r0 + wr + wn - 1) / a.group : w_lo;
  // exp2(c s - m) with c > 0, so that the maximum of c s is that of s: a negative scale turns the queries' sign
  const float c = fabsf(a.c) < 0x1p-126f ? 0x1p-126f : fabsf(a.c);  // (NaN stays)
  v4i q[QS];
  {
    const char* src = a.q + (s.row0 + tok) * a.q_row + head * a.q_head;
    const int turn = a.c < 0.0f ? (int)0x80008000u : 0;
#pragma unroll
    for (int k = 0; k < QS; ++k) {
      q[k] = *(const v4i*)(src + (k * 16 + hl * 8) * 2);
      q[k] = mine ? q[k] ^ turn : v4i{0, 0, 0, 0};
    }
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
  // lane i (of four) holds the page of a tile's i-th 16 keys, as the table has it; checked when it is used, an iteration later
  const auto pages_of = [&](int tile) {
    const int k = key_of(tile) + 16 * (lane & 3);
    return table[((unsigned)k < (unsigned)s.len ? k : 0) >> a.page_shift];
  };
  // which of them are there
  const auto there_of = [&](int tile, int pages) {
    return (int)__ballot(tile < end && key_of(tile) + 16 * (lane & 3) < s.len && (unsigned)pages < (unsigned)a.pages) & 15;
  };
  // a tile that some rows see in part
  const auto partial = [&](int tile, int there) {
    const int k0 = key_of(tile);
    return there != 15 || k0 + BN > s.len || !sees_all(a, p_lo, p_hi, k0, k0 + BN - 1);
  };

  // Places of this lane's operands, and of its codes: piece c of a row is piece 0 with c's bits turned over.
  int k_base = c32 * ROW + (hl ^ key_place(c32)) * 16, v_base;
  {
    const int l16 = lane & 15, r = 4 * hl + l16 / 4;  // (8 rows further the place is the same)
    v_base = r * ROW + (((lane >> 4 & 1) * 2 + l16 % 4 / 2) ^ value_place(r)) * 16 + l16 % 2 * 8;
  }
  constexpr int RPC = 512 / D, WIDEN = 16 / RPC;  // rows that are widened at once, 8 codes a lane; turns for 16
  int kw_base, vw_base;
  {
    const int r = lane / (D / 8), at = lane % (D / 8);
    kw_base = (16 * wave + r) * ROW + (at ^ key_place(r)) * 16;
    vw_base = (16 * wave + r) * ROW + (at ^ value_place(r)) * 16;
  }

  // This wave's 16 keys of a tile, straight from memory, 1 KiB an instruction.  16 bits: lane i brings the 16-byte piece that belongs
  // at its end.  Codes, half as many bytes: into the second half of their place, from which they are widened when they are there.
  constexpr int PIECES = (E4M3 ? D : ROW) / 16;  // of a row
  constexpr int RPL = 64 / PIECES;               // rows of an instruction
  constexpr int N = E4M3 ? CODES : LOADS;
  int k_off[N], v_off[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int r = j * RPL + lane / PIECES, at = lane % PIECES;  // (16 rows further the places are the same)
    k_off[j] = r * a.k_slot + (E4M3 ? at : at ^ key_place(r)) * 16;
    v_off[j] = r * a.v_slot + (E4M3 ? at : at ^ value_place(r)) * 16;
  }
  constexpr int RAW = E4M3 ? CODES * 1024 : 0;
  float sr = 0.0f;  // scales: of the keys in lanes 0 .. 15, of the values in lanes 16 .. 31
  const auto load = [&](int tile, int pages, int there, int buf) {
    const int64_t page = there >> wave & 1 ? __builtin_amdgcn_readlane(pages, wave) : 0, slot = (key_of(tile) + 16 * wave) & in_page;
    const char* ks = a.k + page * a.k_page + hk * a.k_head + slot * a.k_slot;
    const char* vs = a.v + page * a.v_page + hk * a.v_head + slot * a.v_slot;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      to_shared(ks, &kl[buf][16 * wave * ROW + RAW + j * 1024], k_off[j]);
      to_shared(vs, &vl[buf][16 * wave * ROW + RAW + j * 1024], v_off[j]);
    }
    if constexpr (E4M3) {
      const float* src = (lane & 16) ? a.vs + page * a.vs_page + hk * a.vs_head : a.ks + page * a.ks_page + hk * a.ks_head;
      sr = src[slot + (lane & 15)];  // (looked at when the codes are, an iteration later)
    }
  };
  // (256 elements, whose block has its compute unit to itself, read them before the second product and widen them behind it: 608 us
  // for one prompt of 6000 tokens with 16 + 4 heads, else 643; 128, with 19 registers more for it, 2500 us instead of 2440 as below)
  constexpr bool EARLY = E4M3 && D == 256;
  v2i ku[E4M3 ? WIDEN : 1], vu[E4M3 ? WIDEN : 1];
  const auto codes = [&](int buf) __attribute__((always_inline)) {
    if constexpr (E4M3) {
#pragma unroll
      for (int j = 0; j < WIDEN; ++j) {
        ku[j] = *(const v2i*)(kl[buf] + 16 * wave * ROW + RAW + j * 512 + lane * 8);
        vu[j] = *(const v2i*)(vl[buf] + 16 * wave * ROW + RAW + j * 512 + lane * 8);
      }
    }
  };
  // What a tile that has arrived still needs.  Codes become 16-bit numbers.  In a tile that is not seen as a whole, values that nobody
  // may see become zero, and so do infinities and NaN (see finite_only).
  const auto settle_as = [&](int tile, int buf, int there, auto part_of) __attribute__((always_inline)) {
    const bool part = part_of;
    bool fine = true;
    const int k0 = key_of(tile) + 16 * wave;
    const auto clean = [&](uint32_t u, int r) {
      const bool in = (there >> wave & 1) && k0 + r < s.len;
      const uint32_t v = in ? finite_only<PT>(u) : 0u;
      fine = fine && (v == u || !in);
      return v;
    };
    if constexpr (E4M3) {
      if constexpr (!EARLY) codes(buf);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (all of them are read before the first is written over)
      // (rows j RPC + r with r < RPC, a power of two: their places are those of r with the bits of j RPC turned over)
#pragma unroll
      for (int j = 0; j < WIDEN; ++j) {
        uint32_t y[4], z[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          widen4<QT>((uint32_t)ku[j][i], y[2 * i], y[2 * i + 1]);
          widen4<PT>((uint32_t)vu[j][i], z[2 * i], z[2 * i + 1]);
        }
        if (part) {
#pragma unroll
          for (int i = 0; i < 4; ++i) z[i] = clean(z[i], j * RPC + lane / (D / 8));
        }
        __builtin_memcpy(kl[buf] + j * RPC * ROW + (kw_base ^ key_place(j * RPC) * 16), y, 16);
        __builtin_memcpy(vl[buf] + j * RPC * ROW + (vw_base ^ value_place(j * RPC) * 16), z, 16);
      }
      if (lane < 32) sc[buf][lane >> 4][16 * wave + (lane & 15)] = (lane & 16) ? sr : sr * c;
    } else if (part) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        v4i* at = (v4i*)(vl[buf] + 16 * wave * ROW + j * 1024 + lane * 16);
        v4i u = *at;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = (int)clean((uint32_t)u[i], j * RPL + lane / PIECES);
        *at = u;
      }
    }
    if (part && __any(!fine) && lane == 0) odd = 1;
  };
  // (e4m3: both forms of this and of `powers` are written out, since a test inside waits for each read from shared memory by itself:
  // 2 x 2048 tokens behind 30000 keys 2440 us, else 2650)
  const auto settle = [&](int tile, int buf, int there, bool part) __attribute__((always_inline)) {
    if (!E4M3) settle_as(tile, buf, there, part);
    else if (part) settle_as(tile, buf, there, std::true_type{});
    else settle_as(tile, buf, there, std::false_type{});
  };

  if (threadIdx.x == 0) odd = 0;
  int pages = pages_of(begin), there = there_of(begin, pages);
  if (begin < end) {
    load(begin, pages, there, begin & 1);
    pages = pages_of(begin + 1);
  }
  __syncthreads();
  for (int tile = begin; tile < end; ++tile) {
    const int buf = tile & 1, k0 = key_of(tile);
    const bool part = partial(tile, there);
    if (!E4M3 || tile == begin) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (EARLY && tile == begin) codes(buf);
    if (E4M3 ? tile == begin : part) settle(tile, buf, there, part);
    // this tile is here, and nobody reads the one before it any more
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int there_now = there;
    const bool more = tile + 1 < end;
    if (more) {
      there = there_of(tile + 1, pages);
      load(tile + 1, pages, there, buf ^ 1);
      pages = pages_of(tile + 2);
    }
    // (computed anew in every iteration instead of being kept in registers that are needed)
    if constexpr (E4M3 || D == 256) asm volatile("" : "+v"(k_base), "+v"(v_base), "+v"(kw_base), "+v"(vw_base));
    const bool whole = !part || (there_now == 15 && k0 + BN <= s.len && sees_all(a, w_lo, w_hi, k0, k0 + BN - 1));
    // S^T
    v16f st[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) st[0][i] = st[1][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < QS; ++k)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) st[kt] = mfma32<QT>(*(const v4i*)(kl[buf] + (k_base ^ k * 32) + kt * 32 * ROW), q[k], st[kt]);
    // (six reads ahead of the products)
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int k = 0; k < 2 * QS - 6; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
    // register 4 i + j of st[kt]: key kt * 32 + 8 i + 4 hl + j.  From here on as the exponents that the present maximum leaves.
    const float ms = safe_max(m), ml = ms - LIFT;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4f by = {c, c, c, c};
        if constexpr (E4M3) by = *(const v4f*)&sc[buf][0][kt * 32 + 8 * i + 4 * hl];
#pragma unroll
        for (int j = 0; j < 4; ++j) st[kt][4 * i + j] = __fmaf_rn(st[kt][4 * i + j], by[j], -ml);
      }
    if (!whole) {
      // (one test at a time, and only those that the tile needs)
      const Bounds bd = bounds_of(a, pos, pos, s.len, k0 + 4 * hl);
      const auto keep = [&](auto seen) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[kt][i] = seen(kt * 32 + 8 * (i / 4) + i % 4) ? st[kt][i] : -__builtin_inff();
      };
      if (k0 + BN > s.len || k0 + BN - 1 > w_lo) keep([&](int at) { return at <= bd.hi; });
      if (a.window && k0 <= w_hi - a.window) keep([&](int at) { return at > bd.lo || at < bd.sink; });
      if (there_now != 15) keep([&](int at) { return (there_now >> (at >> 4) & 1) != 0; });
      if (!mine) keep([&](int) { return false; });
    }
    float top = fmaxf(st[0][0], st[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(fmaxf(top, st[0][i]), st[1][i]);
    top = max_x32(top);
    // The maximum is held back: powers up to 2^HOLD are as good as powers up to 1, and O is rescaled a few times at all (8192 tokens 560 us,
    // 600 with O rescaled for every tile; e4m3, 2 x 2048 tokens behind 30000 keys, 2707 and 2795)
    const bool grow = top > HOLD + LIFT || (m == -__builtin_inff() && top > m);
    const bool any = __any(grow);
    const float step = grow ? top - LIFT : 0.0f;
    if (any) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[0][i] -= step;
        st[1][i] -= step;
      }
    }
    if (any) {
      const float m_new = grow ? ms + step : m, f = grow ? exp2_hw(m - m_new) : 1.0f;
#pragma unroll
      for (int d = 0; d < NV; ++d) o[d] *= f;
      l *= f;
      m = m_new;
    }
    v4i pb[4], pl[4];
    float sum = 0.0f;  // (a tile's first, so that what is small beside l is not rounded away one by one)
    const auto powers = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float pr[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            pr[j] = exp2_hw(st[kt][4 * i + j]);
            sum += pr[j];
          }
          if constexpr (E4M3) {
            const v4f vs = *(const v4f*)&sc[buf][1][kt * 32 + 8 * i + 4 * hl];
            // (a key that the row does not see counts nothing, whatever its scale holds)
#pragma unroll
            for (int j = 0; j < 4; ++j) pr[j] = !masked || st[kt][4 * i + j] != -__builtin_inff() ? pr[j] * vs[j] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t hi = pack2<PT>(pr[2 * j], pr[2 * j + 1]);
            pb[kt * 2 + i / 2][i % 2 * 2 + j] = (int)hi;
            if constexpr (TWO)
              pl[kt * 2 + i / 2][i % 2 * 2 + j] =
                  (int)pack2<PT>(pr[2 * j] - __uint_as_float(hi << 16), pr[2 * j + 1] - __uint_as_float(hi & 0xffff0000u));
          }
        }
    };
    if (E4M3 && !whole) powers(std::true_type{});
    else powers(std::false_type{});
    l += sum;
    // O^T: step k of the reduction has keys 16 k + 4 hl + (0..3) and those + 8, as the scores lie
    const auto values = [&](int d, int k) {
      const char* at = vl[buf] + (v_base ^ d * 64) + 16 * k * ROW;
      const s4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)at);
      const s4v w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(at + 8 * ROW));
      v4i f;
      __builtin_memcpy(&f, &u, 8);
      __builtin_memcpy((char*)&f + 8, &w, 8);
      return f;
    };
    if (EARLY && more) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      codes(buf ^ 1);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int d = 0; d < NV; ++d) {
        const v4i f = values(d, k);
        o[d] = mfma32<PT>(f, pb[k], o[d]);
        if constexpr (TWO) o[d] = mfma32<PT>(f, pl[k], o[d]);
      }
    if (E4M3 && more) {
      if (!EARLY) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      settle(tile + 1, buf ^ 1, there, partial(tile + 1, there));
    }
  }

  l = sum_x32(l);
  if (uniform(odd)) {
#pragma unroll 1
    for (int tile = begin; tile < end; ++tile) {
      const int pages = pages_of(tile), there = there_of(tile, pages);
      if (!partial(tile, there)) continue;
#pragma unroll 1
      for (int i = 0; i < BN; ++i) {
        const int key = key_of(tile) + i;
        if (!(there >> (i >> 4) & 1) || key >= s.len) continue;
        const int page = __builtin_amdgcn_readlane(pages, i >> 4);
        const bool seen = mine && inside(bounds_of(a, pos, pos, s.len, key), 0);
        const char* src = a.v + page * a.v_page + hk * a.v_head + (int64_t)(key & in_page) * a.v_slot;
#pragma unroll
        for (int d = 0; d < NV; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int at = d * 32 + 8 * k + 4 * hl;
            uint32_t u[2];
            if constexpr (E4M3) widen4<PT>(*(const uint32_t*)(src + at), u[0], u[1]);
            else __builtin_memcpy(u, src + 2 * at, 8);
#pragma unroll
            for (int n = 0; n < 4; ++n) o[d][4 * k + n] = add_odd<PT>(o[d][4 * k + n], (u16)(u[n / 2] >> 16 * (n % 2)), seen);
          }
      }
    }
  }
  if (sa.splits) {
    if (part_no == 0 && threadIdx.x == 0) {
      Cut d{};
      d.rows = nrows;
      d.first = pair * sa.parts;
      d.last = d.first + sa.parts - 1;
      d.row0 = s.row0;
      d.pair_row0 = r0;
      d.head = hk;
      ((Cut*)sa.ws)[pair] = d;
    }
    if (!mine) return;
    float* share = share_of<D>(sa, pair * sa.parts + part_no);
    const int r = wr + c32;
#pragma unroll
    for (int d = 0; d < NV; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(v4f*)(share + r * D + d * 32 + 8 * i + 4 * hl) = v4f{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (hl == 0) *(float2*)(share + BM * D + 2 * r) = make_float2(m, l);
    return;
  }
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

int fmsmo_paged_prompt(const SplitArgs& sa, int dtype, bool e4m3, int dim, fmsmo_stream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)sa.tiles * sa.p.kv_heads * sa.parts);
  const auto go = [&](auto t, auto e, auto d) {
    hipLaunchKernelGGL((paged_prompt_kernel<decltype(t)::value, decltype(e)::value, decltype(d)::value>), dim3(blocks), dim3(256), 0,
                       (hipStream_t)stream, sa);
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

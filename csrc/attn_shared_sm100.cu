// Attention of a batch whose sequences share a long prefix (tcgen05, head_dim 128), over the slot-addressed pool.
//
// Softmax over a union of key sets: with (m, l, O) = (maximum, sum of 2^(s - m), sum of 2^(s - m) v) of each set, the union has
// m = max m_i, l = sum l_i 2^(m_i - m), O = sum O_i 2^(m_i - m), output O / l.  So the shared prefix [0, P) is attended by the rows
// of ALL sequences together (128 rows a tile whatever sequences they are from, its keys read once), every sequence attends to its
// own keys [P, L), and the parts are joined.  Where every sequence's rows fill tiles of their own there is nothing to gain by that, and a
// sequence's rows take both ranges in one go.
//
// Work is a line of units, a unit being 96 keys for a pair of row tiles: items (pair of tiles, KV head) one after the other, an
// item's units in key order behind a few that stand for what it costs beside them.  Every CTA takes an equal piece of the line, so
// lengths, which only the device knows, balance by themselves; where a piece begins or ends inside an item its parts go through a
// workspace and attn_shared_merge_kernel.
//
// A CTA: two softmax groups (warps 0-3, 4-7; one row a thread), warps 8 and 11 issue the MMAs of either product, warps 9 and 10
// load K and V (and Q) by TMA (boxes of 16 rows where slots follow one another, gathers of four rows where not).  A job is one row
// tile against 96 keys; jobs alternate between the groups: the two tiles of a pair on the same keys, or, for a single tile, every
// other block of keys.  The groups use one set of score columns in turn: a group has its row in registers 300 cycles after the
// scores are there, and then the next job's may overwrite them.  Every wait is bounded (status word).
//
// What bounds it: the way of a job's scores, product to registers to the next job's product, with the second product of the job
// before in between: 1,380 cycles a job of 128 rows x 96 keys, of which the tensor pipe is busy for 770 (56 %), the special function
// unit for 800 (58 %) and the schedulers for 620 (45 %).  16 trees of 128 nodes behind
// 8192 keys (floor 176 us): 254 us, 300 under the power cap.  Times of other forms relative to it, each timed in turn with it: 80 keys and
// scores of their own for each group 1.06, scores of their own and one set of probabilities 1.03, 128 keys (which spill) 1.10, 64 keys
// and probabilities in two buffers 1.20, a quarter of the exponentials as polynomials 1.07.
#include "gemm_common.cuh"

#include <math.h>
#include <algorithm>

namespace js {

constexpr int SD = 128;              // head dim
constexpr int SROWS = 128;           // rows of a tile
constexpr int SKEYS = 96;            // keys of a unit
constexpr int KSLOTS = 3, VSLOTS = 3, SSLOTS = KSLOTS + VSLOTS;      // rings of K and V tiles
constexpr int kItemCost = 8;         // what an item costs beside its jobs, in jobs: setting out, and results out of tensor memory
constexpr int kQTile = SROWS * 256, kKTile = SKEYS * 256;      // bytes of a Q, K or V tile: 2 halves x rows x 128 B
constexpr int SWARPS = 12, STHREADS = 32 * SWARPS;      // three warps to a quarter of the SM: 168 registers a thread
constexpr int kSharedSmem = 2 * kQTile + SSLOTS * kKTile + 512;
// Tensor memory: scores of a job in columns 0-95, which the groups use in turn; probabilities of group g from 128 + 64 g, its output from 256 + 128 g
constexpr int kColP = 128, kColO = 256;

struct SharedAttn {
  const __nv_bfloat16* q;      // (T, Hq, 128), ldq elements between tokens
  const int *slot_map, *seq_rows, *cu_q, *past_lens, *mask_bits;
  __nv_bfloat16* out;          // (T, Hq * 128)
  int* plan;                   // length of a piece of the line; where every item begins on it
  uint8_t* parted;             // (tile of the sequences' rows, head): its output is in parts (without a prefix)
  float *po, *so;              // partial outputs of prefix and sequence segments: (segment, side, 16, row, 8), as a row a thread writes them
  float2 *pml, *sml;           // their (maximum, sum): (segment, side, row)
  int* status;
  long long ldq;
  int B, T, Hq, Hkv, S, max_seqs, max_len, W, causal, G, npt, ctas;
  int prefix;                  // keys of the prefix items (0: none)
  int first_key;               // where the sequences' own items begin
  int prefix_items, seq_items, seq_rows_kept;      // bounds on item numbers; rows of a sequence segment's tile that the workspace holds
  float scale_log2;
};

struct SharedMaps {
  CUtensorMap k16, v16;        // boxes of 16 rows x 64 columns
  CUtensorMap k1, v1;          // boxes of one row, for gathers
  CUtensorMap q;               // boxes of npt tokens x G heads x 64 columns
};

JS_DEVICE int sa_wait(uint64_t* bar, uint32_t parity, int* status, int code, uint32_t* gave_up) {
  return mbar_wait_warp(bar, parity, status, code, gave_up);
}

// The last uses of a ring of barriers: what a warp has started has ended before its CTA leaves, also where another wait ran out first.
template <int SLOTS>
JS_DEVICE void sa_settle(uint64_t* ring, int uses, int* status, int code) {
#pragma unroll 1
  for (int j = max(0, uses - SLOTS); j < uses; ++j) mbar_wait(&ring[j % SLOTS], (j / SLOTS) & 1, status, code);
}

// ---------------------------------------------------------------- the line of units
struct SaSeq { int q_begin, n, past, first, end, row; };      // rows, committed keys, key range, slot-map row
JS_DEVICE SaSeq sa_seq(const SharedAttn& p, int b) {
  SaSeq s;
  if (b < 0) {                 // the prefix, for the rows of all sequences
    s.q_begin = 0;
    s.n = max(0, min(p.cu_q[p.B], p.T));
    s.past = s.end = p.prefix;
    s.first = 0;
    s.row = 0;                 // sa_prefix_row says
  } else {
    s.q_begin = min(max(0, p.cu_q[b]), p.T);
    s.n = max(0, min(p.cu_q[b + 1], p.T) - s.q_begin);
    s.past = min(max(0, p.past_lens[b]), p.max_len);
    s.end = min(s.past + s.n, p.max_len);
    s.first = p.first_key;
    s.row = p.seq_rows[b];
  }
  return s;
}
// The slot-map row that the prefix is read through: the first sequence's that has rows (others may have none any more).  A whole warp asks.
JS_DEVICE int sa_prefix_row(const SharedAttn& p) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < p.B; base += 32) {
    const unsigned some = __ballot_sync(0xffffffffu, base + lane < p.B && sa_seq(p, base + lane).n > 0);
    if (some != 0) return p.seq_rows[base + __ffs(some) - 1];
  }
  return -1;
}
// keys a pair of tiles sees end here
JS_DEVICE int sa_end(const SharedAttn& p, const SaSeq& s, int b, int pair) {
  return b >= 0 && p.causal ? min(s.end, s.past + (pair + 1) * 2 * p.npt) : s.end;
}
JS_DEVICE int sa_units(const SharedAttn& p, const SaSeq& s, int b, int pair) {
  return max(0, sa_end(p, s, b, pair) - s.first + SKEYS - 1) / SKEYS;
}
JS_DEVICE int sa_pairs(const SharedAttn& p, const SaSeq& s) { return (s.n + 2 * p.npt - 1) / (2 * p.npt); }
// An item's length on the line: its jobs (two a unit where both tiles have rows) behind what it costs beside them (nothing without units)
JS_DEVICE int sa_weight(const SharedAttn& p, const SaSeq& s, int pair) { return s.n - pair * 2 * p.npt > p.npt ? 2 : 1; }
JS_DEVICE int sa_length(const SharedAttn& p, const SaSeq& s, int b, int pair) {
  const int n = sa_units(p, s, b, pair);
  return n > 0 ? n * sa_weight(p, s, pair) + kItemCost : 0;
}
JS_DEVICE int sa_total(const SharedAttn& p, int b) {       // length of one head's items
  const SaSeq s = sa_seq(p, b);
  const int pairs = sa_pairs(p, s);
  if (pairs == 0) return 0;
  if (b < 0 || !p.causal) return (pairs - 1) * sa_length(p, s, b, 0) + sa_length(p, s, b, pairs - 1);
  int n = 0;
  for (int i = 0; i < pairs; ++i) n += sa_length(p, s, b, i);
  return n;
}
// Item numbers grow along the line (with gaps): a sequence starts behind the pairs of all rows before it.
JS_DEVICE int sa_item(const SharedAttn& p, const SaSeq& s, int b, int pair, int h) {
  return (b < 0 ? pair : p.prefix_items / p.Hkv + s.q_begin / (2 * p.npt) + b + pair) * p.Hkv + h;
}
// The line is cut into pieces of one length, one for each CTA (none for the last ones where it is short).
JS_DEVICE int sa_piece(const SharedAttn& p, int total) { return max(1, (total + p.ctas - 1) / p.ctas); }

// Units of an item that begin ahead of place t in it
JS_DEVICE int sa_unit(int t, bool two) { return (max(0, t - kItemCost) + two) >> two; }

// A CTA's piece of the line, item by item; every role walks it for itself.
struct SaWalk {
  int b, pair, h, t, left;     // place in an item, what is left of the piece
  int at;                      // place on the line
  int parity;                  // group of the next job
  SaSeq s;
  int units, first, nt, span;  // of the item; this segment's units from the first one; its part of the line
  int group0;                  // the group of the segment's first job
  bool two;                    // both tiles of the pair have rows
};
JS_DEVICE void sa_begin(const SharedAttn& p, SaWalk& w) { if (w.left > 0) w.s = sa_seq(p, w.b); }
JS_DEVICE void sa_done(SaWalk& w) {
  w.left -= w.span;
  w.t += w.span;
  w.at += w.span;
  if (!w.two) w.parity ^= w.nt & 1;
}
// the next segment; sa_done has been called for the one before
JS_DEVICE bool sa_next(const SharedAttn& p, SaWalk& w) {
  while (w.left > 0) {
    for (;;) {
      const int length = w.pair < sa_pairs(p, w.s) ? sa_length(p, w.s, w.b, w.pair) : 0;
      if (w.t < length) break;
      w.t = 0;
      if (length == 0 || ++w.h == p.Hkv) {
        w.h = 0;
        ++w.pair;
      }
      while (w.pair >= sa_pairs(p, w.s)) {
        w.pair = 0;
        if (++w.b >= p.B) return false;
        w.s = sa_seq(p, w.b);
      }
    }
    w.units = sa_units(p, w.s, w.b, w.pair);
    w.two = sa_weight(p, w.s, w.pair) == 2;
    w.span = min(w.left, (w.units << w.two) + kItemCost - w.t);
    // a unit that a cut goes through is the earlier CTA's
    w.first = sa_unit(w.t, w.two);
    w.nt = sa_unit(w.t + w.span, w.two) - w.first;
    w.group0 = w.parity;
    if (w.nt > 0) return true;
    sa_done(w);
  }
  return false;
}

JS_DEVICE void sa_mma_tmem_a(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
JS_DEVICE void sa_tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// 32 bytes, a whole sector of the L2 cache, in one store
JS_DEVICE void sa_store32(void* to, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}
JS_DEVICE void sa_tmem_st32(uint32_t taddr, const uint32_t* r) {
  sa_tmem_st16(taddr, r);
  sa_tmem_st16(taddr + 16, r + 16);
}
JS_DEVICE void sa_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
JS_DEVICE float sa_exp2(float x) {      // denormal results flush to zero; exp2(-inf) = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
JS_DEVICE float sa_max3(float a, float b, float c) {      // NaN if one is: a row with a NaN score stays NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two fp32 in a register pair: half as many instructions
JS_DEVICE uint64_t sa_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
JS_DEVICE void sa_unpack(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
JS_DEVICE uint64_t sa_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
JS_DEVICE uint64_t sa_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
JS_DEVICE void sa_tma_heads(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int head, int token) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(head), "r"(token) : "memory");
}
JS_DEVICE void sa_tma_box(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
JS_DEVICE void sa_tma_rows(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y0, int y1, int y2, int y3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y0), "r"(y1), "r"(y2), "r"(y3) : "memory");
}
// MN-major operand stored as two 64-column halves of 128-byte rows, 128-byte swizzle; the halves `half_stride` bytes apart
JS_DEVICE uint64_t sa_desc_mn(uint32_t smem_addr, uint32_t half_stride) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(half_stride >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// Keys [k, k + 32) that a row sees, bit by bit: all committed ones, and new ones by the causal rule or the row's ancestor bits
JS_DEVICE uint32_t sa_visible(const SharedAttn& p, const SaSeq& s, bool prefix, int end, int node, const int* bits, int k) {
  const int j = k - s.past;                                    // place of the first among the new rows
  uint32_t v = j <= -32 ? 0xffffffffu : j < 0 ? (1u << -j) - 1u : 0u;
  if (!prefix && j > -32) {
    if (p.causal) {
      const int c = node - j;
      if (c >= 31) v = 0xffffffffu; else if (c >= 0) v |= (1u << (c + 1)) - 1u;
    } else {
      auto word = [&](int i) { return i >= 0 && i < p.W ? static_cast<uint32_t>(bits[i]) : 0u; };
      if (j < 0) v |= word(0) << -j;
      else v = __funnelshift_r(word(j >> 5), word((j >> 5) + 1), j & 31);
    }
  }
  const int left = end - k;                                    // keys at or past the end do not exist
  if (left < 32) v &= left <= 0 ? 0u : (1u << left) - 1u;
  return v;
}

__global__ void __launch_bounds__(STHREADS, 1) attn_shared_kernel(const SharedAttn p, const __grid_constant__ SharedMaps maps) {
  extern __shared__ __align__(1024) uint8_t smem[];        // swizzled tiles begin at multiples of 1024
  uint8_t *sQ = smem, *sKV = smem + 2 * kQTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + SSLOTS * kKTile);
  uint64_t *kv_full = bars, *kv_empty = bars + SSLOTS;                        // a slot of the ring
  uint64_t *q_full = bars + 2 * SSLOTS, *q_empty = q_full + 2;                // a Q buffer
  uint64_t *s_full = q_empty + 2, *s_read = s_full + 2, *p_full = s_read + 2, *pv_done = p_full + 2;      // a group
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
  uint32_t* gave_up_words = tmem_slot + 1;
  int* start = reinterpret_cast<int*>(gave_up_words + 16);                    // the first unit: b, pair, h, t; units in all; scan scratch
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t* gave_up = gave_up_words + warp;

  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's piece of the line
  if (tid == 0) {
    for (int s = 0; s < SSLOTS; ++s) { mbar_init(&kv_full[s], 1); mbar_init(&kv_empty[s], 1); }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&q_full[g], 1);
      mbar_init(&q_empty[g], 1);
      mbar_init(&s_full[g], 1);
      mbar_init(&s_read[g], 128);
      mbar_init(&p_full[g], 128);
      mbar_init(&pv_done[g], 1);
    }
    for (int w = 0; w < 16; ++w) gave_up_words[w] = 0;
    fence_barrier_init();
  }
  int* scan = start + 8;                        // a total per warp
  const int prefix_units = p.prefix > 0 ? sa_total(p, -1) * p.Hkv : 0;
  // units of the sequences ahead of this thread's (of every 384), and of all of them
  auto ahead = [&](int value, int& all) {
    int inc = value;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += other;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int before = inc - value;
    all = 0;
    for (int i = 0; i < SWARPS; ++i) {
      if (i < warp) before += scan[i];
      all += scan[i];
    }
    return before;
  };
  for (int b = tid; blockIdx.x == 0 && b < p.B; b += STHREADS) {
    const SaSeq s = sa_seq(p, b);
    if (s.n > 0 && s.past < p.prefix) report(p.status, kShortPrefix);
    const int past = p.past_lens[b];           // s.past is cut to the slot map's columns: a sequence that does not fit in them loses keys
    if (s.n > 0 && (past < 0 || past > p.max_len - s.n)) report(p.status, kBadSlot);
  }
  const int mine = tid < p.B ? sa_total(p, tid) * p.Hkv : 0;
  int total;
  const int mine_ahead = ahead(mine, total);
  for (int base = STHREADS; base < p.B; base += STHREADS) {
    int all;
    ahead(base + tid < p.B ? sa_total(p, base + tid) * p.Hkv : 0, all);
    total += all;
  }
  total += prefix_units;
  const int piece = sa_piece(p, total), u0 = min(static_cast<int>(blockIdx.x) * piece, total), u1 = min(u0 + piece, total);
  if (u0 < prefix_units) {
    if (tid == 0) {
      const SaSeq s = sa_seq(p, -1);
      int pair = 0, at = u0, length = sa_length(p, s, -1, 0);      // all pairs but the last are alike
      if (length > 0) pair = min(at / (length * p.Hkv), sa_pairs(p, s) - 1);
      at -= pair * length * p.Hkv;
      length = sa_length(p, s, -1, pair);
      start[0] = -1;
      start[1] = pair;
      start[2] = at / length;
      start[3] = at % length;
    }
  } else if (u0 < u1) {
    int run = prefix_units;
    for (int base = 0; base < p.B; base += STHREADS) {
      const int b = base + tid;
      int v = mine, before = mine_ahead, all = 0;
      if (p.B > STHREADS) {
        v = b < p.B ? sa_total(p, b) * p.Hkv : 0;
        before = ahead(v, all);
      }
      before += run;
      run += all;
      if (u0 >= before && u0 < before + v) {
        const SaSeq s = sa_seq(p, b);
        int pair = 0, at = u0 - before;
        while (at >= sa_length(p, s, b, pair) * p.Hkv) at -= sa_length(p, s, b, pair++) * p.Hkv;
        const int length = sa_length(p, s, b, pair);
        start[0] = b;
        start[1] = pair;
        start[2] = at / length;
        start[3] = at % length;
      }
    }
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (tid == 0 && blockIdx.x == 0) p.plan[0] = piece;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  SaWalk w;
  w.left = u1 - u0;
  w.at = u0;
  if (w.left > 0) {
    w.b = start[0];
    w.pair = start[1];
    w.h = start[2];
    w.t = start[3];
  }
  w.parity = 0;
  sa_begin(p, w);

  if (warp == 9 || warp == 10) {
    // ================================================================ loaders: warp 9 takes the K tiles, warp 10 the V tiles and, ahead of an item's first, its Q tiles
    const bool values = warp == 10;
    const CUtensorMap *box = values ? &maps.v16 : &maps.k16, *one = values ? &maps.v1 : &maps.k1;
    // One tile ahead: the slots of the next one, which may be another sequence's, are asked for before this one is issued.
    struct Tile {
      int slot[SKEYS / 32], row0, keys;                  // keys: to the end of what the item sees, from the tile's first
      int token, h, sides;                      // a segment's first tile: its Q tiles (sides 0: another tile)
    };
    const int* slots = nullptr;
    if (w.left > 0 && w.b < 0) w.s.row = sa_prefix_row(p);      // a walk that takes prefix items starts with them
    int at = 0;                                 // tile of the segment
    auto open = [&] {
      at = 0;
      if (!sa_next(p, w)) return false;
      const bool known = w.s.row >= 0 && w.s.row < p.max_seqs;
      if (!known) report(p.status, kBadSlot);
      slots = p.slot_map + static_cast<size_t>(known ? w.s.row : 0) * p.max_len;
      if (values && lane == 0 && w.first == 0) p.plan[1 + sa_item(p, w.s, w.b, w.pair, w.h)] = w.at - w.t;      // where the item begins
      return true;
    };
    auto ask = [&](Tile& t) {
      const int first = w.s.first + (w.first + at) * SKEYS, end = sa_end(p, w.s, w.b, w.pair);
      t.keys = end - first;
      t.row0 = w.h * p.S;
      t.token = w.s.q_begin + w.pair * 2 * p.npt;
      t.h = w.h;
      t.sides = at > 0 ? 0 : w.two ? 2 : 1;
#pragma unroll
      for (int part = 0; part < SKEYS / 32; ++part) t.slot[part] = __ldg(slots + min(first + 32 * part + lane, end - 1));      // keys past the end repeat the last one
      if (++at < w.nt) return true;
      sa_done(w);
      return open();
    };
    Tile tile, next{};
    bool have = open(), more = have && ask(tile), ok = true;
    int uses = 0, n = 0;                        // Q buffers filled so far: buffer uses % 2; tiles issued
    for (; have; ++n) {
      have = more;
      if (more) more = ask(next);
      for (int side = 0; values && side < tile.sides && ok; ++side, ++uses) {
        const int buf = uses & 1;
        ok = sa_wait(&q_empty[buf], ((uses >> 1) & 1) ^ 1, p.status, kTimeoutEmpty, gave_up);
        if (!ok) break;
        // A box holds the G heads of npt tokens.  Those behind the sequence's last one are another's or zero: a row's scores and output
        // are its own, and nobody reads these.
        if (elect_one()) {
          mbar_expect_tx(&q_full[buf], p.npt * p.G * SD * 2);
          const uint32_t dst = smem_u32(sQ + buf * kQTile);
          const int token = tile.token + side * p.npt;
          sa_tma_heads(dst, &maps.q, &q_full[buf], 0, tile.h * p.G, token);
          sa_tma_heads(dst + SROWS * 128, &maps.q, &q_full[buf], 64, tile.h * p.G, token);
        }
        __syncwarp();
      }
      if (!ok) break;
      // Groups of 16 keys: those in one page load as a box, others four rows at a time, and those behind the last key not at all (the
      // second product leaves them out, and the scores of the first are masked).
      unsigned paged = 0;
      int page[SKEYS / 16];
#pragma unroll
      for (int part = 0; part < SKEYS / 32; ++part) {
        int& slot = tile.slot[part];
        if (slot < 0 || slot >= p.S) { report(p.status, kBadSlot); slot = 0; }
        const int first = __shfl_sync(0xffffffffu, slot, lane & 16);
        // keys have to be there but need not be seen: the last group's box may go on behind the last key
        const bool fits = slot == first + (lane & 15) || (!values && 32 * part + lane >= tile.keys && first + 15 < p.S);
        const uint32_t in_row = __ballot_sync(0xffffffffu, fits);
        if ((in_row & 0xffffu) == 0xffffu) paged |= 1u << (2 * part);
        if ((in_row >> 16) == 0xffffu) paged |= 2u << (2 * part);
        page[2 * part] = tile.row0 + __shfl_sync(0xffffffffu, slot, 0);
        page[2 * part + 1] = tile.row0 + __shfl_sync(0xffffffffu, slot, 16);
      }
      const int groups = min(SKEYS / 16, (tile.keys + 15) / 16);
      const int s = values ? KSLOTS + n % VSLOTS : n % KSLOTS;
      if (!sa_wait(&kv_empty[s], ((n / (values ? VSLOTS : KSLOTS)) & 1) ^ 1, p.status, kTimeoutEmpty, gave_up)) break;
      const uint32_t dst = smem_u32(sKV + s * kKTile);
      if (elect_one()) {
        mbar_expect_tx(&kv_full[s], groups * 4096);
#pragma unroll
        for (int part = 0; part < SKEYS / 16; ++part) {
          if (part >= groups || !((paged >> part) & 1u)) continue;
          sa_tma_box(dst + part * 2048, box, &kv_full[s], 0, page[part]);
          sa_tma_box(dst + part * 2048 + SKEYS * 128, box, &kv_full[s], 64, page[part]);
        }
      }
      __syncwarp();
      const unsigned rest = ((1u << groups) - 1u) & ~paged;
      if (rest != 0) {
#pragma unroll
        for (int part = 0; part < SKEYS / 16; ++part) {
          if (!((rest >> part) & 1u)) continue;
#pragma unroll
          for (int g = 4 * part; g < 4 * part + 4; ++g) {
            int y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = tile.row0 + __shfl_sync(0xffffffffu, tile.slot[g / 8], 4 * (g & 7) + e);
            if (elect_one()) {
              sa_tma_rows(dst + g * 512, one, &kv_full[s], 0, y[0], y[1], y[2], y[3]);
              sa_tma_rows(dst + g * 512 + SKEYS * 128, one, &kv_full[s], 64, y[0], y[1], y[2], y[3]);
            }
            __syncwarp();
          }
        }
      }
      tile = next;
    }
    static_assert(KSLOTS == VSLOTS, "one ring size for both loaders");
    sa_settle<KSLOTS>(values ? kv_full + KSLOTS : kv_full, n, p.status, kTimeoutFull);
    if (values) sa_settle<2>(q_full, uses, p.status, kTimeoutFull);
  } else if (warp == 8) {
    // ================================================================ issuer of the first product: S = Q K^T of a job once the group's scores before it are read
    // (One warp for both products held the MMAs up: its waits take as long as they run.)
    constexpr uint32_t idesc = umma_idesc_bf16(SROWS, SKEYS);
    const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ)), k_desc = umma_desc_sw128(smem_u32(sKV));
    int n = 0, tile = 0, use = 0;               // jobs; K tiles and Q buffers of the segments before
    bool ok = true;
    while (ok && sa_next(p, w)) {
      const int sides = w.two ? 2 : 1, jobs = w.nt * sides;
      for (int job = 0; job < jobs; ++job, ++n) {
        const int g = n & 1, side = w.two ? job & 1 : 0, buf = (use + side) & 1, slot = tile + (w.two ? job >> 1 : job), s = slot % KSLOTS;
        if (job < sides && !(ok = sa_wait(&q_full[buf], ((use + side) >> 1) & 1, p.status, kTimeoutFull, gave_up))) break;
        if (side == 0 && !(ok = sa_wait(&kv_full[s], (slot / KSLOTS) & 1, p.status, kTimeoutFull, gave_up))) break;
        if (n > 0 && !(ok = sa_wait(&s_read[g ^ 1], ((n - 1) >> 1) & 1, p.status, kTimeoutAccum, gave_up))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = q_desc + static_cast<uint64_t>(buf * (kQTile >> 4)), b = k_desc + static_cast<uint64_t>(s * (kKTile >> 4));
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16(tmem, a + (k >> 2) * (SROWS * 128 >> 4) + 2 * (k & 3), b + (k >> 2) * (SKEYS * 128 >> 4) + 2 * (k & 3), idesc, k != 0);
          umma_commit(&s_full[g]);
          if (side == sides - 1) umma_commit(&kv_empty[s]);
          if (job + sides >= jobs) umma_commit(&q_empty[buf]);
        }
        __syncwarp();
      }
      tile += w.nt;
      use += sides;
      sa_done(w);
    }
    sa_settle<2>(s_full, n, p.status, kTimeoutAccum);
  } else if (warp == 11) {
    // ================================================================ issuer of the second product: O += P V
    constexpr uint32_t idesc = umma_idesc_bf16(SROWS, SD) | (1u << 16);
    const uint64_t v_desc = sa_desc_mn(smem_u32(sKV), SKEYS * 128);
    int n = 0, tile = 0;
    bool ok = true;
    while (ok && sa_next(p, w)) {
      const int end = sa_end(p, w.s, w.b, w.pair);
      const int sides = w.two ? 2 : 1, jobs = w.nt * sides;
      for (int job = 0; job < jobs; ++job, ++n) {
        const int g = n & 1, slot = tile + (w.two ? job >> 1 : job), s = KSLOTS + slot % VSLOTS;
        if (!(ok = sa_wait(&kv_full[s], (slot / VSLOTS) & 1, p.status, kTimeoutFull, gave_up))) break;
        if (!(ok = sa_wait(&p_full[g], (n >> 1) & 1, p.status, kTimeoutAccum, gave_up))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t b = v_desc + static_cast<uint64_t>(s * (kKTile >> 4));
          const int keys = end - (w.s.first + (w.first + (w.two ? job >> 1 : job)) * SKEYS);
#pragma unroll
          for (int k = 0; k < SKEYS / 16; ++k)
            if (16 * k < keys) sa_mma_tmem_a(tmem + kColO + g * 128, tmem + kColP + g * 64 + k * 8, b + k * (2048 >> 4), idesc, k != 0 || job >= 2);
          umma_commit(&pv_done[g]);
          if (!w.two || (job & 1)) umma_commit(&kv_empty[s]);
        }
        __syncwarp();
      }
      tile += w.nt;
      sa_done(w);
    }
    sa_settle<2>(pv_done, n, p.status, kTimeoutAccum);
  } else {
    // ================================================================ softmax and epilogue: one row a thread
    const int g = warp >> 2, row = (warp & 3) * 32 + lane, tok = row / p.G, sub = row % p.G;
    const uint32_t t_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + t_lane, tp = ts + kColP + g * 64, to = tmem + t_lane + kColO + g * 128;
    int jobs_done = 0;                          // of this group: the phase of its barriers
    bool ok = true;
    bool more = sa_next(p, w);
    while (ok && more) {
      const bool prefix = w.b < 0;
      const int rel = g ^ w.group0, side = w.two ? rel : 0;
      const int node = (w.pair * 2 + side) * p.npt + tok, head = w.h * p.G + sub;
      const bool valid = tok < p.npt && node < w.s.n;
      const int end = sa_end(p, w.s, w.b, w.pair);
      const int* bits = !p.causal && valid && !prefix ? p.mask_bits + static_cast<size_t>(w.s.q_begin + node) * p.W : nullptr;
      float m_run = -INFINITY, l_run = 0.f;
      int jobs = 0;
      const bool busy = __any_sync(0xffffffffu, valid);      // a warp without rows only keeps the barriers going
      for (int i = w.two ? 0 : rel; i < w.nt && ok; i += w.two ? 1 : 2, ++jobs, ++jobs_done) {
        const int k0 = w.s.first + (w.first + i) * SKEYS;
        const bool all = k0 + SKEYS <= min(w.s.past, end);      // every row of the item sees the whole block
        uint32_t see[SKEYS / 32] = {};
        if (!all && valid) {
#pragma unroll
          for (int c = 0; c < SKEYS / 32; ++c) see[c] = sa_visible(p, w.s, prefix, end, node, bits, k0 + 32 * c);
        }
        ok = sa_wait(&s_full[g], jobs_done & 1, p.status, kTimeoutAccum, gave_up);
        if (!ok) break;
        tc_fence_after();
        if (!busy) {
          mbar_arrive(&s_read[g]);
          if (jobs_done > 0) ok = sa_wait(&pv_done[g], (jobs_done - 1) & 1, p.status, kTimeoutAccum, gave_up);      // an arrival counts for the job that it is for
          if (!ok) break;
          mbar_arrive(&p_full[g]);
          continue;
        }
        uint32_t sr[SKEYS];
#pragma unroll
        for (int c = 0; c < SKEYS; c += 32) tmem_ld_32x32(ts + c, sr + c);
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(&s_read[g]);
        if (!all) {                             // scores of keys the row does not see
#pragma unroll
          for (int j = 0; j < SKEYS; ++j)
            if (!((see[j >> 5] >> (j & 31)) & 1u)) sr[j] = 0xff800000u;      // -inf
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < SKEYS; j += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx4[e] = sa_max3(mx4[e], __uint_as_float(sr[j + 2 * e]), __uint_as_float(sr[j + 2 * e + 1]));
        const float mx = sa_max3(sa_max3(mx4[0], mx4[1], mx4[2]), mx4[3], -INFINITY) * p.scale_log2;
        // integer running maximum in the log2 domain: probabilities are exact powers of two apart whatever the pieces
        const float m_new = sa_max3(m_run, ceilf(mx), -INFINITY), m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = sa_exp2(m_run - m_safe);
        m_run = m_new;
        const uint64_t scale2 = sa_pack(p.scale_log2, p.scale_log2), shift2 = sa_pack(-m_safe, -m_safe);
        uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int part = 0; part < SKEYS / 32; ++part) {
          uint32_t pr[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = part * 16 + i;
            float p0, p1;
            const uint64_t x = sa_fma2(sa_pack(__uint_as_float(sr[2 * j]), __uint_as_float(sr[2 * j + 1])), scale2, shift2);
            sa_unpack(x, p0, p1);
            p0 = sa_exp2(p0);
            p1 = sa_exp2(p1);
            sum2[j & 3] = sa_add2(sum2[j & 3], sa_pack(p0, p1));
            const __nv_bfloat162 v = __floats2bfloat162_rn(p0, p1);      // the MMA's operand: bf16, the sum keeps fp32
            pr[i] = *reinterpret_cast<const uint32_t*>(&v);
          }
          if (part == 0 && jobs_done > 0) {      // this group's PV before: its probabilities are read, its output is complete
            ok = sa_wait(&pv_done[g], (jobs_done - 1) & 1, p.status, kTimeoutAccum, gave_up);
            if (!ok) break;
            tc_fence_after();
          }
          sa_tmem_st16(tp + 16 * part, pr);
        }
        if (!ok) break;
        if (__any_sync(0xffffffffu, valid && jobs > 0 && alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < SD; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32(to + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            sa_tmem_st32(to + c, o);
          }
        }
        sa_tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[g]);
        float sum_lo, sum_hi;
        sa_unpack(sa_add2(sa_add2(sum2[0], sum2[1]), sa_add2(sum2[2], sum2[3])), sum_lo, sum_hi);
        l_run = l_run * alpha + (sum_lo + sum_hi);
      }
      if (!ok) break;
      // ---- the segment's result: the output where this CTA saw all keys of the rows, else a part
      const int item = sa_item(p, w.s, w.b, w.pair, w.h);
      const bool direct = w.two && w.nt == w.units && !prefix && p.prefix == 0;
      const int rows = prefix ? SROWS : p.seq_rows_kept;
      const size_t seg = static_cast<size_t>(blockIdx.x) + (prefix ? item : item - p.prefix_items);
      const size_t at = (seg * 2 + rel) * rows + row;
      const bool keep = valid && !direct && row < rows;
      __nv_bfloat16* out = direct ? p.out + (static_cast<size_t>(w.s.q_begin + node) * p.Hq + head) * SD : nullptr;
      float* part = (prefix ? p.po : p.so) + ((seg * 2 + rel) * rows * SD + row * 8);
      if (keep) (prefix ? p.pml : p.sml)[at] = make_float2(m_run, l_run);
      else if (valid && !direct) report(p.status, kRowsOverflow);      // more rows in a sequence than the caller's bound
      if (p.prefix == 0 && (warp & 3) == 0 && lane == 0 && (w.two || rel == 0))
        p.parted[(w.s.q_begin / p.npt + w.b + w.pair * 2 + side) * p.Hkv + w.h] = !direct;
      sa_done(w);
      more = sa_next(p, w);                     // what it asks memory for comes while the last product ends
      if (jobs > 0) {
        ok = sa_wait(&pv_done[g], (jobs_done - 1) & 1, p.status, kTimeoutAccum, gave_up);
        if (!ok) break;
        tc_fence_after();
        const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
#pragma unroll 1
        for (int c = 0; busy && c < SD; c += 64) {
          uint32_t o[64];
          tmem_ld_32x32(to + c, o);
          tmem_ld_32x32(to + c + 32, o + 32);
          tmem_ld_wait();
          if (direct && valid) {
#pragma unroll
            for (int j = 0; j < 64; j += 16) {
              uint32_t pk[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * e]) * inv, __uint_as_float(o[j + 2 * e + 1]) * inv);
                pk[e] = *reinterpret_cast<const uint32_t*>(&v);
              }
              sa_store32(out + c + j, pk);
            }
          } else if (keep) {
#pragma unroll
            for (int j = 0; j < 64; j += 8) sa_store32(part + static_cast<size_t>(c + j) * rows, o + j);
          }
        }
      }
    }
    sa_tmem_st_wait();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the rows of a tile: a block takes up to kMergeRows rows of one head.
constexpr int kMergeRows = 32, kMergeWarps = 8;
__global__ void __launch_bounds__(32 * kMergeWarps) attn_shared_merge_kernel(const SharedAttn p) {
  // Until the wait below only the call's inputs are read: the kernel before, which is launched without overlap, began when they were there.
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, row0 = blockIdx.z * kMergeRows;
  {                                            // rows behind the last sequence are zero
    const int first = max(0, min(p.cu_q[p.B], p.T));
    uint4* out = reinterpret_cast<uint4*>(p.out + static_cast<size_t>(first) * p.Hq * SD);
    const size_t n = static_cast<size_t>(p.T - first) * p.Hq * SD / 8, blocks = static_cast<size_t>(gridDim.x) * gridDim.y * gridDim.z;
    const size_t block = (static_cast<size_t>(blockIdx.z) * gridDim.y + h) * gridDim.x + blockIdx.x;
    for (size_t i = block * blockDim.x + threadIdx.x; i < n; i += blocks * blockDim.x) out[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // Every block waits, also one without a row: this kernel ends behind the one before, and what follows it on the stream waits for this one alone.
  if (p.prefix == 0) {                         // most tiles were written by their CTA
    pdl_wait();
    if (p.parted[blockIdx.x * p.Hkv + h] == 0) return;
  }
  // tiles are numbered like pairs: those of a sequence start behind the tiles of all rows before it
  int b = -1;                                  // the last sequence that starts at or before this tile
  for (int base = 0; base < p.B; base += 32) {
    const unsigned some = __ballot_sync(0xffffffffu, base + lane < p.B && min(max(p.cu_q[base + lane], 0), p.T) / p.npt + base + lane <= static_cast<int>(blockIdx.x));
    b += __popc(some);
    if (some != 0xffffffffu) break;
  }
  if (b < 0) {
    pdl_wait();
    return;
  }
  const SaSeq s = sa_seq(p, b);
  const int tile = blockIdx.x - (s.q_begin / p.npt + b), node0 = tile * p.npt;
  const int rows = min(p.npt, s.n - node0) * p.G;
  pdl_wait();
  if (rows <= row0) return;
  const int piece = p.plan[0], pair = tile >> 1, units = sa_units(p, s, b, pair);
  const bool two = s.n - pair * 2 * p.npt > p.npt;
  int c0 = 0, own = 0, item = 0, own_begin = 0;      // first CTA and number of CTAs with a part of the sequence's own keys
  if (units > 0) {
    item = sa_item(p, s, b, pair, h);
    // On the line, whatever the plan says: a CTA that a wait ran out in leaves its items' places unwritten, and nothing is read past the parts.
    const int u = own_begin = min(max(p.plan[1 + item], 0), p.ctas * piece - 1);
    c0 = min((u + kItemCost) / piece, p.ctas - 1);
    own = min((u + kItemCost + ((units - 1) << two)) / piece, p.ctas - 1) - c0 + 1;
    item -= p.prefix_items;
  }
  if (own == 1 && two && p.prefix == 0) return;       // written by its CTA
  const SaSeq all = p.prefix > 0 ? sa_seq(p, -1) : s;
  const int all_units = p.prefix > 0 ? sa_units(p, all, -1, 0) : 0;
  const int own_parts = two ? own : 2 * own;
  // a row and 16 columns a thread, a warp's lanes on neighbouring rows; with fewer rows than lanes, lanes share a row's parts among them
  const int there = min(rows - row0, kMergeRows);
  int wide = 1;
  while (wide < there) wide <<= 1;
  const int row = row0 + (lane & (wide - 1)), share = 32 / wide;
  const bool live = row < row0 + there;
  const int tok = (live ? row : row0) / p.G, t = s.q_begin + node0 + tok, sub = (live ? row : row0) - tok * p.G;
  int pc0 = 0, shared_parts = 0, p_item = 0, p_row = 0, p_begin = 0;
  bool p_two = false;
  if (all_units > 0) {
    const int p_tile = t / p.npt, p_pair = p_tile >> 1;
    p_item = sa_item(p, all, -1, p_pair, h);
    p_two = sa_weight(p, all, p_pair) == 2;
    p_begin = p_pair * p.Hkv * sa_length(p, all, -1, 0) + h * sa_length(p, all, -1, p_pair);
    pc0 = (p_begin + kItemCost) / piece;
    shared_parts = ((p_begin + kItemCost + ((all_units - 1) << p_two)) / piece - pc0 + 1) * (p_two ? 1 : 2);
    p_row = (t - p_tile * p.npt) * p.G + sub + (p_two ? (p_tile & 1) * SROWS : 0);
  }
  const int parts = live ? shared_parts + own_parts : 0;
  float m = -INFINITY, l = 0.f, acc[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  auto exp_of = [](float v, float top) { return top == -INFINITY ? (v == v ? 0.f : v) : exp2f(v - top); };      // NaN scores leave a sum without a maximum
#pragma unroll 2
  for (int k = lane / wide; k < parts; k += share) {
    const bool common = k < shared_parts, pair_of = common ? p_two : two;
    const int j = common ? k : k - shared_parts, c = (common ? pc0 : c0) + (pair_of ? j : j >> 1), begin = common ? p_begin : own_begin;
    // a cut piece may hold no unit's beginning, and then no part
    if (sa_unit(c * piece - begin, pair_of) == sa_unit((c + 1) * piece - begin, pair_of) || (!common && row >= p.seq_rows_kept)) continue;
    const int kept = common ? SROWS : p.seq_rows_kept, at_row = common ? p_row % SROWS : row;
    const size_t seg = static_cast<size_t>(c + (common ? p_item : item)) * 2 + (common ? (p_two ? p_row / SROWS : j & 1) : two ? tile & 1 : j & 1);
    const float2 ml = (common ? p.pml : p.sml)[seg * kept + at_row];
    const float4* from = reinterpret_cast<const float4*>((common ? p.po : p.so) + (seg * SD + 16 * warp) * kept + 8 * at_row);
    const float4 x[4] = {from[0], from[1], from[2 * kept], from[2 * kept + 1]};
    if (ml.y == 0.f) continue;                 // no visible key: the part's output may be unwritten
    const float top = fmaxf(m, ml.x), old = exp_of(m, top), add = exp_of(ml.x, top);
    m = top;
    l = l * old + ml.y * add;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      acc[4 * q] = fmaf(x[q].x, add, acc[4 * q] * old);
      acc[4 * q + 1] = fmaf(x[q].y, add, acc[4 * q + 1] * old);
      acc[4 * q + 2] = fmaf(x[q].z, add, acc[4 * q + 2] * old);
      acc[4 * q + 3] = fmaf(x[q].w, add, acc[4 * q + 3] * old);
    }
  }
  for (int o = wide; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    const float top = fmaxf(m, m2), f = exp_of(m, top), f2 = exp_of(m2, top);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = acc[j] * f + __shfl_xor_sync(0xffffffffu, acc[j], o) * f2;
  }
  if (!live || lane >= wide) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t pk[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(acc[2 * j] * inv, acc[2 * j + 1] * inv);
    pk[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
  sa_store32(p.out + (static_cast<size_t>(t) * p.Hq + h * p.G + sub) * SD + 16 * warp, pk);
}

// Queries as (tokens, heads, 128), tokens ldq elements apart
static int make_head_map(CUtensorMap* m, const void* q, int T, int Hq, long long ldq, int npt, int G) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[3] = {SD, static_cast<cuuint64_t>(Hq), static_cast<cuuint64_t>(T)}, strides[2] = {SD * 2, static_cast<cuuint64_t>(ldq) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(npt)}, step[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -2;
}

static long long shared_round(long long bytes) { return (bytes + 255) / 256 * 256; }

// What a launch lays out in its workspace; returns the bytes.
static long long shared_layout(SharedAttn* p, uint8_t* ws, int max_q) {
  const int pair_rows = 2 * p->npt;
  p->prefix_items = p->prefix > 0 ? (p->T + pair_rows - 1) / pair_rows * p->Hkv : 0;
  p->seq_items = (p->T / pair_rows + p->B + 1) * p->Hkv;
  p->seq_rows_kept = max_q >= p->npt ? SROWS : max_q * p->G;
  const long long prefix_rows = p->prefix > 0 ? 2ll * SROWS * (p->ctas + p->prefix_items) : 0;
  const long long rows = 2ll * p->seq_rows_kept * (p->ctas + p->seq_items);
  long long at = 0;
  auto take = [&](long long bytes) { uint8_t* r = ws + at; at += shared_round(bytes); return r; };
  p->plan = reinterpret_cast<int*>(take(4ll * (1 + p->prefix_items + p->seq_items)));
  p->parted = take((p->T / p->npt + p->B + 1ll) * p->Hkv);
  p->pml = reinterpret_cast<float2*>(take(8 * prefix_rows));
  p->sml = reinterpret_cast<float2*>(take(8 * rows));
  p->po = reinterpret_cast<float*>(take(4 * SD * prefix_rows));
  p->so = reinterpret_cast<float*>(take(4 * SD * rows));
  return at;
}

// Attending to the prefix for all rows together pays where sequences leave much of their own tiles empty: tiles of all rows together
// against those of B sequences, whose last ones are half full on average.  Together / alone, us: 64 x 1 row behind 8192 keys 53 / 317, 8 x 1
// behind 1024 17.6 / 22; 16 trees (32 over 8 heads) behind 2048 of 16 rows 34 / 41, of 32 46 / 47, of 48 58 / 56 (the last that go
// together), of 64 66 / 58, of 128 behind 8192 289 / 265; 6 prompts of 33 - 901 rows 236 / 188.  It knows nothing of lengths, and misses
// some: 16 trees of 96 rows behind 8192 keys would gain (220 / 266), two of 16 behind 4096 lose (43 / 34); below some 100 keys and for one
// sequence it makes no difference (8 x 1 row behind 64 keys 17.3 / 17.4, one row 15.5 / 15.4).
static bool shared_pays(int B, int T, int npt) {
  const long long together = T, own = std::max(static_cast<long long>(B) * npt, T + static_cast<long long>(B) * npt / 2);
  return 4 * together <= 3 * own;
}

static int shared_setup(SharedAttn* p, int max_q, int prefix_len, int ctas) {
  if (p->B < 0 || p->T < 0 || p->Hkv < 1 || p->Hq < 1 || p->Hq % p->Hkv || prefix_len < 0 || prefix_len > p->max_len || max_q < 1 || ctas < 1) return -10;
  p->G = p->Hq / p->Hkv;
  if (p->G > SROWS) return -11;
  p->npt = SROWS / p->G;
  p->ctas = ctas;
  // The sequences' own items begin at a multiple of 16 positions, where pages do, so that their keys load in boxes.
  p->prefix = p->first_key = shared_pays(p->B, p->T, p->npt) ? prefix_len / 16 * 16 : 0;
  // places on the line are 32-bit: at most this many items, of at most that length
  const double items = (2.0 * (p->T / (2 * p->npt)) + p->B + 2) * p->Hkv;
  return items * (2.0 * (p->max_len / SKEYS + 1) + kItemCost) < 2e9 ? 0 : -16;
}

}  // namespace js

// Bytes of workspace that js_shared_attention wants for these sizes; negative: refused.
extern "C" long long js_shared_attention_ws(int B, int T, int Hq, int Hkv, int max_len, int prefix_len, int max_q, int ctas) {
  using namespace js;
  SharedAttn p{};
  p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.max_len = max_len;
  const int rc = shared_setup(&p, max_q, prefix_len, ctas);
  return rc != 0 ? rc : shared_layout(&p, nullptr, max_q);
}

// q (T, Hq, 128) bf16, ldq elements between tokens; pools (Hkv, S, 128); slot_map (max_seqs, max_len); seq_rows, past_lens (B); cu_q (B + 1);
// mask_bits (T, W), or null when causal; out (T, Hq * 128).  Positions [0, prefix_len) hold the same slots in all rows of the slot map that
// are named; max_q bounds a sequence's rows.  ws: js_shared_attention_ws bytes.  q and the pools on 16-byte boundaries, out and ws on 32.
extern "C" int js_shared_attention(const void* q, long long ldq, const void* k_pool, const void* v_pool, const int* slot_map, const int* seq_rows,
                                   const int* cu_q, const int* past_lens, const int* mask_bits, void* out, void* ws, long long ws_bytes,
                                   int* status, int B, int T, int Hq, int Hkv, int S, int max_seqs, int max_len, int W, int causal, float scale,
                                   int prefix_len, int max_q, int ctas, cudaStream_t stream) {
  using namespace js;
  if (T == 0 || B == 0) return 0;
  SharedAttn p{};
  p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.max_len = max_len;
  if (const int rc = shared_setup(&p, max_q, prefix_len, ctas)) return rc;
  // copies start on 16-byte boundaries, results and parts leave 32 bytes at a time
  if (ldq % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(ws)) & 31)) return -12;
  if (!causal && (mask_bits == nullptr || W < 1)) return -13;
  if (!(scale > 0.f) || S < 1 || max_seqs < 1) return -10;
  if (shared_layout(&p, reinterpret_cast<uint8_t*>(ws), max_q) > ws_bytes) return -14;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.ldq = ldq;
  p.slot_map = slot_map; p.seq_rows = seq_rows; p.cu_q = cu_q; p.past_lens = past_lens; p.mask_bits = mask_bits;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.status = status;
  p.S = S; p.max_seqs = max_seqs; p.W = W; p.causal = causal;
  p.scale_log2 = scale * 1.4426950408889634f;
  SharedMaps maps;
  const uint64_t rows = static_cast<uint64_t>(Hkv) * S;
  if (rows >= (1ull << 31) || make_map(&maps.k16, k_pool, rows, SD, SD, 16) || make_map(&maps.v16, v_pool, rows, SD, SD, 16) ||
      make_map(&maps.k1, k_pool, rows, SD, SD, 1) || make_map(&maps.v1, v_pool, rows, SD, SD, 1) ||
      make_head_map(&maps.q, q, T, Hq, ldq, p.npt, p.G)) return -15;
  static int configured[kMaxDevicesCached] = {};
  if (ensure_dyn_smem(attn_shared_kernel, kSharedSmem, configured) != 0) return -3;
  attn_shared_kernel<<<ctas, STHREADS, kSharedSmem, stream>>>(p, maps);
  if (cudaGetLastError() != cudaSuccess) return -4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(T / p.npt + B, Hkv, (p.seq_rows_kept + kMergeRows - 1) / kMergeRows);
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_shared_merge_kernel, p) == cudaSuccess ? 0 : -5;
}

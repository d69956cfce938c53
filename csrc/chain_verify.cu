// Drafted chains against the target's probabilities, from given random numbers.
//
// Sequence b drafted x_0 .. x_{n-1}; draft row i holds the logits x_i was drawn from, target row i the target's logits at the same
// place, and one more target row stands behind the last draft.  With p_i = softmax(target row i / T), q_i = softmax(draft row i / Td):
// x_i is accepted when all before it were and u_i q_i(x_i) < p_i(x_i).  With a drafts accepted, the next token is drawn by
// inverse CDF with v from p_n when a == n, else from max(p_a - q_a, 0): the committed tokens are then samples of the target.
// A temperature below 1e-5 is a point mass at the lowest most likely index.  A row with a NaN says as little as one without a logit above -inf.
//
// chain_stats_kernel reads the rows of some drafts (maximum, sum of exponentials) and decides about them; chain_token_kernel draws
// the token, a cluster per sequence.  A block of the first kernel asks whether an earlier draft of its sequence is known to be
// rejected before it reads; blocks start in the order of their drafts, eight at a time, so that most rows behind a rejection are not
// read (64 chains of 4 to 16 drafts over 151936 fp32 values 149 us; four at a time 157, sixteen 150, all 170).  Sums that only decide
// `u q < p` are fp32: a probability is off by some 1e-6 of itself at most (a term e bits below the maximum by 3.5 e 2^-24 of itself, the
// hardware's exponential by 2^-22, what is added up by a few 2^-24); the drafted token's own exponential is fp64.  The running sum
// that a token is found in is fp64, as its index would change with every rounding among 150,000 terms.
//
// What bounds it: few sequences, latency (one chain of 3 drafts 25 us, 12 us in either kernel); many, reading (90 of those 149 us) and
// the draw (60 us), whose warps wait for values, barriers of the cluster and fp64 chains (16 sequences: fp64 pipe 30 % of the time that
// an SM has work, 47 % on the busiest SM).
#include "common.cuh"

#include <math.h>
#include <type_traits>

namespace js {

// A block of the first kernel reads 16 KB of either row at once.  fp32: 128 threads, six blocks an SM (64 sequences 149 us, 167 with four of 256
// threads); bf16 has twice the values, that want the registers of 256 threads (16 sequences 55 us, 74 with 128).
constexpr int kChunkBytes = 16384;
template <typename T>
struct StatShape { static constexpr int kThreads = 256, kResident = 4; };
template <>
struct StatShape<float> { static constexpr int kThreads = 128, kResident = 6; };
constexpr int kAhead = 8;            // drafts of a sequence that blocks of their own read
constexpr int kChainThreads = 512;
constexpr double kGreedyBelow = 1e-5;      // fp32 1e-5 lies below it
constexpr int kNoneRejected = 0x7fffffff;

struct ChainParams {
  const void *target, *draft;          // (D + B, V), (D, V)
  long long ldt, ldd;
  const int *drafts, *cu;              // (D), (B + 1)
  const float *accept_u, *sample_u;    // (D), (B)
  const float *temp, *draft_temp;      // (B), or null: the scalars
  double temp_all, draft_temp_all;
  float4* stats;                       // (rows, chunks) of both matrices, the draft's behind the target's: maximum, sum, index of the maximum;
                                       // chunk 0 has the row's own figures in the end
  int* rejected;                       // (B) kNoneRejected - i for the first draft i known to be rejected, 0: none; zero at the start
  int* arrived;                        // (D + B) chunks of a target row (and its draft row) that are there; zero at the start
  int* accepted;
  long long* token;
  int* status;
  int B, D, V, chunks;
};

template <typename T>
JS_DEVICE float chain_f(T v);
template <>
JS_DEVICE float chain_f<float>(float v) { return v; }
template <>
JS_DEVICE float chain_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr double kLog2e = 1.4426950408889634, kHottest = 1e30;      // temperatures end there
JS_DEVICE double chain_temp(const float* each, double all, int b) { return fmin(each != nullptr ? each[b] : all, kHottest); }

// drafts of sequence b: first and number (bad offsets are cut to what is there)
JS_DEVICE int chain_span(const ChainParams& p, int b, int& first) {
  first = min(max(p.cu[b], 0), p.D);
  return max(0, min(p.cu[b + 1], p.D) - first);
}

// log2(e) / T.  Exponents of a row's sum are (x - maximum) * scale, subtracted first: so nothing overflows, and a row that a large finite mask
// fills says what it says (one operation a value more than a rounded base costs 64 sequences 2 of 149 us).  An exponent of -e bits is off by 5 e 2^-24
// at most: half a step each for T, log2(e), their quotient, the difference and the product.
JS_DEVICE float chain_scale(double temp) { return temp < kGreedyBelow ? 1.f : static_cast<float>(kLog2e) / static_cast<float>(temp); }
JS_DEVICE float chain_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

JS_DEVICE float chain_max(float a, float b) {      // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
struct RowStat { float m, s; int at; };      // maximum (NaN if a logit is), sum of the exponentials relative to it, lowest index of the maximum
JS_DEVICE RowStat join(const RowStat& a, const RowStat& b, float scale) {
  RowStat r;
  r.m = chain_max(a.m, b.m);
  r.at = a.m > b.m ? a.at : b.m > a.m ? b.at : min(a.at, b.at);
  r.s = (a.m == r.m ? a.s : a.s != 0.f ? a.s * chain_exp2((a.m - r.m) * scale) : 0.f) +
        (b.m == r.m ? b.s : b.s != 0.f ? b.s * chain_exp2((b.m - r.m) * scale) : 0.f);
  return r;
}
JS_DEVICE RowStat warp_join(RowStat r, float scale) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const RowStat other{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o), __shfl_xor_sync(0xffffffffu, r.at, o)};
    r = join(r, other, scale);
  }
  return r;
}

// probability of the element at `index`, whose logit is `x`
JS_DEVICE double chain_prob(float x, int index, double temp, const RowStat& st) {
  if (temp < kGreedyBelow) return index == st.at ? 1.0 : 0.0;
  return st.s != 0.f ? exp2((static_cast<double>(x) - st.m) * (kLog2e / temp)) / st.s : 0.0;      // NaN beside a logit of +inf
}

// A row as the 16-byte blocks that hold it: a copy starts and ends with a block, and never leaves the blocks that the row has a part in.
struct ChainRow {
  const uint8_t* start;
  int bytes, ahead;            // of all blocks; values of the first block ahead of the row
  template <typename T>
  JS_DEVICE void set(const T* row, int V) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15);
    start = reinterpret_cast<const uint8_t*>(from);
    ahead = static_cast<int>(reinterpret_cast<uintptr_t>(row) - from) / static_cast<int>(sizeof(T));
    bytes = (static_cast<int>((ahead + V) * sizeof(T)) + 15) & ~15;
  }
};

JS_DEVICE float chain_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
JS_DEVICE float warp_max_f32(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// One chunk of the rows of drafts z, z + Z, ... of a sequence: block (chunk, sequence, z).
template <typename T>
__global__ void __launch_bounds__(StatShape<T>::kThreads, StatShape<T>::kResident) chain_stats_kernel(ChainParams p) {
  constexpr int N = 16 / sizeof(T), kStatThreads = StatShape<T>::kThreads, kStatBlocks = kChunkBytes / 16 / kStatThreads, kWarps = kStatThreads / 32;
  __shared__ float tops[2][kWarps], sums[2][kWarps];
  __shared__ int where[2], go;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, chunk = blockIdx.x, b = blockIdx.y;
  pdl_launch_dependents();
  int first;
  const int n = chain_span(p, b, first);
  if (static_cast<int>(blockIdx.z) > n) return;
  const double temps[2] = {chain_temp(p.temp, p.temp_all, b), chain_temp(p.draft_temp, p.draft_temp_all, b)};
  const float scales[2] = {chain_scale(temps[0]), chain_scale(temps[1])};
  for (int i = blockIdx.z; i <= n; i += gridDim.z) {
    // Behind a known rejection nobody needs the rows; whether they are read all the same goes by time, results do not.
    __syncthreads();
    if (tid == 0) go = kNoneRejected - *reinterpret_cast<volatile int*>(p.rejected + b) >= i;
    if (tid < 2) where[tid] = 0x7fffffff;
    __syncthreads();
    if (!go) return;
    const long long trow = static_cast<long long>(first) + b + i, drow = static_cast<long long>(first) + i;
    const T* rows[2] = {reinterpret_cast<const T*>(p.target) + trow * p.ldt, reinterpret_cast<const T*>(p.draft) + drow * p.ldd};
    uint4 raw[2][kStatBlocks];
    int ahead[2];
#pragma unroll
    for (int row = 0; row < 2; ++row) {
      ChainRow r{nullptr, 0, 0};
      if (row == 0 || i < n) r.set(rows[row], p.V);
      ahead[row] = r.ahead;
      const int left = r.bytes - chunk * kChunkBytes;
#pragma unroll
      for (int q = 0; q < kStatBlocks; ++q) {
        const int at = (q * kStatThreads + tid) * 16;
        constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;      // -inf
        raw[row][q] = make_uint4(kNone, kNone, kNone, kNone);
        if (at < left) raw[row][q] = __ldg(reinterpret_cast<const uint4*>(r.start + static_cast<size_t>(chunk) * kChunkBytes + at));
      }
    }
    constexpr int kChunk = kChunkBytes / static_cast<int>(sizeof(T));
    auto value = [&](int row, int q, int c) {  // value c of this thread's block q
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[row][q]);
      if constexpr (sizeof(T) == 4) return __uint_as_float(w[c]);
      else return __uint_as_float(c & 1 ? w[c >> 1] & 0xffff0000u : w[c >> 1] << 16);
    };
    auto index = [&](int row, int q, int c) { return chunk * kChunk + (q * kStatThreads + tid) * N + c - ahead[row]; };
#pragma unroll
    for (int row = 0; row < 2; ++row) {
      if (ahead[row] == 0 && (chunk + 1) * kChunk <= p.V) continue;
      // a chunk at an end of the row: what is not the row's is -inf
#pragma unroll
      for (int q = 0; q < kStatBlocks; ++q) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&raw[row][q]);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const int at = index(row, q, c);
          if (at >= 0 && at < p.V) continue;
          if constexpr (sizeof(T) == 4) w[c] = 0xff800000u;
          else w[c >> 1] = c & 1 ? (w[c >> 1] & 0xffffu) | 0xff800000u : (w[c >> 1] & 0xffff0000u) | 0xff80u;
        }
      }
    }
    float tops2[2];
#pragma unroll
    for (int row = 0; row < 2; ++row) {
      float top = -INFINITY;
#pragma unroll
      for (int q = 0; q < kStatBlocks; ++q)
#pragma unroll
        for (int c = 0; c < N; c += 2) top = chain_max3(top, value(row, q, c), value(row, q, c + 1));
      top = warp_max_f32(top);
      if (lane == 0) tops[row][warp] = top;
    }
    __syncthreads();
#pragma unroll
    for (int row = 0; row < 2; ++row) {
      float top = warp_max_f32(tops[row][lane % kWarps]);
      if (row == 1 && i == n) top = -INFINITY;
      tops2[row] = top;
      float sum = 0.f;
      if (top != -INFINITY) {
        float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < kStatBlocks; ++q)
#pragma unroll
          for (int c = 0; c < N; ++c) e[c & 3] += chain_exp2((value(row, q, c) - top) * scales[row]);
        sum = (e[0] + e[1]) + (e[2] + e[3]);
        if (temps[row] < kGreedyBelow) {       // only a point mass wants to know where the maximum is
#pragma unroll
          for (int q = 0; q < kStatBlocks; ++q)
#pragma unroll
            for (int c = 0; c < N; ++c) if (value(row, q, c) == top) atomicMin(&where[row], index(row, q, c));
        }
      }
      sum = warp_sum(sum);
      if (lane == 0) sums[row][warp] = sum;
    }
    __syncthreads();
    if (warp != 0) continue;
    RowStat st{tops2[0], 0.f, where[0]}, sd{tops2[1], 0.f, where[1]};
    for (int w = 0; w < kWarps; ++w) {
      st.s += sums[0][w];
      sd.s += sums[1][w];
    }
    float4 *tstat = p.stats + trow * p.chunks, *dstat = p.stats + (p.D + p.B + drow) * p.chunks;
    if (p.chunks > 1) {                        // the last chunk to arrive joins them all, in order
      int there = 0;
      if (lane == 0) {
        __stcg(tstat + chunk, make_float4(st.m, st.s, __int_as_float(st.at), 0.f));
        if (i < n) __stcg(dstat + chunk, make_float4(sd.m, sd.s, __int_as_float(sd.at), 0.f));
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(there) : "l"(p.arrived + trow) : "memory");
      }
      if (__shfl_sync(0xffffffffu, there, 0) != p.chunks - 1) continue;
      __threadfence();
      auto all = [&](const float4* at, float scale) {
        RowStat r{-INFINITY, 0.f, 0x7fffffff};
        for (int c = lane; c < p.chunks; c += 32) {
          const float4 v = __ldcg(at + c);
          r = join(r, RowStat{v.x, v.y, __float_as_int(v.z)}, scale);
        }
        return warp_join(r, scale);
      };
      st = all(tstat, scales[0]);
      if (i < n) sd = all(dstat, scales[1]);
      __syncwarp();
    }
    if (lane != 0) continue;
    // a row with a NaN says as little as one without a logit above -inf
    if (st.m != st.m) st = RowStat{-INFINITY, 0.f, 0x7fffffff};
    if (sd.m != sd.m) sd = RowStat{-INFINITY, 0.f, 0x7fffffff};
    tstat[0] = make_float4(st.m, st.s, __int_as_float(st.at), 0.f);
    if (i == n) continue;
    dstat[0] = make_float4(sd.m, sd.s, __int_as_float(sd.at), 0.f);
    const int tok = p.drafts[drow];
    const bool known = tok >= 0 && tok < p.V;
    if (!known) report(p.status, kBadToken);
    if (!known || !(p.accept_u[drow] * chain_prob(chain_f(rows[1][tok]), tok, temps[1], sd) < chain_prob(chain_f(rows[0][tok]), tok, temps[0], st)))
      atomicMax(p.rejected + b, kNoneRejected - i);
  }
}

// 2^(t / 512) for t from -512 * 1020 to 0 (results stay above the smallest normal number, 2^-1022): t = n + r, a table of 2^(j/512) and the
// series of 2^(r/512) to the second power, |r| <= 1/2 (P. Tang's table-driven scheme): relative error below 6e-11, of either sign.
constexpr int kExpTable = 512;
// Probabilities are cut below 2^-790 of the most likely one's, and count there as something from 2^-990 to 2^-790: divided by a sum of up to 2^28
// terms they stay in the table's domain, and that many of them add up to less than 2^-760, below which a sum counts as zero.
constexpr double kCut = -790.0 * kExpTable, kNoSum = 0x1p-760;
JS_DEVICE double exp2_table(double t, const double* table) {
  constexpr double kRound = 6755399441055744.0;              // 1.5 * 2^52: the integer part of the sum's low word
  constexpr double c1 = 0.69314718055994531 / kExpTable;
  const double shifted = t + kRound;
  const int n = __double2loint(shifted);
  const double r = t - (shifted - kRound);
  const double e = fma(r, fma(r, c1 * c1 / 2.0, c1), 1.0) * table[n & (kExpTable - 1)];
  return __hiloint2double(__double2hiint(e) + ((n >> 9) << 20), __double2loint(e));
}

// Table steps a logit, and half the logit at which a row is cut, rounded down (logits are halved, so that the cut of any finite maximum is finite and
// -inf lies below it).  Where the next value below the maximum has 2^-100 of its probability or less, that is as good as nothing: the slope stops
// there, so that rounding takes the cut down by 2^-200 at most (below a negative power of two values lie twice as far from each other as above).
struct ChainAxis {
  double slope;
  float least;
  JS_DEVICE ChainAxis(float top, double temp) {
    const double step = top == -3.402823466e38f ? 0x1p104 : static_cast<double>(top) - nextafterf(top, -INFINITY);
    slope = fmin(kExpTable * kLog2e / temp, 100.0 * kExpTable / step);
    least = __double2float_rd(0.5 * (top + kCut / slope));
  }
};

// CLUSTER CTAs share a sequence's last row.
template <typename T, int CLUSTER>
__global__ void __launch_bounds__(kChainThreads, 2) chain_token_kernel(ChainParams p) {
  constexpr int kWarps = kChainThreads / 32;
  __shared__ double table[kExpTable], part[kWarps], part2[kWarps], sums[CLUSTER][2];
  __shared__ int passing, holding;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  const int b = blockIdx.x / CLUSTER;
  static_assert(kExpTable == kChainThreads, "an entry a thread");
  table[tid] = exp2(static_cast<double>(tid) / kExpTable);
  if (tid == 0) {
    passing = 0x7fffffff;
    holding = -1;
  }
  pdl_wait();
  int first;
  const int n = chain_span(p, b, first);
  const double tt = chain_temp(p.temp, p.temp_all, b), td = chain_temp(p.draft_temp, p.draft_temp_all, b);
  const int a = min(n, kNoneRejected - p.rejected[b]);
  const bool left = a < n;                // draw from the difference
  const long long trow = first + b + a, drow = first + a;
  const float4 tstat = p.stats[trow * p.chunks], dstat = left ? p.stats[(p.D + p.B + drow) * p.chunks] : make_float4(0.f, 0.f, 0.f, 0.f);
  const int t_at = __float_as_int(tstat.z), d_at = __float_as_int(dstat.z);      // where a point mass lies
  if (rank == 0 && tid == 0) p.accepted[b] = a;
  __syncthreads();
  const T* x = reinterpret_cast<const T*>(p.target) + trow * p.ldt;
  const T* y = reinterpret_cast<const T*>(p.draft) + drow * p.ldd;
  if (tt < kGreedyBelow || tstat.x == -INFINITY) {              // the same for the whole cluster; without a logit above -inf: no token
    if (rank == 0 && tid == 0) p.token[b] = t_at < p.V ? t_at : -1;
    return;
  }
  // The draft's share of a weight: none behind the last draft and beside a row without a logit above -inf; a point mass takes all of its index
  // (p <= 1) and nothing elsewhere.
  const bool point = left && td < kGreedyBelow, both = left && !point && dstat.x != -INFINITY;
  const int skip = point ? d_at : -1;
  const ChainAxis ta(tstat.x, tt), da(both ? dstat.x : 0.f, td);
  double tc = -tstat.x * ta.slope, dc = both ? -dstat.x * da.slope : 0.0;
  auto ep = [&](float v) { return exp2_table(fma(static_cast<double>(fmaxf(0.5f * v, ta.least)), 2.0 * ta.slope, tc), table); };
  auto eq = [&](float v) { return exp2_table(fma(static_cast<double>(fmaxf(0.5f * v, da.least)), 2.0 * da.slope, dc), table); };
  // A CTA takes a slice of the vocabulary and a warp a slice of that, so sums follow the order of the indices.
  const int lo = static_cast<long long>(p.V) * rank / CLUSTER, size = static_cast<int>(static_cast<long long>(p.V) * (rank + 1) / CLUSTER) - lo;
  auto warp_lo = [&](int w) { return lo + static_cast<int>(static_cast<long long>(size) * w / kWarps); };
  // f(index, target logit, draft logit) for this warp's elements; four at a time, as fp64 chains are long
  auto each = [&](auto two, auto f) {
    constexpr bool kTwo = decltype(two)::value;
    const int end = warp_lo(warp + 1);
    int i = warp_lo(warp) + lane;
    for (; i + 96 < end; i += 128) {
      float v[4], w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = chain_f(x[i + 32 * j]);
        w[j] = kTwo ? chain_f(y[i + 32 * j]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i + 32 * j, v[j], w[j]);
    }
    for (; i < end; i += 32) f(i, chain_f(x[i]), kTwo ? chain_f(y[i]) : 0.f);
  };
  // the warps' sums into `to`; their sum in order
  auto block_sum = [&](double v, double* to) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) to[warp] = v > kNoSum ? v : 0.0;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kWarps; ++w) v += to[w];
    return v;
  };
  // this CTA's pair of sums to every CTA of the cluster
  auto exchange = [&](double s0, double s1) {
    cluster_sync();                       // every CTA of the cluster runs, and is done with the sums of before
    if (tid < CLUSTER) {
      const uint32_t at = map_to_cta(smem_u32(&sums[rank][0]), tid);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(s0) : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at + 8), "d"(s1) : "memory");
    }
    __syncwarp();
    cluster_sync();
  };
  double sum = 0.0;
  if (both) {
    double sp = 0.0, sq = 0.0;
    each(std::true_type{}, [&](int, float v, float w) {
      sp += ep(v);
      sq += eq(w);
    });
    sp = block_sum(sp, part);
    sq = block_sum(sq, part2);
    exchange(sp, sq);
    sp = sq = 0.0;
    for (int c = 0; c < CLUSTER; ++c) {
      sp += sums[c][0];
      sq += sums[c][1];
    }
    tc -= kExpTable * log2(sp);           // probabilities from here on
    dc -= kExpTable * log2(sq);
    each(std::true_type{}, [&](int, float v, float w) { sum += fmax(ep(v) - eq(w), 0.0); });
  } else {
    each(std::false_type{}, [&](int i, float v, float) { sum += i != skip ? ep(v) : 0.0; });
  }
  auto weight = [&](int i) {
    const float v = chain_f(x[i]);
    if (!(0.5f * v > ta.least) || i == skip) return 0.0;
    return both ? fmax(ep(v) - eq(chain_f(y[i])), 0.0) : ep(v);
  };
  sum = block_sum(sum, part);
  exchange(sum, 0.0);
  double total = 0.0;
  for (int c = 0; c < CLUSTER; ++c) total += sums[c][0];
  if (!(total > 0.0)) {                   // rounding left nothing of the difference: the target's most likely token
    if (rank != 0) return;
    for (int i = p.V - 1 - tid; i >= 0; i -= kChainThreads) if (chain_f(x[i]) == tstat.x) atomicMin(&passing, i);
    __syncthreads();
    if (tid == 0) p.token[b] = passing < p.V ? passing : -1;
    return;
  }
  // The first of `count` parts whose running sum passes the goal, or (where rounding lets none pass it) the last one with a weight;
  // `run` becomes the sum ahead of it.
  const double goal = static_cast<double>(p.sample_u[b]) * total;
  auto find = [&](int count, auto value, double& run) {
    int last = 0;
    double ahead = run;
    for (int c = 0; c < count; ++c) {
      const double v = value(c);
      if (v > 0.0) {
        last = c;
        ahead = run;
        if (run + v > goal) break;
      }
      run += v;
    }
    run = ahead;
    return last;
  };
  double run = 0.0;
  if (find(CLUSTER, [&](int c) { return sums[c][0]; }, run) != rank) return;
  const int w = find(kWarps, [&](int c) { return part[c]; }, run);
  // the warp's slice once more, a few neighbouring elements a thread
  const int from = warp_lo(w), to = warp_lo(w + 1), per = (to - from + kChainThreads - 1) / kChainThreads;
  const int mine = min(to, from + tid * per), stop = min(to, mine + per);
  sum = 0.0;
  for (int i = mine; i < stop; ++i) sum += weight(i);
  double inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += other;
  }
  __syncthreads();
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  double ahead = run;
  for (int c = 0; c < warp; ++c) ahead += part[c];
  if (sum > 0.0) {
    if (ahead + inc > goal) atomicMin(&passing, tid);
    atomicMax(&holding, tid);
  }
  __syncthreads();
  if (tid == (passing != 0x7fffffff ? passing : holding)) {
    ahead += inc - sum;
    p.token[b] = mine + find(stop - mine, [&](int c) { return weight(mine + c); }, ahead);
  }
}

template <typename T, int CLUSTER>
static int launch_token(const ChainParams& p, cudaStream_t stream) {
  auto kern = chain_token_kernel<T, CLUSTER>;
  if (CLUSTER > 8) {
    static int allowed[kMaxDevicesCached] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -3;
    if (dev >= kMaxDevicesCached || !__atomic_load_n(&allowed[dev], __ATOMIC_ACQUIRE)) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return -3;
      if (dev < kMaxDevicesCached) __atomic_store_n(&allowed[dev], 1, __ATOMIC_RELEASE);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.B * CLUSTER);
  cfg.blockDim = dim3(kChainThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CLUSTER;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? 0 : -5;
}

template <typename T>
static int launch_chain(const ChainParams& p, cudaStream_t stream) {
  chain_stats_kernel<T><<<dim3(p.chunks, p.B, kAhead), StatShape<T>::kThreads, 0, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return -4;
  // As many CTAs a sequence as are there at once, two an SM (16 is more than a portable cluster has).  us with 16, 8, 4 and 2: one sequence 25, 29, 38,
  // 56; 16 sequences 54, 59, 63, 86; 48 (32001 words) 54, 39, 38, 39; 64 184, 158, 149, 170.
  constexpr int kAtOnce = 2 * 148;
  if (p.B * 16 <= kAtOnce) return launch_token<T, 16>(p, stream);
  return p.B * 8 <= kAtOnce ? launch_token<T, 8>(p, stream) : launch_token<T, 4>(p, stream);
}

}  // namespace js

// Float4s of scratch for `rows` rows of V values: a chunk each.
static int chain_chunks(int V, int size) { return (V * size + 15 + js::kChunkBytes) / js::kChunkBytes; }
extern "C" long long js_chain_verify_ws(int B, int D, int V, int is_bf16) {
  return (2ll * D + B) * chain_chunks(V, is_bf16 ? 2 : 4) * 16 + (static_cast<long long>(D) + 2 * B) * 4;
}

// target (D + B, V), draft (D, V) fp32 or bf16 (is_bf16), rows ldt / ldd elements apart; drafts (D), cu (B + 1) int32; accept_u (D),
// sample_u (B) fp32 in [0, 1); temp, draft_temp (B) fp32 or null (the scalars hold).  ws: js_chain_verify_ws bytes.  accepted (B) int32, token
// (B) int64.
extern "C" int js_chain_verify(const void* target, long long ldt, const void* draft, long long ldd, int is_bf16, const int* drafts,
                               const int* cu, const float* accept_u, const float* sample_u, const float* temp, double temp_all,
                               const float* draft_temp, double draft_temp_all, void* ws, int* accepted, long long* token,
                               int* status, int B, int D, int V, cudaStream_t stream) {
  using namespace js;
  if (B < 0 || B > 0xffff || D < 0 || V < 1 || V > (1 << 28)) return -10;
  if (B == 0) return 0;
  const int chunks = chain_chunks(V, is_bf16 ? 2 : 4);
  float4* stats = reinterpret_cast<float4*>(ws);
  int* rejected = reinterpret_cast<int*>(stats + (2ll * D + B) * chunks);
  ChainParams p{target, draft, ldt, ldd, drafts, cu, accept_u, sample_u, temp, draft_temp, temp_all, draft_temp_all,
                stats, rejected, rejected + B, accepted, token, status, B, D, V, chunks};
  if (cudaMemsetAsync(rejected, 0, sizeof(int) * (static_cast<size_t>(D) + 2 * B), stream) != cudaSuccess) return -3;
  return is_bf16 ? launch_chain<__nv_bfloat16>(p, stream) : launch_chain<float>(p, stream);
}

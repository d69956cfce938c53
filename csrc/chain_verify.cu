// Drafted chains against the target's probabilities, from given random numbers.
//
// Sequence b drafted x_0 .. x_{n-1}; draft row i holds the logits x_i was drawn from, target row i the target's logits at the same
// place, and one more target row stands behind the last draft.  With p_i = softmax(target row i / T), q_i = softmax(draft row i / Td):
// x_i is accepted when all before it were and u_i q_i(x_i) < p_i(x_i).  With a drafts accepted, the next token is drawn by
// inverse CDF with v from p_n when a == n, else from max(p_a - q_a, 0): the committed tokens are then samples of the target.
// A temperature below 1e-5 is a point mass at the lowest most likely index.
//
// Two launches.  chain_stats_kernel reads the rows once (maximum, sum of exponentials, index of the maximum), the rows of the first
// drafts before those of later ones; a row behind a draft already known to be rejected is left out.  chain_token_kernel decides, and draws the
// token with a cluster per sequence.  Sums that only decide `u q < p` are fp32 (a decision is off by 1e-7 of a probability); the
// running sum that a token is found in is fp64, as its index would change with every rounding among 150,000 terms.
#include "common.cuh"

#include <math.h>

namespace js {

constexpr int kChainThreads = 512;
constexpr int kChainCluster = 8;      // CTAs that share a sequence's last row
constexpr float kGreedyBelow = 1e-5f;

struct ChainParams {
  const void *target, *draft;          // (D + B, V), (D, V)
  long long ldt, ldd;
  const int *drafts, *cu;              // (D), (B + 1)
  const float *accept_u, *sample_u;    // (D), (B)
  const float *temp, *draft_temp;      // (B), or null: the scalars
  double temp_all, draft_temp_all;
  float4* stats;                       // (rows, chunks) of both matrices, the draft's behind the target's: maximum, sum, index of the maximum
  int* rejected;                       // (B) a bound on the first rejected draft (all ones bytes 0x7f: none known)
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

JS_DEVICE double chain_temp(const float* each, double all, int b) { return each != nullptr ? each[b] : all; }

// drafts of sequence b: first and number (bad offsets are cut to what is there)
JS_DEVICE int chain_span(const ChainParams& p, int b, int& first) {
  first = min(max(p.cu[b], 0), p.D);
  return max(0, min(p.cu[b + 1], p.D) - first);
}

// Base-2 exponent of a difference of logits: log2(e) / T as the sum of two fp32, so that the factor's rounding does not weigh on every term
struct ChainScale { float hi, lo; };
JS_DEVICE ChainScale chain_scale(double temp) {
  const double f = temp < kGreedyBelow ? 1.0 : 1.4426950408889634 / temp;
  const float hi = static_cast<float>(f);
  return ChainScale{hi, static_cast<float>(f - hi)};
}
JS_DEVICE float chain_exp(float d, const ChainScale& f) {
  d = fmaxf(d, -1e30f);      // -inf would meet the other part's sign
  return exp2f(fmaf(d, f.hi, d * f.lo));
}

struct RowStat { float m, s; int at; };      // maximum, sum of the exponentials relative to it, lowest index of the maximum
JS_DEVICE RowStat join(const RowStat& a, const RowStat& b, const ChainScale& f) {
  RowStat r;
  r.m = fmaxf(a.m, b.m);
  r.at = a.m > b.m ? a.at : b.m > a.m ? b.at : min(a.at, b.at);
  r.s = (a.m == r.m ? a.s : a.s != 0.f ? a.s * chain_exp(a.m - r.m, f) : 0.f) +
        (b.m == r.m ? b.s : b.s != 0.f ? b.s * chain_exp(b.m - r.m, f) : 0.f);
  return r;
}

// The figures of elements [lo, hi) of a row, by the whole block
template <typename T>
JS_DEVICE RowStat row_stat(const T* x, int lo, int hi, const ChainScale& f, RowStat* red) {
  constexpr int N = 16 / sizeof(T);
  RowStat r{-INFINITY, 0.f, 0x7fffffff};
  auto one = [&](float v, int i) {
    if (v > r.m) {
      r.s = r.s * chain_exp(r.m - v, f) + 1.f;
      r.m = v;
      r.at = i;
    } else {
      r.s += chain_exp(v - r.m, f);
    }
  };
  // elements ahead of the first 16-byte boundary, then vectors, then the rest
  const int lead = min(hi - lo, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) & 15) / sizeof(T)));
  const int n_vec = (hi - lo - lead) / N, tail = lo + lead + n_vec * N;
  if (threadIdx.x < lead) one(chain_f(x[lo + threadIdx.x]), lo + threadIdx.x);
  const uint4* v = reinterpret_cast<const uint4*>(x + lo + lead);
#pragma unroll 4
  for (int i = threadIdx.x; i < n_vec; i += kChainThreads) {
    const uint4 w = __ldg(v + i);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < N; ++j) one(chain_f(e[j]), lo + lead + i * N + j);
  }
  if (tail + static_cast<int>(threadIdx.x) < hi) one(chain_f(x[tail + threadIdx.x]), tail + threadIdx.x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const RowStat other{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o), __shfl_xor_sync(0xffffffffu, r.at, o)};
    r = join(r, other, f);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = r;
  __syncthreads();
  r = red[0];
  for (int w = 1; w < kChainThreads / 32; ++w) r = join(r, red[w], f);
  return r;
}

// probability of the element at `index`, whose logit is `x`
JS_DEVICE double chain_prob(float x, int index, double temp, const RowStat& st) {
  if (temp < kGreedyBelow) return index == st.at ? 1.0 : 0.0;
  return st.s > 0.f ? exp2((static_cast<double>(x) - st.m) * (1.4426950408889634 / temp)) / st.s : 0.0;
}

template <typename T>
__global__ void __launch_bounds__(kChainThreads) chain_stats_kernel(ChainParams p) {
  __shared__ RowStat red[kChainThreads / 32];
  __shared__ int longest, known;
  const int tid = threadIdx.x;
  if (tid == 0) longest = 0;
  __syncthreads();
  int most = 0;
  for (int b = tid; b < p.B; b += kChainThreads) { int f; most = max(most, chain_span(p, b, f)); }
  if (most > 0) atomicMax(&longest, most);
  __syncthreads();
  const long long tasks = static_cast<long long>(longest + 1) * p.B * p.chunks;
  for (long long k = blockIdx.x; k < tasks; k += gridDim.x) {
    const int chunk = k % p.chunks, b = (k / p.chunks) % p.B, i = k / p.chunks / p.B;
    int first;
    const int n = chain_span(p, b, first);
    if (i > n) continue;
    __syncthreads();
    if (tid == 0) known = *reinterpret_cast<volatile int*>(p.rejected + b);
    __syncthreads();
    if (known < i) continue;              // nobody needs these rows; whether they are read all the same goes by time, results do not
    const int lo = static_cast<long long>(p.V) * chunk / p.chunks, hi = static_cast<long long>(p.V) * (chunk + 1) / p.chunks;
    const long long trow = first + b + i;
    const T* x = reinterpret_cast<const T*>(p.target) + trow * p.ldt;
    const double tt = chain_temp(p.temp, p.temp_all, b), td = chain_temp(p.draft_temp, p.draft_temp_all, b);
    const RowStat st = row_stat(x, lo, hi, chain_scale(tt), red);
    if (tid == 0) p.stats[trow * p.chunks + chunk] = make_float4(st.m, st.s, __int_as_float(st.at), 0.f);
    if (i == n) continue;
    const long long drow = first + i;
    const T* y = reinterpret_cast<const T*>(p.draft) + drow * p.ldd;
    const RowStat sd = row_stat(y, lo, hi, chain_scale(td), red);
    if (tid == 0) {
      p.stats[(p.D + p.B + drow) * p.chunks + chunk] = make_float4(sd.m, sd.s, __int_as_float(sd.at), 0.f);
      const int tok = p.drafts[drow];
      if (p.chunks == 1 && (tok < 0 || tok >= p.V ||
          !(p.accept_u[drow] * chain_prob(chain_f(y[tok]), tok, td, sd) < chain_prob(chain_f(x[tok]), tok, tt, st))))
        atomicMin(p.rejected + b, i);
    }
  }
}

// 2^t for t <= 0 (0 below 2^-1000): t = n / 32 + r, a table of 2^(j/32) and the series of e^(r ln 2) to the fourth power, |r| <= 1/64
// (P. Tang's table-driven scheme): relative error below 2e-12.
JS_DEVICE double exp2_table(double t, const double* table) {
  if (!(t > -1000.0)) return 0.0;
  const double shifted = t * 32.0 + 6755399441055744.0;      // 1.5 * 2^52: the integer part of the sum's low word
  const int n = __double2loint(shifted);
  const double r = (t * 32.0 - (shifted - 6755399441055744.0)) * (0.69314718055994531 / 32.0);
  const double e = fma(r, fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0);
  const double scale = __hiloint2double(((n >> 5) + 1023) << 20, 0);
  return e * table[n & 31] * scale;
}

template <typename T>
__global__ void __launch_bounds__(kChainThreads) chain_token_kernel(ChainParams p) {
  constexpr int kWarps = kChainThreads / 32;
  __shared__ double table[32], part[kWarps], sums[kChainCluster][2];
  __shared__ RowStat tstat, dstat;
  __shared__ int first_bad, passing, holding;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  const int b = blockIdx.x / kChainCluster;
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  int first;
  const int n = chain_span(p, b, first);
  const double tt = chain_temp(p.temp, p.temp_all, b), td = chain_temp(p.draft_temp, p.draft_temp_all, b);
  const T* target = reinterpret_cast<const T*>(p.target);
  const T* draft = reinterpret_cast<const T*>(p.draft);
  auto stat_of = [&](long long row, const ChainScale& f) {
    RowStat r{-INFINITY, 0.f, 0x7fffffff};
    for (int c = 0; c < p.chunks; ++c) {
      const float4 v = p.stats[row * p.chunks + c];
      r = join(r, RowStat{v.x, v.y, __float_as_int(v.z)}, f);
    }
    return r;
  };
  const ChainScale tf = chain_scale(tt), df = chain_scale(td);
  if (tid == 0) {
    first_bad = min(n, p.rejected[b]);
    passing = 0x7fffffff;
    holding = -1;
  }
  __syncthreads();
  // Every CTA of the cluster decides for itself.  Rows behind the first rejection may hold no figures: what is decided there does not count.
  for (int i = tid; i < n; i += kChainThreads) {
    const int tok = p.drafts[first + i];
    const long long trow = first + b + i, drow = first + i;
    bool good = tok >= 0 && tok < p.V;
    if (good)
      good = p.accept_u[drow] * chain_prob(chain_f(draft[drow * p.ldd + tok]), tok, td, stat_of(p.D + p.B + drow, df)) <
             chain_prob(chain_f(target[trow * p.ldt + tok]), tok, tt, stat_of(trow, tf));
    else if (rank == 0)
      report(p.status, kBadToken);
    if (!good) atomicMin(&first_bad, i);
  }
  __syncthreads();
  const int a = first_bad;
  const bool left = a < n;                // draw from the difference
  const long long trow = first + b + a, drow = first + a;
  if (tid == 0) {
    tstat = stat_of(trow, tf);
    if (left) dstat = stat_of(p.D + p.B + drow, df);
    if (rank == 0) p.accepted[b] = a;
  }
  __syncthreads();
  const T* x = target + trow * p.ldt;
  const T* y = draft + drow * p.ldd;
  const int most_likely = tstat.at < p.V ? tstat.at : -1;       // -1: no index has a probability
  if (tt < kGreedyBelow || most_likely < 0) {                   // the same for the whole cluster
    if (rank == 0 && tid == 0) p.token[b] = most_likely;
    return;
  }
  const double ts = 1.4426950408889634 / tt, ds = 1.4426950408889634 / td;
  const float tm = tstat.m, dm = left ? dstat.m : 0.f;
  const bool draft_point = td < kGreedyBelow;
  auto ep = [&](int i) { return exp2_table((static_cast<double>(chain_f(x[i])) - tm) * ts, table); };
  auto eq = [&](int i) {
    return draft_point ? (i == dstat.at ? 1.0 : 0.0) : exp2_table((static_cast<double>(chain_f(y[i])) - dm) * ds, table);
  };
  // A CTA takes a slice of the vocabulary and a warp a slice of that, so sums follow the order of the indices.
  const int lo = static_cast<long long>(p.V) * rank / kChainCluster, size = static_cast<int>(static_cast<long long>(p.V) * (rank + 1) / kChainCluster) - lo;
  auto warp_lo = [&](int w) { return lo + static_cast<int>(static_cast<long long>(size) * w / kWarps); };
  auto warp_sum64 = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  // the warps' sums into `part`; their sum in order
  auto block_sum = [&](double v) {
    v = warp_sum64(v);
    __syncthreads();
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kWarps; ++w) v += part[w];
    return v;
  };
  // this CTA's pair of sums to every CTA of the cluster
  auto exchange = [&](double s0, double s1) {
    cluster_sync();                       // every CTA of the cluster runs, and is done with the sums of before
    if (tid < kChainCluster) {
      const uint32_t at = map_to_cta(smem_u32(&sums[rank][0]), tid);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(s0) : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at + 8), "d"(s1) : "memory");
    }
    __syncwarp();
    cluster_sync();
  };
  double ip = 1.0, iq = 0.0;
  if (left) {
    double sp = 0.0, sq = 0.0;
    for (int i = lo + tid; i < lo + size; i += kChainThreads) {
      sp += ep(i);
      sq += eq(i);
    }
    sp = block_sum(sp);
    sq = block_sum(sq);
    exchange(sp, sq);
    sp = sq = 0.0;
    for (int c = 0; c < kChainCluster; ++c) {
      sp += sums[c][0];
      sq += sums[c][1];
    }
    ip = 1.0 / sp;
    iq = sq > 0.0 ? 1.0 / sq : 0.0;
  }
  auto weight = [&](int i) {
    const double w = left ? ep(i) * ip - eq(i) * iq : ep(i);
    return w > 0.0 ? w : 0.0;
  };
  double sum = 0.0;
  for (int i = warp_lo(warp) + lane; i < warp_lo(warp + 1); i += 32) sum += weight(i);
  sum = block_sum(sum);
  exchange(sum, 0.0);
  double total = 0.0;
  for (int c = 0; c < kChainCluster; ++c) total += sums[c][0];
  if (!(total > 0.0)) {                   // rounding left nothing of the difference
    if (rank == 0 && tid == 0) p.token[b] = most_likely;
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
  if (find(kChainCluster, [&](int c) { return sums[c][0]; }, run) != rank) return;
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
    const int i = find(stop - mine, [&](int c) { return weight(mine + c); }, ahead);
    p.token[b] = mine + i;
  }
}

template <typename T>
static int launch_chain(const ChainParams& p, int grid, cudaStream_t stream) {
  chain_stats_kernel<T><<<grid, kChainThreads, 0, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return -4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.B * kChainCluster);
  cfg.blockDim = dim3(kChainThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kChainCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, chain_token_kernel<T>, p) == cudaSuccess ? 0 : -5;
}

}  // namespace js

// target (D + B, V), draft (D, V) fp32 or bf16 (is_bf16), rows ldt / ldd elements apart; drafts (D), cu (B + 1) int32; accept_u (D),
// sample_u (B) fp32 in [0, 1); temp, draft_temp (B) fp32 or null (the scalars hold).  stats: (2 D + B) * chunks float4,
// rejected: B ints, both scratch.  accepted (B) int32, token (B) int64.
extern "C" int js_chain_verify(const void* target, long long ldt, const void* draft, long long ldd, int is_bf16, const int* drafts,
                               const int* cu, const float* accept_u, const float* sample_u, const float* temp, double temp_all,
                               const float* draft_temp, double draft_temp_all, void* stats, int* rejected, int* accepted, long long* token,
                               int* status, int B, int D, int V, int chunks, int grid, cudaStream_t stream) {
  using namespace js;
  if (B < 0 || D < 0 || V < 1 || chunks < 1 || grid < 1) return -10;
  if (B == 0) return 0;
  ChainParams p{target, draft, ldt, ldd, drafts, cu, accept_u, sample_u, temp, draft_temp, temp_all, draft_temp_all,
                reinterpret_cast<float4*>(stats), rejected, accepted, token, status, B, D, V, chunks};
  if (cudaMemsetAsync(rejected, 0x7f, sizeof(int) * B, stream) != cudaSuccess) return -3;
  return is_bf16 ? launch_chain<__nv_bfloat16>(p, grid, stream) : launch_chain<float>(p, grid, stream);
}

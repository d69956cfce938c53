// Pages, slot maps and the rows of a forward from request lengths, on the device.
//
// Request b holds slots for its first m_b positions (whole pages of s), has p_b committed ones and gets c_b new rows:
//   need_b = max(0, ceil((p_b + c_b) / s) - ceil(m_b / s)),   cu_q, cu_pages = running sums of c and need.
// Page k of its new ones is free_pages[cu_pages[b] + k]; the new positions' entries of the slot map, and position and slot of
// every new row, follow from that without reading what another block writes (rows below ceil(m_b / s) * s read entries that
// the launch leaves alone).  So one launch does everything: a block serves one request, and sums the requests before it for
// itself (12 bytes a request out of L2), which costs less than a second launch or a look-back chain for the batches that a
// server runs.  Bound by launch latency until slot maps of megabytes are written (16 requests of a row each: 3.3 us).  Four neighbours share a
// division and a page number and leave in one 16-byte store: 256 prompts, 25 MB of slot map and rows, 14 us (25 us with a store a value).
#include "common.cuh"

namespace js {

constexpr int kPlanThreads = 256;

struct SlotPlan {
  const int *past, *counts, *mapped, *rows, *free_pages;
  int *slot_map, *cu_q, *cu_pages, *positions, *slots, *status;
  int B, F, page, max_seqs, max_len, T;
};

JS_DEVICE unsigned pages_of(unsigned positions, unsigned page) { return positions / page + (positions % page != 0u); }
JS_DEVICE int capped_int(long long v) { return v > 0x7fffffffll ? 0x7fffffff : static_cast<int>(v); }

// rows and new pages of request b (negative lengths count as none)
JS_DEVICE void plan_need(const SlotPlan& p, int b, unsigned& past, unsigned& count, unsigned& held, unsigned& need) {
  past = max(0, p.past[b]);
  count = max(0, p.counts[b]);
  held = pages_of(max(0, p.mapped[b]), p.page);
  const unsigned want = pages_of(past + count, p.page);
  need = want > held ? want - held : 0u;
}

__global__ void __launch_bounds__(kPlanThreads) slot_plan_kernel(SlotPlan p) {
  __shared__ long long sum_q[kPlanThreads / 32], sum_p[kPlanThreads / 32];
  __shared__ int seen_row;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
  if (tid == 0) seen_row = 0;
  __syncthreads();
  const int row = b < p.B ? p.rows[b] : -1;
  long long q = 0, pages = 0;
  bool again = false;
  for (int j = tid; j < b && j < p.B; j += kPlanThreads) {
    unsigned past, count, held, need;
    plan_need(p, j, past, count, held, need);
    q += count;
    pages += need;
    again |= p.rows[j] == row && (count > 0 || need > 0);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    q += __shfl_xor_sync(0xffffffffu, q, o);
    pages += __shfl_xor_sync(0xffffffffu, pages, o);
  }
  if (lane == 0) { sum_q[warp] = q; sum_p[warp] = pages; }
  if (again) seen_row = 1;
  __syncthreads();
  q = pages = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) { q += sum_q[w]; pages += sum_p[w]; }

  unsigned past = 0, count = 0, held = 0, need = 0;
  if (b < p.B) plan_need(p, b, past, count, held, need);
  if (first == 0) {
    p.cu_q[b] = capped_int(q);
    p.cu_pages[b] = capped_int(pages);
    if (b == p.B - 1) { p.cu_q[p.B] = capped_int(q + count); p.cu_pages[p.B] = capped_int(pages + need); }
  }
  const bool sound = row >= 0 && row < p.max_seqs && seen_row == 0;      // a slot-map row serves one request
  if (b < p.B && !sound && first == 0 && (count > 0 || need > 0)) report(p.status, kBadSlot);      // without rows and pages it only fills up a batch
  const unsigned page = p.page;
  // page `k` of the request's new ones
  auto granted = [&](unsigned k) {
    const int id = pages + k < p.F ? p.free_pages[pages + k] : -1;
    if (id < 0) report(p.status, kNoPage);
    return id < 0 ? -1 : id;
  };
  int* map = p.slot_map + (sound ? static_cast<size_t>(row) * p.max_len : 0);
  if (sound) {
    const unsigned long long base = static_cast<unsigned long long>(held) * page;
    const unsigned long long stop = min(base + static_cast<unsigned long long>(need) * page, static_cast<unsigned long long>(p.max_len));
    unsigned long long done = base;
    if ((page | p.max_len) % 4 == 0 && reinterpret_cast<uintptr_t>(map) % 16 == 0) {      // four positions of a page in one store
      for (unsigned long long i = base + 4ull * first; i < stop; i += 4ull * step) {
        const unsigned k = static_cast<unsigned>(i) / page;
        const int id = granted(k - held), at = id * static_cast<int>(page) + static_cast<int>(static_cast<unsigned>(i) - k * page);
        *reinterpret_cast<int4*>(map + i) = id < 0 ? make_int4(-1, -1, -1, -1) : make_int4(at, at + 1, at + 2, at + 3);
      }
      done = stop;
    }
    for (unsigned long long i = done + first; i < stop; i += step) {
      const unsigned k = static_cast<unsigned>(i) / page;
      const int id = granted(k - held);
      map[i] = id < 0 ? -1 : id * static_cast<int>(page) + static_cast<int>(static_cast<unsigned>(i) - k * page);
    }
  }
  // four rows at a time, on 16-byte boundaries of the results
  const long long end = min(q + static_cast<long long>(count), static_cast<long long>(p.T));
  for (long long t0 = (q & ~3ll) + 4ll * first; t0 < end; t0 += 4ll * step) {
    const long long from = max(t0, q), to = min(t0 + 4, end);
    unsigned pos = past + static_cast<unsigned>(from - q), k = pos / page, off = pos - k * page;
    int id = 0;
    bool look = true;
    int at[4], slot[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t0 + j < from || t0 + j >= to) continue;
      at[j] = capped_int(pos);
      slot[j] = -1;
      if (sound && pos < static_cast<unsigned>(p.max_len)) {
        if (k < held) slot[j] = map[pos];
        else {
          if (look) id = granted(k - held);
          look = false;
          if (id >= 0) slot[j] = id * static_cast<int>(page) + static_cast<int>(off);
        }
      } else {
        report(p.status, kBadSlot);
      }
      ++pos;
      if (++off == page) {
        off = 0;
        ++k;
        look = true;
      }
    }
    if (to - from == 4) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(at[0], at[1], at[2], at[3]);
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (t0 + j < from || t0 + j >= to) continue;
        p.positions[t0 + j] = at[j];
        p.slots[t0 + j] = slot[j];
      }
    }
  }
  if (first == 0 && q + count > p.T) report(p.status, kRowsOverflow);
  if (b >= p.B - 1) {      // rows behind the last sequence
    for (long long i = q + count + first; i < p.T; i += step) {
      p.positions[i] = 0;
      p.slots[i] = -1;
    }
  }
}

}  // namespace js

// past, counts, mapped, rows (B); free_pages (F); slot_map (max_seqs, max_len); cu_q, cu_pages (B + 1); positions, slots (T), on
// 16-byte boundaries.  All int32.  `chunks` blocks serve a request.
extern "C" int js_slot_plan(const int* past, const int* counts, const int* mapped, const int* rows, const int* free_pages, int* slot_map,
                            int* cu_q, int* cu_pages, int* positions, int* slots, int* status, int B, int F, int page, int max_seqs,
                            int max_len, int T, int chunks, cudaStream_t stream) {
  using namespace js;
  if (B < 0 || F < 0 || T < 0 || page < 1 || max_seqs < 0 || max_len < 0 || chunks < 1 || B > 65535) return -10;
  SlotPlan p{past, counts, mapped, rows, free_pages, slot_map, cu_q, cu_pages, positions, slots, status, B, F, page, max_seqs, max_len, T};
  slot_plan_kernel<<<dim3(chunks, B > 0 ? B : 1), kPlanThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

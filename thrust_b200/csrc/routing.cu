// Statistics of routing tokens to experts: how many tokens each expert gets, the balance loss, its gradient.
//
// The loss of a sequence is experts / (k n^2) * sum_e count[e] * sum_t p[t][e] with p = softmax(logits), so one pass
// over the logits gives column sums of p, one over the ids a histogram, and both end in `experts` numbers. The backward
// pass is local to a row: p * (w - p . w). All of it is bound by HBM (or by the launch, for a decoding batch).
//
// Layout. A row of logits is spread over 1 to 32 lanes, eight experts to a lane and step, so that a lane loads 16 bytes
// of a 16-bit type at once, sums over a row are shuffles among its lanes, and the column sums stay in the lane's own
// registers for all rows of a CTA. Registers are summed over warps in a fixed order, and the CTAs' sums are added as
// 64-bit integers, whose order does not matter: reproducible, and finished by whichever CTA is last. Rows are fetched a
// step ahead of the arithmetic, which is what bounds these kernels: 150 instructions a row of 256 experts, half of them
// exponentials, conversions and shuffles. Measured (calls): loss of 65536 x 256 bf16 with 8 ids a row 22.5 us (floor
// 5.6; float32 24 us, floor 10.9), gradient of 131072 x 128 bf16 20.5 us (floor 10.3; float32 28.6 us, floor 20.5; 262144 x
// 256 bf16 in 63 us, 4.3 TB/s), 262144 x 8 ids of 64 bits 12 us in the kernel (floor 2.6; shared-memory atomics and a memory
// latency for each batch of ids). A CTA takes its sequences one after the other: 4096 x 8 in 256 sequences 84 us a call.
//
// Bits. The softmax is in 32 bits with the approximate exponential (off by 2^-22) and reciprocal (2^-23), which keeps the
// instructions few that bound these kernels: below 4 units of 2^-23 of a probability for logits near the largest, plus the
// rounding of the difference, which grows with it as the probability falls. Column sums are in 32 bits over a lane's own
// rows of one CTA, 300 additions for a million rows of 256 experts, and exact from there on. The loss is a 32-bit sum of at
// most 1024 terms, none below zero, that is rounded to 32 bits anyway.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "model_common.cuh"

namespace tb200 {
namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / kWarp;
constexpr uint32_t kMaxCountExperts = 8192;  // counters of a CTA in 32 KB
constexpr uint32_t kMaxBalanceExperts = 1024;

struct Ids {
  const void* ids;
  uint64_t stride;
  uint32_t k;
  int bytes;
};
__device__ __forceinline__ int64_t id_at(const Ids& d, uint64_t row, uint32_t slot) {
  const uint64_t i = row * d.stride + slot;
  return d.bytes == 4 ? (int64_t)static_cast<const int32_t*>(d.ids)[i] : static_cast<const int64_t*>(d.ids)[i];
}

// The ids of rows [r0, r1) into a CTA's counters. Eight ids a thread are on their way before the first is counted: a
// CTA that waits for one after the other spends a memory latency on each.
__device__ __forceinline__ void count_rows(const Ids& d, const uint8_t* mask, uint64_t r0, uint64_t r1, uint32_t experts,
                                           unsigned* counters) {
  constexpr int U = 8;
  const bool dense = d.stride == d.k && mask == nullptr;
  // pieces of rows whose ids are numbered in 32 bits: a division of 64 bits costs more than the rest
  for (uint64_t at = r0; at < r1;) {
    const uint64_t most = (1u << 30) / d.k + 1;
    const uint64_t end = r1 - at < most ? r1 : at + most;
    const uint32_t n = (uint32_t)((end - at) * d.k);
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += U * kRouteThreads) {
      int64_t id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t i = i0 + u * kRouteThreads;
        id[u] = -1;
        if (i >= n) continue;
        if (dense) {
          id[u] = id_at(d, at, i);
        } else {
          const uint32_t row = i / d.k;
          if (mask == nullptr || mask[at + row]) id[u] = id_at(d, at + row, i - row * d.k);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (id[u] >= 0 && id[u] < (int64_t)experts) atomicAdd(&counters[id[u]], 1u);
    }
    at = end;
  }
}

// ---- tokens per expert ------------------------------------------------------------------------------

__device__ __forceinline__ void write_counts(const unsigned long long* sums, const unsigned* counters, uint32_t experts,
                                             uint64_t* counts, uint64_t* begins) {
  // exclusive prefix sums by strips: thread t has the experts of strip t
  __shared__ unsigned long long s_strip[kRouteThreads];
  const uint32_t per = (experts + kRouteThreads - 1) / kRouteThreads;
  const uint32_t e0 = min(threadIdx.x * per, experts), e1 = min(e0 + per, experts);
  auto at = [&](uint32_t e) { return sums ? __ldcg(&sums[e]) : (unsigned long long)counters[e]; };
  unsigned long long mine = 0;
  for (uint32_t e = e0; e < e1; ++e) {
    const unsigned long long v = at(e);
    counts[e] = v;
    mine += v;
  }
  if (begins == nullptr) return;
  s_strip[threadIdx.x] = mine;
  __syncthreads();
  for (int off = 1; off < kRouteThreads; off *= 2) {
    const unsigned long long v = threadIdx.x >= off ? s_strip[threadIdx.x - off] : 0;
    __syncthreads();
    s_strip[threadIdx.x] += v;
    __syncthreads();
  }
  unsigned long long run = s_strip[threadIdx.x] - mine;
  for (uint32_t e = e0; e < e1; ++e) {
    begins[e] = run;
    run += at(e);
  }
  if (threadIdx.x == kRouteThreads - 1) begins[experts] = s_strip[threadIdx.x];
}

__global__ void __launch_bounds__(kRouteThreads)
expert_counts_kernel(Ids ids, const uint8_t* mask, uint64_t rows, uint64_t rows_of_cta, uint32_t experts,
                     uint64_t* counts, uint64_t* begins, TempHeader* hdr, unsigned long long* sums) {
  extern __shared__ unsigned s_count[];
  __shared__ unsigned s_last;
  for (uint32_t e = threadIdx.x; e < experts; e += kRouteThreads) s_count[e] = 0;
  __syncthreads();
  const uint64_t r0 = blockIdx.x * rows_of_cta, r1 = min(r0 + rows_of_cta, rows);
  if (r0 < r1) count_rows(ids, mask, r0, r1, experts, s_count);
  __syncthreads();
  if (gridDim.x == 1) {  // the scratch is not cleared for a single CTA
    if (threadIdx.x == 0) hdr->status = TB200_OK;
    write_counts(nullptr, s_count, experts, counts, begins);
    return;
  }
  for (uint32_t e = threadIdx.x; e < experts; e += kRouteThreads)
    if (s_count[e]) atomicAdd(&sums[e], (unsigned long long)s_count[e]);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(&hdr->ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  write_counts(sums, nullptr, experts, counts, begins);
}

// ---- rows of logits over lanes ------------------------------------------------------------------------

// A row over L (a power of two) lanes: element i of step j is expert (j * L + lane) * 8 + i. Places beyond the last expert
// hold -inf, like disabled experts. Eight elements stay in the words that they came in until they are worked on.
template <typename T> constexpr int kWordsOf8 = sizeof(T) * 8 / 4;
template <typename T, int J>
struct RowPack {
  unsigned w[J * kWordsOf8<T>];
};
template <typename T> __device__ constexpr unsigned none_word();
template <> __device__ constexpr unsigned none_word<float>() { return 0xff800000u; }
template <> __device__ constexpr unsigned none_word<__half>() { return 0xfc00fc00u; }
template <> __device__ constexpr unsigned none_word<__nv_bfloat16>() { return 0xff80ff80u; }

template <typename T>
__device__ __forceinline__ void unpack8(const unsigned* w, float* f) {
#pragma unroll
  for (int i = 0; i < kWordsOf8<T>; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of a float32
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <typename T, int J, int L, bool VEC>
__device__ __forceinline__ void load_row(const char* row, bool on, uint32_t lane, uint32_t experts, RowPack<T, J>& out) {
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t e = (j * L + lane) * 8;
    unsigned* w = &out.w[j * kWordsOf8<T>];
#pragma unroll
    for (int i = 0; i < kWordsOf8<T>; ++i) w[i] = none_word<T>();
    if constexpr (VEC) {
      if (on && e < experts) {
#pragma unroll
        for (int i = 0; i < kWordsOf8<T> / 4; ++i) {
          const uint4 v = __ldcs(reinterpret_cast<const uint4*>(row + e * sizeof(T)) + i);
          w[4 * i] = v.x;
          w[4 * i + 1] = v.y;
          w[4 * i + 2] = v.z;
          w[4 * i + 3] = v.w;
        }
      }
    } else {
      Pack<T, 8> p;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        p.v[i] = on && e + i < experts ? reinterpret_cast<const T*>(row)[e + i] : from_f32<T>(__int_as_float(0xff800000));
#pragma unroll
      for (int i = 0; i < kWordsOf8<T>; ++i) w[i] = reinterpret_cast<const unsigned*>(&p)[i];
    }
  }
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int off = 1; off < L; off *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int off = 1; off < L; off *= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
// Softmax of a row in 32 bits: p[e] = e[e] * the value returned. A row of nothing but -inf has no probabilities: zero.
template <typename T, int J, int L>
__device__ __forceinline__ float softmax_row(const RowPack<T, J>& row, float (&e)[J * 8]) {
  const float none = __int_as_float(0xff800000);
  float top = none;
#pragma unroll
  for (int j = 0; j < J; ++j) unpack8<T>(&row.w[j * kWordsOf8<T>], &e[j * 8]);
#pragma unroll
  for (int i = 0; i < J * 8; ++i) top = fmaxf(top, e[i]);
  top = lanes_max<L>(top);
  float unit[J * 8], base[J * 8];
  fill_n(unit, kLog2e);
  fill_n(base, top == none ? 0.0f : -top);  // the difference first: logits near the end of the type's range stay in it
  add_n(e, e, base);
  mul_n(e, e, unit);
  float part[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < J * 8; i += 2) {
    e[i] = exp2_fast(e[i]);
    e[i + 1] = exp2_fast(e[i + 1]);
    add2(part[0], part[1], part[0], part[1], e[i], e[i + 1]);
  }
  const float sum = lanes_sum<L>(part[0] + part[1]);
  float scale;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(scale) : "f"(sum));  // the sum is 1 at least, or zero
  return sum == 0.0f ? 0.0f : scale;
}

// Rows that a warp has on their way at once, for each of its row groups.
template <typename T, int J> constexpr int kRowsAtOnce = J == 1 ? (sizeof(T) == 2 ? 3 : 2) : 1;

struct Spans {  // packed sequences over the rows, or one sequence
  const void* offsets;
  int bytes;
  uint64_t sequences, rows;
};
__device__ __forceinline__ int64_t raw_offset(const Spans& s, uint64_t i) {
  return s.bytes == 4 ? (int64_t)static_cast<const int32_t*>(s.offsets)[i] : static_cast<const int64_t*>(s.offsets)[i];
}
__device__ __forceinline__ uint64_t begin_of(const Spans& s, uint64_t i) {  // of sequence i; i = sequences: the end
  if (s.bytes == 0) return i == 0 ? 0 : s.rows;
  const int64_t v = raw_offset(s, i);
  return v < 0 ? 0 : (uint64_t)v > s.rows ? s.rows : (uint64_t)v;
}
__device__ __forceinline__ uint64_t sequence_of(const Spans& s, uint64_t row) {  // last one that begins at or before row
  if (s.bytes == 0) return 0;
  uint64_t lo = 0, hi = s.sequences;  // first boundary behind row, less one
  while (lo < hi) {
    const uint64_t mid = (lo + hi + 1) / 2;
    if (begin_of(s, mid) <= row) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// ---- balance loss -------------------------------------------------------------------------------------

struct BalanceArgs {
  RowsOf z;
  Ids ids;
  const uint8_t* mask;
  Spans spans;
  uint64_t rows_of_cta;
  uint32_t experts;
  float scale;  // fixed point: one is `scale`
  float* loss;
  uint64_t* counts;
  float* weights;
  TempHeader* hdr;
  unsigned long long* sums;    // [sequences][experts] of probabilities
  unsigned long long* totals;  // [sequences][experts] of ids
  unsigned long long* tokens;  // [sequences]
  unsigned* done;              // [sequences] pieces of a sequence that are in
  unsigned* poison;            // [sequences] a probability was NaN
};

// Outputs of empty sequences, which belong to no CTA's rows, and the report of bad offsets: a warp for 32 sequences.
__device__ __noinline__ void empty_sequences(Spans spans, uint32_t experts, float* loss, uint64_t* counts, float* weights,
                                             int* status) {
  const unsigned lane = lane_id();
  bool bad = blockIdx.x == 0 && threadIdx.x == 0 &&
             raw_offset(spans, spans.sequences) != (int64_t)begin_of(spans, spans.sequences);
  for (uint64_t base = (blockIdx.x * (uint64_t)kRouteWarps + threadIdx.x / kWarp) * kWarp; base < spans.sequences;
       base += (uint64_t)gridDim.x * kRouteThreads) {
    const uint64_t s = base + lane;
    bool empty = false;
    if (s < spans.sequences) {
      const uint64_t b = begin_of(spans, s), e = begin_of(spans, s + 1);
      bad = bad || raw_offset(spans, s) != (int64_t)b || (s == 0 && b != 0) || e < b;
      empty = e <= b;
      if (empty) loss[s] = 0.0f;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, empty); left != 0; left &= left - 1) {
      const uint64_t row = (base + __ffs(left) - 1) * experts;
      for (uint32_t i = lane; i < experts; i += kWarp) {
        counts[row + i] = 0;
        weights[row + i] = 0.0f;
      }
    }
  }
  if (bad) atomicExch(status, (int)TB200_ERR_INVALID_ARGUMENT);
}

template <typename T, int J, int L, bool VEC>
__global__ void __launch_bounds__(kRouteThreads, J == 1 ? 3 : 1) balance_kernel(BalanceArgs a) {
  __shared__ unsigned s_count[kMaxBalanceExperts];
  __shared__ float s_sum[kRouteWarps][J * 256];
  __shared__ unsigned s_tokens[kRouteWarps];
  __shared__ float s_loss[kRouteWarps];
  __shared__ unsigned s_last;
  const unsigned lane = lane_id(), warp = threadIdx.x / kWarp;
  constexpr uint32_t groups = kWarp / L;
  const uint32_t in_row = lane % L, group = lane / L;
  const uint64_t r0 = blockIdx.x * a.rows_of_cta, r1 = min(r0 + a.rows_of_cta, a.spans.rows);

  if (gridDim.x == 1) {  // the scratch is not cleared for a single CTA
    unsigned* words = reinterpret_cast<unsigned*>(a.sums);
    const uint64_t cells = a.spans.sequences * a.experts;
    for (uint64_t i = threadIdx.x; i < cells * 4 + a.spans.sequences * 4; i += kRouteThreads) words[i] = 0;
    if (threadIdx.x == 0) a.hdr->status = TB200_OK;
    __threadfence();
    __syncthreads();
  }
  if (a.spans.bytes && blockIdx.x * (uint64_t)kRouteThreads < a.spans.sequences)
    empty_sequences(a.spans, a.experts, a.loss, a.counts, a.weights, &a.hdr->status);
  if (r0 >= r1) return;

  for (uint64_t s = sequence_of(a.spans, r0); s < a.spans.sequences; ++s) {
    const uint64_t begin = begin_of(a.spans, s), end = begin_of(a.spans, s + 1);
    if (begin >= r1) break;
    const uint64_t from = max(begin, r0), to = min(end, r1);
    if (from >= to) continue;
    for (uint32_t e = threadIdx.x; e < a.experts; e += kRouteThreads) s_count[e] = 0;
    float acc[J * 8] = {};
    unsigned kept = 0;
    // the next rows are on their way while these are worked on
    constexpr int U = kRowsAtOnce<T, J>;
    RowPack<T, J> pack[U], ahead[U];
    bool on[U], on_ahead[U];
    const uint32_t here = (uint32_t)(to - from);
    const char* const rows_here = a.z.data + from * a.z.row * sizeof(T);
    const uint32_t row_bytes = (uint32_t)(a.z.row * sizeof(T));
    auto fetch = [&](uint32_t base, RowPack<T, J>(&into)[U], bool(&counts)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t row = base + u * kRouteWarps * groups + group;
        counts[u] = row < here && (a.mask == nullptr || a.mask[from + row]);
        load_row<T, J, L, VEC>(rows_here + (uint64_t)row * row_bytes, counts[u], in_row, a.experts, into[u]);
      }
    };
    fetch(warp * groups, pack, on);
    __syncthreads();
    count_rows(a.ids, a.mask, from, to, a.experts, s_count);
    for (uint32_t base = warp * groups; base < here; base += U * kRouteWarps * groups) {
      fetch(base + U * kRouteWarps * groups, ahead, on_ahead);
#pragma unroll
      for (int u = 0; u < U; ++u) {  // rows that do not count hold -inf alone
        float e[J * 8], scale[J * 8];
        fill_n(scale, softmax_row<T, J, L>(pack[u], e));
        fma_n(acc, e, scale, acc);
        kept += on[u] && in_row == 0;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        pack[u] = ahead[u];
        on[u] = on_ahead[u];
      }
    }
    // over the row groups of a warp, then over the warps, in a fixed order
#pragma unroll
    for (int i = 0; i < J * 8; ++i)
      for (int off = L; off < kWarp; off *= 2) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], off);
    for (int off = 16; off > 0; off /= 2) kept += __shfl_xor_sync(0xffffffffu, kept, off);
    if (group == 0) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[warp][(j * L + in_row) * 8 + i] = acc[j * 8 + i];
    }
    if (lane == 0) s_tokens[warp] = kept;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.experts; e += kRouteThreads) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kRouteWarps; ++w) sum += s_sum[w][e];
      if (!(sum == sum)) atomicOr(&a.poison[s], 1u);
      else if (sum > 0.0f) atomicAdd(&a.sums[s * a.experts + e], __float2ull_rn(sum * a.scale));
      if (s_count[e]) atomicAdd(&a.totals[s * a.experts + e], (unsigned long long)s_count[e]);
    }
    if (threadIdx.x == 0) {
      unsigned n = 0;
      for (int w = 0; w < kRouteWarps; ++w) n += s_tokens[w];
      if (n) atomicAdd(&a.tokens[s], (unsigned long long)n);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      const unsigned pieces = (unsigned)((end - 1) / a.rows_of_cta - begin / a.rows_of_cta + 1);
      s_last = atomicAdd(&a.done[s], 1u) == pieces - 1;
    }
    __syncthreads();
    if (s_last) {
      __threadfence();
      const double n = (double)__ldcg(&a.tokens[s]);
      const double unit = n > 0 ? (double)a.experts / ((double)a.ids.k * n * n) : 0.0;
      float part = 0.0f;
      for (uint32_t e = threadIdx.x; e < a.experts; e += kRouteThreads) {
        const unsigned long long c = __ldcg(&a.totals[s * a.experts + e]);
        const float w = (float)(unit * (double)c);
        a.counts[s * a.experts + e] = c;
        a.weights[s * a.experts + e] = w;
        part += w * (float)((double)__ldcg(&a.sums[s * a.experts + e]) / (double)a.scale);
      }
      part = lanes_sum<kWarp>(part);
      if (lane == 0) s_loss[warp] = part;
      __syncthreads();
      if (threadIdx.x == 0) {
        float loss = 0.0f;
        for (int w = 0; w < kRouteWarps; ++w) loss += s_loss[w];
        a.loss[s] = __ldcg(&a.poison[s]) ? __int_as_float(0x7fc00000) : loss;
      }
    }
    __syncthreads();
  }
}

struct BalanceBackArgs {
  RowsOf z, dz;
  const float* weights;
  const float* dloss;
  const uint8_t* mask;
  Spans spans;
  uint64_t rows_of_warp;
  uint32_t experts;
};

template <typename T, int J, int L, bool VEC>
__global__ void __launch_bounds__(kRouteThreads, J == 1 ? 3 : 1) balance_backward_kernel(BalanceBackArgs a) {
  const unsigned lane = lane_id();
  constexpr uint32_t groups = kWarp / L;
  const uint32_t in_row = lane % L, group = lane / L;
  const uint64_t warp = blockIdx.x * (uint64_t)kRouteWarps + threadIdx.x / kWarp;
  const uint64_t r0 = warp * a.rows_of_warp, r1 = min(r0 + a.rows_of_warp, a.spans.rows);
  if (r0 >= r1) return;
  uint64_t s = ~0ull;     // the sequence whose weights are held,
  uint32_t held_to = 0;   // its end among the warp's rows,
  bool some = false;      // and whether there is one
  float w[J * 8] = {};
  float scale = 0.0f;
  constexpr int U = kRowsAtOnce<T, J>;
  RowPack<T, J> pack[U], ahead[U];
  bool on[U], on_ahead[U];
  const uint32_t here = (uint32_t)(r1 - r0), row_bytes = (uint32_t)(a.z.row * sizeof(T)), out_bytes = (uint32_t)(a.dz.row * sizeof(T));
  const char* const rows_here = a.z.data + r0 * a.z.row * sizeof(T);
  char* const out_here = a.dz.data + r0 * a.dz.row * sizeof(T);
  auto fetch = [&](uint32_t at, RowPack<T, J>(&into)[U], bool(&counts)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t row = at + u * groups + group;
      counts[u] = row < here && (a.mask == nullptr || a.mask[r0 + row]);
      load_row<T, J, L, VEC>(rows_here + (uint64_t)row * row_bytes, counts[u], in_row, a.experts, into[u]);
    }
  };
  fetch(0, pack, on);
  for (uint32_t at = 0; at < here; at += U * groups) {
    fetch(at + U * groups, ahead, on_ahead);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t row = at + u * groups + group;
      const bool valid = row < here;
      if (valid && row >= held_to) {
        const uint64_t at_row = r0 + row;
        if (s == ~0ull) s = sequence_of(a.spans, at_row);
        while (s < a.spans.sequences && at_row >= begin_of(a.spans, s + 1)) ++s;
        const uint64_t end = s < a.spans.sequences ? begin_of(a.spans, s + 1) : a.spans.rows;
        held_to = end - r0 < here ? (uint32_t)(end - r0) : here;
        some = s < a.spans.sequences && at_row >= begin_of(a.spans, s);
        scale = some ? a.dloss[s] : 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t e = (j * L + in_row) * 8 + i;
            w[j * 8 + i] = some && e < a.experts ? a.weights[s * a.experts + e] : 0.0f;
          }
      }
      const bool kept = on[u] && some;
      float e[J * 8];
      const float share = softmax_row<T, J, L>(pack[u], e);
      float part[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < J * 8; i += 2) fma2(part[0], part[1], e[i], e[i + 1], w[i], w[i + 1], part[0], part[1]);
      const float dot = lanes_sum<L>(part[0] + part[1]) * share;
      float less[J * 8], factor[J * 8], d[J * 8];
      fill_n(less, -dot);
      fill_n(factor, scale * share);
      add_n(d, w, less);
      mul_n(e, e, factor);
      mul_n(d, d, e);
      if (!kept) fill_n(d, 0.0f);  // not by a factor of zero: rows of no sequence may hold NaN or infinities
      if (!valid) continue;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t first = (j * L + in_row) * 8;
        char* to = out_here + (uint64_t)row * out_bytes + first * sizeof(T);
        Pack<T, 8> out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out.v[i] = from_f32<T>(d[j * 8 + i]);
        if constexpr (VEC) {
          if (first < a.experts) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(out) / 16); ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(&out)[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (first + i < a.experts) reinterpret_cast<T*>(to)[i] = out.v[i];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      pack[u] = ahead[u];
      on[u] = on_ahead[u];
    }
  }
}

template <int WHICH, typename... T> struct Tag {};

uint32_t lanes_of(uint32_t experts) {  // lanes that share a row
  uint32_t lanes = 1;
  while (lanes < kWarp && lanes * 8 < experts) lanes *= 2;
  return lanes;
}
// Calls f(type tag, J, L, VEC) for a row of this type and size.
template <typename F>
int by_row(int dtype, uint32_t experts, bool vec, F f) {
  using std::integral_constant;
  auto sized = [&](auto tag, auto v) -> int {
    constexpr integral_constant<int, 1> one{};
    if (experts > 512) return f(tag, integral_constant<int, 4>{}, integral_constant<int, 32>{}, v);
    if (experts > 256) return f(tag, integral_constant<int, 2>{}, integral_constant<int, 32>{}, v);
    switch (lanes_of(experts)) {
      case 1: return f(tag, one, integral_constant<int, 1>{}, v);
      case 2: return f(tag, one, integral_constant<int, 2>{}, v);
      case 4: return f(tag, one, integral_constant<int, 4>{}, v);
      case 8: return f(tag, one, integral_constant<int, 8>{}, v);
      case 16: return f(tag, one, integral_constant<int, 16>{}, v);
      default: return f(tag, one, integral_constant<int, 32>{}, v);
    }
  };
  auto typed = [&](auto tag) -> int { return vec ? sized(tag, std::true_type{}) : sized(tag, std::false_type{}); };
  if (dtype == TB200_F32) return typed(float{});
  if (dtype == TB200_F16) return typed(__half{});
  return typed(__nv_bfloat16{});
}

int check_ids(const void* ids, uint64_t rows, uint32_t k, uint64_t stride, int bytes) {
  if (bytes != 4 && bytes != 8) return TB200_ERR_INVALID_ARGUMENT;
  if (k == 0 || (rows > 1 && stride < k) || rows > (1ull << 40) || k > (1u << 20)) return TB200_ERR_INVALID_ARGUMENT;
  if (rows && (!ids || reinterpret_cast<uintptr_t>(ids) % bytes)) return TB200_ERR_INVALID_ARGUMENT;
  return TB200_OK;
}

}  // namespace
}  // namespace tb200

extern "C" int tb200_expert_counts(void* d_temp, size_t* temp_bytes, const void* d_ids, uint64_t rows, uint32_t k,
                                   uint64_t id_stride, int id_bytes, const uint8_t* d_mask, uint32_t experts,
                                   uint64_t* d_counts, uint64_t* d_begins, tb200_stream_t stream) {
  using namespace tb200;
  if (temp_bytes == nullptr || experts == 0) return TB200_ERR_INVALID_ARGUMENT;
  if (experts > kMaxCountExperts) return TB200_ERR_UNSUPPORTED;
  const size_t need = kHeaderBytes + align_up(experts * sizeof(unsigned long long), 256);
  if (d_temp == nullptr) {
    *temp_bytes = need;
    return TB200_OK;
  }
  if (*temp_bytes < need) return TB200_ERR_TEMP_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(d_temp) % 256) return TB200_ERR_INVALID_ARGUMENT;
  int rc = check_ids(d_ids, rows, k, id_stride, id_bytes);
  if (rc) return rc;
  if (!d_counts || (reinterpret_cast<uintptr_t>(d_counts) | reinterpret_cast<uintptr_t>(d_begins)) % 8) return TB200_ERR_INVALID_ARGUMENT;
  int sms = 0;
  rc = sm_count_of_device(&sms);
  if (rc) return rc;
  // a CTA for each 4096 ids, as many as two waves hold
  uint64_t ctas = (rows * k + 4095) / 4096;
  if (ctas > 2ull * sms) ctas = 2ull * sms;
  if (ctas > rows) ctas = rows;
  if (ctas == 0) ctas = 1;
  const uint64_t per = rows ? (rows + ctas - 1) / ctas : 1;
  ctas = rows ? (rows + per - 1) / per : 1;
  if (ctas > 1) TB200_CUDA_TRY(cudaMemsetAsync(d_temp, 0, need, stream));
  const Ids ids{d_ids, id_stride, k, id_bytes};
  expert_counts_kernel<<<(unsigned)ctas, kRouteThreads, experts * sizeof(unsigned), stream>>>(
      ids, d_mask, rows, per, experts, d_counts, d_begins, static_cast<TempHeader*>(d_temp),
      reinterpret_cast<unsigned long long*>(static_cast<char*>(d_temp) + kHeaderBytes));
  trace_mark(stream, kTraceExpertCounts);
  return (int)cudaGetLastError();
}

extern "C" int tb200_balance_loss(void* d_temp, size_t* temp_bytes, const tb200_rows* logits, int dtype, const void* d_ids,
                                  uint32_t k, uint64_t id_stride, int id_bytes, const uint8_t* d_mask,
                                  const void* d_offsets, int offset_bytes, uint64_t sequences, uint64_t rows,
                                  uint32_t experts, float* d_loss, uint64_t* d_counts, float* d_weights,
                                  tb200_stream_t stream) {
  using namespace tb200;
  if (temp_bytes == nullptr || experts == 0) return TB200_ERR_INVALID_ARGUMENT;
  if (model_bytes(dtype) == 0 || experts > kMaxBalanceExperts || sequences > 0x7fffffffull) return TB200_ERR_UNSUPPORTED;
  if (offset_bytes != 0 && offset_bytes != 4 && offset_bytes != 8) return TB200_ERR_INVALID_ARGUMENT;
  if (offset_bytes == 0 && sequences != 1) return TB200_ERR_INVALID_ARGUMENT;
  const uint64_t cells = sequences * experts;
  const size_t need = kHeaderBytes + align_up(cells * 16 + sequences * 16, 256);
  if (d_temp == nullptr) {
    *temp_bytes = need;
    return TB200_OK;
  }
  if (*temp_bytes < need) return TB200_ERR_TEMP_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(d_temp) % 256) return TB200_ERR_INVALID_ARGUMENT;
  int rc = check_ids(d_ids, rows, k, id_stride, id_bytes);
  if (rc) return rc;
  if (rows >= (1ull << 31) || (rows && logits && logits->row_stride > (1u << 28))) return TB200_ERR_UNSUPPORTED;
  const int tb = model_bytes(dtype);
  if (rows && !good_rows(logits, tb)) return TB200_ERR_INVALID_ARGUMENT;
  if (offset_bytes && (!d_offsets || reinterpret_cast<uintptr_t>(d_offsets) % offset_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  if (sequences && (!d_loss || !d_counts || !d_weights)) return TB200_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(d_counts) % 8 ||
      (reinterpret_cast<uintptr_t>(d_loss) | reinterpret_cast<uintptr_t>(d_weights)) % 4) return TB200_ERR_INVALID_ARGUMENT;
  if (rows == 0 || sequences == 0) {
    rc = status_without_rows(d_temp, d_offsets, offset_bytes, sequences, rows, stream);
    if (rc || sequences == 0) return rc;
    TB200_CUDA_TRY(cudaMemsetAsync(d_loss, 0, sequences * sizeof(float), stream));
    TB200_CUDA_TRY(cudaMemsetAsync(d_counts, 0, cells * sizeof(uint64_t), stream));
    return (int)cudaMemsetAsync(d_weights, 0, cells * sizeof(float), stream);
  }
  int sms = 0;
  rc = sm_count_of_device(&sms);
  if (rc) return rc;
  BalanceArgs a{};
  a.z = rows_of(logits, true);
  a.ids = Ids{d_ids, id_stride, k, id_bytes};
  a.mask = d_mask;
  a.spans = Spans{d_offsets, offset_bytes, sequences, rows};
  a.experts = experts;
  int bits = 62;  // a sum of all rows stays below 2^62
  while (bits > 1 && (rows >> (62 - bits)) != 0) --bits;
  a.scale = ldexpf(1.0f, bits);
  a.loss = d_loss;
  a.counts = d_counts;
  a.weights = d_weights;
  a.hdr = static_cast<TempHeader*>(d_temp);
  a.sums = reinterpret_cast<unsigned long long*>(static_cast<char*>(d_temp) + kHeaderBytes);
  a.totals = a.sums + cells;
  a.tokens = a.totals + cells;
  a.done = reinterpret_cast<unsigned*>(a.tokens + sequences);
  a.poison = a.done + sequences;
  const bool vec = experts % 8 == 0 && rows_on(a.z, tb, 16);
  return by_row(dtype, experts, vec, [&](auto tag, auto j, auto l, auto v) -> int {
    auto kernel = balance_kernel<decltype(tag), decltype(j)::value, decltype(l)::value, decltype(v)::value>;
    int per_sm = 0;
    const int rc = resident_ctas<Tag<0, decltype(tag), decltype(j), decltype(l), decltype(v)>>(kernel, kRouteThreads, 0, &per_sm);
    if (rc) return rc;
    // as many CTAs as fit, each with one row at least for every row group of its warps
    const uint64_t slots = (uint64_t)per_sm * sms, least = (uint64_t)kRouteWarps * (kWarp / decltype(l)::value);
    a.rows_of_cta = (rows + slots - 1) / slots;
    if (a.rows_of_cta < least) a.rows_of_cta = least;
    // One CTA does all of one sequence with up to 2^15 probabilities and 2^13 ids: no clear of the scratch in front. That
    // saves a call 2 to 3 us, and costs up to 3 us where the GPU has work queued or replays a graph. Measured, one CTA
    // against many, a call / in a graph: 1024 x 8 with 2 ids a row 17.5 against 19.5 / 7.4 against 10.0 us, 4096 x 8 with 2
    // ids 17.7 against 19.5 / 12.0 against 10.2, 128 x 256 with 8 ids 17.6 against 21.1 / 10.8 against 7.6. Not more ids
    // (4096 x 8 with 8: 22.7 against 19.4 / 21.8 against 10.4) nor more sequences, which a CTA takes one after the
    // other (4096 x 8 with 2 ids in 16 sequences: 92 against 20 / 90 against 11).
    if (sequences == 1 && rows * experts <= 32768 && rows * k <= 8192) a.rows_of_cta = rows;
    const unsigned grid = (unsigned)((rows + a.rows_of_cta - 1) / a.rows_of_cta);
    if (grid > 1) TB200_CUDA_TRY(cudaMemsetAsync(d_temp, 0, need, stream));
    kernel<<<grid, kRouteThreads, 0, stream>>>(a);
    trace_mark(stream, kTraceBalanceLoss);
    return (int)cudaGetLastError();
  });
}

extern "C" int tb200_balance_loss_backward(const tb200_rows* logits, int dtype, const float* d_weights,
                                           const float* d_dloss, const uint8_t* d_mask, const void* d_offsets,
                                           int offset_bytes, uint64_t sequences, uint64_t rows, uint32_t experts,
                                           const tb200_rows* dlogits, tb200_stream_t stream) {
  using namespace tb200;
  const int tb = model_bytes(dtype);
  if (experts == 0) return TB200_ERR_INVALID_ARGUMENT;
  if (tb == 0 || experts > kMaxBalanceExperts || sequences > 0x7fffffffull || rows >= (1ull << 31)) return TB200_ERR_UNSUPPORTED;
  if (offset_bytes != 0 && offset_bytes != 4 && offset_bytes != 8) return TB200_ERR_INVALID_ARGUMENT;
  if (offset_bytes == 0 && sequences != 1) return TB200_ERR_INVALID_ARGUMENT;
  if (rows == 0) return TB200_OK;
  if (!good_rows(logits, tb) || !good_rows(dlogits, tb)) return TB200_ERR_INVALID_ARGUMENT;
  if (logits->row_stride > (1u << 28) || dlogits->row_stride > (1u << 28)) return TB200_ERR_UNSUPPORTED;
  if (offset_bytes && (!d_offsets || reinterpret_cast<uintptr_t>(d_offsets) % offset_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  if (sequences && (!d_weights || !d_dloss)) return TB200_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(d_weights) | reinterpret_cast<uintptr_t>(d_dloss)) % 4) return TB200_ERR_INVALID_ARGUMENT;
  BalanceBackArgs a{};
  a.z = rows_of(logits, true);
  a.dz = rows_of(dlogits, true);
  a.weights = d_weights;
  a.dloss = d_dloss;
  a.mask = d_mask;
  a.spans = Spans{d_offsets, offset_bytes, sequences, rows};
  a.experts = experts;
  int sms = 0;
  const int rc = sm_count_of_device(&sms);
  if (rc) return rc;
  const bool vec = experts % 8 == 0 && rows_on(a.z, tb, 16) && rows_on(a.dz, tb, 16);
  return by_row(dtype, experts, vec, [&](auto tag, auto j, auto l, auto v) -> int {
    auto kernel = balance_backward_kernel<decltype(tag), decltype(j)::value, decltype(l)::value, decltype(v)::value>;
    int per_sm = 0;
    const int rc = resident_ctas<Tag<1, decltype(tag), decltype(j), decltype(l), decltype(v)>>(kernel, kRouteThreads, 0, &per_sm);
    if (rc) return rc;
    // as many warps as fit, each with one row at least for every row group
    const uint64_t slots = (uint64_t)per_sm * sms * kRouteWarps, least = kWarp / decltype(l)::value;
    a.rows_of_warp = (rows + slots - 1) / slots;
    if (a.rows_of_warp < least) a.rows_of_warp = least;
    const uint64_t warps = (rows + a.rows_of_warp - 1) / a.rows_of_warp;
    kernel<<<(unsigned)((warps + kRouteWarps - 1) / kRouteWarps), kRouteThreads, 0, stream>>>(a);
    trace_mark(stream, kTraceBalanceLoss);
    return (int)cudaGetLastError();
  });
}

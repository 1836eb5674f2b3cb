// One row of the gated linear recurrence for each of many sequences: state = a * state + x in a pool of states.
//
// Bound by HBM where there are many rows (a state is read and written in 32 bits, which no order of work avoids) and by
// the launch where there are few. Threads take four channels of one row; a CTA works on one row, so that rows which
// name the same state are put in order by a CTA alone: the CTA of the first of them applies them all. Looking through the
// slots of all rows costs a CTA two loads a thread for 512 rows, and grows with their square: 4096 rows of 4096 channels
// 80 us (39 without slots), 16384 x 2048 463 us (75), 65536 x 2048 6.9 ms (0.28). Measured: one row of 2048 channels 3.6 us,
// 512 rows of 4096 channels 8.4 us (3.0 TB/s of 25 MB; half of that time is a kernel's own latency). A single step uses the
// series of a gate near one, since every step rounds the gate anew; a log gate g below -0.3 takes the fast exponential, off
// by 2 + 1.2 |g| units of 2^-23 of the gate, which a state with such gates has forgotten after four steps.
#include <cuda_runtime.h>

#include <cstdint>

#include "model_common.cuh"

namespace tb200 {
namespace {

constexpr int kStepThreads = 256;
constexpr uint64_t kStepMaxIndexed = 65536;  // every row looks through the slots of all rows

struct StepArgs {
  float* state;
  uint64_t slots, slot_stride, rows;
  const void* index;
  int index_bytes, log_gate;
  uint32_t channels, head_size;
  RowsOf gate, x, y;
};

__device__ __forceinline__ int64_t slot_of(const StepArgs& p, uint64_t row) {
  if (p.index_bytes == 0) return (int64_t)row;
  return p.index_bytes == 4 ? (int64_t)static_cast<const int32_t*>(p.index)[row] : static_cast<const int64_t*>(p.index)[row];
}

template <typename T, typename G, int V, bool SHARED>
__global__ void __launch_bounds__(kStepThreads) step_kernel(StepArgs p) {
  constexpr int GV = SHARED ? 1 : V;
  const uint64_t row = blockIdx.x;
  const bool logg = p.log_gate != 0;
  const uint32_t c0 = (blockIdx.y * kStepThreads + threadIdx.x) * V;
  const bool live = c0 < p.channels;
  const int64_t slot = slot_of(p, row);
  const bool good = slot >= 0 && (uint64_t)slot < p.slots;
  bool more = false;  // rows behind this one that work on the same state
  if (p.index_bytes != 0 && good) {
    bool before = false;
    for (uint64_t r = threadIdx.x; r < p.rows; r += kStepThreads)
      if (r != row && slot_of(p, r) == slot) (r < row ? before : more) = true;
    if (__syncthreads_or(before)) return;
    more = __syncthreads_or(more);
  }
  if (!live) return;
  float out[V];
  if (!good) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.0f;
    store_floats<T, V>(p.y.data, row * p.y.row + c0, out);
    return;
  }
  float* at = p.state + (uint64_t)slot * p.slot_stride + c0;
  Pack<float, V> h = *reinterpret_cast<const Pack<float, V>*>(at);
  for (uint64_t r = row; r < p.rows; ++r) {
    if (r != row && slot_of(p, r) != slot) continue;
    const Pack<G, GV> g = load_pack<G, GV>(p.gate.data, r * p.gate.row + (SHARED ? c0 / p.head_size : c0));
    const Pack<T, V> x = load_pack<T, V>(p.x.data, r * p.x.row + c0);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float c = hold_gate(to_f32<G>(g.v[SHARED ? 0 : i]), logg);
      out[i] = h.v[i] = advance(c, held_near(c, logg), h.v[i], to_f32<T>(x.v[i]));
    }
    store_floats<T, V>(p.y.data, r * p.y.row + c0, out);
    if (!more) break;
  }
  *reinterpret_cast<Pack<float, V>*>(at) = h;
}

template <typename T, typename G>
int launch_step(const StepArgs& p, uint32_t heads, cudaStream_t stream) {
  const bool shared = heads != p.channels;
  bool wide = p.channels % 4 == 0 && rows_on(p.x, sizeof(T), 4 * sizeof(T)) && rows_on(p.y, sizeof(T), 4 * sizeof(T)) &&
              reinterpret_cast<uintptr_t>(p.state) % 16 == 0 && p.slot_stride % 4 == 0;
  wide = wide && (shared ? p.head_size % 4 == 0 : rows_on(p.gate, sizeof(G), 4 * sizeof(G)));
  const uint32_t per_cta = kStepThreads * (wide ? 4 : 1);
  const dim3 grid((unsigned)p.rows, (p.channels + per_cta - 1) / per_cta);
  if (grid.y > 65535) return TB200_ERR_UNSUPPORTED;
  if (wide) {
    if (shared) step_kernel<T, G, 4, true><<<grid, kStepThreads, 0, stream>>>(p);
    else step_kernel<T, G, 4, false><<<grid, kStepThreads, 0, stream>>>(p);
  } else {
    if (shared) step_kernel<T, G, 1, true><<<grid, kStepThreads, 0, stream>>>(p);
    else step_kernel<T, G, 1, false><<<grid, kStepThreads, 0, stream>>>(p);
  }
  trace_mark(stream, kTraceRecurrenceStep);
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace tb200

extern "C" int tb200_linear_recurrence_step(float* d_state, uint64_t slots, uint64_t slot_stride, const void* d_slots,
                                            int slot_bytes, const tb200_rows* gate, const tb200_rows* x,
                                            const tb200_rows* y, uint64_t rows, uint64_t channels, uint64_t heads,
                                            int dtype, int gate_dtype, int log_gate, tb200_stream_t stream) {
  using namespace tb200;
  const int tb = model_bytes(dtype), gb = model_bytes(gate_dtype);
  if (tb == 0 || (gate_dtype != dtype && gate_dtype != TB200_F32)) return TB200_ERR_UNSUPPORTED;
  if (slot_bytes != 0 && slot_bytes != 4 && slot_bytes != 8) return TB200_ERR_INVALID_ARGUMENT;
  if (channels == 0 || heads == 0 || channels % heads || slot_stride < channels) return TB200_ERR_INVALID_ARGUMENT;
  if (channels > (1u << 24) || rows > 0x7fffffffull) return TB200_ERR_UNSUPPORTED;
  if (slot_bytes != 0 && rows > kStepMaxIndexed) return TB200_ERR_UNSUPPORTED;
  if (slot_bytes == 0 && rows > slots) return TB200_ERR_INVALID_ARGUMENT;
  if (rows == 0) return TB200_OK;
  if (!good_rows(gate, gb) || !good_rows(x, tb) || !good_rows(y, tb)) return TB200_ERR_INVALID_ARGUMENT;
  if ((slots && !d_state) || reinterpret_cast<uintptr_t>(d_state) % 4) return TB200_ERR_INVALID_ARGUMENT;
  if (slot_bytes && (!d_slots || reinterpret_cast<uintptr_t>(d_slots) % slot_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  StepArgs p{};
  p.state = d_state;
  p.slots = slots;
  p.slot_stride = slot_stride;
  p.rows = rows;
  p.index = d_slots;
  p.index_bytes = slot_bytes;
  p.log_gate = log_gate;
  p.channels = (uint32_t)channels;
  p.head_size = (uint32_t)(channels / heads);
  p.gate = rows_of(gate, true);
  p.x = rows_of(x, true);
  p.y = rows_of(y, true);
  if (dtype == TB200_F32) return launch_step<float, float>(p, (uint32_t)heads, stream);
  if (dtype == TB200_BF16)
    return gate_dtype == TB200_F32 ? launch_step<__nv_bfloat16, float>(p, (uint32_t)heads, stream)
                                   : launch_step<__nv_bfloat16, __nv_bfloat16>(p, (uint32_t)heads, stream);
  return gate_dtype == TB200_F32 ? launch_step<__half, float>(p, (uint32_t)heads, stream)
                                 : launch_step<__half, __half>(p, (uint32_t)heads, stream);
}

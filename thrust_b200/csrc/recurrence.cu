// Gated linear recurrence y[t] = a[t] * y[t-1] + x[t] by sequence and channel, forward and backward.
//
// A stretch of rows maps the state in front of it to the state behind it: h -> A * h + B, with A the product of its
// gates and B what the stretch makes of a zero state. The backward pass is the same in the other direction: with
// P = a[t] * G[t] as the state (G[t] = dy[t] + P[t+1]), a stretch maps the P behind it to the P of its first row,
// with the same A. So one kernel serves both: logical rows run with the recurrence, forward in memory or backward.
//
// The unit of work is a tile of kWarps * R rows by a block of channels. Every warp keeps R rows in registers, a lane V
// neighbouring channels of them: one pass over the rows gives the stretch's (A, B), the warps' stretches are joined
// through shared memory, and a second pass over the same registers gives the outputs. Every input is read once and
// every output written once: the kernel is bound by HBM.
//
// Gates close to one. A state remembers 1 / (1 - a) rows, so an error of a counts relative to 1 - a: a rounding of
// 2^-25 in a = 0.9995 is 6e-5 of it, and a library exponential whose last bit leans to one side adds up over the whole
// memory. With log gates in [-0.3, 0] the state therefore advances by its change, h + ((a - 1) * h + x), with a - 1
// from its own series, and A is the exponential of the SUM of the gates, in the same two forms; with plain gates
// A - 1 is carried beside A. States, products and sums are held in 32 bits; outputs are rounded once.
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "model_common.cuh"

namespace tb200 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * kWarp;

struct RecArgs {
  const void* offsets;
  int offset_bytes;
  int log_gate, fill;
  uint64_t sequences;   // of them
  uint64_t length;      // rows of a sequence; packed: of all
  uint64_t chain_rows;  // rows of a chain: of one sequence, or of all sequences behind one another
  int chain_is_sequence;
  uint32_t channels, heads, head_size;
  uint32_t block_heads, parts;  // heads in a block of channels; blocks that share one head
  RowsOf gate, in, out;         // forward: x -> y; backward: dy -> dx
  RowsOf y, dgate;              // backward only
  const float* first;           // forward: initial states; backward: gradient of the final states
  const float* initial;         // backward: initial states (y[-1])
  float* last;                  // forward: final states; backward: gradient of the initial states
  float* partial;               // backward, a head over several blocks: their sums, [rows][heads][parts]
  TempHeader* hdr;
  uint32_t blocks, chains;      // blocks of channels, chains
  uint64_t tiles;               // of a chain
  unsigned long long* maps;     // [tile][chain][block][channel]: what the tile does to a state (0: not there yet)
  unsigned* states;             // [tile][chain][block][channel]: the state behind the tile (0: not there yet)
};

// A of a stretch in one word: A - 1 with the lowest bit set where A >= 1/2, else A with it clear. The bit costs at
// most one unit of the last place, of A - 1 where that is what matters.
__device__ __forceinline__ unsigned word_of(float a, float m) {
  return a >= 0.5f ? (__float_as_uint(m) | 1u) : (__float_as_uint(a) & ~1u);
}
__device__ __forceinline__ float apply(unsigned word, float h, float b) {  // A * h + b
  const float u = fmaf(__uint_as_float(word), h, b);
  return (word & 1u) ? h + u : u;
}

// Descriptors hold the complement, so that cleared scratch means "not there yet"; the two values whose complement
// would be zero are NaNs and give way to other NaNs.
__device__ __forceinline__ unsigned long long map_bits(unsigned word, float b) {
  if (word == 0xffffffffu) word = 0xfffffffdu;
  return ~((unsigned long long)word << 32 | __float_as_uint(b));
}
__device__ __forceinline__ unsigned state_bits(float h) {
  const unsigned u = __float_as_uint(h);
  return ~(u == 0xffffffffu ? 0x7fffffffu : u);
}

// The state in front of a tile, for one channel: from the nearest known state among the tiles in front, through the maps
// of the tiles between, in the order of the rows. A known state is itself the one in front of its tile put through that
// tile's map, so the value is the same wherever the walk begins, to the bit. At most kReach tiles back; where no state is
// known there, the wait is for one to come closer, which the tile right behind the last known state always brings about.
constexpr int kReach = 8;
__device__ float state_in_front(const unsigned long long* maps, const unsigned* states, uint64_t step, uint64_t tile, int* status) {
  const int n = tile < kReach ? (int)tile : kReach;
  for (unsigned polls = 0;; ++polls) {
    unsigned long long m[kReach];
    unsigned s[kReach];
#pragma unroll
    for (int j = 0; j < kReach; ++j) {
      s[j] = j < n ? ld_relaxed_u32(states - (j + 1) * step) : 0u;
      m[j] = j < n ? ld_relaxed_u64(maps - (j + 1) * step) : 0ull;
    }
    float h = 0.0f;
    bool known = false;
#pragma unroll
    for (int j = kReach - 1; j >= 0; --j) {
      if (s[j] != 0u) {
        h = __uint_as_float(~s[j]);
        known = true;
      } else if (m[j] != 0ull) {
        h = apply((unsigned)(~m[j] >> 32), h, __uint_as_float((unsigned)~m[j]));
      } else {
        known = false;
      }
    }
    if (known) return h;
    if ((polls & 63u) == 63u && ld_relaxed_s32(status) != 0) return h;  // someone else gave up
    if (polls >= kSpinLimit) {
      note_timeout(status, kSiteLookback, tile, 0);
      return h;
    }
    backoff(polls);
  }
}

constexpr int kMaxRows = 16;  // rows of a lane, at most
struct Marks {           // of the rows of a tile of packed sequences
  int seq[kWarps * kMaxRows];  // sequence of a first or last row
  unsigned char kind[kWarps * kMaxRows];  // bit 0: first row of its sequence, bit 1: last
};

__device__ __forceinline__ uint64_t offset_at(const RecArgs& p, uint64_t i) {
  const int64_t v = p.offset_bytes == 4 ? (int64_t)static_cast<const int32_t*>(p.offsets)[i]
                                        : static_cast<const int64_t*>(p.offsets)[i];
  return v < 0 ? 0 : (uint64_t)v > p.length ? p.length : (uint64_t)v;
}

// Marks the first and last rows of sequences among rows [r0, r1), in memory order; hands the states of empty sequences
// that lie here through for channels [c0, c0 + count). One warp does it; the others wait at the barrier behind.
__device__ void mark_rows(const RecArgs& p, uint64_t r0, uint64_t r1, bool at_end, uint32_t c0, uint32_t count, Marks& m) {
  const unsigned lane = lane_id();
  for (int i = lane; i < (int)sizeof(m.kind) / 4; i += kWarp) reinterpret_cast<unsigned*>(m.kind)[i] = 0;
  __syncwarp();
  // first boundary at or behind r0: every step looks at 32 boundaries at once
  uint64_t lo = 0, hi = p.sequences + 1;
  while (lo < hi) {
    const uint64_t stride = (hi - lo + kWarp - 1) / kWarp;
    const uint64_t at = lo + (lane + 1) * stride - 1;  // the last of the lane's stretch
    const unsigned in_front = __ballot_sync(0xffffffffu, at < hi && offset_at(p, at) < r0);
    const int skip = __popc(in_front);  // stretches that lie wholly in front of r0
    lo += skip * stride;
    const uint64_t end = lo + stride - 1;  // the next stretch ends at or behind r0, unless it is cut
    if (end < hi) hi = end;
  }
  for (uint64_t j = lo + lane; j <= p.sequences; j += kWarp) {
    const uint64_t v = offset_at(p, j);
    if (v > r1) break;
    if (j > 0 && v > r0 && offset_at(p, j - 1) < v) {  // sequence j - 1 ends in front of boundary j
      m.seq[v - 1 - r0] = (int)(j - 1);
      atomicOr(reinterpret_cast<unsigned*>(m.kind) + (v - 1 - r0) / 4, 2u << (8 * ((v - 1 - r0) % 4)));
    }
    if (j < p.sequences && (v < r1 || at_end)) {
      const uint64_t end = offset_at(p, j + 1);
      if (end > v && v < r1 && v >= r0) {
        m.seq[v - r0] = (int)j;
        atomicOr(reinterpret_cast<unsigned*>(m.kind) + (v - r0) / 4, 1u << (8 * ((v - r0) % 4)));
      } else if (end <= v && p.last != nullptr) {
        for (uint32_t c = c0; c < c0 + count; ++c) p.last[j * p.channels + c] = p.first ? p.first[j * p.channels + c] : 0.0f;
      }
    }
  }
}

template <typename T, typename G, int V, bool SHARED, bool BACK, int R>
__global__ void __launch_bounds__(kThreads, 2) recurrence_kernel(RecArgs p) {
  constexpr int WIDTH = kWarp * V;
  constexpr int GV = SHARED ? 1 : V;  // gates of a lane in a row
  constexpr int TILE = kWarps * R;
  constexpr unsigned ALL = (unsigned)((1ull << R) - 1);
  static_assert(R <= kMaxRows, "marks are sized for this");
  __shared__ Marks s_marks;
  __shared__ unsigned s_word[kWarps][WIDTH];
  __shared__ float s_b[kWarps][WIDTH];
  __shared__ float s_carry[kWarps][WIDTH];
  __shared__ int s_reset[kWarps];  // a sequence begins among the warp's rows
  __shared__ int s_need[kWarps];   // the warp has rows in front of that
  __shared__ unsigned s_ticket;

  const unsigned lane = lane_id(), warp = threadIdx.x / kWarp;
  const bool logg = p.log_gate != 0;

  // Tiles are handed out in the order of the recurrence, all chains and blocks of channels of one stretch of rows before
  // the next: whatever a tile waits for is worked on by a CTA that runs already.
  unsigned id = blockIdx.x;
  if (p.tiles > 1) {
    if (threadIdx.x == 0) s_ticket = atomicAdd(&p.hdr->ticket, 1u);
    __syncthreads();
    id = s_ticket;
  } else if (id == 0) {  // the scratch is not cleared where no tile waits for another
    if (threadIdx.x == 0) p.hdr->status = TB200_OK;
    __syncthreads();
  }
  const uint32_t block = id % p.blocks;
  const uint32_t chain = id / p.blocks % p.chains;
  const uint64_t tile = id / p.blocks / p.chains;

  // the block's channels
  uint32_t c0, count;
  if (!SHARED) {
    c0 = block * WIDTH;
    count = min((uint32_t)WIDTH, p.channels - c0);
  } else if (p.parts == 1) {
    const uint32_t h0 = block * p.block_heads;
    c0 = h0 * p.head_size;
    count = min(p.block_heads, p.heads - h0) * p.head_size;
  } else {
    const uint32_t h0 = block / p.parts, part = block % p.parts;
    c0 = h0 * p.head_size + part * WIDTH;
    count = min((uint32_t)WIDTH, p.head_size - part * WIDTH);
  }
  const uint32_t ch = c0 + lane * V;
  const bool live = lane * V < count;
  const uint32_t head = SHARED ? ch / p.head_size : 0;
  const uint32_t gate_at = SHARED ? head : ch;

  // ---- load: the warp's rows run from `row` with the recurrence, `n` of them exist ----------------------
  const uint64_t q = tile * TILE + warp * R;
  const int n = q >= p.chain_rows ? 0 : p.chain_rows - q < R ? (int)(p.chain_rows - q) : R;
  const int64_t row = BACK ? (int64_t)p.chain_rows - 1 - (int64_t)q : (int64_t)q;  // below zero only where n is 0
  auto at = [&](const RowsOf& a, uint32_t column) { return (int64_t)(chain * a.seq + column) + row * (int64_t)a.row; };
  auto next = [](const RowsOf& a) { return BACK ? -(int64_t)a.row : (int64_t)a.row; };

  Pack<G, GV> gate[R];
  Pack<T, V> x[R];
  Pack<T, V> before[BACK ? R : 1];  // y of the row in front, in memory
  {
    int64_t eg = at(p.gate, gate_at), ex = at(p.in, ch), ey = BACK ? at(p.y, ch) - (int64_t)p.y.row : 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (live && r < n) {
        gate[r] = load_pack<G, GV>(p.gate.data, eg);
        x[r] = load_pack<T, V>(p.in.data, ex);
        if constexpr (BACK)
          if (row - r > 0) before[r] = load_pack<T, V>(p.y.data, ey);
      }
      eg += next(p.gate);
      ex += next(p.in);
      if constexpr (BACK) ey += next(p.y);
    }
  }

  // ---- first and last rows of sequences: bit r of a mask is the warp's row r ------------------------------
  unsigned m_inside = (unsigned)((1ull << n) - 1), m_first = 0, m_last = 0;
  int seq = chain;  // of row `lane`, where that is a first or last one
  if (p.offsets != nullptr) {
    if (id == 0) {  // bad offsets are reported, and cannot lead outside the arrays
      bool bad = false;
      for (uint64_t i = threadIdx.x; i <= p.sequences; i += kThreads) {
        const int64_t v = p.offset_bytes == 4 ? (int64_t)static_cast<const int32_t*>(p.offsets)[i]
                                              : static_cast<const int64_t*>(p.offsets)[i];
        bad = bad || v < 0 || (uint64_t)v > p.length || (i == 0 ? v != 0 : (uint64_t)v < offset_at(p, i - 1));
      }
      if (bad) atomicExch(&p.hdr->status, (int)TB200_ERR_INVALID_ARGUMENT);
    }
    const uint64_t lo = tile * TILE, hi = min(lo + TILE, p.chain_rows);
    const uint64_t r0 = BACK ? p.chain_rows - hi : lo, r1 = BACK ? p.chain_rows - lo : hi;
    if (warp == 0) mark_rows(p, r0, r1, r1 == p.chain_rows, c0, count, s_marks);
    __syncthreads();
    const uint64_t mine = (uint64_t)(BACK ? row - (int)lane : row + (int)lane);
    const bool valid = (int)lane < n;
    const unsigned kind = valid ? s_marks.kind[mine - r0] : 0;
    if (kind) seq = s_marks.seq[mine - r0];
    m_first = __ballot_sync(0xffffffffu, kind & 1);
    m_last = __ballot_sync(0xffffffffu, kind & 2);
    m_inside = __ballot_sync(0xffffffffu, valid && mine >= offset_at(p, 0) && mine < offset_at(p, p.sequences));
  } else if (p.chain_is_sequence) {
    if (n > 0) {
      const unsigned low = q == 0 ? 1u : 0u, high = q + n == p.chain_rows ? 1u << (n - 1) : 0u;
      m_first = BACK ? high : low;
      m_last = BACK ? low : high;
    }
  } else if (n > 0) {  // sequences of equal length behind one another
    const uint64_t mine = (uint64_t)(BACK ? row - (int)min((int)lane, n - 1) : row + (int)min((int)lane, n - 1));
    const uint64_t s = p.chain_rows >> 32 ? mine / p.length : (uint32_t)mine / (uint32_t)p.length;
    const uint64_t t = mine - s * p.length;
    seq = (int)s;
    m_first = __ballot_sync(0xffffffffu, (int)lane < n && t == 0);
    m_last = __ballot_sync(0xffffffffu, (int)lane < n && t == p.length - 1);
  }
  const unsigned m_begin = BACK ? m_last : m_first, m_end = BACK ? m_first : m_last;  // with the recurrence
  const bool plain_rows = m_inside == ALL && (m_begin | m_end) == 0;  // nothing but rows of one sequence

  // the state that a sequence begins with
  auto first_state = [&](int r, float (&h)[V]) {
    const int s = __shfl_sync(0xffffffffu, seq, r);
    const float* from = p.first + (uint64_t)s * p.channels + ch;
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = live ? from[i] : 0.0f;
  };

  // ---- first pass: the stretch's A and B --------------------------------------------------------------------
  float a[R][GV];  // the gates themselves from here on
  float A[GV], M[GV], B[V];
  {
    float sum[GV];
#pragma unroll
    for (int i = 0; i < GV; ++i) A[i] = 1.0f, M[i] = 0.0f, sum[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) B[i] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!plain_rows && !(m_inside >> r & 1)) continue;
      const bool begin = !plain_rows && (m_begin >> r & 1);
      if (begin) {
        if (p.first) {
          first_state(r, B);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) B[i] = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < GV; ++i) {
        const float g = to_f32<G>(gate[r].v[i]);
        if (logg) {
          sum[i] += g;
          a[r][i] = __expf(g);
        } else {
          A[i] *= g;
          M[i] = fmaf(M[i], g, g - 1.0f);
          a[r][i] = g;
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float ai = a[r][SHARED ? 0 : i], xv = to_f32<T>(x[r].v[i]);
        if constexpr (BACK) {
          B[i] = ai * (xv + B[i]);
        } else {
          B[i] = begin && !p.first ? xv : fmaf(ai, B[i], xv);
        }
      }
    }
    if (logg) {
#pragma unroll
      for (int i = 0; i < GV; ++i) {
        const float c = hold_gate(sum[i], true);
        const bool near = held_near(c, true);
        A[i] = near ? 1.0f + c : c;
        M[i] = near ? c : c - 1.0f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s_word[warp][lane * V + i] = word_of(A[SHARED ? 0 : i], M[SHARED ? 0 : i]);
    s_b[warp][lane * V + i] = B[i];
  }
  if (lane == 0) {
    s_reset[warp] = m_begin != 0;
    s_need[warp] = (m_inside & ((m_begin & -m_begin) - 1u)) != 0;  // rows in front of the first begin; all without one
  }
  __syncthreads();

  // ---- the states in front of the warps' stretches --------------------------------------------------------------
  if (threadIdx.x < WIDTH) {
    // the whole tile's map; behind a begin only B counts
    bool reset = false, need = false;
    float ta = 1.0f, tm = 0.0f, tb = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const unsigned word = s_word[w][threadIdx.x];
      const float v = __uint_as_float(word), b = s_b[w][threadIdx.x];
      const float wa = (word & 1u) ? 1.0f + v : v, wm = (word & 1u) ? v : v - 1.0f;
      need = need || (!reset && s_need[w]);
      reset = reset || s_reset[w];
      tb = s_reset[w] ? b : apply(word, tb, b);
      ta *= wa;
      tm = fmaf(tm, wa, wm);
    }
    float h = 0.0f;
    if (p.tiles > 1) {
      const uint64_t to = (uint64_t)id * WIDTH + threadIdx.x, step = (uint64_t)p.chains * p.blocks * WIDTH;
      const unsigned word = word_of(ta, tm);
      const bool last_tile = tile + 1 == p.tiles;
      if (!last_tile) {
        if (reset || tile == 0) st_relaxed_u32(p.states + to, state_bits(tb));
        else st_relaxed_u64(p.maps + to, map_bits(word, tb));
      }
      if (need && tile > 0) {
        h = state_in_front(p.maps + to, p.states + to, step, tile, &p.hdr->status);
        if (!reset && !last_tile) st_relaxed_u32(p.states + to, state_bits(apply(word, h, tb)));
      } else if (!need && !reset && tile > 0 && !last_tile) {
        // no row of the tile belongs to a sequence: nobody behind it needs a state before a sequence begins
        st_relaxed_u32(p.states + to, state_bits(0.0f));
      }
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      s_carry[w][threadIdx.x] = h;
      h = s_reset[w] ? s_b[w][threadIdx.x] : apply(s_word[w][threadIdx.x], h, s_b[w][threadIdx.x]);
    }
  }
  __syncthreads();

  // ---- second pass: outputs ----------------------------------------------------------------------------------
  float h[V];
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = s_carry[warp][lane * V + i];
  int64_t eo = at(p.out, ch), ed = BACK ? at(p.dgate, gate_at) : 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = plain_rows || (m_inside >> r & 1);
    if (in || (p.fill && r < n)) {
      const bool begin = !plain_rows && (m_begin >> r & 1);
      const bool end = !plain_rows && (m_end >> r & 1);
      if (begin) {
        if (p.first) {
          first_state(r, h);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) h[i] = 0.0f;
        }
      }
      const int s = plain_rows ? 0 : __shfl_sync(0xffffffffu, seq, r);
      float out[V], dg[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xv = to_f32<T>(x[r].v[i]), ai = a[r][SHARED ? 0 : i];
        if constexpr (BACK) {
          float prev = to_f32<T>(before[r].v[i]);
          if (end) prev = p.initial && live ? p.initial[(uint64_t)s * p.channels + ch + i] : 0.0f;
          out[i] = xv + h[i];
          h[i] = ai * out[i];
          dg[i] = (logg ? h[i] : out[i]) * prev;
        } else {
          h[i] = begin && !p.first ? xv : fmaf(ai, h[i], xv);
          out[i] = h[i];
        }
      }
      if (!in) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = dg[i] = 0.0f;
      }
      if (live) store_floats<T, V>(p.out.data, eo, out);
      if constexpr (BACK) {
        if constexpr (!SHARED) {
          if (live) store_floats<G, V>(p.dgate.data, ed, dg);
        } else {
          // the head's lanes are neighbours; the first of them gathers the sum
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < V; ++i) sum += dg[i];
          if (!live) sum = 0.0f;
          const uint32_t per = p.parts == 1 ? p.head_size / V : kWarp;
          const uint32_t place = lane % per;
          for (uint32_t off = 1; off < per; off *= 2) {
            const float other = __shfl_down_sync(0xffffffffu, sum, off);
            if (place + off < per) sum += other;
          }
          if (live && place == 0) {
            if (p.parts == 1) {
              const float one[1] = {sum};
              store_floats<G, 1>(p.dgate.data, ed, one);
            } else {
              const uint64_t flat = chain * p.chain_rows + (uint64_t)(row - r);
              p.partial[(flat * p.heads + head) * p.parts + block % p.parts] = sum;
            }
          }
        }
      }
      if (in && end && p.last && live) {
#pragma unroll
        for (int i = 0; i < V; ++i) p.last[(uint64_t)s * p.channels + ch + i] = h[i];
      }
    }
    eo += next(p.out);
    if constexpr (BACK) ed += next(p.dgate);
  }
}

// dgate of heads that span several blocks of channels: the blocks' sums, in their order.
template <typename G>
__global__ void __launch_bounds__(kThreads) join_gate_kernel(RecArgs p, uint64_t rows) {
  const uint64_t n = rows * p.heads;
  const uint64_t used = p.offsets && !p.fill ? offset_at(p, p.sequences) : rows;
  for (uint64_t i = blockIdx.x * (uint64_t)kThreads + threadIdx.x; i < n; i += (uint64_t)gridDim.x * kThreads) {
    const uint64_t row = i / p.heads, head = i - row * p.heads;
    if (row >= used) continue;
    float sum[1] = {0.0f};
    for (uint32_t k = 0; k < p.parts; ++k) sum[0] += p.partial[i * p.parts + k];
    const uint64_t b = p.offsets ? 0 : row / p.length, t = row - b * p.length;
    store_floats<G, 1>(p.dgate.data, b * p.dgate.seq + t * p.dgate.row + head, sum);
  }
}

// Blocks of channels for V channels a lane.
void divide_channels(RecArgs& p, uint32_t width) {
  if (p.heads == p.channels) {
    p.blocks = (p.channels + width - 1) / width;
    p.parts = 1;
  } else if (p.head_size <= width) {
    p.block_heads = width / p.head_size;
    p.parts = 1;
    p.blocks = (p.heads + p.block_heads - 1) / p.block_heads;
  } else {
    p.parts = (p.head_size + width - 1) / width;
    p.blocks = p.heads * p.parts;
  }
}

constexpr int kRows = 8;  // rows of a lane
constexpr uint64_t kTileRows = kWarps * kRows;

struct Call {
  tb200_recurrence_shape shape;
  RecArgs args;
  uint64_t rows;     // of all sequences
  char* descriptors;
};

template <typename T, typename G, int V, bool SHARED, bool BACK>
int launch_kernel(Call& k, cudaStream_t stream) {
  RecArgs& p = k.args;
  constexpr uint32_t WIDTH = kWarp * V;
  divide_channels(p, WIDTH);
  const uint64_t ctas = p.tiles * p.chains * p.blocks;
  if (ctas > 0x7fffffffull) return TB200_ERR_UNSUPPORTED;
  if (p.tiles > 1) {
    const size_t states = ctas * WIDTH;
    p.states = reinterpret_cast<unsigned*>(k.descriptors);
    p.maps = reinterpret_cast<unsigned long long*>(k.descriptors + states * sizeof(unsigned));
    TB200_CUDA_TRY(cudaMemsetAsync(p.hdr, 0, kHeaderBytes + states * (sizeof(unsigned) + sizeof(unsigned long long)), stream));
  }
  recurrence_kernel<T, G, V, SHARED, BACK, kRows><<<(unsigned)ctas, kThreads, 0, stream>>>(p);
  trace_mark(stream, kTraceRecurrence);
  TB200_CUDA_TRY(cudaGetLastError());
  if (BACK && SHARED && p.parts > 1) {
    const uint64_t n = k.rows * p.heads;
    const uint64_t grid = (n + kThreads - 1) / kThreads;
    join_gate_kernel<G><<<(unsigned)(grid < 4096 ? grid : 4096), kThreads, 0, stream>>>(p, k.rows);
    trace_mark(stream, kTraceRecurrence);
    TB200_CUDA_TRY(cudaGetLastError());
  }
  return TB200_OK;
}

template <typename T, typename G, bool BACK>
int launch_typed(Call& k, cudaStream_t stream) {
  RecArgs& p = k.args;
  const bool shared = p.heads != p.channels;
  constexpr int ST = 4 * sizeof(T), SG = 4 * sizeof(G);
  // four channels a lane where every row of every array begins on that many elements and a head's channels divide so
  bool wide = p.channels % 4 == 0 && rows_on(p.in, sizeof(T), ST) && rows_on(p.out, sizeof(T), ST);
  if (BACK) wide = wide && rows_on(p.y, sizeof(T), ST);
  if (shared) {
    wide = wide && p.head_size % 4 == 0;
  } else {
    wide = wide && rows_on(p.gate, sizeof(G), SG);
    if (BACK) wide = wide && rows_on(p.dgate, sizeof(G), SG);
  }
  if (shared)
    return wide ? launch_kernel<T, G, 4, true, BACK>(k, stream) : launch_kernel<T, G, 1, true, BACK>(k, stream);
  return wide ? launch_kernel<T, G, 4, false, BACK>(k, stream) : launch_kernel<T, G, 1, false, BACK>(k, stream);
}

template <bool BACK>
int launch(Call& k, cudaStream_t stream) {
  const int t = k.shape.dtype, g = k.shape.gate_dtype;
  if (t == TB200_F32) return launch_typed<float, float, BACK>(k, stream);
  if (t == TB200_BF16)
    return g == TB200_F32 ? launch_typed<__nv_bfloat16, float, BACK>(k, stream)
                          : launch_typed<__nv_bfloat16, __nv_bfloat16, BACK>(k, stream);
  return g == TB200_F32 ? launch_typed<__half, float, BACK>(k, stream) : launch_typed<__half, __half, BACK>(k, stream);
}

// Whether the sequences of all arrays lie directly behind one another. A size query names no arrays: it has to be
// answered for those that need the most scratch.
bool dense(const tb200_recurrence_shape* s, std::initializer_list<const tb200_rows*> arrays) {
  for (const tb200_rows* r : arrays)
    if (s && r && s->sequences > 1 && r->sequence_stride != s->rows * r->row_stride) return false;
  return true;
}

// The checks that both directions share.
int prepare(void* d_temp, size_t* temp_bytes, const tb200_recurrence_shape* shape, bool back, bool dense, Call& k) {
  if (temp_bytes == nullptr || shape == nullptr) return TB200_ERR_INVALID_ARGUMENT;
  const tb200_recurrence_shape& s = *shape;
  if (model_bytes(s.dtype) == 0 || (s.gate_dtype != s.dtype && s.gate_dtype != TB200_F32)) return TB200_ERR_UNSUPPORTED;
  if (s.offset_bytes != 0 && s.offset_bytes != 4 && s.offset_bytes != 8) return TB200_ERR_INVALID_ARGUMENT;
  if (s.channels == 0 || s.heads == 0 || s.channels % s.heads) return TB200_ERR_INVALID_ARGUMENT;
  if (s.channels > (1u << 24) || s.sequences > 0x7fffffffull || s.rows > (1ull << 40)) return TB200_ERR_UNSUPPORTED;
  k.shape = s;
  k.rows = s.offset_bytes ? s.rows : s.sequences * s.rows;
  RecArgs& p = k.args;
  p = RecArgs{};
  p.offset_bytes = s.offset_bytes;
  p.log_gate = s.log_gate;
  p.fill = s.fill_outside;
  p.sequences = s.sequences;
  p.length = s.rows;
  p.channels = (uint32_t)s.channels;
  p.heads = (uint32_t)s.heads;
  p.head_size = (uint32_t)(s.channels / s.heads);
  // Sequences of equal length are chains of their own, unless they are so short that their tiles would be mostly empty
  // and lie behind one another (strides, which a size query does not see): then all of them are one chain, as packed
  // ones are.
  p.chain_is_sequence = s.offset_bytes == 0 && (s.rows > kTileRows / 2 || !dense);
  p.chains = p.chain_is_sequence ? (uint32_t)s.sequences : 1;
  p.chain_rows = p.chain_is_sequence ? s.rows : k.rows;
  p.tiles = (p.chain_rows + kTileRows - 1) / kTileRows;

  // Descriptors lie directly behind the header, where one clear reaches both; the sums of heads that span several
  // blocks lie behind them. The pointers' alignment decides on four or one channels a lane: room for either.
  size_t descriptors = 0, sums = 0;
  for (uint32_t width = kWarp; width <= 4 * kWarp; width *= 4) {
    divide_channels(p, width);
    if (p.tiles > 1) {
      const size_t d = p.tiles * p.chains * p.blocks * width * (sizeof(unsigned) + sizeof(unsigned long long));
      if (d > descriptors) descriptors = d;
    }
    if (back && p.parts > 1) {
      const size_t b = k.rows * p.heads * p.parts * sizeof(float);
      if (b > sums) sums = b;
    }
  }
  descriptors = align_up(descriptors, 256);
  const size_t need = kHeaderBytes + descriptors + align_up(sums, 256);
  if (d_temp == nullptr) {
    *temp_bytes = need;
    return TB200_OK;
  }
  if (*temp_bytes < need) return TB200_ERR_TEMP_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(d_temp) % 256) return TB200_ERR_INVALID_ARGUMENT;
  p.hdr = static_cast<TempHeader*>(d_temp);
  k.descriptors = static_cast<char*>(d_temp) + kHeaderBytes;
  p.partial = reinterpret_cast<float*>(k.descriptors + descriptors);
  return TB200_OK;
}

// States of sequences that have no rows at all.
int hand_through(const Call& k, const float* from, float* to, cudaStream_t stream) {
  const size_t bytes = k.shape.sequences * k.shape.channels * sizeof(float);
  if (to == nullptr || bytes == 0) return TB200_OK;
  if (from == nullptr) return (int)cudaMemsetAsync(to, 0, bytes, stream);
  return from == to ? TB200_OK : (int)cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, stream);
}

}  // namespace
}  // namespace tb200

extern "C" int tb200_linear_recurrence(void* d_temp, size_t* temp_bytes, const tb200_recurrence_shape* shape,
                                       const void* d_offsets, const tb200_rows* gate, const tb200_rows* x,
                                       const tb200_rows* y, const float* d_initial, float* d_final,
                                       tb200_stream_t stream) {
  using namespace tb200;
  Call k{};
  const int rc = prepare(d_temp, temp_bytes, shape, false, dense(shape, {gate, x, y}), k);
  if (rc || d_temp == nullptr) return rc;
  const bool packed = k.shape.offset_bytes != 0;
  if (packed && (!d_offsets || reinterpret_cast<uintptr_t>(d_offsets) % k.shape.offset_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  const bool some = k.rows != 0 && k.shape.sequences + (packed && k.shape.fill_outside) != 0;
  const int tb = model_bytes(k.shape.dtype);
  if (some && !(good_rows(gate, model_bytes(k.shape.gate_dtype)) && good_rows(x, tb) && good_rows(y, tb)))
    return TB200_ERR_INVALID_ARGUMENT;
  if (!some) {
    TB200_CUDA_TRY(cudaMemsetAsync(d_temp, 0, kHeaderBytes, stream));
    return hand_through(k, d_initial, d_final, stream);
  }
  RecArgs& p = k.args;
  p.offsets = packed ? d_offsets : nullptr;
  p.gate = rows_of(gate, packed);
  p.in = rows_of(x, packed);
  p.out = rows_of(y, packed);
  p.first = d_initial;
  p.last = d_final;
  return launch<false>(k, stream);
}

extern "C" int tb200_linear_recurrence_backward(void* d_temp, size_t* temp_bytes, const tb200_recurrence_shape* shape,
                                                const void* d_offsets, const tb200_rows* gate, const tb200_rows* y,
                                                const tb200_rows* dy, const tb200_rows* dx, const tb200_rows* dgate,
                                                const float* d_initial, const float* d_dfinal, float* d_dinitial,
                                                tb200_stream_t stream) {
  using namespace tb200;
  Call k{};
  const int rc = prepare(d_temp, temp_bytes, shape, true, dense(shape, {gate, y, dy, dx, dgate}), k);
  if (rc || d_temp == nullptr) return rc;
  const bool packed = k.shape.offset_bytes != 0;
  if (packed && (!d_offsets || reinterpret_cast<uintptr_t>(d_offsets) % k.shape.offset_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  const bool some = k.rows != 0 && k.shape.sequences + (packed && k.shape.fill_outside) != 0;
  const int tb = model_bytes(k.shape.dtype), gb = model_bytes(k.shape.gate_dtype);
  if (some && !(good_rows(gate, gb) && good_rows(y, tb) && good_rows(dy, tb) && good_rows(dx, tb) && good_rows(dgate, gb)))
    return TB200_ERR_INVALID_ARGUMENT;
  if (!some) {
    TB200_CUDA_TRY(cudaMemsetAsync(d_temp, 0, kHeaderBytes, stream));
    return hand_through(k, d_dfinal, d_dinitial, stream);
  }
  RecArgs& p = k.args;
  p.offsets = packed ? d_offsets : nullptr;
  p.gate = rows_of(gate, packed);
  p.in = rows_of(dy, packed);
  p.out = rows_of(dx, packed);
  p.y = rows_of(y, packed);
  p.dgate = rows_of(dgate, packed);
  p.initial = d_initial;
  p.first = d_dfinal;
  p.last = d_dinitial;
  return launch<true>(k, stream);
}

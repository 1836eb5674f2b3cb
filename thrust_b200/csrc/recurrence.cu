// Gated linear recurrence y[t] = a[t] * y[t-1] + x[t] by sequence and channel, forward and backward.
//
// A stretch of rows maps the state in front of it to the state behind it: h -> A * h + B, with A the product of its
// gates and B what the stretch makes of a zero state. The backward pass is the same in the other direction: with
// P = a[t] * G[t] as the state (G[t] = dy[t] + P[t+1]), a stretch maps the P behind it to the P of its first row,
// with the same A. So one kernel serves both: logical rows run with the recurrence, forward in memory or backward.
//
// The unit of work is a tile of 64 (wide types: 32) rows by 128 channels. A warp has eight (four) of its rows, a lane four
// neighbouring channels of them. A first pass over a tile gives every stretch's (A, B); threads with one channel each put
// the stretches together, publish the tile's map and find the state in front of the tile; a second pass gives the
// outputs. The rows wait in shared memory between the passes, so every input is read from memory once and every output
// written once: the floor is HBM's.
//
// Few long sequences are cut along time, so a tile has to learn the state in front of it from tiles that other CTAs work
// on. What that costs is latency, a microsecond or two a step through L2, and it is hidden by keeping rows in flight: one
// CTA on an SM takes tiles one after the other, two tiles' rows are on their way as boxes of a tensor map, the next one's
// map is computed and published while the state in front of the one before is looked for. Tiles are drawn by ticket in
// the order of the recurrence, all channels of one stretch of time before the next.
//
// Gates close to one. A state remembers 1 / (1 - a) rows, so an error of a counts relative to 1 - a: a rounding of
// 2^-25 in a = 0.9995 is 6e-5 of it, and an exponential whose last bit leans to one side adds up over the whole memory.
// Within a stretch of eight rows that stays a rounding; only the product A of a stretch is applied over and over. So A is
// held as A - 1 where it is near one: the exponential of the SUM of log gates less one, from its own series, or carried
// beside the product of plain gates. States, products and sums are held in 32 bits; outputs are rounded once.
//
// Measured (one B200, 6.56 TB/s copy): forward 65536 x 2048 bf16 with 32-bit log gates 281 us, 3.8 TB/s, with one
// sequence only 9 tiles of each block of channels are in work at once and 14 % of the looks wait for the tile in
// front (float32 521 us, 3.1 TB/s); backward of 8 x 4096 x 2048 bf16 141 us, 4.8 TB/s, bound by latency in the compute warps
// (12 warps an SM, issue slots 37 % busy). 4 x 4096 x 2048 forward and backward: bf16 70 and 82 us (floors 31 and 51), float32
// 126 and 151 us (61 and 102). Rows that are not on 16 bytes take one channel a lane, a quarter of the bytes for the same
// latency: 4 x 4096 x 2047 bf16 212 and 691 us (its values go through registers, which the backward pass spills: 460 to 472
// bytes stored a thread), float32 230 and 234 us. Tried and slower: rows parked in registers (spills; 707 us), one tile a CTA (452 us), 16-byte
// cp.async for the rows (373 us: the copies' issue took as long as a pass), 16 tiles looked at every time (327 us), sums
// over a head by shuffles (the compiler's form of them in this loop takes 300 cycles each).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "model_common.cuh"

namespace tb200 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * kWarp;

struct Divisor {  // n / d for n below 2^31, by a multiplication
  uint32_t factor, shift;
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(factor, n) + n) >> shift; }
};
Divisor divisor(uint32_t d) {
  uint32_t shift = 0;
  while ((1ull << shift) < d) ++shift;
  return Divisor{(uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}

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
  Divisor by_blocks, by_chains, by_gates;  // by_gates: heads in a block
  // bytes from a row to the next one with the recurrence
  int next_gate, next_in, next_out, next_y, next_dgate;
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
// tile's map, so the value is the same wherever the walk begins, to the bit. Eight tiles back, and eight more where all
// the maps of the first eight but none of their states are known (few chains, many tiles of each in work); where no
// state is known there either, the wait is for one to come closer, which the tile right behind the last known state
// always brings about.
constexpr int kReach = 8;
struct InFront {  // what is known of eight tiles in front, nearest first
  unsigned long long maps[kReach];
  unsigned states[kReach];
  __device__ __forceinline__ void look(const unsigned long long* m, const unsigned* s, uint64_t step, unsigned tile) {
#pragma unroll
    for (int j = 0; j < kReach; ++j) {
      s -= step;
      m -= step;
      states[j] = j < tile ? ld_relaxed_u32(s) : 0u;
      maps[j] = j < tile ? ld_relaxed_u64(m) : 0ull;
    }
  }
  // For a whole warp: the distance of the nearest state that all its channels know, with all maps nearer than it; kReach
  // where there are only maps, more where some are missing.
  __device__ __forceinline__ int nearest() const {
    unsigned all_states = 0, all_maps = 0;
#pragma unroll
    for (int j = 0; j < kReach; ++j) {
      all_states |= (unsigned)__all_sync(0xffffffffu, states[j] != 0u) << j;
      all_maps |= (unsigned)__all_sync(0xffffffffu, maps[j] != 0ull) << j;
    }
    const int from = __ffs(all_states | 1u << kReach) - 1;
    return (~all_maps & ((1u << from) - 1u)) != 0 ? kReach + 1 : from;
  }
  // From the state at a distance, or from h where that is kReach, through the nearer maps.
  __device__ __forceinline__ float through(int from, float h) const {
#pragma unroll
    for (int j = kReach - 1; j >= 0; --j) {
      if (j > from) continue;
      h = j == from ? __uint_as_float(~states[j])
                    : apply((unsigned)(~maps[j] >> 32), h, __uint_as_float((unsigned)~maps[j]));
    }
    return h;
  }
};
// One look. True where the state is known.
__device__ __forceinline__ bool look_for_state(const unsigned long long* maps, const unsigned* states, uint64_t step,
                                               unsigned tile, float& h) {
  InFront near;
  near.look(maps, states, step, tile);
  int from = near.nearest();
  if (from > kReach) return false;
  if (from == kReach) {
    if (tile <= kReach) return false;
    InFront far;
    far.look(maps - kReach * step, states - kReach * step, step, tile - kReach);
    from = far.nearest();
    if (from >= kReach) return false;
    h = far.through(from, 0.0f);
    from = kReach;
  }
  h = near.through(from, h);
  return true;
}
__device__ __forceinline__ float wait_for_state(const unsigned long long* maps, const unsigned* states, uint64_t step,
                                                unsigned tile, int* status) {
  float h = 0.0f;
  for (unsigned polls = 0; !look_for_state(maps, states, step, tile, h); ++polls) {
    if ((polls & 63u) == 63u && __any_sync(0xffffffffu, ld_relaxed_s32(status) == (int)TB200_ERR_WAIT_TIMEOUT)) break;  // someone else gave up
    if (polls >= kSpinLimit) {
      note_timeout(status, kSiteLookback, tile, 0);
      break;
    }
    backoff(polls);
  }
  return h;
}

template <int TILE>
struct Marks {  // of the rows of a tile of packed sequences
  int seq[TILE];             // sequence of a first or last row
  unsigned char kind[TILE];  // bit 0: first row of its sequence, bit 1: last
  uint64_t from, to;         // the rows of all sequences
  bool plain;                // the tile is full, and all its rows are inner ones of one sequence
};

__device__ __forceinline__ uint64_t offset_at(const RecArgs& p, uint64_t i) {
  const int64_t v = p.offset_bytes == 4 ? (int64_t)static_cast<const int32_t*>(p.offsets)[i]
                                        : static_cast<const int64_t*>(p.offsets)[i];
  return v < 0 ? 0 : (uint64_t)v > p.length ? p.length : (uint64_t)v;
}

// Marks the first and last rows of sequences among rows [r0, r1), in memory order; hands the states of empty sequences
// that lie here through for channels [c0, c0 + count). True where the rows are inner ones of one sequence. For one warp.
template <int TILE>
__device__ bool mark_rows(const RecArgs& p, uint64_t r0, uint64_t r1, bool at_end, uint32_t c0, uint32_t count, Marks<TILE>& m) {
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
  if (lo > 0 && lo <= p.sequences && offset_at(p, lo) > r1) return true;  // inner rows of one sequence
  for (uint64_t base = lo; base <= p.sequences; base += kWarp) {
    const uint64_t j = base + lane;
    const bool here = j <= p.sequences && offset_at(p, j) <= r1;
    bool empty = false;
    if (here) {
      const uint64_t v = offset_at(p, j);
      if (j > 0 && v > r0 && offset_at(p, j - 1) < v) {  // sequence j - 1 ends in front of boundary j
        m.seq[v - 1 - r0] = (int)(j - 1);
        atomicOr(reinterpret_cast<unsigned*>(m.kind) + (v - 1 - r0) / 4, 2u << (8 * ((v - 1 - r0) % 4)));
      }
      if (j < p.sequences && (v < r1 || at_end)) {
        const uint64_t end = offset_at(p, j + 1);
        if (end > v && v < r1 && v >= r0) {
          m.seq[v - r0] = (int)j;
          atomicOr(reinterpret_cast<unsigned*>(m.kind) + (v - r0) / 4, 1u << (8 * ((v - r0) % 4)));
        }
        empty = end <= v;
      }
    }
    for (unsigned left = __ballot_sync(0xffffffffu, empty && p.last != nullptr); left != 0; left &= left - 1) {
      const uint64_t row = (base + __ffs(left) - 1) * p.channels;  // all lanes hand its states through
      for (uint32_t c = c0 + lane; c < c0 + count; c += kWarp) p.last[row + c] = p.first ? p.first[row + c] : 0.0f;
    }
    if (!__all_sync(0xffffffffu, here)) break;
  }
  return false;
}

// Asynchronous copies of a lane's own channels into its own place in shared memory: no barrier, only the lane's wait.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// A tile, as one thread works it out for all: where its first row (with the recurrence) begins in every array, at the
// block's first channel. The others follow at RecArgs::next_* bytes.
struct TileInfo {
  const char *gate, *in, *y;  // y: the row in front in memory, which may not exist
  char *out, *dgate;
  int64_t row;          // the first row's place in the chain, in memory order
  uint32_t id, tile;    // id >= the number of tiles: there is none
  uint32_t chain, block;
  uint32_t c0, count;   // the block's channels
  uint32_t head;        // its first head
  int rows;             // how many of the tile's rows exist
  bool plain;           // all, and none is a first or last one; what packed sequences add to that stands in their marks
};
template <typename T, typename G, int WIDTH, int TILE, bool SHARED, bool BACK>
__device__ __forceinline__ void describe(const RecArgs& p, unsigned id, unsigned total, TileInfo& o) {
  o.id = id;
  if (id >= total) return;
  const unsigned rest = p.by_blocks.of(id), block = id - rest * p.blocks;
  const unsigned tile = p.by_chains.of(rest), chain = rest - tile * p.chains;
  o.tile = tile;
  o.chain = chain;
  o.block = block;
  uint32_t head = 0, c0 = block * WIDTH, count = min((uint32_t)WIDTH, p.channels - c0);
  if (SHARED && p.parts == 1) {
    head = block * p.block_heads;
    c0 = head * p.head_size;
    count = min(p.block_heads, p.heads - head) * p.head_size;
  } else if (SHARED) {
    head = block / p.parts;
    const uint32_t part = block - head * p.parts;
    c0 = head * p.head_size + part * WIDTH;
    count = min((uint32_t)WIDTH, p.head_size - part * WIDTH);
  }
  o.c0 = c0;
  o.count = count;
  o.head = head;
  const uint64_t first = (uint64_t)tile * TILE, left = p.chain_rows - first;
  o.rows = left < TILE ? (int)left : TILE;
  const int64_t row = BACK ? (int64_t)(p.chain_rows - 1 - first) : (int64_t)first;
  o.row = row;
  o.plain = left > TILE && first != 0 && p.chain_is_sequence;
  auto place = [&](const RowsOf& a, uint32_t column) { return (int64_t)(chain * a.seq + column) + row * (int64_t)a.row; };
  const uint32_t gate = SHARED ? head : c0;
  o.gate = p.gate.data + place(p.gate, gate) * (int64_t)sizeof(G);
  o.in = p.in.data + place(p.in, c0) * (int64_t)sizeof(T);
  o.out = p.out.data + place(p.out, c0) * (int64_t)sizeof(T);
  if constexpr (BACK) {
    o.y = p.y.data + (place(p.y, c0) - (int64_t)p.y.row) * (int64_t)sizeof(T);
    o.dgate = p.dgate.data + place(p.dgate, gate) * (int64_t)sizeof(G);
  }
}
// Which of the warp's rows are what: bit r of a mask is row r.
struct RowKinds {
  unsigned inside, begin, end;  // rows of a sequence; its first and last one with the recurrence
};
template <int TILE, bool BACK>
__device__ void marks_of_tile(const RecArgs& p, const TileInfo& w, Marks<TILE>& m) {  // for one warp
  const uint64_t lo = (uint64_t)w.tile * TILE, hi = min(lo + TILE, p.chain_rows);
  const uint64_t r0 = BACK ? p.chain_rows - hi : lo, r1 = BACK ? p.chain_rows - lo : hi;
  const bool none = mark_rows(p, r0, r1, r1 == p.chain_rows, w.c0, w.count, m);
  if (lane_id() == 0) {
    m.from = offset_at(p, 0);
    m.to = offset_at(p, p.sequences);
    m.plain = none && w.rows == TILE;
  }
}

// Bytes of shared memory that tiles may take, beside the joins and marks.
constexpr int kStageBudget = 200 << 10;
constexpr int kStages = 4;  // a tile in each: parked, landed, and two on their way
// Rows of a lane: eight, or four where four tiles of eight rows a lane would not fit.
constexpr int rows_of_lane(int bytes_of_row) { return kStages * 8 * bytes_of_row * kThreads <= kStageBudget ? 8 : 4; }

template <typename T, typename G, int V, bool SHARED, bool BACK>
struct Shape {
  static constexpr int GV = SHARED ? 1 : V;  // gates of a lane in a row
  static constexpr int ROW = (int)(sizeof(Pack<T, V>) * (BACK ? 2 : 1) + sizeof(Pack<G, GV>));
  static constexpr int R = rows_of_lane(ROW);
  // Four channels a lane: tiles come as boxes of a tensor map. One: every thread copies its own channels, 4 bytes and
  // more asynchronously, less through registers. Shared gates always take the latter way.
  static constexpr bool BOXES = V == 4;
  static constexpr bool X_ASYNC = sizeof(T) >= 4, G_ASYNC = !SHARED && sizeof(G) >= 4;
  // the exponentials of log gates take the place of gates of 32 bits
  static constexpr bool KEEPS_EXP = sizeof(G) == 4 && !SHARED;
  static constexpr int kX = R * kThreads * (int)sizeof(Pack<T, V>);
  static constexpr int kGate = R * kThreads * (int)sizeof(Pack<G, GV>);
  static constexpr int kStage = kX * (BACK ? 2 : 1) + kGate;
  [[maybe_unused]] static constexpr int kBoxes = kX * (BACK ? 2 : 1) + (SHARED ? 0 : kGate);
  static constexpr int kJoin = kWarps * kWarp * V * 4;
  static constexpr size_t kBytes = (size_t)kStages * kStage + 4 * kJoin;
  static_assert(kStages * kStage <= kStageBudget && kStage % 128 == 0 && kX % 128 == 0, "room and alignment of the stages");
};

// A box of rows and channels of one sequence into shared memory. x is a multiple of 16 bytes; rows and channels outside the
// array come as zeros. Never used with multicast.
__device__ __forceinline__ void box_load(void* to, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(smem_u32(to)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

// Barriers: the states in front of a tile's stretches are there, by the parity of the tile; among the warps that join.
enum : int { kStatesReady = 1, kJoined = 3 };
__device__ __forceinline__ bool mbar_test(unsigned long long* bar, unsigned parity) {  // without waiting
  unsigned ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ void barrier_arrive(int id, int count) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory");
}

// Waits for a phase of one of the CTA's own barriers; where that takes about a second, carries on with the status raised.
// Boxes land and warps arrive whatever became of other CTAs, so nothing that the status says ends a wait: boxes may be on
// their way, and in scratch that no tile waits in the status is whatever was there until block 0 sets it, among its first
// instructions and so long before a wait can run out. Once a wait of the CTA ran out, its others wait a 64th of that.
__device__ __forceinline__ void mbar_wait(unsigned long long* bar, unsigned parity, int* status, volatile int* gave_up) {
  for (unsigned spins = 0; !mbar_try_wait(bar, parity); ++spins) {
    if ((spins & 1023u) != 1023u) continue;
    if (spins >= (*gave_up ? kSpinLimit / 64 : kSpinLimit)) {
      *gave_up = 1;
      note_timeout(status, kSiteMbarrier, smem_u32(bar), parity);
      return;
    }
  }
}

// One CTA on an SM, which takes tile after tile. Eight warps compute: the first pass over tile i as soon as its rows have
// landed, then the second pass over tile i - 1, once the state in front of it is known. One thread for each channel
// joins: it hands the state in front of tile i - 1 on if it is known by now, puts the stretches of tile i together and
// publishes its map, all while the others compute. Order between the two kinds: s_ready (maps of all stretches are
// there; all warps are done with tile i - 2, whose stage takes the rows of tile i + 2) and the named barriers
// kStatesReady (states in front of all stretches are there; descriptions of the tiles up to i + 2 as well).
template <typename T, typename G, int V, bool SHARED, bool BACK>
__global__ void __launch_bounds__(kThreads + kWarp * V, 1)
recurrence_kernel(const __grid_constant__ RecArgs p, const __grid_constant__ CUtensorMap map_gate,
                  const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_y) {
  using S = Shape<T, G, V, SHARED, BACK>;
  constexpr int WIDTH = kWarp * V, GV = S::GV, R = S::R, TILE = kWarps * R;
  constexpr int CTA = kThreads + WIDTH;
  constexpr unsigned ALL = (1u << R) - 1;
  extern __shared__ __align__(128) char s_dynamic[];
  __shared__ Marks<TILE> s_marks[4];  // a ring
  // of the stretches: bit 0, a sequence begins among the rows; bit 1, there are rows in front of that
  __shared__ __align__(8) unsigned char s_kinds[2][kWarps];
  __shared__ int s_seq[2][kWarps][R];  // sequences of first and last rows, by the parity of the tile
  __shared__ TileInfo s_tiles[8];  // of the CTA, a ring
  __shared__ float s_heads[SHARED && BACK ? kWarps : 1][SHARED && BACK ? R : 1][kWarp + 1];
  __shared__ unsigned long long s_landed[kStages];  // a stage's boxes
  __shared__ unsigned long long s_ready[2];         // the maps of all warps' stretches, by the parity of the tile
  __shared__ int s_gave_up;                         // a wait for one of these ran out
  auto* s_word = reinterpret_cast<unsigned(*)[kWarps][WIDTH]>(s_dynamic + kStages * S::kStage);
  auto* s_b = reinterpret_cast<float(*)[kWarps][WIDTH]>(s_dynamic + kStages * S::kStage + 2 * S::kJoin);

  // Tiles are handed out in the order of the recurrence, all chains and blocks of channels of one stretch of rows before
  // the next: whatever a tile waits for is worked on by a CTA that runs already, and a tile's map never waits for more
  // than the tiles in front of it in its own CTA.
  const bool chained = p.tiles > 1;
  const unsigned total = (unsigned)p.tiles * p.chains * p.blocks;
  auto draw = [&](unsigned behind) { return chained ? atomicAdd(&p.hdr->ticket, 1u) : behind + gridDim.x; };
  auto describe_tile = [&](unsigned id, unsigned i) { describe<T, G, WIDTH, TILE, SHARED, BACK>(p, id, total, s_tiles[i & 7]); };

  const bool joins = threadIdx.x >= kThreads;
  const int lane = (int)lane_id(), warp = (int)(threadIdx.x / kWarp);
  const bool logg = p.log_gate != 0;
  // the lane's place in a row, in bytes; shared gates: its head's place among the block's
  const int lane_x = lane * V * (int)sizeof(T);
  const int lane_head = SHARED && p.parts == 1 ? lane * V / (int)p.head_size : 0;
  const int lane_g = SHARED ? lane_head * (int)sizeof(G) : lane * V * (int)sizeof(G);
  const int head_lanes = SHARED ? (p.parts == 1 ? (int)p.head_size / V : kWarp) : 1;
  constexpr int GATES = SHARED ? kWarp : WIDTH;  // places for gates in a row of a stage

  // row r of the warp in a stage; rows lie in the order of memory
  auto place = [&](int r) { return BACK ? TILE - 1 - (warp * R + r) : warp * R + r; };
  auto stage_x = [&](int k, int r) { return reinterpret_cast<Pack<T, V>*>(s_dynamic + k * S::kStage + place(r) * WIDTH * (int)sizeof(T) + lane_x); };
  auto stage_y = [&](int k, int r) { return reinterpret_cast<Pack<T, V>*>(s_dynamic + k * S::kStage + S::kX + place(r) * WIDTH * (int)sizeof(T) + lane_x); };
  char* const gates = s_dynamic + S::kX * (BACK ? 2 : 1);
  auto stage_g = [&](int k, int r) { return reinterpret_cast<Pack<G, GV>*>(gates + k * S::kStage + place(r) * GATES * (int)sizeof(G) + lane_g); };
  auto row_of = [&](auto* base, int next, int r) { return base + (int64_t)(warp * R + r) * next; };

  // Brings a tile's rows on their way to a stage. One thread asks for the boxes; the rest every computing warp
  // fetches for itself, and what comes through registers gets to the stage with `settle`.
  struct Late {
    G gate[S::G_ASYNC || S::BOXES && !SHARED ? 1 : R];
    T x[S::X_ASYNC || S::BOXES ? 1 : R];
    T before[S::X_ASYNC || S::BOXES || !BACK ? 1 : R];
  } late;
  const int block_gates = SHARED ? (p.parts == 1 ? (int)p.block_heads : 1) : 0;  // of a row
  constexpr int ASKS = CTA - kWarp;  // the thread that asks for the boxes
  auto fetch_boxes = [&](const TileInfo& w, int k) {
    unsigned long long* bar = &s_landed[k];
    char* to = s_dynamic + k * S::kStage;
    const int y = BACK ? (int)w.row - (TILE - 1) : (int)w.row, z = p.chain_is_sequence ? (int)w.chain : 0;
    mbar_expect_tx(bar, S::kBoxes);
    box_load(to, &map_in, (int)w.c0, y, z, bar);
    if constexpr (BACK) box_load(to + S::kX, &map_y, (int)w.c0, y - 1, z, bar);
    if constexpr (!SHARED) box_load(to + S::kX * (BACK ? 2 : 1), &map_gate, (int)w.c0, y, z, bar);
  };
  auto fetch = [&](const TileInfo& w, int k) {
    const int n = w.rows - warp * R;  // rows of this warp
    if constexpr (SHARED) {
      // the warp's gates, one a lane: row by row, the block's heads of a row side by side
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int v = j * kWarp + lane, r = (int)p.by_gates.of(v), h = v - r * block_gates;
        if (j * kWarp >= R * block_gates) break;
        if (r < R && r < n && w.head + h < p.heads) late.gate[j] = load_pack<G, 1>(row_of(w.gate, p.next_gate, r), h).v[0];
      }
    }
    if constexpr (!S::BOXES) {
      if (lane >= (int)w.count) return;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= n) break;
        const char* x = row_of(w.in + lane_x, p.next_in, r);
        if constexpr (S::X_ASYNC) copy_async<sizeof(T)>(stage_x(k, r), x); else late.x[r] = load_pack<T, 1>(x, 0).v[0];
        if constexpr (!SHARED) {
          const char* g = row_of(w.gate + lane_g, p.next_gate, r);
          if constexpr (S::G_ASYNC) copy_async<sizeof(G)>(stage_g(k, r), g); else late.gate[r] = load_pack<G, 1>(g, 0).v[0];
        }
        if constexpr (BACK) {
          if (w.row - warp * R - r > 0) {
            const char* y = row_of(w.y + lane_x, p.next_y, r);
            if constexpr (S::X_ASYNC) copy_async<sizeof(T)>(stage_y(k, r), y); else late.before[r] = load_pack<T, 1>(y, 0).v[0];
          }
        }
      }
    }
  };
  auto settle = [&](int k) {
    if constexpr (SHARED) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int v = j * kWarp + lane, r = (int)p.by_gates.of(v), h = v - r * block_gates;
        if (j * kWarp >= R * block_gates) break;
        if (r < R) reinterpret_cast<G*>(gates + k * S::kStage)[place(r) * GATES + h] = late.gate[j];
      }
    }
    if constexpr (!S::BOXES) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (!S::G_ASYNC && !SHARED) stage_g(k, r)->v[0] = late.gate[r];
        if constexpr (!S::X_ASYNC) {
          stage_x(k, r)->v[0] = late.x[r];
          if constexpr (BACK) stage_y(k, r)->v[0] = late.before[r];
        }
      }
    }
    __syncwarp();  // lanes read one another's gates
  };

  if (threadIdx.x == ASKS) {
    for (int k = 0; k < kStages; ++k) mbar_init(&s_landed[k], 1);
    for (int k = 0; k < 2; ++k) mbar_init(&s_ready[k], kWarps);
    mbar_init_fence();
    s_gave_up = 0;
  }
  if (threadIdx.x == kThreads) describe_tile(chained ? draw(0) : blockIdx.x, 0);
  __syncthreads();
  if (s_tiles[0].id >= total) return;
  if (!joins) {
    fetch(s_tiles[0], 0);
    copies_issued();
    settle(0);
  } else {
    if (S::BOXES && threadIdx.x == ASKS) fetch_boxes(s_tiles[0], 0);
    if (threadIdx.x == kThreads) {
      const unsigned id1 = draw(s_tiles[0].id), id2 = draw(id1);
      describe_tile(id1, 1);
      describe_tile(id2, 2);
      if (!chained && blockIdx.x == 0) p.hdr->status = TB200_OK;  // scratch that no tile waits in is not cleared
    }
    __syncwarp();
    if (p.offsets && warp == kWarps)
      for (int i = 0; i < 2 && s_tiles[i].id < total; ++i) marks_of_tile<TILE, BACK>(p, s_tiles[i], s_marks[i]);
  }
  __syncthreads();

  if (joins) {
    // ================================ the threads that join: one for each channel ==============================
    const unsigned c = threadIdx.x - kThreads;
    const uint64_t step = (uint64_t)p.chains * p.blocks * WIDTH;
    if (p.offsets != nullptr && s_tiles[0].id == 0) {  // bad offsets are reported, and cannot lead outside the arrays
      bool bad = false;
      for (uint64_t i = c; i <= p.sequences; i += WIDTH) {
        const int64_t v = p.offset_bytes == 4 ? (int64_t)static_cast<const int32_t*>(p.offsets)[i]
                                              : static_cast<const int64_t*>(p.offsets)[i];
        bad = bad || v < 0 || (uint64_t)v > p.length || (i == 0 ? v != 0 : (uint64_t)v < offset_at(p, i - 1));
      }
      if (bad) atomicExch(&p.hdr->status, (int)TB200_ERR_INVALID_ARGUMENT);
    }
    if (S::BOXES && threadIdx.x == ASKS && s_tiles[1].id < total) fetch_boxes(s_tiles[1], 1);
    // of the tile before: its own map and its warps', whether its state is to be published, whether it needs the one in front
    unsigned p_id = 0, p_tile = 0, p_word = 0, p_words[kWarps] = {};
    float p_b = 0.0f, p_bs[kWarps] = {};
    unsigned long long p_begins = 0;
    bool p_state = false, p_wait = false;
    for (unsigned i = 0;; ++i) {
      const int k = i & 1;
      const unsigned id = s_tiles[i & 7].id;
      const bool some = id < total;
      unsigned drawn = total;  // the answer is looked at much later
      if (c == 0) {
        const unsigned newest = s_tiles[(i + 2) & 7].id;
        if (newest < total) drawn = draw(newest);
      }
      const uint64_t p_at = (uint64_t)p_id * WIDTH + c;
      // ---- the states in front of the stretches of the tile before: at once where they are known by now, ---------
      // ---- else after this tile's map is out -----------------------------------------------------------------------
      float in_front = 0.0f;
      bool known = true;
      unsigned long long* maps_ready = &s_ready[k];
      if (p_wait) {
        do {  // as long as there is nothing else to do
          known = look_for_state(p.maps + p_at, p.states + p_at, step, p_tile, in_front);
        } while (!known && some && !__any_sync(0xffffffffu, mbar_test(maps_ready, i >> 1 & 1)));
      }
      auto hand_on = [&] {
        if (i > 0) {
          if (p_state) st_relaxed_u32(p.states + p_at, state_bits(apply(p_word, in_front, p_b)));
          float h = in_front;
#pragma unroll
          for (int v = 0; v < kWarps; ++v) {
            s_b[k ^ 1][v][c] = h;
            const float on = apply(p_words[v], h, p_bs[v]);
            h = p_begins >> (8 * v) & 1 ? p_bs[v] : on;
          }
        }
        barrier_arrive(kStatesReady + (k ^ 1), CTA);
      };
      if (known) hand_on();

      // ---- this tile's map; behind a begin only B counts --------------------------------------------------
      unsigned word = 0, tile = 0, words[kWarps] = {};
      float tb = 0.0f, bs[kWarps] = {};
      unsigned long long begins = 0;
      bool need = false;
      if (some) {
        tile = s_tiles[i & 7].tile;
        mbar_wait(maps_ready, i >> 1 & 1, &p.hdr->status, &s_gave_up);
        // all warps are done with the tile before the parked one: its stage is free
        if (S::BOXES && threadIdx.x == ASKS && s_tiles[(i + 2) & 7].id < total) fetch_boxes(s_tiles[(i + 2) & 7], (i + 2) % kStages);
        const unsigned long long kinds = *reinterpret_cast<const unsigned long long*>(s_kinds[k]);
        begins = kinds & 0x0101010101010101ull;
        need = (kinds >> 1 & 0x0101010101010101ull & (((begins & -begins) << 1) - 1)) != 0;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
          words[v] = s_word[k][v][c];
          bs[v] = s_b[k][v][c];
        }
        if (chained) {
          float ta = 1.0f, tm = 0.0f;
#pragma unroll
          for (int v = 0; v < kWarps; ++v) {
            const float m = __uint_as_float(words[v]);
            const float wa = (words[v] & 1u) ? 1.0f + m : m, wm = (words[v] & 1u) ? m : m - 1.0f;
            const float on = apply(words[v], tb, bs[v]);
            tb = begins >> (8 * v) & 1 ? bs[v] : on;
            ta *= wa;
            tm = fmaf(tm, wa, wm);
          }
          word = word_of(ta, tm);
          if (tile + 1 < p.tiles) {
            const uint64_t to = (uint64_t)id * WIDTH + c;
            // no row of any sequence: nobody behind needs a state before a sequence begins, so any will do
            if (begins || tile == 0 || !need) st_relaxed_u32(p.states + to, state_bits(tb));
            else st_relaxed_u64(p.maps + to, map_bits(word, tb));
          }
        }
      }
      if (!known) {
        in_front = wait_for_state(p.maps + p_at, p.states + p_at, step, p_tile, &p.hdr->status);
        hand_on();
      }
      if (!some) return;
      if (c == 0) describe_tile(drawn, i + 3);
      if (p.offsets && warp == kWarps && s_tiles[(i + 2) & 7].id < total)
        marks_of_tile<TILE, BACK>(p, s_tiles[(i + 2) & 7], s_marks[(i + 2) & 3]);
      p_id = id;
      p_tile = tile;
      p_word = word;
      p_b = tb;
      p_begins = begins;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) p_words[v] = words[v], p_bs[v] = bs[v];
      p_wait = need && tile > 0;
      p_state = p_wait && !begins && tile + 1 < p.tiles;
      // what one thread has described, and no thread far ahead of the others
      if constexpr (WIDTH > kWarp) named_barrier(kJoined, WIDTH); else __syncwarp();
    }
  }

  // ==================================== the warps that compute ================================================
  RowKinds pk{};
  bool parked = false, unsettled = false, p_plain = false;
  for (unsigned i = 0;; ++i) {
    const int k = i & 1;
    const TileInfo& w = s_tiles[i & 7];
    const bool some = w.id < total;
    const int stage = i % kStages, s1 = (i + 1) % kStages, s2 = (i + 2) % kStages, p_stage = (i + 3) % kStages;
    if ((!S::BOXES || SHARED) && i == 0) {
      if (s_tiles[1].id < total) {
        fetch(s_tiles[1], s1);
        unsettled = true;
      }
      copies_issued();
    }
    const bool plain = p.offsets ? s_marks[i & 3].plain : w.plain;
    RowKinds kinds{ALL, 0, 0};
    if (some) {
      // ---- first and last rows of sequences ---------------------------------------------------------------
      if (!plain) {
        const int n = max(0, min(R, w.rows - warp * R));
        const bool valid = lane < n;
        int seq = w.chain;  // of row `lane`, where that is a first or last one
        const int64_t mine = valid ? (BACK ? w.row - warp * R - lane : w.row + warp * R + lane) : 0;  // lane r: row r
        unsigned m_first = 0, m_last = 0;
        kinds.inside = (1u << n) - 1;
        if (p.offsets != nullptr) {
          const uint64_t lo = (uint64_t)w.tile * TILE, hi = min(lo + TILE, p.chain_rows);
          const int64_t r0 = BACK ? p.chain_rows - hi : lo;
          const unsigned kind = valid ? s_marks[i & 3].kind[mine - r0] : 0;
          if (kind) seq = s_marks[i & 3].seq[mine - r0];
          m_first = __ballot_sync(0xffffffffu, kind & 1);
          m_last = __ballot_sync(0xffffffffu, kind & 2);
          kinds.inside = __ballot_sync(0xffffffffu, valid && (uint64_t)mine >= s_marks[i & 3].from && (uint64_t)mine < s_marks[i & 3].to);
        } else if (p.chain_is_sequence) {
          m_first = __ballot_sync(0xffffffffu, valid && mine == 0);
          m_last = __ballot_sync(0xffffffffu, valid && (uint64_t)mine == p.chain_rows - 1);
        } else {  // sequences of equal length behind one another
          const uint64_t s = p.chain_rows >> 32 ? (uint64_t)mine / p.length : (uint32_t)mine / (uint32_t)p.length;
          const uint64_t t = (uint64_t)mine - s * p.length;
          seq = (int)s;
          m_first = __ballot_sync(0xffffffffu, valid && t == 0);
          m_last = __ballot_sync(0xffffffffu, valid && t == p.length - 1);
        }
        kinds.begin = BACK ? m_last : m_first;
        kinds.end = BACK ? m_first : m_last;
        if (lane < R) s_seq[k][warp][lane] = seq;
        __syncwarp();
      }

      // ---- first pass: the stretch's A and B ----------------------------------------------------------------
      if constexpr (S::BOXES) mbar_wait(&s_landed[stage], i / kStages & 1, &p.hdr->status, &s_gave_up);
      else asm volatile("cp.async.wait_group 1;" ::: "memory");  // all but the copies of the tile behind
      // all values first: nothing below comes between the loads
      Pack<G, GV> gate[R];
      Pack<T, V> x[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        gate[r] = *stage_g(stage, r);
        x[r] = *stage_x(stage, r);
      }
      float A[GV], M[GV], B[V], sum[GV];
      fill_n(A, 1.0f);
      fill_n(M, 0.0f);
      fill_n(sum, 0.0f);
      fill_n(B, 0.0f);
      auto first_pass = [&](auto inner, auto log_gate) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (!inner && !(kinds.inside >> r & 1)) continue;
          const bool begin = !inner && (kinds.begin >> r & 1);
          if (begin) {
            const uint64_t s = s_seq[k][warp][r];
#pragma unroll
            for (int e = 0; e < V; ++e)
              B[e] = p.first && lane * V < (int)w.count ? p.first[s * p.channels + w.c0 + lane * V + e] : 0.0f;
          }
          float a[GV], av[V], xv[V];
#pragma unroll
          for (int e = 0; e < GV; ++e) a[e] = to_f32<G>(gate[r].v[e]);
#pragma unroll
          for (int e = 0; e < V; ++e) xv[e] = to_f32<T>(x[r].v[e]);
          if (log_gate) {  // errors stay within the stretch of a warp's rows, so the fast exponential will do
            float unit[GV];
            fill_n(unit, kLog2e);
            add_n(sum, sum, a);
            mul_n(a, a, unit);
#pragma unroll
            for (int e = 0; e < GV; ++e) a[e] = exp2_fast(a[e]);
            if constexpr (S::KEEPS_EXP) *stage_g(stage, r) = pack_of<G, GV>(a);  // for the second pass
          } else {
            float less[GV], one[GV];
            fill_n(one, -1.0f);
            add_n(less, a, one);
            mul_n(A, A, a);
            fma_n(M, M, a, less);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) av[e] = a[SHARED ? 0 : e];
          if constexpr (BACK) {
            add_n(B, xv, B);
            mul_n(B, av, B);
          } else if (begin && !p.first) {
#pragma unroll
            for (int e = 0; e < V; ++e) B[e] = xv[e];
          } else {
            fma_n(B, av, B, xv);
          }
        }
      };
      if (plain) {
        if (logg) first_pass(std::true_type{}, std::true_type{}); else first_pass(std::true_type{}, std::false_type{});
      } else {
        first_pass(std::false_type{}, logg);
      }
      if (logg) {
#pragma unroll
        for (int e = 0; e < GV; ++e) {
          const float c = hold_gate(sum[e], true);
          const bool near = held_near(c, true);
          A[e] = near ? 1.0f + c : c;
          M[e] = near ? c : c - 1.0f;
        }
      }
      Pack<unsigned, V> words;
#pragma unroll
      for (int e = 0; e < V; ++e) words.v[e] = word_of(A[SHARED ? 0 : e], M[SHARED ? 0 : e]);
      *reinterpret_cast<Pack<unsigned, V>*>(&s_word[k][warp][lane * V]) = words;
      *reinterpret_cast<Pack<float, V>*>(&s_b[k][warp][lane * V]) = pack_of<float, V>(B);
      if (lane == 0) {
        const bool in_front = (kinds.inside & ((kinds.begin & -kinds.begin) - 1u)) != 0;
        s_kinds[k][warp] = (unsigned char)((kinds.begin != 0) | in_front << 1);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_ready[k]);
    }
    if (unsettled) settle(s1);  // what was fetched a step ago, for the tile behind this one
    unsettled = false;

    named_barrier(kStatesReady + (k ^ 1), CTA);
    auto fetch_two_ahead = [&] {
      const TileInfo& ahead = s_tiles[(i + 2) & 7];
      if (some && ahead.id < total) {
        fetch(ahead, s2);
        unsettled = true;
      }
      copies_issued();
    };
    if constexpr (!S::BOXES || SHARED) fetch_two_ahead();  // into the stage that the tile before the parked one has left

    // ---- second pass: the parked tile's outputs ---------------------------------------------------------------
    if (parked) {
      const TileInfo& pw = s_tiles[(i - 1) & 7];
      const bool live = lane * V < (int)pw.count;
      const uint32_t ch = pw.c0 + lane * V;
      const Pack<float, V> in_front = *reinterpret_cast<const Pack<float, V>*>(&s_b[k ^ 1][warp][lane * V]);
      float h[V];
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = in_front.v[e];
      Pack<G, GV> gate[R];
      Pack<T, V> x[R], before[BACK ? R : 1];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        gate[r] = *stage_g(p_stage, r);
        x[r] = *stage_x(p_stage, r);
        if constexpr (BACK) before[r] = *stage_y(p_stage, r);
      }
      char* to = pw.out + lane_x;
      char* to_g = BACK ? pw.dgate + lane_g : nullptr;
      float head_sum[SHARED && BACK ? R : 1] = {};
      auto second_pass = [&](auto inner, auto log_gate) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool in = inner || (pk.inside >> r & 1);
          if (!in && !(p.fill && warp * R + r < pw.rows)) continue;
          const bool begin = !inner && (pk.begin >> r & 1);
          const bool end = !inner && (pk.end >> r & 1);
          const uint64_t s = inner ? 0 : s_seq[k ^ 1][warp][r];
          if (begin) {
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = p.first && live ? p.first[s * p.channels + ch + e] : 0.0f;
          }
          float a[GV], av[V], xv[V], out[V], dg[V];
#pragma unroll
          for (int e = 0; e < GV; ++e) a[e] = to_f32<G>(gate[r].v[e]);
          if (!S::KEEPS_EXP && log_gate) {
            float unit[GV];
            fill_n(unit, kLog2e);
            mul_n(a, a, unit);
#pragma unroll
            for (int e = 0; e < GV; ++e) a[e] = exp2_fast(a[e]);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) av[e] = a[SHARED ? 0 : e], xv[e] = to_f32<T>(x[r].v[e]);
          if constexpr (BACK) {
            float prev[V];
#pragma unroll
            for (int e = 0; e < V; ++e) prev[e] = to_f32<T>(before[r].v[e]);
            if (end) {
#pragma unroll
              for (int e = 0; e < V; ++e) prev[e] = p.initial && live ? p.initial[s * p.channels + ch + e] : 0.0f;
            }
            add_n(out, xv, h);
            mul_n(h, av, out);
            if (log_gate) mul_n(dg, h, prev); else mul_n(dg, out, prev);
          } else {
            if (begin && !p.first) {
#pragma unroll
              for (int e = 0; e < V; ++e) h[e] = xv[e];
            } else {
              fma_n(h, av, h, xv);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) out[e] = h[e];
          }
          if (!in) {
            fill_n(out, 0.0f);
            fill_n(dg, 0.0f);
          }
          if ((inner && !SHARED) || live) store_floats<T, V>(row_of(to, p.next_out, r), 0, out);
          if constexpr (BACK) {
            if constexpr (!SHARED) {
              if (inner || live) store_floats<G, V>(row_of(to_g, p.next_dgate, r), 0, dg);
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e) head_sum[r] += dg[e];
              if (!live) head_sum[r] = 0.0f;
            }
          }
          if (in && end && p.last && live) {
#pragma unroll
            for (int e = 0; e < V; ++e) p.last[s * p.channels + ch + e] = h[e];
          }
        }
      };
      if (!SHARED && p_plain && !live) {
        // nothing to write
      } else if (p_plain) {
        if (logg) second_pass(std::true_type{}, std::true_type{}); else second_pass(std::true_type{}, std::false_type{});
      } else {
        second_pass(std::false_type{}, logg);
      }
      if constexpr (SHARED && BACK) {
        // the lanes' sums meet in shared memory: a lane adds up one row of one head, in the order of the channels
        // (shuffles here are compiled to a form that takes 300 cycles each)
        float(*sums)[kWarp + 1] = s_heads[warp];
#pragma unroll
        for (int r = 0; r < R; ++r) sums[r][lane] = head_sum[r];
        __syncwarp();
        for (int v = lane; v < R * block_gates; v += kWarp) {
          const int r = (int)p.by_gates.of(v), h = v - r * block_gates;
          const bool there = p_plain || (pk.inside >> r & 1) || (p.fill && warp * R + r < pw.rows);
          if (!there || h * head_lanes * V >= (int)pw.count) continue;
          float one[1] = {0.0f};
          for (int l = 0; l < head_lanes; ++l) one[0] += sums[r][h * head_lanes + l];
          if (p.parts == 1) {
            store_floats<G, 1>(row_of(pw.dgate, p.next_dgate, r), h, one);
          } else {
            const uint64_t flat = pw.chain * p.chain_rows + (uint64_t)(pw.row - warp * R - r);
            p.partial[(flat * p.heads + pw.head) * p.parts + pw.block % p.parts] = one[0];
          }
        }
        __syncwarp();
      }
    }
    if (!some) return;
    if (S::KEEPS_EXP && S::BOXES) fence_proxy_async_smem();  // exponentials were stored where boxes will land
    parked = true;
    p_plain = plain;
    pk = kinds;
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

// Blocks of channels and tiles for a CTA that is `width` channels wide.
void divide(RecArgs& p, uint32_t width, int bytes_of_row) {
  const uint64_t tile_rows = (uint64_t)kWarps * rows_of_lane(bytes_of_row);
  p.tiles = (p.chain_rows + tile_rows - 1) / tile_rows;
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

constexpr uint64_t kShortRows = 32;  // sequences up to this length fill at most half a tile

struct Call {
  tb200_recurrence_shape shape;
  RecArgs args;
  uint64_t rows;     // of all sequences
  char* descriptors;
};

// ---- tensor maps ------------------------------------------------------------------------------------------------------

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
EncodeTiled encode_tiled() {  // asked of the runtime, so that the library does not link the driver
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}
template <typename T> constexpr CUtensorMapDataType map_type();
template <> constexpr CUtensorMapDataType map_type<float>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT32; }
template <> constexpr CUtensorMapDataType map_type<__half>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }
template <> constexpr CUtensorMapDataType map_type<__nv_bfloat16>() { return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }

// Boxes of `rows` rows by 128 channels of an array of [sequences][rows][channels]. False where it cannot be had.
template <typename T>
bool map_of(CUtensorMap* map, const RowsOf& a, const RecArgs& p, int rows) {
  constexpr uint64_t E = sizeof(T);
  const uint64_t sequences = p.chain_is_sequence ? p.sequences : 1;
  const uint64_t apart = sequences > 1 ? a.seq * E : a.row * E;
  if (!rows_on(a, E, 16) || a.row == 0 || apart == 0 || apart >= (1ull << 40) || a.row * E >= (1ull << 40)) return false;
  const cuuint64_t dims[3] = {p.channels, p.chain_rows, sequences};
  const cuuint64_t strides[2] = {a.row * E, apart};
  const cuuint32_t box[3] = {4 * kWarp, (cuuint32_t)rows, 1}, ones[3] = {1, 1, 1};
  return encode_tiled()(map, map_type<T>(), 3, a.data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
struct Maps {
  CUtensorMap gate, in, y;
};

template <typename T, typename G, int V, bool SHARED, bool BACK>
struct Tag {};
template <typename T, typename G, int V, bool SHARED, bool BACK>
int launch_kernel(Call& k, const Maps& maps, cudaStream_t stream) {
  RecArgs& p = k.args;
  constexpr uint32_t WIDTH = kWarp * V;
  divide(p, WIDTH, Shape<T, G, V, SHARED, BACK>::ROW);
  const uint64_t ctas = p.tiles * p.chains * p.blocks;
  if (ctas > 0x7fffffffull) return TB200_ERR_UNSUPPORTED;
  if (p.tiles > 1) {
    const size_t states = ctas * WIDTH;
    p.states = reinterpret_cast<unsigned*>(k.descriptors);
    p.maps = reinterpret_cast<unsigned long long*>(k.descriptors + states * sizeof(unsigned));
    TB200_CUDA_TRY(cudaMemsetAsync(p.hdr, 0, kHeaderBytes + states * (sizeof(unsigned) + sizeof(unsigned long long)), stream));
  }
  p.by_blocks = divisor(p.blocks);
  p.by_chains = divisor(p.chains);
  p.by_gates = divisor(SHARED && p.parts == 1 ? p.block_heads : 1);
  const auto next = [](const RowsOf& a, int elem) { return (int)(a.row * elem) * (BACK ? -1 : 1); };
  for (const RowsOf* a : {&p.gate, &p.in, &p.out, &p.y, &p.dgate})
    if (a->row > (1u << 28)) return TB200_ERR_UNSUPPORTED;  // a tile's rows are reached by 32-bit steps
  p.next_gate = next(p.gate, sizeof(G));
  p.next_in = next(p.in, sizeof(T));
  p.next_out = next(p.out, sizeof(T));
  p.next_y = next(p.y, sizeof(T));
  p.next_dgate = next(p.dgate, sizeof(G));
  constexpr size_t smem = Shape<T, G, V, SHARED, BACK>::kBytes;
  constexpr int threads = kThreads + kWarp * V;
  auto kernel = recurrence_kernel<T, G, V, SHARED, BACK>;
  int per_sm = 0, sms = 0;
  int rc = resident_ctas<Tag<T, G, V, SHARED, BACK>>(kernel, threads, smem, &per_sm);
  if (rc == TB200_OK) rc = sm_count_of_device(&sms);
  if (rc) return rc;
  const uint64_t slots = (uint64_t)per_sm * sms;
  kernel<<<(unsigned)(ctas < slots ? ctas : slots), threads, smem, stream>>>(p, maps.gate, maps.in, maps.y);
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
  // Four channels a lane, in boxes, where boxes can be had of everything that is read (rows and the blocks' first
  // channels on 16 bytes), rows are written in whole groups of four and a head's channels divide so; else one.
  constexpr int ST = 4 * sizeof(T), SG = 4 * sizeof(G);
  Maps maps{};
  bool wide = p.channels % 4 == 0 && p.chain_rows < (1ull << 31) && encode_tiled() != nullptr && rows_on(p.out, sizeof(T), ST);
  if (shared) {
    wide = wide && p.head_size % 4 == 0;
    divide(p, 4 * kWarp, 0);
    const uint32_t block = p.parts == 1 ? p.block_heads * p.head_size : p.head_size;
    wide = wide && block * sizeof(T) % 16 == 0;
  } else if (BACK) {
    wide = wide && rows_on(p.dgate, sizeof(G), SG);
  }
  const int rows = kWarps * (shared ? Shape<T, G, 4, true, BACK>::R : Shape<T, G, 4, false, BACK>::R);
  wide = wide && map_of<T>(&maps.in, p.in, p, rows);
  if (BACK) wide = wide && map_of<T>(&maps.y, p.y, p, rows);
  if (!shared) wide = wide && map_of<G>(&maps.gate, p.gate, p, rows);
  if (shared)
    return wide ? launch_kernel<T, G, 4, true, BACK>(k, maps, stream) : launch_kernel<T, G, 1, true, BACK>(k, maps, stream);
  return wide ? launch_kernel<T, G, 4, false, BACK>(k, maps, stream) : launch_kernel<T, G, 1, false, BACK>(k, maps, stream);
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
  if (s.offset_bytes == 0 && s.sequences != 0 && s.rows > (1ull << 40) / s.sequences) return TB200_ERR_UNSUPPORTED;
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
  p.chain_is_sequence = s.offset_bytes == 0 && (s.rows > kShortRows || !dense);
  p.chains = p.chain_is_sequence ? (uint32_t)s.sequences : 1;
  p.chain_rows = p.chain_is_sequence ? s.rows : k.rows;

  // Descriptors lie directly behind the header, where one clear reaches both; the sums of heads that span several
  // blocks lie behind them. The pointers' alignment decides on four or one channels a lane: room for either.
  size_t descriptors = 0, sums = 0;
  const int tb = model_bytes(s.dtype), gb = model_bytes(s.gate_dtype);
  for (int v = 1; v <= 4; v *= 4) {
    const uint32_t width = kWarp * v;
    divide(p, width, v * tb * (back ? 2 : 1) + (s.heads == s.channels ? v : 1) * gb);
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

bool good_states(std::initializer_list<const float*> states) {  // each may be absent
  uintptr_t all = 0;
  for (const float* s : states) all |= reinterpret_cast<uintptr_t>(s);
  return all % sizeof(float) == 0;
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
  if (!good_states({d_initial, d_final})) return TB200_ERR_INVALID_ARGUMENT;
  const bool packed = k.shape.offset_bytes != 0;
  if (packed && (!d_offsets || reinterpret_cast<uintptr_t>(d_offsets) % k.shape.offset_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  const bool some = k.rows != 0 && k.shape.sequences + (packed && k.shape.fill_outside) != 0;
  const int tb = model_bytes(k.shape.dtype);
  if (some && !(good_rows(gate, model_bytes(k.shape.gate_dtype)) && good_rows(x, tb) && good_rows(y, tb)))
    return TB200_ERR_INVALID_ARGUMENT;
  if (!some) {
    const int rc = status_without_rows(d_temp, d_offsets, k.shape.offset_bytes, k.shape.sequences, k.rows, stream);
    if (rc) return rc;
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
  if (!good_states({d_initial, d_dfinal, d_dinitial})) return TB200_ERR_INVALID_ARGUMENT;
  const bool packed = k.shape.offset_bytes != 0;
  if (packed && (!d_offsets || reinterpret_cast<uintptr_t>(d_offsets) % k.shape.offset_bytes)) return TB200_ERR_INVALID_ARGUMENT;
  const bool some = k.rows != 0 && k.shape.sequences + (packed && k.shape.fill_outside) != 0;
  const int tb = model_bytes(k.shape.dtype), gb = model_bytes(k.shape.gate_dtype);
  if (some && !(good_rows(gate, gb) && good_rows(y, tb) && good_rows(dy, tb) && good_rows(dx, tb) && good_rows(dgate, gb)))
    return TB200_ERR_INVALID_ARGUMENT;
  if (!some) {
    const int rc = status_without_rows(d_temp, d_offsets, k.shape.offset_bytes, k.shape.sequences, k.rows, stream);
    if (rc) return rc;
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

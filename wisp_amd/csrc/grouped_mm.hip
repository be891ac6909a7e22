// Matrix products grouped by expert with ragged sizes.
//
//   out[i] = w[e] x[i]   for the rows i in [ends[e - 1], ends[e])
//
// bfloat16: float32 sums of exact products, rounded once.  Block FP8: x and w
// are e4m3 codes, x with a float32 scale s per row and 128 columns, w with one
// per 128 x 128 block; per 128 columns kb
//   acc += dot(x[kb], w[kb]) * (s[i][kb] * ws[n / 128][kb])
// in float32, rounded to bfloat16.
//
// A chunk is 128 bytes of every row: 64 columns in bfloat16, two steps of
// v_mfma_f32_16x16x32_bf16; 128 columns in FP8, one v_mfma_f32_16x16x128_f8f6f4
// and one block of the scales.  The weights are the A operand, so a lane holds
// consecutive outputs of one row of x.
#include <type_traits>

#include "common.h"

namespace wisp {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kChunk = 128;   // bytes of a row per chunk
constexpr int kBlock = 128;   // rows and columns of a block of FP8 weights
constexpr int kWaves = 4;     // of a block
constexpr int kWaveRows = 64;  // weight rows of a wave
constexpr int kPanel = kWaves * kWaveRows;

struct Args {
  const uint8_t* x;
  const float* s;      // FP8: [rows, groups], s_ld floats apart
  const uint8_t* w;    // expert e at + e * w_stride bytes, rows w_ld bytes apart
  const float* ws;     // FP8: expert e at + e * ws_stride floats, [ceil(N / 128), groups]
  const int32_t* ends;
  void* out;           // [rows, N]
  int64_t x_ld, w_stride, w_ld, ws_stride, s_ld;  // bytes; floats for the scales
  int E, M, N;
  int row_bytes;       // of a row's columns
  int groups;          // FP8: scales of a row
  bool out_f32, zero_tail;
};

// ---------------------------------------------------------------------------
// Ranges of memory as buffers: what lies behind the end reads as zero
// ---------------------------------------------------------------------------

#ifdef __HIP_DEVICE_COMPILE__
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __attribute__((always_inline)) inline Buffer buffer(const void* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)p;  // (the same for the whole wave)
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), 0,
                                           __builtin_amdgcn_readfirstlane((int)bytes), 0x00027000);
}
__device__ __attribute__((always_inline)) inline u32x4 load16(Buffer b, int voff, int soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, voff, soff, 0));
}
__device__ __attribute__((always_inline)) inline float load4(Buffer b, int voff, int soff) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, voff, soff, 0));
}
__device__ __attribute__((always_inline)) inline void store16b(u32x4 v, Buffer b, int voff,
                                                                 int soff) {
  __builtin_amdgcn_raw_buffer_store_b128(v, b, voff, soff, 0);
}
__device__ __attribute__((always_inline)) inline void store4b(uint32_t v, Buffer b, int voff,
                                                                 int soff) {
  __builtin_amdgcn_raw_buffer_store_b32(v, b, voff, soff, 0);
}
__device__ __attribute__((always_inline)) inline void store2b(uint16_t v, Buffer b, int voff,
                                                                 int soff) {
  __builtin_amdgcn_raw_buffer_store_b16(v, b, voff, soff, 0);
}
__device__ __attribute__((always_inline)) inline f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __attribute__((always_inline)) inline f32x4 mfma_fp8(u32x4 a0, u32x4 a1, u32x4 b0,
                                                                u32x4 b1) {
  const i32x8 a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3],
                   (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
  const i32x8 b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3],
                   (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  // formats 0/0: e4m3; zero scale operands: the unscaled instruction
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, z, 0, 0, 0, 0, 0, 0);
}
#else  // the host pass does not know these builtins
typedef int Buffer;
__device__ inline Buffer buffer(const void*, uint32_t) { return 0; }
__device__ inline u32x4 load16(Buffer, int, int) { return u32x4{}; }
__device__ inline float load4(Buffer, int, int) { return 0.f; }
__device__ inline void store16b(u32x4, Buffer, int, int) {}
__device__ inline void store4b(uint32_t, Buffer, int, int) {}
__device__ inline void store2b(uint16_t, Buffer, int, int) {}
__device__ inline f32x4 mfma_bf16(u32x4, u32x4, f32x4 c) { return c; }
__device__ inline f32x4 mfma_fp8(u32x4, u32x4, u32x4, u32x4) { return f32x4{}; }
#endif

// Two float32 as bfloat16 (nearest, ties to even), the first in the low half.
__device__ inline uint32_t bf16_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// ---------------------------------------------------------------------------
// The groups
// ---------------------------------------------------------------------------

// Per expert its first row, its rows and the tiles before it.
struct Table {
  int start[kMaxExperts], rows[kMaxExperts], base[kMaxExperts + 1];
  int last;  // one past the last group's last row
};

// Ends outside [0, M] count as 0 or M, one below an earlier one as that one:
// groups never overlap and stay inside the buffer whatever ends holds.  Called
// by one wave.
__device__ inline void fill_table(Table* tab, const Args& a, int toks) {
  const int lane = threadIdx.x & 63;
  int top = 0, base = 0;
  for (int e0 = 0; e0 < a.E; e0 += 64) {
    int end = e0 + lane < a.E ? min(max(a.ends[e0 + lane], 0), a.M) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(end, d);
      end = lane >= d ? max(end, o) : end;
    }
    end = max(end, top);
    const int before = __shfl_up(end, 1);
    const int start = lane ? before : top;
    const int n = (end - start + toks - 1) / toks;
    int incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d);
      incl += lane >= d ? o : 0;
    }
    if (e0 + lane < a.E) {
      tab->start[e0 + lane] = start;
      tab->rows[e0 + lane] = end - start;
      tab->base[e0 + lane + 1] = base + incl;
    }
    top = __builtin_amdgcn_readlane(end, 63);
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  if (lane == 0) {
    tab->base[0] = 0;
    tab->last = top;
  }
}

// One output tile: an expert, a panel of its weight rows, and rows of x.
struct Work {
  int expert, panel, row0, rows;  // rows 0: none left
};

// Works are ordered by expert, then panel, then tile of rows; a group of n
// tiles splits into equal ones (rounded up to 16 rows).
__device__ inline Work find_work(const Table* tab, int w, int E, int npanels, int toks) {
  const int lane = threadIdx.x & 63;
  const int j = w / npanels;  // a tile of the work's expert
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int end = tab->base[min(e0 + lane, E - 1) + 1];
    const uint64_t hit = __ballot(end > j);
    if (hit) {
      const int e = e0 + __builtin_ctzll(hit);
      const int b = __builtin_amdgcn_readfirstlane(tab->base[e]);
      const int n = __builtin_amdgcn_readfirstlane(tab->base[e + 1]) - b;
      const int m = __builtin_amdgcn_readfirstlane(tab->rows[e]);
      const int start = __builtin_amdgcn_readfirstlane(tab->start[e]);
      const int off = w - b * npanels;
      const int per = ((m + n - 1) / n + 15) & ~15;
      const int m0 = (off % n) * per;
      // (rounding up may leave the last tiles fewer rows, or none)
      return Work{e, off / n, start + min(m0, m), max(min(per, m - m0), 0)};
    }
  }
  return Work{-1, 0, 0, 0};
}

// Blocks go to the XCDs round-robin; each XCD takes runs of kRun consecutive
// works, so blocks that read the same weights or rows share an L2.
constexpr int kRun = 32;
__device__ inline int work_of(int b, int j) {
  const int i = (b >> 3) + j * ((int)gridDim.x >> 3);
  return ((i / kRun) * 8 + (b & 7)) * kRun + i % kRun;
}

// Zeros into the rows behind the last group, all blocks together.
__device__ inline void zero_rows(const Args& a, int last) {
  const int64_t wide = a.out_f32 ? 4 : 2;
  uint8_t* p = (uint8_t*)a.out + last * (int64_t)a.N * wide;
  const int64_t bytes = (a.M - last) * (int64_t)a.N * wide;
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  const int64_t head = min((int64_t)(-(uintptr_t)p & 15), bytes), body = (bytes - head) / 16;
  if (at < head / 2) reinterpret_cast<uint16_t*>(p)[at] = 0;
  for (int64_t i = at; i < body; i += step)
    reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0, 0, 0, 0);
  const int64_t rest = (bytes - head - body * 16) / 2;
  if (at < rest) reinterpret_cast<uint16_t*>(p + head + body * 16)[at] = 0;
}

// Byte of 16-byte piece cb of row r of an LDS tile of 128-byte rows.  Rows
// shift their pieces, so that the 16 rows a fragment reads at one piece spread
// over the banks.
__device__ inline int at(int r, int cb) { return r * kChunk + ((cb ^ (r & 7)) << 4); }

// A tile's outputs, from row row0 of out on: rows behind the tile's are behind
// the buffer's end, and so is where a column behind N is sent.
struct Outputs {
  Buffer b;
  int N, wide;
};
__device__ __attribute__((always_inline)) inline Outputs outputs(const Args& a, int64_t row0,
                                                                 int rows) {
  const int wide = a.out_f32 ? 4 : 2;
  return Outputs{buffer((uint8_t*)a.out + row0 * a.N * wide, (uint32_t)(rows * a.N * wide)), a.N,
                 wide};
}
constexpr int kNowhere = INT32_MIN;  // an offset behind every end, with any tile's added

// 16 consecutive outputs (4 groups of 4), columns [n, n + 16) of row
// 16 * t + col.  (The tile's part of the offset is the wave's: per lane, the
// compiler would hold every tile's in a register through the products.)
template <bool F32, bool WHOLE>
__device__ __attribute__((always_inline)) inline void store16(const Outputs& o, int t, int col,
                                                              int n, const f32x4 (&v)[4]) {
  const int at = (col * o.N + n) * o.wide, soff = 16 * t * o.N * o.wide;
  if constexpr (F32) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if constexpr (WHOLE) {
        store16b(__builtin_bit_cast(u32x4, v[g]), o.b, n + 4 * g < o.N ? at + 16 * g : kNowhere,
                 soff);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          store4b(__float_as_uint(v[g][j]), o.b,
                  n + 4 * g + j < o.N ? at + 16 * g + 4 * j : kNowhere, soff);
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 x = v[2 * h], y = v[2 * h + 1];
      const u32x4 u = {bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(y[0], y[1]),
                       bf16_pair(y[2], y[3])};
      if constexpr (WHOLE) {
        store16b(u, o.b, n + 8 * h < o.N ? at + 16 * h : kNowhere, soff);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          store2b((uint16_t)(u[i / 2] >> (16 * (i & 1))), o.b,
                  n + 8 * h + i < o.N ? at + 16 * h + 2 * i : kNowhere, soff);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The tiles: 256 weight rows by up to 16 * NT rows of x
// ---------------------------------------------------------------------------
//
// Persistent blocks of four waves.  A wave owns 64 weight rows and reads them
// from memory straight into its registers, a chunk ahead: no other wave of the
// block needs them.  The rows of x, which all four need, go through LDS, two
// chunks a stage.  The loads of a block run ahead over the ends of its tiles.
// A wave's MFMA row i of group g is weight row 16 * (i / 4) + 4 * g + i % 4, so
// that a lane ends with 16 consecutive outputs of a row of x.

template <int NT>
struct Shape {
  static constexpr int kToks = 16 * NT;
  static constexpr int kCopies = kToks / 8 / kWaves;  // of a wave, 8 rows each
  static constexpr int kTile = kToks * kChunk;        // one chunk of the rows of x
  static constexpr int kScales = 4 * kToks * 4;       // FP8: two stages of two chunks
  static constexpr int kLds = 4 * kTile + kScales + (int)sizeof(Table);
};

// What a kernel writes: 16-byte pieces of bfloat16 (N a multiple of 8) or of
// float32 (of 4), or single values.
enum Out { kBf16, kF32, kNarrow };

template <bool FP8, int NT, Out OUT>
__global__ __launch_bounds__(256, NT == 16 ? 1 : 2) void grouped_tile_kernel(const Args a) {
  using Sh = Shape<NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* scales = reinterpret_cast<float*>(smem + 4 * Sh::kTile);
  Table* tab = reinterpret_cast<Table*>(smem + 4 * Sh::kTile + Sh::kScales);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  if (wave == 0) fill_table(tab, a, Sh::kToks);
  __syncthreads();
  const int npanels = (a.N + kPanel - 1) / kPanel;
  const int chunks = (a.row_bytes + kChunk - 1) / kChunk, pairs = (chunks + 1) / 2;

  // lane offsets into the weights and the rows of x
  const int wvoff = (16 * (col >> 2) + (col & 3)) * (int)a.w_ld + 16 * quarter;
  const int xrow = wave * 8 + (lane >> 3);
  const int xvoff = xrow * (int)a.x_ld + 16 * (lane & 7);

  // the three works in flight: computed, weights loading, rows loading
  struct Place {
    Work work;
    int pair;
  };
  int turn = 0;
  auto next = [&](Place p) -> Place {
    if (p.work.expert >= 0 && ++p.pair < pairs) return p;
    do {
      p.work = find_work(tab, work_of(blockIdx.x, turn++), a.E, npanels, Sh::kToks);
    } while (p.work.expert >= 0 && p.work.rows == 0);
    p.pair = 0;
    return p;
  };

  u32x4 wf[2][2][4];            // [chunk of a pair][half of it][group]
  u32x4 xs[2][Sh::kCopies];
  float xscale[2], wscale[2];

  auto load_w = [&](const Place& p, int c) {
    const int64_t r0 = p.work.panel * kPanel + wave * kWaveRows;
    const int64_t left = a.N - r0;  // (none: every load is behind the end)
    const Buffer b = buffer(a.w + (p.work.expert < 0 ? 0 : p.work.expert * a.w_stride) +
                                (left > 0 ? r0 * a.w_ld : 0),
                            p.work.expert < 0 || left <= 0
                                ? 0u
                                : (uint32_t)((left - 1) * a.w_ld + a.row_bytes));
    const int o = (2 * p.pair + c) * kChunk;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        wf[c][h][g] = load16(b, wvoff, 4 * g * (int)a.w_ld + o + 64 * h);
    if constexpr (FP8) {
      const Buffer sb = buffer(a.ws + (p.work.expert < 0 ? 0 : p.work.expert * a.ws_stride),
                               p.work.expert < 0 ? 0u
                                                 : (uint32_t)(4 * a.groups *
                                                              ((a.N + kBlock - 1) / kBlock)));
      wscale[c] = load4(sb, 0, 4 * ((int)(r0 / kBlock) * a.groups + 2 * p.pair + c));
    }
  };
  auto load_x = [&](const Place& p) {
    const Buffer b = buffer(a.x + p.work.row0 * a.x_ld,
                            p.work.rows ? (uint32_t)((p.work.rows - 1) * a.x_ld + a.row_bytes)
                                        : 0u);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int o = (2 * p.pair + c) * kChunk;
#pragma unroll
      for (int i = 0; i < Sh::kCopies; ++i)
        xs[c][i] = load16(b, xvoff, 32 * i * (int)a.x_ld + o);
    }
    if constexpr (FP8) {
      const Buffer sb = buffer(a.s + p.work.row0 * a.s_ld,
                               p.work.rows ? (uint32_t)(4 * ((p.work.rows - 1) * a.s_ld + a.groups))
                                           : 0u);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        xscale[c] = load4(sb, min(tid, Sh::kToks - 1) * (int)a.s_ld * 4, 4 * (2 * p.pair + c));
    }
  };
  // (columns behind the row's end are another row's: zeroed)
  auto store_x = [&](const Place& p, int stage) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int left = a.row_bytes - (2 * p.pair + c) * kChunk;
      if (left < kChunk && 16 * (lane & 7) >= left)
#pragma unroll
        for (int i = 0; i < Sh::kCopies; ++i) xs[c][i] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < Sh::kCopies; ++i)
        *reinterpret_cast<u32x4*>(smem + (2 * stage + c) * Sh::kTile +
                                  at(32 * i + xrow, lane & 7)) = xs[c][i];
      if constexpr (FP8)
        if (tid < Sh::kToks)
          scales[(2 * stage + c) * Sh::kToks + tid] = left > 0 ? xscale[c] : 0.f;
    }
  };

  f32x4 acc[4][NT];

  // A stage is multiplied in blocks of four 16-byte fragments a lane: bf16, one
  // half chunk of four tiles of 16 rows; FP8, one chunk of two.  The fragments of
  // a block are read while the one before it is multiplied; the last block of
  // a stage is multiplied behind the barrier, over the first reads of the next.
  constexpr int kSteps = FP8 ? 2 : 4;               // of a stage, along the columns
  constexpr int kWide = FP8 ? 2 : 4;                // tiles of 16 rows of a block
  constexpr int kBlocks = kSteps * (NT / kWide);
  u32x4 f[2][4];
  float fs[2][2];
  auto read = [&](int i, int stage, int b) {
    const int step = b / (NT / kWide), t0 = b % (NT / kWide) * kWide;
    const uint8_t* tile = smem + (2 * stage + (FP8 ? step : step / 2)) * Sh::kTile;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + (FP8 ? k / 2 : k), h = FP8 ? k & 1 : step & 1;
      f[i][k] = *reinterpret_cast<const u32x4*>(tile + at(16 * t + col, 4 * h + quarter));
    }
    if constexpr (FP8)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        fs[i][t] = scales[(2 * stage + step) * Sh::kToks + 16 * (t0 + t) + col];
  };
  auto multiply = [&](int i, int b, int nt) {
    const int step = b / (NT / kWide), t0 = b % (NT / kWide) * kWide;
    if (t0 >= nt) return;
    if constexpr (!FP8) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          acc[g][t0 + t] = mfma_bf16(wf[step / 2][step & 1][g], f[i][t], acc[g][t0 + t]);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float sc = fs[i][t] * wscale[step];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 d = mfma_fp8(wf[step][0][g], wf[step][1][g], f[i][2 * t], f[i][2 * t + 1]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[g][t0 + t][j] = __builtin_fmaf(d[j], sc, acc[g][t0 + t][j]);
        }
      }
    }
  };

  Place cur = next(Place{Work{-1, 0, 0, 0}, 0});
  if (cur.work.expert >= 0) {
    load_x(cur);
    load_w(cur, 0);
    load_w(cur, 1);
    store_x(cur, 0);
    Place wnext = next(cur);
    load_x(wnext);
    __syncthreads();
    read(0, 0, 0);
    int stage = 0;
    do {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[g][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      const Work work = cur.work;
      const int nt = (work.rows + 15) / 16;
      for (int pair = 0; pair < pairs; ++pair) {
        const Place xnext = next(wnext);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int left = a.row_bytes - (2 * pair + c) * kChunk;
          if (left < kChunk) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (64 * h + 16 * quarter >= left)
#pragma unroll
                for (int g = 0; g < 4; ++g) wf[c][h][g] = u32x4{0, 0, 0, 0};
          }
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          if (b + 1 < kBlocks) {
            read((b + 1) & 1, stage, b + 1);
          } else {
            block_lds_sync();
            read((b + 1) & 1, stage ^ 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          multiply(b & 1, b, nt);
          __builtin_amdgcn_sched_barrier(0);
          if (b == kBlocks / 4) {
            store_x(wnext, stage ^ 1);
            load_x(xnext);
          }
          if (b + 1 == kBlocks / 2) load_w(wnext, 0);
          if (b + 1 == kBlocks) load_w(wnext, 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        stage ^= 1;
        cur = wnext;
        wnext = xnext;
      }
      const Outputs o = outputs(a, work.row0, work.rows);
      const int n = work.panel * kPanel + wave * kWaveRows + 16 * quarter;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4 v[4] = {acc[0][t], acc[1][t], acc[2][t], acc[3][t]};
        if constexpr (OUT != kNarrow)
          store16<OUT == kF32, true>(o, t, col, n, v);
        else if (a.out_f32)
          store16<true, false>(o, t, col, n, v);
        else
          store16<false, false>(o, t, col, n, v);
      }
    } while (cur.work.expert >= 0);
  }
  if (a.zero_tail) zero_rows(a, tab->last);
}

template <bool FP8, int NT, Out OUT>
hipError_t launch_tile(const Args& a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_lds(&grouped_tile_kernel<FP8, NT, OUT>, Shape<NT>::kLds,
                                 Shape<NT>::kLds, &done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((grouped_tile_kernel<FP8, NT, OUT>), dim3(NT == 16 ? 256 : 512), dim3(256),
                     Shape<NT>::kLds, st, a);
  return hipGetLastError();
}

int refuse(int rc, const char* why, const char* where) {
  wisp_set_last_error(why, where);
  return rc;
}

template <bool FP8, Out OUT>
hipError_t launch_of(const Args& a, hipStream_t st) {
  // rows an expert has if the rows are spread evenly
  const int per = a.M / a.E;
  if constexpr (!FP8) {
    if (per > 128) return launch_tile<false, 16, OUT>(a, st);
  }
  return launch_tile<FP8, 4, OUT>(a, st);
}

template <bool FP8>
int grouped(const Args& a, hipStream_t st) {
  hipError_t e;
  if (a.N % (a.out_f32 ? 4 : 8))
    e = launch_tile<FP8, 4, kNarrow>(a, st);
  else if (a.out_f32)
    e = launch_of<false, kF32>(a, st);
  else
    e = launch_of<FP8, kBf16>(a, st);
  WISP_HIP_TRY(e);
  return WISP_OK;
}

// What both entry points check; elem: bytes of a column.
const char* unsupported(int64_t x_ld, int64_t w_ld, int64_t w_stride, int64_t N, int64_t K,
                        int elem, const void* x, const void* w) {
  if (K % (16 / elem)) return "a row of x and of w must be whole 16-byte pieces";
  if (x_ld * elem % 16 || w_ld * elem % 16 || w_stride * elem % 16 || (uintptr_t)x % 16 ||
      (uintptr_t)w % 16)
    return "x, w and their strides must be 16-byte aligned";
  // (32-bit offsets inside a tile of x and inside an expert's weights)
  if (N * w_ld * elem >= (int64_t)1 << 31 || x_ld * elem >= (int64_t)1 << 22 || N >= 1 << 21)
    return "an expert's weights of 2 GiB, rows of x 4 MiB apart or 2^21 outputs";
  return nullptr;
}

}  // namespace
}  // namespace wisp

extern "C" int wisp_grouped_mm(const void* x, int64_t x_ld, const void* w, int64_t w_stride,
                               int64_t w_ld, const int32_t* ends, int E, int M, int N, int K,
                               void* out, int out_dtype, int zero_tail, wisp_stream_t stream) {
  using namespace wisp;
  const char* where = "wisp_grouped_mm";
  if (E < 1 || M < 0 || N < 0 || K < 1 || (out_dtype != WISP_BF16 && out_dtype != WISP_F32))
    return refuse(WISP_ERR_INVALID, "invalid sizes", where);
  if (M == 0 || N == 0) return WISP_OK;
  if (!x || !w || !ends || !out || x_ld < K || w_ld < K || w_stride < 0)
    return refuse(WISP_ERR_INVALID, "a buffer is missing or a stride too small", where);
  if (E > kMaxExperts) return refuse(WISP_ERR_UNSUPPORTED, "more than 512 experts", where);
  if (const char* why = unsupported(x_ld, w_ld, w_stride, N, K, 2, x, w))
    return refuse(WISP_ERR_UNSUPPORTED, why, where);
  const Args a = {(const uint8_t*)x, nullptr, (const uint8_t*)w, nullptr, ends, out, 2 * x_ld,
                  2 * w_stride, 2 * w_ld, 0, 0, E, M, N, 2 * K, 0, out_dtype == WISP_F32,
                  zero_tail != 0};
  return grouped<false>(a, (hipStream_t)stream);
}

extern "C" int wisp_grouped_mm_fp8(const uint8_t* q, int64_t q_ld, const float* s, int64_t s_ld,
                                   const uint8_t* w, int64_t w_stride, int64_t w_ld,
                                   const float* ws, int64_t ws_stride, const int32_t* ends, int E,
                                   int M, int N, int K, void* out, int zero_tail,
                                   wisp_stream_t stream) {
  using namespace wisp;
  const char* where = "wisp_grouped_mm_fp8";
  if (E < 1 || M < 0 || N < 0 || K < 1) return refuse(WISP_ERR_INVALID, "invalid sizes", where);
  if (M == 0 || N == 0) return WISP_OK;
  const int groups = (K - 1) / kBlock + 1;
  if (!q || !s || !w || !ws || !ends || !out || q_ld < K || w_ld < K || w_stride < 0 ||
      s_ld < groups || ws_stride < 0)
    return refuse(WISP_ERR_INVALID, "a buffer is missing or a stride too small", where);
  if (E > kMaxExperts) return refuse(WISP_ERR_UNSUPPORTED, "more than 512 experts", where);
  if (const char* why = unsupported(q_ld, w_ld, w_stride, N, K, 1, q, w))
    return refuse(WISP_ERR_UNSUPPORTED, why, where);
  if (s_ld >= (int64_t)1 << 20)
    return refuse(WISP_ERR_UNSUPPORTED, "scales of x 4 MiB apart", where);
  const Args a = {q, s, w, ws, ends, out, q_ld, w_stride, w_ld, ws_stride, s_ld, E, M, N, K,
                  groups, false, zero_tail != 0};
  return grouped<true>(a, (hipStream_t)stream);
}

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
#include <algorithm>

#include "common.h"

namespace wisp {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kChunk = 128;   // bytes of a row per chunk
constexpr int kBlock = 128;   // rows and columns of a block of FP8 weights
constexpr int kWaves = 4;     // of a block
constexpr int kPanel = 256;   // weight rows of the large tiles

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
// 16 bytes at p, the same for the whole wave, plus a lane's offset.
__device__ __attribute__((always_inline)) inline u32x4 load_global(const uint8_t* p, uint32_t off) {
  typedef const __attribute__((address_space(1))) uint8_t* Bytes;
  return *(const __attribute__((address_space(1))) u32x4*)((Bytes)p + off);
}
__device__ __attribute__((always_inline)) inline float load_global4(const uint8_t* p,
                                                                     uint32_t off) {
  typedef const __attribute__((address_space(1))) uint8_t* Bytes;
  return *(const __attribute__((address_space(1))) float*)((Bytes)p + off);
}
__device__ __attribute__((always_inline)) inline const uint8_t* uniform(const uint8_t* p) {
  const uint64_t a = (uint64_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return (const uint8_t*)(((uint64_t)hi << 32) | lo);
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
__device__ __attribute__((always_inline)) inline void store8b(u32x2 v, Buffer b, int voff,
                                                                 int soff) {
  __builtin_amdgcn_raw_buffer_store_b64(v, b, voff, soff, 0);
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
__device__ __attribute__((always_inline)) inline f32x16 mfma_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
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
__device__ inline u32x4 load_global(const uint8_t*, uint32_t) { return u32x4{}; }
__device__ inline float load_global4(const uint8_t*, uint32_t) { return 0.f; }
__device__ inline const uint8_t* uniform(const uint8_t* p) { return p; }
__device__ inline u32x4 load16(Buffer, int, int) { return u32x4{}; }
__device__ inline float load4(Buffer, int, int) { return 0.f; }
__device__ inline void store16b(u32x4, Buffer, int, int) {}
__device__ inline void store8b(u32x2, Buffer, int, int) {}
__device__ inline void store4b(uint32_t, Buffer, int, int) {}
__device__ inline void store2b(uint16_t, Buffer, int, int) {}
__device__ inline f32x4 mfma_bf16(u32x4, u32x4, f32x4 c) { return c; }
__device__ inline f32x16 mfma_bf16(u32x4, u32x4, f32x16 c) { return c; }
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
// by one wave.  (Sums behind a group's rows are unsigned, here and in find_work: of
// 2^31 - 1 rows they pass 2^31, at most by a fourth.)
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
    const int n = (int)(((uint32_t)(end - start) + toks - 1) / toks);
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
__device__ inline Work find_work(const Table* tab, int w, int E, int npanels) {
  const int lane = threadIdx.x & 63;
  const int j = w / npanels;  // a tile of the work's expert
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int end = tab->base[min(e0 + lane, E - 1) + 1];
    const uint64_t hit = __ballot(end > j);
    if (hit) {
      const int e = e0 + __builtin_ctzll(hit);
      const int b = __builtin_amdgcn_readfirstlane(tab->base[e]);
      const int n = __builtin_amdgcn_readfirstlane(tab->base[e + 1]) - b;
      const uint32_t m = __builtin_amdgcn_readfirstlane(tab->rows[e]);
      const int start = __builtin_amdgcn_readfirstlane(tab->start[e]);
      const int off = w - b * npanels;
      const uint32_t per = ((m + n - 1) / n + 15) & ~15u;
      const uint32_t m0 = min((off % n) * per, m);
      // (rounding up may leave the last tiles fewer rows, or none)
      return Work{e, off / n, start + (int)m0, (int)min(per, m - m0)};
    }
  }
  return Work{-1, 0, 0, 0};
}

// Blocks go to the XCDs round-robin; each XCD takes runs of up to 32 consecutive
// works, so blocks that read the same weights or rows share an L2.  The runs are
// as many for every XCD, and as long: with runs of 32 always, 128 works would
// leave four XCDs with their L2 and their share of the memory's rate idle.
__device__ inline int run_length(int works) {
  const int turns = (works + 255) / 256;
  return max((works + 8 * turns - 1) / max(8 * turns, 1), 1);
}
__device__ inline int work_of(int b, int j, int run) {
  const int i = (b >> 3) + j * ((int)gridDim.x >> 3), turn = i / run;
  return (turn * 8 + (b & 7)) * run + i - turn * run;
}

// A pair of chunks of a work, left of them to go with this one.
struct Place {
  Work work;
  int pair, left;
};
__device__ inline Place nowhere() { return Place{Work{-1, 0, 0, 0}, 0, 0}; }

// The pairs of a block's works, one after the other.  Every 24 panels in a row
// start at a pair of their own and wrap around: blocks that all start at column 0
// crowd a few memory channels (Qwen3 w13 of 512 tokens 179 us, so 144), and panels
// that each start elsewhere read the rows of x that they share at different times,
// out of the L2 again (1024 tokens 161 us, so 154; 8192 tokens 463, 449).  24 is four
// experts of that layer in the large tiles, measured there; other sizes take it as it
// is.  So the order of a sum, and the last bits of its row, go by the expert's place in
// the call as well as by the kernel.
constexpr uint32_t kGolden = 2654435769u;  // 2^32 / 1.618..: any first n are spread evenly
template <int TOKS>
struct Walk {
  const Table* tab;
  int E, npanels, pairs, run, turn;
  __device__ __attribute__((always_inline)) inline Place next(Place p) {
    p.pair = p.pair + 1 == pairs ? 0 : p.pair + 1;
    if (--p.left > 0) return p;
    do {
      p.work = find_work(tab, work_of(blockIdx.x, turn++, run), E, npanels);
    } while (p.work.expert >= 0 && p.work.rows == 0);
    const uint32_t set = (uint32_t)(max(p.work.expert, 0) * npanels + p.work.panel) / 24;
    p.pair = (int)((uint64_t)(set * kGolden) * (uint32_t)pairs >> 32);
    p.left = pairs;
    return p;
  }
};

// Zeros into the rows behind the last group, all blocks (of a grid in x) together.
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

// Byte of 16-byte piece cb of row r of an LDS tile of 128-byte rows.  Rows shift
// their pieces so that no two of 16 lanes that a read serves in one cycle meet in a
// bank: lanes 0-3, 12-15, 20-27 of each half, the other 16 of it.  at: fragments of
// 16 rows, in order or 16 * a + 4 * g + b (below), lane l / 16 at its own piece.
// at32x and at32w: of 32 rows at one piece, in order, and 16 * h + 4 * a + b.
// (SQ_LDS_BANK_CONFLICT of the reads is 0; with one rule for all, the reads of
// 32 rows took 8 cycles instead of 4.)
__device__ inline int at(int r, int cb) {
  const int shift = (r & 3) | ((r >> 2 ^ r >> 4) & 1) << 2;
  return r * kChunk + ((cb ^ shift) << 4);
}
__device__ inline int at32x(int r, int cb) { return r * kChunk + ((cb ^ (r >> 1 & 7)) << 4); }
__device__ inline int at32w(int r, int cb) {
  const int shift = (r >> 1 & 1) | (r >> 4 & 1) << 1 | (r >> 2 & 1) << 2;
  return r * kChunk + ((cb ^ shift) << 4);
}

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

// 4 * G consecutive outputs, columns [n, n + 4 * G) of row t0 + r; WHOLE: N is a
// whole number of the pieces stored.  (t0, the same for the wave, goes into the
// scalar offset: per lane, the compiler would hold every tile's offset in a
// register through the products.)
template <bool F32, bool WHOLE, int G>
__device__ __attribute__((always_inline)) inline void store_outputs(const Outputs& o, int t0,
                                                                    int r, int n,
                                                                    const f32x4 (&v)[G]) {
  const int at = (r * o.N + n) * o.wide, soff = t0 * o.N * o.wide;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if constexpr (F32 && WHOLE) {
      store16b(__builtin_bit_cast(u32x4, v[g]), o.b, n + 4 * g < o.N ? at + 16 * g : kNowhere,
               soff);
    } else if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        store4b(__float_as_uint(v[g][j]), o.b, n + 4 * g + j < o.N ? at + 16 * g + 4 * j : kNowhere,
                soff);
    } else if constexpr (WHOLE && G > 1) {
      if (g % 2 == 0) {
        const f32x4 x = v[g], y = v[g + 1];
        const u32x4 u = {bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(y[0], y[1]),
                         bf16_pair(y[2], y[3])};
        store16b(u, o.b, n + 4 * g < o.N ? at + 8 * g : kNowhere, soff);
      }
    } else if constexpr (WHOLE) {
      store8b(u32x2{bf16_pair(v[g][0], v[g][1]), bf16_pair(v[g][2], v[g][3])}, o.b,
              n < o.N ? at : kNowhere, soff);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        store2b((uint16_t)(bf16_pair(v[g][j], 0.f) & 0xffff), o.b,
                n + 4 * g + j < o.N ? at + 8 * g + 2 * j : kNowhere, soff);
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows an expert: 64 * G weight rows by 64 rows of x
// ---------------------------------------------------------------------------
//
// What bounds these calls is the weights' stream (Qwen3 w13 of 512 tokens: 144 us,
// 5.6 TB/s; Mixtral's of 200 tokens 355 us, 5.3).  Persistent blocks of four
// waves; a wave owns 16 * G weight rows and reads them from memory straight into
// its registers, one to two chunks ahead: no other wave of the block needs them.
// The rows of x, which all four need, go through LDS, two chunks a stage.  The
// loads of a block run ahead over the ends of its tiles.  MFMA row i of a wave's
// group g is weight row 4 * G * (i / 4) + 4 * g + i % 4, so that a lane ends with
// 4 * G consecutive outputs of a row of x.

template <int NT, int G>
struct Shape {
  static constexpr int kPanel = kWaves * 16 * G;  // weight rows
  static constexpr int kToks = 16 * NT;
  static constexpr int kCopies = kToks / 8 / kWaves;  // of a wave, 8 rows each
  static constexpr int kTile = kToks * kChunk;        // one chunk of the rows of x
  static constexpr int kScales = 4 * kToks * 4;       // FP8: two stages of two chunks
  static constexpr int kLds = 4 * kTile + kScales + (int)sizeof(Table);
};

// What a kernel writes: 16-byte pieces of bfloat16 (N a multiple of 8) or of
// float32 (of 4), or single values.
enum Out { kBf16, kF32, kNarrow };

template <bool FP8, int NT, int G, Out OUT>
__global__ __launch_bounds__(256, 2) void grouped_tile_kernel(const Args a) {
  using Sh = Shape<NT, G>;
  constexpr int kPanel = Sh::kPanel;
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
  const int wvoff = (4 * G * (col >> 2) + (col & 3)) * (int)a.w_ld + 16 * quarter;
  const int xrow = wave * 8 + (lane >> 3);
  const int xvoff = xrow * (int)a.x_ld + 16 * (lane & 7);

  // (three places in flight: computed, weights loading, rows loading)
  Walk<Sh::kToks> walk{tab, a.E, npanels, pairs, run_length(tab->base[a.E] * npanels), 0};
  auto next = [&](const Place& p) { return walk.next(p); };

  u32x4 wf[2][2][G];            // [chunk of a pair][half of it][group]
  u32x4 xs[2][Sh::kCopies];
  float xscale[2], wscale[2];

  auto load_w = [&](const Place& p, int c) {
    const int64_t r0 = p.work.panel * kPanel + wave * 16 * G;
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
      for (int g = 0; g < G; ++g)
        wf[c][h][g] = load16(b, wvoff, 4 * g * (int)a.w_ld + o + 64 * h);
    if constexpr (FP8) {
      const Buffer sb = buffer(a.ws + (p.work.expert < 0 ? 0 : p.work.expert * a.ws_stride),
                               p.work.expert < 0 ? 0u
                                                 : (uint32_t)(4 * a.groups *
                                                              ((a.N + kBlock - 1) / kBlock)));
      // (behind the row's end the next block's would follow: none)
      wscale[c] = load4(sb, 2 * p.pair + c < a.groups ? 0 : kNowhere,
                        4 * ((int)(r0 / kBlock) * a.groups + 2 * p.pair + c));
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

  f32x4 acc[G][NT];

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
        for (int g = 0; g < G; ++g)
          acc[g][t0 + t] = mfma_bf16(wf[step / 2][step & 1][g], f[i][t], acc[g][t0 + t]);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float sc = fs[i][t] * wscale[step];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const f32x4 d = mfma_fp8(wf[step][0][g], wf[step][1][g], f[i][2 * t], f[i][2 * t + 1]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[g][t0 + t][j] = __builtin_fmaf(d[j], sc, acc[g][t0 + t][j]);
        }
      }
    }
  };

  Place cur = next(nowhere());
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
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[g][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      const Work work = cur.work;
      const int nt = (work.rows + 15) / 16;
      for (int pair = 0; pair < pairs; ++pair) {
        const Place xnext = next(wnext);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int left = a.row_bytes - (2 * cur.pair + c) * kChunk;
          if (left < kChunk) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (64 * h + 16 * quarter >= left)
#pragma unroll
                for (int g = 0; g < G; ++g) wf[c][h][g] = u32x4{0, 0, 0, 0};
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
      const int n = work.panel * kPanel + wave * 16 * G + 4 * G * quarter;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 v[G];
#pragma unroll
        for (int g = 0; g < G; ++g) v[g] = acc[g][t];
        if constexpr (OUT != kNarrow)
          store_outputs<OUT == kF32, true>(o, 16 * t, col, n, v);
        else if (!FP8 && a.out_f32)
          store_outputs<true, false>(o, 16 * t, col, n, v);
        else
          store_outputs<false, false>(o, 16 * t, col, n, v);
      }
    } while (cur.work.expert >= 0);
  }
  if (a.zero_tail) zero_rows(a, tab->last);
}

// ---------------------------------------------------------------------------
// bfloat16, many rows an expert: 256 weight rows by 64 * L rows of x
// ---------------------------------------------------------------------------
//
// One block a CU, four waves (2 x 2): a wave owns 128 weight rows and every other
// 32 rows of x, in 4 x L tiles of v_mfma_f32_32x32x16_bf16, the instruction that
// one wave a SIMD feeds best (on random values 2016 TFLOP/s, 1777 with 16x16x32).
// Both operands go through registers to LDS, 8 lanes a row, loaded three chunks
// ahead of their use: a wave that read its operands straight from memory, 16 rows
// of 64 bytes a load, would keep the address unit busy for 64 cycles a load
// instead of 16.  A chunk is four steps of 16 columns; between a step's matrix
// instructions go the reads of the next step's fragments, as early as they can,
// and a share of the chunk's stores and loads.  The last matrix instructions of a
// chunk's last step are multiplied behind the barrier, over the next reads.
// MFMA row 8 * a + 4 * h + b of a group of 32 is weight row 16 * h + 4 * a + b, so
// that a lane ends with 16 consecutive outputs of a row of x.
//
// Qwen3 w13 of 65536 rows, 128 experts (412 GFLOP): 449 to 457 us, 902 to 916 TFLOP/s;
// Mixtral w13 of 4000 rows (940 GFLOP): 977 us, 962 TFLOP/s.  Of 100 cycles the matrix
// units are busy for 58 and LDS for 34, at 1.74 GHz.  Without the loads the products
// take 287 us: the copies, which wait in registers and cost a write of 16 cycles a KB
// into LDS, are covered in part only; memory is read 1.25 GB of 1.07 needed.
// One more 64 rows of x a tile (L 4) spills registers and takes 465 us and more.
template <int L>
struct Big {
  static constexpr int kToks = 64 * L;
  static constexpr int kRows = kPanel + kToks;       // of a stage
  static constexpr int kStage = kRows * kChunk;
  static constexpr int kCopies = kRows / 32;         // of a wave, 8 rows each
  static constexpr int kLds = 2 * kStage + (int)sizeof(Table);
};

// TAIL: rows that are not whole pairs of chunks.
template <int L, bool TAIL>
__global__ __launch_bounds__(256, 1) void grouped_big_kernel(const Args a) {
  using Sh = Big<L>;
  extern __shared__ __align__(16) uint8_t smem[];
  Table* tab = reinterpret_cast<Table*>(smem + 2 * Sh::kStage);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave >> 1, wt = wave & 1;
  if (wave == 0) fill_table(tab, a, Sh::kToks);
  __syncthreads();
  const int npanels = (a.N + kPanel - 1) / kPanel;
  const int pairs = (a.row_bytes + 2 * kChunk - 1) / (2 * kChunk);  // of chunks

  // copies: this lane's row and piece of every 32 rows
  const int crow = wave * 8 + (lane >> 3), ccol = 16 * (lane & 7);
  uint8_t* const wdst = smem + at32w(crow, lane & 7);
  uint8_t* const xdst = smem + kPanel * kChunk + at32x(crow, lane & 7);
  // fragments: this lane's row of every 32
  const int col = lane & 31, high = lane >> 5;
  const int frow = 16 * (col >> 2 & 1) + 4 * (col >> 3) + (col & 3);

  Walk<Sh::kToks> walk{tab, a.E, npanels, pairs, run_length(tab->base[a.E] * npanels), 0};
  auto next = [&](const Place& p) { return walk.next(p); };
  // Where a work's rows start, and this lane's offsets of its copies from there;
  // rows behind the last are that one again (what they give is not stored).
  const uint8_t *wbase, *xbase;
  uint32_t off[Sh::kCopies];
  auto aim = [&](const Work& w) {
    const int64_t r0 = w.panel * kPanel;
    wbase = uniform(a.w + (w.expert < 0 ? 0 : w.expert * a.w_stride + r0 * a.w_ld));
    xbase = uniform(a.x + w.row0 * a.x_ld);
    const int wlast = w.expert < 0 ? 0 : (int)min(a.N - r0, (int64_t)kPanel) - 1;
    const int xlast = max(w.rows, 1) - 1;
#pragma unroll
    for (int i = 0; i < Sh::kCopies; ++i)
      off[i] = i < 8 ? min(32 * i + crow, wlast) * (uint32_t)a.w_ld
                     : min(32 * (i - 8) + crow, xlast) * (uint32_t)a.x_ld;
  };

  u32x4 cp[2][Sh::kCopies];  // two chunks on their way to LDS: weights, then rows of x
  f32x16 acc[4][L];
  u32x4 wf[2][4], xf[2][L];

  // Chunk c of a place's pair into cp[c].
  auto load = [&](int pair, int c, int i) {
    const int o = (2 * pair + c) * kChunk;
    const uint8_t* base = i < 8 ? wbase : xbase;
    if constexpr (TAIL)  // (columns behind the row's end: its last ones)
      cp[c][i] = load_global(base, off[i] + min(o + ccol, a.row_bytes - 16));
    else
      cp[c][i] = load_global(base + o, off[i] + ccol);
  };
  // chunk c of a pair has stage c
  auto store = [&](int pair, int c, int i) {
    u32x4 v = cp[c][i];
    if constexpr (TAIL) {
      // columns behind the row's end count as zero, in both operands
      const uint32_t keep = (2 * pair + c) * kChunk + ccol < a.row_bytes ? ~0u : 0u;
      v &= u32x4{keep, keep, keep, keep};
    }
    *reinterpret_cast<u32x4*>((i < 8 ? wdst + 32 * i * kChunk : xdst + 32 * (i - 8) * kChunk) +
                              c * Sh::kStage) = v;
  };
  auto read = [&](int c, int step, int i) {
    const int to = step & 1;
    if (i < 4)
      wf[to][i] = *reinterpret_cast<const u32x4*>(
          smem + c * Sh::kStage + at32w(128 * wr + 32 * i + frow, 2 * step + high));
    else
      xf[to][i - 4] = *reinterpret_cast<const u32x4*>(
          smem + c * Sh::kStage + kPanel * kChunk +
          at32x(32 * wt + 64 * (i - 4) + col, 2 * step + high));
  };

  Place cur = next(nowhere());
  if (cur.work.expert >= 0) {
    aim(cur.work);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < Sh::kCopies; ++i) load(cur.pair, c, i);
    Place n1 = next(cur);
    if (n1.left == pairs) aim(n1.work);
#pragma unroll
    for (int i = 0; i < Sh::kCopies; ++i) {
      store(cur.pair, 0, i);
      load(n1.pair, 0, i);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4 + L; ++i) read(0, 0, i);
    do {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int t = 0; t < L; ++t) acc[g][t] = f32x16{};
      const Work work = cur.work;
      for (int pair = 0; pair < pairs; ++pair) {
        const Place n2 = next(n1);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c == 1 && n2.left == pairs) aim(n2.work);
#pragma unroll
          for (int step = 0; step < 4; ++step)
#pragma unroll
            for (int i = 0; i < 2 * L; ++i) {  // two matrix instructions each
              if (step < 3) {
#pragma unroll
                for (int k = 2 * i; k < 2 * i + 2; ++k)
                  if (k < 4 + L) read(c, step + 1, k);
              } else if (i == 2 * L - 2) {
                block_lds_sync();
#pragma unroll
                for (int k = 0; k < 4 + L; ++k) read(c ^ 1, 0, k);
              }
#pragma unroll
              for (int m = 2 * i; m < 2 * i + 2; ++m)
                acc[m % 4][m / 4] = mfma_bf16(wf[step & 1][m % 4], xf[step & 1][m / 4],
                                              acc[m % 4][m / 4]);
              // This place's share of the copies, all of them before the barrier:
              // the next chunk leaves for its stage, and the one that follows it
              // by two is loaded.
              constexpr int kPlaces = 8 * L - 2;
              const int place = 2 * L * step + i;
              if (place < kPlaces) {
#pragma unroll
                for (int k = place * Sh::kCopies / kPlaces;
                     k < (place + 1) * Sh::kCopies / kPlaces; ++k) {
                  store(c == 0 ? cur.pair : n1.pair, c ^ 1, k);
                  load(c == 0 ? n1.pair : n2.pair, c ^ 1, k);
                }
              }
              // (the loads stay here: the compiler would sink them to their use)
              __builtin_amdgcn_sched_barrier(0);
            }
        }
        cur = n1;
        n1 = n2;
      }
      const Outputs o = outputs(a, work.row0, work.rows);
#pragma unroll
      for (int t = 0; t < L; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            v[q] = f32x4{acc[g][t][4 * q], acc[g][t][4 * q + 1], acc[g][t][4 * q + 2],
                         acc[g][t][4 * q + 3]};
          const int n = work.panel * kPanel + 128 * wr + 32 * g + 16 * high;
          if (a.out_f32)
            store_outputs<true, true>(o, 64 * t, 32 * wt + col, n, v);
          else
            store_outputs<false, true>(o, 64 * t, 32 * wt + col, n, v);
        }
    } while (cur.work.expert >= 0);
  }
  if (a.zero_tail) zero_rows(a, tab->last);
}

template <int L, bool TAIL>
hipError_t launch_big(const Args& a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_lds(&grouped_big_kernel<L, TAIL>, Big<L>::kLds, Big<L>::kLds,
                                 &done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((grouped_big_kernel<L, TAIL>), dim3(256), dim3(256), Big<L>::kLds, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Block FP8, many rows an expert: 256 weight rows by 256 rows of x
// ---------------------------------------------------------------------------
//
// The same copies, two chunks ahead.  The sums are scaled ones, which the vector
// units add, so they need vector registers: eight waves (2 x 4) of 128 weight rows
// (one row of blocks of the weights' scales) by 64 rows of x.  A chunk is one
// column of blocks and one v_mfma_f32_16x16x128_f8f6f4 a tile of 16 x 16, whose
// result is scaled into the sums while the next weight rows are multiplied.  MFMA
// row 4 * a + b of group 4 * c + g is weight row 64 * c + 16 * a + 4 * g + b, so
// that a lane ends with 16 consecutive outputs of a row of x.
//
// Mixtral w13 of 4000 rows (940 GFLOP): 525 to 570 us, 1650 to 1790 TFLOP/s.  Of 100 cycles the
// matrix units are busy for 56 and LDS for 37; the scaling (four fused adds behind a
// matrix instruction of 32 cycles) takes half as many vector cycles as that again,
// and all of it overlaps only as two waves a SIMD let it.  Without the loads 389 us.
// Four waves of 256 x 128 take 706 us; the 32 x 32 instruction's 16 sums a tile do
// not fit the registers (3826 us with spills).
struct Big8 {
  static constexpr int kWaves = 8;
  static constexpr int kToks = 256;
  static constexpr int kRows = kPanel + kToks;
  static constexpr int kStage = kRows * kChunk + kToks * 4;  // and the rows' scales
  static constexpr int kCopies = kRows / 64;  // of a wave, 8 rows each
  static constexpr int kLds = 2 * kStage + (int)sizeof(Table);
};

template <bool TAIL>
__global__ __launch_bounds__(512, 2) void grouped_big_fp8_kernel(const Args a) {
  using Sh = Big8;
  extern __shared__ __align__(16) uint8_t smem[];
  Table* tab = reinterpret_cast<Table*>(smem + 2 * Sh::kStage);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 2, wt = wave & 3;
  if (wave == 0) fill_table(tab, a, Sh::kToks);
  __syncthreads();
  const int npanels = (a.N + kPanel - 1) / kPanel;
  const int pairs = (a.row_bytes + 2 * kChunk - 1) / (2 * kChunk);  // of chunks

  const int crow = wave * 8 + (lane >> 3), ccol = 16 * (lane & 7);
  uint8_t* const cdst = smem + at(crow, lane & 7);
  const int col = lane & 15, quarter = lane >> 4;
  const int frow = 16 * (col >> 2) + (col & 3);

  Walk<Sh::kToks> walk{tab, a.E, npanels, pairs, run_length(tab->base[a.E] * npanels), 0};
  auto next = [&](const Place& p) { return walk.next(p); };
  const uint8_t *wbase, *xbase;
  const float *sbase, *wsbase;
  int wlast, xlast;  // (lane offsets are made from these at each load: no register is left)
  auto aim = [&](const Work& w) {
    const int64_t r0 = w.panel * kPanel;
    const int e = max(w.expert, 0);
    wbase = uniform(a.w + (w.expert < 0 ? 0 : e * a.w_stride + r0 * a.w_ld));
    xbase = uniform(a.x + w.row0 * a.x_ld);
    sbase = (const float*)uniform((const uint8_t*)(a.s + w.row0 * a.s_ld));
    // (a wave whose weight rows are all behind N scales by the last block)
    const int block = min((int)(r0 / kBlock) + wr, (a.N - 1) / kBlock);
    wsbase = (const float*)uniform(
        (const uint8_t*)(a.ws + e * a.ws_stride + (int64_t)block * a.groups));
    wlast = w.expert < 0 ? 0 : (int)min(a.N - r0, (int64_t)kPanel) - 1;
    xlast = max(w.rows, 1) - 1;
  };

  u32x4 cp[Sh::kCopies];
  float cs, cws, ws;  // scales on their way: of a row of x, of the weights' block
  f32x4 acc[8][4];
  auto load = [&](int pair, int c, int i) {
    const int o = (2 * pair + c) * kChunk;
    int row = crow;
    asm volatile("" : "+v"(row));  // (or the compiler holds both chunks' offsets in registers)
    const uint8_t* base = i < 4 ? wbase : xbase;
    const uint32_t at = i < 4 ? __umul24(min(64 * i + row, wlast), (uint32_t)a.w_ld)
                              : __umul24(min(64 * (i - 4) + row, xlast), (uint32_t)a.x_ld);
    if constexpr (TAIL)  // (columns behind the row's end: its last ones)
      cp[i] = load_global(base, at + min(o + ccol, a.row_bytes - 16));
    else
      cp[i] = load_global(base + o, at + ccol);
  };
  auto load_scales = [&](int pair, int c) {
    const int g = min(2 * pair + c, a.groups - 1);
    cs = load_global4((const uint8_t*)(sbase + g),
                      4 * __umul24(min(tid & (Sh::kToks - 1), xlast), (uint32_t)a.s_ld));
    cws = load_global4((const uint8_t*)(wsbase + g), 0);
  };
  auto store = [&](int pair, int c, int i) {
    u32x4 v = cp[i];
    if constexpr (TAIL) {
      const uint32_t keep = (2 * pair + c) * kChunk + ccol < a.row_bytes ? ~0u : 0u;
      v &= u32x4{keep, keep, keep, keep};
    }
    *reinterpret_cast<u32x4*>(cdst + c * Sh::kStage + 64 * i * kChunk) = v;
  };
  auto store_scale = [&](int pair, int c) {
    // (a chunk behind the row's end has no scales: nothing times zero)
    if (tid < Sh::kToks)
      reinterpret_cast<float*>(smem + c * Sh::kStage + Sh::kRows * kChunk)[tid] =
          !TAIL || 2 * pair + c < a.groups ? cs : 0.f;
  };
  // 32 columns a lane: pieces quarter and 4 + quarter (of both operands)
  u32x4 wf[2], xf[4][2];
  float xscale[4];
  auto read_w = [&](int c, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      wf[h] = *reinterpret_cast<const u32x4*>(
          smem + c * Sh::kStage +
          at(128 * wr + 64 * (g >> 2) + 4 * (g & 3) + frow, 4 * h + quarter));
  };
  auto read_x = [&](int c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xf[t][h] = *reinterpret_cast<const u32x4*>(
            smem + c * Sh::kStage + kPanel * kChunk +
            at(16 * wt + 64 * t + col, 4 * h + quarter));
      xscale[t] = reinterpret_cast<const float*>(smem + c * Sh::kStage +
                                                 Sh::kRows * kChunk)[16 * wt + 64 * t + col];
    }
  };
  auto add = [&](int g, int t, const f32x4& d, float sc) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[g][t][j] = __builtin_fmaf(d[j], sc, acc[g][t][j]);
    // (here and in vector registers: the compiler would gather a chunk's sums
    // behind its products, and keep them in accumulation registers between)
    asm volatile("" : "+v"(acc[g][t]));
  };

  Place cur = next(nowhere());
  if (cur.work.expert >= 0) {
    // (in the loop's order: a wait counts the loads behind the one it is for, the
    // fewest on any way there)
    aim(cur.work);
    load_scales(cur.pair, 0);
#pragma unroll
    for (int i = 0; i < Sh::kCopies; ++i) load(cur.pair, 0, i);
    store_scale(cur.pair, 0);
    ws = cws;
    load_scales(cur.pair, 1);
#pragma unroll
    for (int i = 0; i < Sh::kCopies; ++i) {
      store(cur.pair, 0, i);
      load(cur.pair, 1, i);
    }
    __syncthreads();
    read_x(0);
    read_w(0, 0);
    do {
#pragma unroll
      for (int g = 0; g < 8; ++g)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[g][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      const Work work = cur.work;
      for (int pair = 0; pair < pairs; ++pair) {
        // (the chunk after this one is on its way, the one after that is loaded)
        const Place n1 = next(cur);
        if (n1.left == pairs) aim(n1.work);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float sc[4];
          // (nothing times zero where neither has a scale; ws is the last group's there)
          if (TAIL && 2 * cur.pair + c >= a.groups) ws = 0.f;
#pragma unroll
          for (int t = 0; t < 4; ++t) sc[t] = xscale[t] * ws;
          store_scale(c == 0 ? cur.pair : n1.pair, c ^ 1);
          ws = cws;
          load_scales(n1.pair, c);
          f32x4 d[4];
#pragma unroll
          for (int g = 0; g < 8; ++g) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              if (g > 0) add(g - 1, t, d[t], sc[t]);
              d[t] = mfma_fp8(wf[0], wf[1], xf[t][0], xf[t][1]);
            }
            if (g < 7) read_w(c, g + 1);  // (the SIMD's other wave multiplies meanwhile)
            // this group's copy
            store(c == 0 ? cur.pair : n1.pair, c ^ 1, g);
            load(n1.pair, c, g);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) add(7, t, d[t], sc[t]);
          block_lds_sync();
          read_x(c ^ 1);
          read_w(c ^ 1, 0);
        }
        cur = n1;
      }
      const Outputs o = outputs(a, work.row0, work.rows);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const f32x4 v[4] = {acc[4 * c][t], acc[4 * c + 1][t], acc[4 * c + 2][t],
                              acc[4 * c + 3][t]};
          store_outputs<false, true>(o, 64 * t, 16 * wt + col,
                               work.panel * kPanel + 128 * wr + 64 * c + 16 * quarter, v);
        }
    } while (cur.work.expert >= 0);
  }
  if (a.zero_tail) zero_rows(a, tab->last);
}

template <bool TAIL>
hipError_t launch_big_fp8(const Args& a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_lds(&grouped_big_fp8_kernel<TAIL>, Big8::kLds, Big8::kLds, &done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((grouped_big_fp8_kernel<TAIL>), dim3(256), dim3(64 * Big8::kWaves),
                     Big8::kLds, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The fewest rows: 16 weight rows a block, the columns split over its waves
// ---------------------------------------------------------------------------
//
// One token's experts have too few panels to fill the GPU: 8 of Qwen3's w13 have
// 192 of 64 rows.  A block takes 16 weight rows of one group and each of its
// waves a fourth of the columns, whose loads are all in flight at once (kBatch
// chunks of both operands); the partial sums meet in LDS, in wave order.  Blocks go
// to the groups in use by their number: j-th in y, which ends name.  Qwen3 w13, one
// token: 17.2 us with the tiles, 10.9 so (4.6 TB/s; one round of blocks).
constexpr int kFewCols = 16;  // rows of x a pass

template <bool FP8, int kBatch>
__global__ __launch_bounds__(256) void grouped_few_kernel(const Args a) {
  __shared__ float part[kWaves][16][kFewCols + 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quarter = lane >> 4;

  // The group: the blockIdx.y-th of those with rows (every wave finds it).
  int expert = -1, row0 = 0, rows = 0, top = 0, seen = 0;
  for (int e0 = 0; e0 < a.E; e0 += 64) {
    int end = e0 + lane < a.E ? min(max(a.ends[e0 + lane], 0), a.M) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(end, d);
      end = lane >= d ? max(end, o) : end;
    }
    end = max(end, top);
    const int before = __shfl_up(end, 1), start = lane ? before : top;
    const uint64_t some = __ballot(end > start);
    const int at = (int)blockIdx.y - seen;  // among these
    const uint64_t mine = __ballot(end > start && __popcll(some & ((1ull << lane) - 1)) == at);
    if (mine) {
      const int l = __builtin_ctzll(mine);
      expert = e0 + l;
      row0 = __builtin_amdgcn_readlane(start, l);
      rows = __builtin_amdgcn_readlane(end, l) - row0;
    }
    seen += __popcll(some);
    top = __builtin_amdgcn_readlane(end, 63);
  }
  if (rows > 0) {
    const int n0 = blockIdx.x * 16;
    const int chunks = (a.row_bytes + kChunk - 1) / kChunk;
    const int c0 = chunks * wave / kWaves, c1 = chunks * (wave + 1) / kWaves;
    const uint8_t* w = a.w + expert * a.w_stride + min(n0 + col, a.N - 1) * a.w_ld;
    const float* ws = FP8 ? a.ws + expert * a.ws_stride + (int64_t)(n0 / kBlock) * a.groups
                          : nullptr;
    for (int m0 = 0; m0 < rows; m0 += kFewCols) {
      const int64_t r = row0 + min(m0 + col, rows - 1);
      const uint8_t* x = a.x + r * a.x_ld;
      const float* s = FP8 ? a.s + r * a.s_ld : nullptr;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      for (int c = c0; c < c1; c += kBatch) {
        u32x4 wf[kBatch][2], xf[kBatch][2];
        float sc[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int at = min(c + i, c1 - 1);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int o = min(at * kChunk + 64 * h + 16 * quarter, a.row_bytes - 16);
            wf[i][h] = *reinterpret_cast<const u32x4*>(w + o);
            xf[i][h] = *reinterpret_cast<const u32x4*>(x + o);
          }
          if constexpr (FP8) sc[i] = s[at] * ws[at];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (c + i >= c1) break;
          // columns behind the row's end count as zero, in both operands
          const int left = a.row_bytes - (c + i) * kChunk;
          if (left < kChunk) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (64 * h + 16 * quarter >= left) wf[i][h] = xf[i][h] = u32x4{0, 0, 0, 0};
          }
          if constexpr (FP8) {
            const f32x4 d = mfma_fp8(wf[i][0], wf[i][1], xf[i][0], xf[i][1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(d[j], sc[i], acc[j]);
          } else {
            acc = mfma_bf16(wf[i][0], xf[i][0], acc);
            acc = mfma_bf16(wf[i][1], xf[i][1], acc);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) part[wave][4 * quarter + j][col] = acc[j];
      __syncthreads();
      const int n = threadIdx.x & 15, m = threadIdx.x >> 4;
      float v = part[0][n][m];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) v += part[i][n][m];
      if (n0 + n < a.N && m0 + m < rows) {
        const int64_t at = (int64_t)(row0 + m0 + m) * a.N + n0 + n;
        if (!FP8 && a.out_f32)
          ((float*)a.out)[at] = v;
        else
          ((uint16_t*)a.out)[at] = bf16_rne(v);
      }
      __syncthreads();
    }
  }
  if (a.zero_tail && blockIdx.y == 0) zero_rows(a, top);
}

template <bool FP8, int kBatch>
hipError_t launch_few(const Args& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)std::min(a.M, a.E));
  hipLaunchKernelGGL((grouped_few_kernel<FP8, kBatch>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <bool FP8>
hipError_t launch_few(const Args& a, hipStream_t st) {
  // a wave's chunks in as few batches as registers allow, the last one full (what
  // it lacks is loaded all the same: Qwen3 w2 of one token, 3 chunks a wave, takes
  // 13.8 us in a batch of 8 and 7.5 in one of 3)
  const int per = ((a.row_bytes + kChunk - 1) / kChunk + kWaves - 1) / kWaves;
  if (per <= 2) return launch_few<FP8, 2>(a, st);
  if (per == 3 || per == 5 || per == 6) return launch_few<FP8, 3>(a, st);
  if constexpr (!FP8)
    if (per > 4) return launch_few<FP8, 8>(a, st);
  return launch_few<FP8, 4>(a, st);
}

template <bool FP8, int G, Out OUT>
hipError_t launch_tile(const Args& a, hipStream_t st) {
  using Sh = Shape<4, G>;
  static_assert(Sh::kLds <= 64 * 1024, "LDS beyond the default limit");
  constexpr int kBlocks = G == 4 ? 2 : G == 2 ? 3 : 4;  // a CU, as registers allow
  hipLaunchKernelGGL((grouped_tile_kernel<FP8, 4, G, OUT>), dim3(256 * kBlocks), dim3(256),
                     Sh::kLds, st, a);
  return hipGetLastError();
}

// Tiles of t rows of an expert, on average over experts of per rows give or take
// their square root: one, and one more for every k * t rows that it has.
float tiles_of(float per, int t) {
  const float h = 1.73f * sqrtf(per);  // (as if evenly spread, of that deviation)
  const int sure = std::max((int)((per - h) / t), 0);
  float n = 1.f + sure;
  for (int k = sure + 1; (float)k * t < per + h; ++k)
    n += std::min((per + h - (float)k * t) / (2 * h), 1.f);
  return n;
}

// The weight rows of the small tiles.
int tile_rows(const Args& a) {
  // The largest panels that give the GPU's blocks a tile each; where experts have
  // several tiles of rows, and the products count too, panels of 128 from fewer on
  // (fp8, 8 experts of 75 rows, 4096 x 14336: 170 us in panels of 64, 151 in 128;
  // 16 of 64 rows, 1536 x 2048: 22.3 and 23.4).
  const int64_t used = std::min(a.M, a.E), works = used * ((a.N + 127) / 128);
  const int64_t rows = (int64_t)(tiles_of((float)a.M / a.E, 64) + 0.6f);
  if (used * ((a.N + 255) / 256) >= 768) return WISP_GROUPED_TILE_256;
  if (works >= 768 || (rows > 1 && works * rows >= 400)) return WISP_GROUPED_TILE_128;
  return WISP_GROUPED_TILE_64;
}

template <bool FP8, Out OUT>
hipError_t launch_tile(int kernel, const Args& a, hipStream_t st) {
  if (kernel == WISP_GROUPED_TILE_256) return launch_tile<FP8, 4, OUT>(a, st);
  if (kernel == WISP_GROUPED_TILE_128) return launch_tile<FP8, 2, OUT>(a, st);
  return launch_tile<FP8, 1, OUT>(a, st);
}

int refuse(int rc, const char* why, const char* where) {
  wisp_set_last_error(why, where);
  return rc;
}

template <int L>
hipError_t launch_big(const Args& a, hipStream_t st) {
  return a.row_bytes % (2 * kChunk) ? launch_big<L, true>(a, st) : launch_big<L, false>(a, st);
}

// The kernel of a call: WISP_GROUPED_*, with WISP_GROUPED_NARROW where single values
// are stored, which the small tiles do.
template <bool FP8>
int choose(const Args& a) {
  // The kernel for the fewest rows (a) against the small tiles (b), in us:
  //                     rows  bf16 a    b   fp8 a    b
  //   128 x 1536 x 2048,  32   37.2  37.4   21.0  21.5
  //                       64   60.9  68.0   36.2  38.5
  //                      128  101.7 100.8   60.2  55.3
  //   128 x 2048 x 768,   96   44.2  52.8   32.7  28.0
  //   8 x 28672 x 4096,   32    304   328    178   174
  //   8 x 4096 x 14336,   64    175   158    111    91
  // and where the tiles cannot fill the GPU, while a group is one pass:
  //   24 x 704 x 1056,   120   10.6  14.0    6.7  12.0
  //                      231   12.1  13.8    7.5  12.0
  //                      360   15.6  13.8    9.9  12.1
  //   16 x 1536 x 2048,  160   24.4  25.0   14.7  16.5
  //   16 x 2048 x 768,    80   12.8  12.4    9.7   9.8
  // (at most 256 rows: all of them may be one expert's, a pass per 16)
  const int most = FP8 ? std::max(16, std::min(32, 2 * a.E)) : std::max(32, std::min(96, 4 * a.E));
  const int64_t works = std::min(a.M, a.E) * (int64_t)((a.N + 63) / 64);
  if (a.M <= most || (a.M <= 64 && works <= 512) ||
      (a.M <= 256 && works < 512 && tiles_of((float)a.M / a.E, kFewCols) == 1.f))
    return WISP_GROUPED_FEW;
  // (pieces of 8 and 16 bytes go to whole dwords: a bfloat16 output that starts between
  // two of them, at an odd element of its buffer, takes single values too)
  if (a.N % (a.out_f32 ? 4 : 8) || (uintptr_t)a.out % 4) return tile_rows(a) | WISP_GROUPED_NARROW;
  // What a chunk of columns takes in each kernel, in 1/100 us, from the works that a
  // CU gets: w on average, as whole turns in the large tiles.  (Works of the small
  // ones: 128 weight rows.  Measured over 4 to 128 experts, 8 sizes of weights, 32
  // to 2000 rows each; the choice is the faster one or within some 5 %, 15 at most.)
  //                        bf16, us: small  128 rows  192 rows   fp8: small  large
  //   128 x 1536 x 2048,  32 rows      146    147       152             81     97
  //                       64           194    161       163            107    102
  //                      128           284    203       189            158    112
  //                      200           401    241       282            222    124
  //   8 x 4096 x 14336,   40           180    207       235            110    168
  //                      100           273    231       241            158    169
  //                      300           719    417       322            390    223
  //   24 x 704 x 1056,    64          13.7   19.5      26.0           12.5   21.3
  //                      375          31.9   24.3      29.5           25.4   24.8
  // None is faster than the weights' stream; where all are that fast, tiles of more
  // rows read x fewer times (bf16, the first layer at 48 rows: 172 us small, 155).
  const float per = (float)a.M / a.E, w1 = a.E * (float)((a.N + 127) / 128) / 256;
  const float panels = (float)(a.E * (int64_t)((a.N + kPanel - 1) / kPanel));
  const float stream = 76 * w1, w = w1 * floorf(tiles_of(per, 64) + 0.6f);
  auto large = [&](int rows, float turn, float work) {
    const float w = panels * tiles_of(per, rows) / 256;
    const float start = 150.f * kChunk / a.row_bytes;  // 1.5 us more than a small one's
    return std::max(turn * ceilf(w) + work * w + start, stream);
  };
  if constexpr (FP8) {
    if (large(256, 140, 80) < std::max(50 + 52 * w, stream)) return WISP_GROUPED_LARGE_256;
  } else {
    const float small = std::max(30 + 44 * w, stream);
    const float two = large(128, 80, 34), three = large(192, 100, 40);
    if (std::min(two, three) < small || (std::min(two, three) == stream && per > 40))
      return two <= three ? WISP_GROUPED_LARGE_128 : WISP_GROUPED_LARGE_192;
  }
  return tile_rows(a);
}

template <bool FP8>
hipError_t launch(const Args& a, hipStream_t st) {
  const int kernel = choose<FP8>(a);
  switch (kernel) {
    case WISP_GROUPED_FEW:
      return launch_few<FP8>(a, st);
    case WISP_GROUPED_LARGE_128:
      if constexpr (!FP8) return launch_big<2>(a, st);
      break;
    case WISP_GROUPED_LARGE_192:
      if constexpr (!FP8) return launch_big<3>(a, st);
      break;
    case WISP_GROUPED_LARGE_256:
      if constexpr (FP8)
        return a.row_bytes % (2 * kChunk) ? launch_big_fp8<true>(a, st)
                                          : launch_big_fp8<false>(a, st);
      break;
  }
  const int tile = kernel & ~WISP_GROUPED_NARROW;
  if (kernel != tile) return launch_tile<FP8, kNarrow>(tile, a, st);
  if constexpr (!FP8)
    if (a.out_f32) return launch_tile<false, kF32>(tile, a, st);
  return launch_tile<FP8, kBf16>(tile, a, st);
}

template <bool FP8>
int grouped(const Args& a, hipStream_t st) {
  WISP_HIP_TRY(launch<FP8>(a, st));
  return WISP_OK;
}

// Elements between experts: 512 times as many fit 64 bits as bytes of any type.
constexpr int64_t kMostApart = (int64_t)1 << 50;

// What both entry points check; elem: bytes of a column.
const char* unsupported(int64_t x_ld, int64_t w_ld, int64_t w_stride, int64_t N, int64_t K,
                        int elem, const void* x, const void* w) {
  // (first, so that no stride's bytes pass 64 bits below, nor a place in the weights)
  if (x_ld >= (int64_t)1 << 22) return "rows of x 4 MiB apart";
  if (w_ld >= (int64_t)1 << 24) return "rows of w 16 MiB apart";
  if (w_stride >= kMostApart) return "experts 2^50 elements apart";
  if (K % (16 / elem)) return "a row of x and of w must be whole 16-byte pieces";
  if (x_ld * elem % 16 || w_ld * elem % 16 || w_stride * elem % 16 || (uintptr_t)x % 16 ||
      (uintptr_t)w % 16)
    return "x, w and their strides must be 16-byte aligned";
  // (32-bit offsets inside a tile of x, inside an expert's weights and in a tile's outputs)
  if (w_ld * elem >= (int64_t)1 << 24 || N * w_ld * elem >= (int64_t)1 << 31)
    return "rows of w 16 MiB apart, or an expert's weights of 2 GiB";
  if (x_ld * elem >= (int64_t)1 << 22) return "rows of x 4 MiB apart";
  if (N >= 1 << 21) return "2^21 outputs of a row";
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
  if (ws_stride >= kMostApart)
    return refuse(WISP_ERR_UNSUPPORTED, "block scales 2^50 elements apart", where);
  if (s_ld >= (int64_t)1 << 20)
    return refuse(WISP_ERR_UNSUPPORTED, "scales of x 4 MiB apart", where);
  const Args a = {q, s, w, ws, ends, out, q_ld, w_stride, w_ld, ws_stride, s_ld, E, M, N, K,
                  groups, false, zero_tail != 0};
  return grouped<true>(a, (hipStream_t)stream);
}

extern "C" int wisp_grouped_mm_kernel(int fp8, int E, int M, int N, int K, const void* out,
                                      int out_dtype) {
  using namespace wisp;
  const int elem = fp8 ? 1 : 2;
  if (E < 1 || E > kMaxExperts || M < 1 || N < 1 || K < 1 ||
      (out_dtype != WISP_BF16 && (fp8 || out_dtype != WISP_F32)) ||
      unsupported(K, K, 0, N, K, elem, nullptr, nullptr))
    return -1;
  Args a{};
  a.out = const_cast<void*>(out);
  a.E = E, a.M = M, a.N = N, a.row_bytes = K * elem;
  a.out_f32 = out_dtype == WISP_F32;
  return fp8 ? choose<true>(a) : choose<false>(a);
}

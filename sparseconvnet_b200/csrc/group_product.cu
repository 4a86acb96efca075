// Products of ragged groups of rows, each with its group's own weights, on tcgen05 tensor cores.
//
//     forward        y[r]  = x[r] W[g] (+ b[g])       for offsets[g] <= r < offsets[g + 1]
//     input          dx[r] = dy[r] W[g]^T
//     weights        dW[g] = sum over the rows of g of x[r]^T dy[r]
//     8 bits         y[r]  = s[r] S[g] (q[r] Q[g]) + b[g]        (e4m3 values, a scale per row and per group and output plane)
//
// The groups' sizes are known on the device only: every block sums the tiles of the groups before it looks for its own
// (one scan at the start of the kernel), and takes every gridDim.x-th tile.  k_group_product does all four; what differs is
// which planes of an operand lie next to each other in memory (K-major: those that are summed over, M- / N-major: the
// others) and, for the weights' gradient, that a tile's sum runs over rows and has to end inside a stage: there the rows
// of the next group are overwritten with zeros before the tensor core sees them (0 times what stands there could be NaN).
// k_group_pair takes wide layers and large groups, k_group_split fp32 rows of few planes.
//
//   arithmetic  16-bit and 8-bit values as they are, fp32 sums.  fp32 values as bf16 parts (k_group_parts): x = h + m + l
//               holds all 24 bits of values from 2^-110 on (below that l ends at bf16's smallest number, 2^-133), and the
//               products h h, h m, m h, h l, l h, m m leave out 2^-24 of a product; two parts and h h, h m, m h leave out 2^-17.  The tensor core cuts its running sum off at every instruction, half a unit
//               of 2^-24 of it on average, so for fp32 results of fp32 and 16-bit values a sum is handed over to the registers
//               of the epilogue warps every kDrain steps, and the products with an m or l have an accumulator of their own
//               (they are 2^-8 as large).  Results of fewer bits, and all results of 8-bit values, take a sum of up to kLong
//               steps as it comes: 512 instructions cut off 5e-5 of it where all products have one sign (measured, 2^-23.4 an
//               instruction), a fifth of fp16's half step.  A longer one, a group of more rows or more planes, is handed over
//               every kLongDrain steps and loses half of that however long it is (200003 rows lost 1e-3 in one piece).
//   tile        128 x TN, TN = 256 for 16- and 8-bit values, 128 where parts or fp32 results take the second half of the
//               tensor memory, 64 where wider tiles would leave SMs without work.  Two accumulators: one is read while the
//               next tile is summed.
//   roles       one warp copies tiles in (TMA, 128-byte swizzle, a ring over all of shared memory), one issues the
//               instructions, eight read the accumulators, scale, add the bias, round and store.
//   measured    32749 rows of 32 groups, 2048 -> 2048 bf16: forward and input gradient 202 us each (1360 TFLOP/s, the tensor
//               cores busy 90% of the time at the 1.53 GHz that the power limit leaves), weights' gradient 262 (59%: a group's
//               256 x 256 results cost as much to write as 500 rows to sum); 65536 rows, 4096 -> 2048 in 8 bits 378 us
//               alone (2.9 PFLOP/s, 93%), 450 to 480 in a row; 37 rows of 8 groups, 1024 -> 1024: 8 us, two trips to L2
//               behind 2 us of set-up; 131071 fp32 rows, 64 -> 96: 31, 35 and 50 us, bound by the splitting warps' latency.
//   small groups  rows behind a group's last are not copied (boxes of 32 rows): their accumulator rows hold anything and are
//               not stored.
//
// Every wait is bounded; what gave up is reported by the next call on the device, or by scn_rows_poll_errors.
#include <cuda.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "rows.cuh"
#include "tc_ptx.cuh"

namespace scn {
namespace {

constexpr int kEpilogueWarps = 8, kThreads = (2 + kEpilogueWarps) * 32;
constexpr int kTileM = 128, kRow = 128;      // bytes of an operand row in a stage
constexpr int kStageRows = 64;               // rows (weights' gradient) or 16-bit values of K in a stage
constexpr int kBoxRows = 32;                 // rows of a copy of the left operand
constexpr int kRing = 196608;                // shared memory of the ring
constexpr int kMostGroups = 1024;
constexpr int kDrain = 4;                    // steps (of four instructions a product) between two hand-overs
constexpr int kLong = 128, kLongDrain = 64;  // long sums of 16- and 8-bit values: from how many steps on, and between two hand-overs
constexpr int kMostStages = 8;

struct GroupParams {
  const void *offsets;
  int off64, groups;
  int n_rows;
  int k, n, m;             // rows: sum over k planes, n results; weights: m x n results, sum over rows
  int n_tiles, m_tiles;    // m_tiles: weights only
  int chunk;               // weights: rows of a unit
  int pick;                // weights: groups that a launch takes, 0: all, 1: those of up to kLong steps, 2: the others
  int tile;                // rows of a unit (rows) or of a tile of the result (weights)
  unsigned idesc;          // without N
  int drain;               // steps between two hand-overs, a power of two
  void *out;
  int out_type, aligned, part_aligned;  // what the results' and the partial sums' rows are aligned to
  int m_rows;              // weights: rows of the result with that of the bias sums, if a tile has room for it
  void *d_bias;
  const float *a, *b;      // fp32 operands that the kernel splits itself
  long long a_stride, b_stride;
  int a_quads, b_quads;    // their rows take 16-byte loads
  float *partial;          // weights: [unit of a group of several units][m_rows][n]
  const void *bias;
  int bias_type;
  const float *row_scale, *col_scale;
  int drop;                // test: leave out the first arrival
  int *flag;               // pinned host memory: set by a kernel that gave up
};

struct Shared {
  unsigned long long full[kMostStages], empty[kMostStages], ready[2], taken[2];
  unsigned long long tail[kMostStages], zeroed[kMostStages];  // pairs
  unsigned tmem;
  int abort, issued;
  unsigned tails, tail_last;  // stages that have been a sum's end, and the parity of the last time
  int warp_sums[32];
  __align__(16) float columns[kEpilogueWarps][128];
  int first[kMostGroups + 3];  // units (of rows) before the group
  int begin[kMostGroups + 2], end[kMostGroups + 2];
  int part[kMostGroups];       // weights: units before the group among the groups of several units, -1: one unit
};

// What a unit of work is
struct Unit {
  int group, row, rows, n0, m0;  // row: first row; rows: of the tile (rows) or of the sum (weights)
  int part;                      // weights: the partial sum that this unit makes, -1: the gradient itself
};

__device__ __forceinline__ void gave_up(const GroupParams &P) {
  *(volatile int *)P.flag = 1;
  __threadfence_system();
}

__device__ __forceinline__ int offset_at(const GroupParams &P, int g) {
  const long long v = P.off64 ? __ldg((const long long *)P.offsets + g) : (long long)__ldg((const int *)P.offsets + g);
  return (int)min(max(v, 0ll), (long long)P.n_rows);
}

__device__ __forceinline__ int units_of(const GroupParams &P, bool weights, int rows) {
  if (weights && P.pick && (rows > kLong * kStageRows) != (P.pick == 2)) return 0;
  const unsigned each = weights ? P.chunk : P.tile;  // (rows + each may pass 2^31)
  const int units = (int)(((unsigned)rows + each - 1) / each);
  return weights ? max(1, units) : units;
}

// Sum (or maximum) of v >= 0 over the threads before this one
template <bool MAX>
__device__ __forceinline__ int over_before(int v, int *warp_sums) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int upto = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto = MAX ? max(upto, o) : upto + o;
  }
  if (lane == 31) warp_sums[warp] = upto;
  int before = __shfl_up_sync(0xffffffffu, upto, 1);
  if (lane == 0) before = 0;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before = MAX ? max(before, warp_sums[w]) : before + warp_sums[w];
  __syncthreads();
  return before;
}

// Where the groups begin and end, and the units before each.  A group begins at the largest offset up to its own, so that
// groups never overlap and their units fit what was made for them, whatever the offsets are.  Rows: groups G and G + 1 are
// the rows behind and in front of all groups, whose results are zeros.
template <bool WEIGHTS>
__device__ __forceinline__ void scan_groups(const GroupParams &P, Shared &S) {
  const int G = P.groups, tid = threadIdx.x;
  if (G + 2 <= 32) {  // one warp, without a barrier until the end: a call on 37 rows 8.4 -> 7.4 us
    if (tid < 32) {
      const int all = WEIGHTS ? G : G + 2;
      int begin = tid <= G ? offset_at(P, tid) : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, begin, d);
        if (tid >= d) begin = max(begin, o);
      }
      const int next = __shfl_down_sync(0xffffffffu, begin, 1), head = __shfl_sync(0xffffffffu, begin, 0);
      const int end = tid < G ? next : tid == G ? P.n_rows : head;
      if (tid > G) begin = 0;
      const int units = tid < all ? units_of(P, WEIGHTS, end - begin) : 0, parts = units > 1 ? units : 0;
      int upto = units, parts_upto = parts;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, d), q = __shfl_up_sync(0xffffffffu, parts_upto, d);
        if (tid >= d) upto += o, parts_upto += q;
      }
      if (tid < all) {
        S.begin[tid] = begin, S.end[tid] = end, S.first[tid] = upto - units;
        if (tid == all - 1) S.first[all] = upto;
        if (WEIGHTS) S.part[tid] = units > 1 ? parts_upto - parts : -1;
      }
    }
    __syncthreads();
    return;
  }
  const int each = (G + 2 + (int)blockDim.x - 1) / (int)blockDim.x;
  const int from = tid * each, to = min(from + each, G + 1);
  int most = 0;
  for (int g = from; g < to; ++g) most = max(most, S.begin[g] = offset_at(P, g));
  most = over_before<true>(most, S.warp_sums);
  for (int g = from; g < to; ++g) S.begin[g] = most = max(most, S.begin[g]);
  __syncthreads();
  const int all = WEIGHTS ? G : G + 2, last = min(from + each, all);
  int sum = 0, parts = 0;
  for (int g = from; g < last; ++g) {
    const int end = g < G ? S.begin[g + 1] : g == G ? P.n_rows : S.begin[0], begin = g <= G ? S.begin[g] : 0;
    S.end[g] = end;
    const int units = units_of(P, WEIGHTS, end - begin);
    sum += units;
    if (units > 1) parts += units;
  }
  int before = over_before<false>(sum, S.warp_sums), parts_before = WEIGHTS ? over_before<false>(parts, S.warp_sums) : 0;
  for (int g = from; g < last; ++g) {
    if (g > G) S.begin[g] = 0;
    const int units = units_of(P, WEIGHTS, S.end[g] - S.begin[g]);
    S.first[g] = before;
    before += units;
    if (WEIGHTS) {
      S.part[g] = units > 1 ? parts_before : -1;
      if (units > 1) parts_before += units;
    }
    if (g == all - 1) S.first[all] = before;
  }
  __syncthreads();
}

// Units in rising order: a role walks its block's units, so the next unit's group is looked for from the present one on (a step
// or two, else by halves).  Between two units every role has this to do before it can go on: with a search over all groups
// and a 64-bit division it took some 800 cycles.
template <bool WEIGHTS, int TN>
struct Walk {
  const GroupParams &P;
  const Shared &S;
  int group = 0;
  __device__ __forceinline__ Walk(const GroupParams &p, const Shared &s) : P(p), S(s) {}
  __device__ __forceinline__ Unit at(long long u) {
    const int all = WEIGHTS ? P.groups : P.groups + 2;
    const int tiles = WEIGHTS ? P.n_tiles * P.m_tiles : P.n_tiles;
    const int r = tiles == 1 ? (int)u : u >> 32 ? (int)(u / tiles) : (int)((unsigned)u / (unsigned)tiles), t = (int)(u - (long long)r * tiles);
    for (int i = 0; i < 3 && S.first[group + 1] <= r; ++i) ++group;  // (first[all] is above every r)
    if (S.first[group + 1] <= r) {
      int lo = group + 1, hi = all - 1;  // the last group that begins at or before r: one without a unit shares its start with the next
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (S.first[mid] <= r)
          lo = mid;
        else
          hi = mid - 1;
      }
      group = lo;
    }
    const int each = WEIGHTS ? P.chunk : P.tile, row = S.begin[group] + (r - S.first[group]) * each;
    const int m = !WEIGHTS || t == 0 ? 0 : (int)((unsigned)t / (unsigned)P.n_tiles);
    return {group, row, min(each, S.end[group] - row), (t - m * P.n_tiles) * TN, m * P.tile,
            WEIGHTS && S.part[group] >= 0 ? S.part[group] + r - S.first[group] : -1};
  }
};

__device__ __forceinline__ void load_tile(unsigned dst, const CUtensorMap *map, int x, int y, int z, int w, unsigned long long *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// a tensor map on its way into the cache that copies read it from
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

template <bool F8>
__device__ __forceinline__ void mma_if(unsigned lead, unsigned d, unsigned a_lo, unsigned a_hi, unsigned b_lo, unsigned b_hi, unsigned idesc,
                                       unsigned accumulate) {
  if (!F8) {
    mma_bf16_if(lead, d, a_lo, a_hi, b_lo, b_hi, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.u32 e, %7, 0;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
  }
}

// 128-byte swizzle; `next`: bytes to the operand's next 64 values along M or N (M- / N-major), not looked at otherwise
__device__ __forceinline__ unsigned desc_lo(unsigned addr, unsigned next) { return ((addr >> 4) & 0x3FFF) | ((next >> 4) << 16); }
constexpr unsigned kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);

// The products of parts, largest first
template <int P>
struct Products {
  static constexpr int N = P == 1 ? 1 : P == 2 ? 3 : 6;
};
__host__ __device__ constexpr int part_a(int i) { return i == 2 || i == 5 ? 1 : i == 4 ? 2 : 0; }  // hh hm mh hl lh mm
__host__ __device__ constexpr int part_b(int i) { return i == 1 || i == 5 ? 1 : i == 3 ? 2 : 0; }

__device__ __forceinline__ float value_at(const void *p, int type, long long i) {
  return type == SCN_TYPE_FLOAT32 ? __ldg((const float *)p + i)
         : type == SCN_TYPE_BFLOAT16 ? __bfloat162float(__ldg((const __nv_bfloat16 *)p + i))
                                     : __half2float(__ldg((const __half *)p + i));
}

// 32 results of a row, `left` of them in the row, in rows that begin at multiples of `aligned` bytes: 8, 16 or 32.  32: whole
// sectors (pieces of 16 bytes reach L2 as two writes of half a sector: group_wide_8bit took 70 us more).  Inlined only (rows.cuh).
template <int WORDS>
__device__ __forceinline__ void store_words32(void *to, int aligned, int left, const unsigned (&w)[WORDS]) {
  constexpr int kPer = 32 / WORDS;  // values of a word
  unsigned *q = (unsigned *)to;
  if (left >= 32 && aligned == 32) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(q + i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]),
                   "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                   : "memory");
  } else if (aligned >= 16) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4)
      if (i * kPer < left) *reinterpret_cast<uint4 *>(q + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 2)
      if (i * kPer < left) *reinterpret_cast<uint2 *>(q + i) = make_uint2(w[i], w[i + 1]);
  }
}
// The same for rows that begin anywhere: through 512 bytes of shared memory, so that a warp writes a row's values side by side (a
// lane that writes its row value by value touches 32 lines with every store: 60000 x 257 -> 333 bf16 took 316 us, now 82).  `to`: the
// lane's row, null if it is not stored.
template <int WORDS>
__device__ __forceinline__ void store_words32_anywhere(void *to, int left, const unsigned (&w)[WORDS], unsigned *shared) {
  constexpr int kRows = 128 / WORDS;  // rows at a time
  const int lane = threadIdx.x % 32;
#pragma unroll 1
  for (int q = 0; q < 32; q += kRows) {
    if (lane >= q && lane < q + kRows) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4 *>(shared + (lane - q) * WORDS + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      void *row = (void *)__shfl_sync(0xffffffffu, (unsigned long long)to, q + r);
      if (row && lane < left) {
        if (WORDS == 32)
          ((unsigned *)row)[lane] = shared[r * WORDS + lane];
        else
          ((unsigned short *)row)[lane] = ((const unsigned short *)shared)[r * 32 + lane];
      }
    }
    __syncwarp();
  }
}
// The whole warp comes here.
__device__ __forceinline__ void store32(void *to, int type, int aligned, int left, const float (&v)[32], float *shared) {
  if (type == SCN_TYPE_FLOAT32) {
    unsigned w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
    if (aligned < 8)
      store_words32_anywhere(to, left, w, (unsigned *)shared);
    else if (to)
      store_words32(to, aligned, left, w);
  } else {
    unsigned w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      w[i] = type == SCN_TYPE_BFLOAT16 ? pair(v[2 * i], v[2 * i + 1], __nv_bfloat16()) : pair(v[2 * i], v[2 * i + 1], __half());
    if (aligned < 8)
      store_words32_anywhere(to, left, w, (unsigned *)shared);
    else if (to)
      store_words32(to, aligned, left, w);
  }
}

// Values of `bytes` in rows of n from p on: what every row's results are aligned to (a run of 32 begins at a multiple of 32)
__host__ __device__ inline int aligned_to(uintptr_t p, long long n, int bytes) {
  const uintptr_t all = p | (uintptr_t)(n * bytes);
  return all % 32 == 0 ? 32 : all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : bytes;
}

// What belongs to a unit's columns and rows, read by a warp of the epilogue while the unit is still being summed: lane l has
// columns l, l + 32 ..
template <int COLS, bool WEIGHTS, bool F8>
struct Terms {
  float bias[COLS / 32], scale[F8 ? COLS / 32 : 1], row_scale;
  bool with_bias, real;
  __device__ __forceinline__ void read(const GroupParams &P, const Unit &u, int c0, int lane_row, int lane) {
    real = !WEIGHTS && u.group < P.groups;
    with_bias = real && P.bias;
    row_scale = F8 && real && lane_row < u.rows ? __ldg(P.row_scale + u.row + lane_row) : 0.f;
#pragma unroll
    for (int j = 0; j < COLS / 32; ++j) {
      const int c = c0 + 32 * j + lane;
      const bool in = real && c < P.n;
      bias[j] = with_bias && in ? value_at(P.bias, P.bias_type, (long long)u.group * P.n + c) : 0.f;
      if (F8) scale[F8 ? j : 0] = in ? __ldg(P.col_scale + (long long)u.group * P.n + c) : 0.f;
    }
  }
};

// 32 results of the row `lane_row` of a unit, from column c = c0 + 32 j on; the whole warp comes here.  `shared`: 128 floats of the
// warp, through which every lane sees all columns' terms.
template <int COLS, bool WEIGHTS, bool F8>
__device__ __forceinline__ void finish32(const GroupParams &P, const Unit &u, const Terms<COLS, WEIGHTS, F8> &terms, int j, int lane_row, int c,
                                         float *shared, float (&v)[32]) {
  const int lane = threadIdx.x % 32;
  if (F8 && terms.real) {
    shared[lane] = terms.scale[F8 ? j : 0];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 s = reinterpret_cast<const float4 *>(shared)[i];
      v[4 * i] *= s.x * terms.row_scale, v[4 * i + 1] *= s.y * terms.row_scale, v[4 * i + 2] *= s.z * terms.row_scale, v[4 * i + 3] *= s.w * terms.row_scale;
    }
    __syncwarp();
  }
  if (!WEIGHTS && terms.with_bias) {
    shared[lane] = terms.bias[j];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = reinterpret_cast<const float4 *>(shared)[i];
      v[4 * i] += b.x, v[4 * i + 1] += b.y, v[4 * i + 2] += b.z, v[4 * i + 3] += b.w;
    }
    __syncwarp();
  }
  auto at = [&](void *p, int type, long long row) { return (void *)((char *)p + (row * P.n + c) * (type == SCN_TYPE_FLOAT32 ? 4 : 2)); };
  if (WEIGHTS) {
    const int m = u.m0 + lane_row;
    const bool part = u.part >= 0;
    const int type = part ? (int)SCN_TYPE_FLOAT32 : P.out_type;
    void *to = nullptr;
    if (m < P.m_rows) to = part ? at(P.partial, type, (long long)u.part * P.m_rows + m) : m < P.m ? at(P.out, type, (long long)u.group * P.m + m) : at(P.d_bias, type, u.group);
    store32(to, type, part ? P.part_aligned : P.aligned, P.n - c, v, shared);
  } else {
    store32(lane_row < u.rows ? at(P.out, P.out_type, u.row + lane_row) : nullptr, P.out_type, P.aligned, P.n - c, v, shared);
  }
}

template <int PARTS, int TN, bool SUMS, bool WEIGHTS, bool B_ROWS, bool F8>
__global__ void __launch_bounds__(kThreads, 1)
k_group_product(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GroupParams P) {
  SCN_GRID_WAIT();
  constexpr int kABytes = kTileM * kRow, kBBytes = TN * kRow, kStage = PARTS * (kABytes + kBBytes), kStages = kRing / kStage;
  static_assert(kStages <= kMostStages && kStages >= 2, "ring");
  constexpr int kAccs = PARTS > 1 ? 2 : 1, kColumns = 256;  // tensor memory: two times 256 columns
  static_assert(kAccs * TN <= kColumns, "accumulators");
  extern __shared__ unsigned char raw[];
  unsigned char *ring = raw + (1024 - smem_u32(raw) % 1024) % 1024;
  __shared__ Shared S;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  volatile int *abort = &S.abort;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&S.full[i], 1), mbar_init(&S.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&S.ready[i], 1), mbar_init(&S.taken[i], kEpilogueWarps);
    S.abort = 0;
    S.issued = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2 && lane == 0) prefetch_map(&map_a), prefetch_map(&map_b);
  if (warp == 1) tmem_alloc(&S.tmem, 512);
  scan_groups<WEIGHTS>(P, S);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = S.tmem;
  const int all = WEIGHTS ? P.groups : P.groups + 2;
  const long long units = (long long)S.first[all] * P.n_tiles * (WEIGHTS ? P.m_tiles : 1);
  constexpr int kPerStage = F8 ? 2 * kStageRows : kStageRows;  // values of K in a stage
  auto steps_of = [&](const Unit &u) { return WEIGHTS ? (u.rows + kStageRows - 1) / kStageRows : u.group < P.groups ? (P.k + kPerStage - 1) / kPerStage : 0; };

  // ==== copies ====
  if (warp == 0) {
    const bool lead = elect_one();
    int step = 0;
    bool ok = true;
    Walk<WEIGHTS, TN> walk(P, S);
    for (long long i = blockIdx.x; i < units && ok; i += gridDim.x) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u);
      const int a_boxes = WEIGHTS ? 2 : (u.rows + kBoxRows - 1) / kBoxRows;
      const unsigned bytes = PARTS * ((WEIGHTS ? kABytes : a_boxes * kBoxRows * kRow) + kBBytes);
      for (int k = 0; k < steps; ++k, ++step) {
        const int st = step % kStages;
        if (step >= kStages && !mbar_wait_warp(&S.empty[st], (step / kStages - 1) & 1, abort)) {
          ok = false;
          break;
        }
        if (lead) {
          const unsigned a = smem_u32(ring) + st * kStage, b = a + PARTS * kABytes;
          mbar_expect_tx(&S.full[st], bytes);
          for (int p = 0; p < PARTS; ++p) {
            if (WEIGHTS) {
              for (int j = 0; j < 2; ++j) load_tile(a + p * kABytes + j * kStageRows * kRow, &map_a, u.m0 + 64 * j, u.row + k * kStageRows, p, 0, &S.full[st]);
              for (int j = 0; j < TN / 64; ++j) load_tile(b + p * kBBytes + j * kStageRows * kRow, &map_b, u.n0 + 64 * j, u.row + k * kStageRows, p, 0, &S.full[st]);
            } else {
              for (int j = 0; j < a_boxes; ++j) load_tile(a + p * kABytes + j * kBoxRows * kRow, &map_a, k * kPerStage, u.row + j * kBoxRows, p, 0, &S.full[st]);
              if (B_ROWS)  // weights [k][n]: 64 values of n to a row
                for (int j = 0; j < TN / 64; ++j) load_tile(b + p * kBBytes + j * kStageRows * kRow, &map_b, u.n0 + 64 * j, k * kStageRows, u.group, p, &S.full[st]);
              else
                load_tile(b + p * kBBytes, &map_b, k * kPerStage, u.n0, u.group, p, &S.full[st]);
            }
          }
          S.issued = step + 1;
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== instructions ====
  else if (warp == 1) {
    const unsigned lead = elect_one();
    int step = 0, turn = 0;
    bool ok = true;
    Walk<WEIGHTS, TN> walk(P, S);
    for (long long i = blockIdx.x; i < units && ok; i += gridDim.x) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u);
      const unsigned idesc = P.idesc | (unsigned)(min(TN, (P.n - u.n0 + 15) / 16 * 16) >> 3) << 17;
      for (int k = 0; k < steps; ++k, ++step) {
        const bool begins = k == 0 || (SUMS && !(k & (P.drain - 1))), ends = k == steps - 1 || (SUMS && !((k + 1) & (P.drain - 1)));
        if (begins && turn >= 2 && !mbar_wait_warp(&S.taken[turn & 1], ((turn >> 1) - 1) & 1, abort)) {
          ok = false;
          break;
        }
        const int st = step % kStages;
        if (!mbar_wait_warp(&S.full[st], (step / kStages) & 1, abort)) {
          ok = false;
          break;
        }
        const unsigned a = smem_u32(ring) + st * kStage, b = a + PARTS * kABytes;
        int instructions = 4;
        if (WEIGHTS) {
          const int left = u.rows - k * kStageRows;
          if (left < kStageRows) {  // the rows behind the sum's last, up to a whole instruction: zeros
            instructions = (left + 15) / 16;
            const int gap = (instructions * 16 - left) * 8;  // 16-byte pieces of one 64 x 64 block
            constexpr int kBlocks = PARTS * (2 + TN / 64);
            for (int q = lane; q < gap * kBlocks; q += 32)
              *reinterpret_cast<uint4 *>(ring + st * kStage + q / gap * (kStageRows * kRow) + left * kRow + q % gap * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        tc_fence_after();
        const unsigned d = tmem + (turn & 1) * kColumns;
        for (int j = 0; j < instructions; ++j) {
#pragma unroll
          for (int q = 0; q < Products<PARTS>::N; ++q) {
            const unsigned pa = a + part_a(q) * kABytes + j * (WEIGHTS ? 16 * kRow : 32), pb = b + part_b(q) * kBBytes + j * (WEIGHTS || B_ROWS ? 16 * kRow : 32);
            const unsigned fresh = begins && j == 0 && (q == 0 || q == 1);
            mma_if<F8>(lead, d + (q ? TN : 0), desc_lo(pa, WEIGHTS ? kStageRows * kRow : 16), kDescHi, desc_lo(pb, WEIGHTS || B_ROWS ? kStageRows * kRow : 16),
                       kDescHi, idesc, !fresh);
          }
        }
        if (!(P.drop && blockIdx.x == 0 && step == 0)) tc_commit_if(lead, &S.empty[st]);
        if (ends) {
          tc_commit_if(lead, &S.ready[turn & 1]);
          ++turn;
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== results ====
  else {
    const int quarter = warp % 4, half = (warp - 2) / 4;  // (a warp reaches the tensor memory's lanes 32 (warp % 4) on)
    constexpr int kMine = TN / 2;
    const int lane_row = quarter * 32 + lane;
    int turn = 0;
    bool ok = true;
    Walk<WEIGHTS, TN> walk(P, S);
    for (long long i = blockIdx.x; i < units && ok; i += gridDim.x) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u), columns = min(P.n - u.n0 - half * kMine, kMine);
      const int turns = steps == 0 ? 0 : SUMS ? (steps - 1) / P.drain + 1 : 1;
      Terms<kMine, WEIGHTS, F8> terms;
      terms.read(P, u, u.n0 + half * kMine, lane_row, lane);
      float sum[SUMS ? kMine : 1];
#pragma unroll
      for (int c = 0; c < (SUMS ? kMine : 1); ++c) sum[c] = 0.f;
      for (int t = 0; t < turns; ++t, ++turn) {
        if (!mbar_wait_warp(&S.ready[turn & 1], (turn >> 1) & 1, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const unsigned from = tmem + ((unsigned)(quarter * 32) << 16) + (turn & 1) * kColumns + half * kMine;
#pragma unroll
        for (int c = 0; c < kMine; c += 32) {
          if (c >= columns) break;
          float v[32];
          tmem_ld32(from + c, v);
          if (SUMS) {
            float low[32];
            if (kAccs == 2) tmem_ld32(from + TN + c, low);
#pragma unroll
            for (int e = 0; e < 32; ++e) sum[SUMS ? c + e : 0] += kAccs == 2 ? v[e] + low[e] : v[e];
          } else {
            finish32(P, u, terms, c / 32, lane_row, u.n0 + half * kMine + c, S.columns[warp - 2], v);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.taken[turn & 1]);
      }
      if (!ok) break;
      if (SUMS || turns == 0) {
#pragma unroll
        for (int c = 0; c < kMine; c += 32) {
          if (c >= columns) break;
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = SUMS ? sum[SUMS ? c + e : 0] : 0.f;
          finish32(P, u, terms, c / 32, lane_row, u.n0 + half * kMine + c, S.columns[warp - 2], v);
        }
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (S.abort) {  // what is under way into this block's memory lands before the block ends
    if (tid == 0) {
      gave_up(P);
      for (int s = 0; s < kStages; ++s)
        if (S.issued > s) mbar_wait(&S.full[s], ((S.issued - 1 - s) / kStages) & 1);
    }
  }
  __syncwarp();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- pairs of blocks ------------------------------------------------------------------------------------------------------
// The same products with two SMs on a tile of 256 x 256 (tcgen05 cta_group::2): each has 128 rows of the left operand, half of
// the right one's columns and the accumulators of its 128 rows, and one of them issues for both.  A block then copies 32 KB
// for what takes 48 KB alone.  That is what bounds wide layers: one block per tile drew 57 bytes per cycle and SM out of L2
// (13.5 TB/s) at 61% of the tensor cores' time.
// The leader's barriers count both blocks' copies and readings; its commits arrive in both blocks.
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned in_block(const void *p, unsigned rank) {  // the peer's (or own) shared memory
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_at(unsigned cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// mbar_wait_warp for barriers that the other block arrives at
__device__ __forceinline__ bool wait_pair(unsigned long long *bar, unsigned parity, const volatile int *abort) {
  const unsigned addr = smem_u32(bar);
  for (unsigned it = 0; it < kWaitLimit; ++it) {
    unsigned done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done != 0)) return true;
    if (__any_sync(0xffffffffu, *abort != 0)) return false;
  }
  return false;
}
// into this block, counted by a barrier of either
__device__ __forceinline__ void load_tile_pair(unsigned dst, const CUtensorMap *map, int x, int y, int z, int w, unsigned cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(cluster_bar)
      : "memory");
}
template <bool F8>
__device__ __forceinline__ void mma_pair_if(unsigned lead, unsigned d, unsigned a_lo, unsigned a_hi, unsigned b_lo, unsigned b_hi, unsigned idesc,
                                            unsigned accumulate) {
  if (!F8)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.u32 e, %7, 0;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t@e tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.u32 e, %7, 0;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void commit_pair_if(unsigned lead, unsigned long long *bar) {  // arrives at `bar` of both blocks
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead), "h"((unsigned short)3)
      : "memory");
}

constexpr int kPairN = 256;  // columns of a pair's tile

template <bool SUMS, bool WEIGHTS, bool B_ROWS, bool F8>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_group_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GroupParams P) {
  SCN_GRID_WAIT();
  constexpr int kABytes = kTileM * kRow, kBBytes = kPairN / 2 * kRow, kStage = kABytes + kBBytes, kStages = kRing / kStage, kColumns = 256;
  static_assert(kStages <= kMostStages, "ring");
  extern __shared__ unsigned char raw[];
  unsigned char *ring = raw + (1024 - smem_u32(raw) % 1024) % 1024;  // (at the same address in both blocks)
  __shared__ Shared S;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const unsigned rank = cluster_rank();
  volatile int *abort = &S.abort;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&S.full[i], 1), mbar_init(&S.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&S.ready[i], 1), mbar_init(&S.taken[i], 2 * kEpilogueWarps);
    for (int i = 0; i < kStages; ++i) mbar_init(&S.tail[i], 1), mbar_init(&S.zeroed[i], 2);
    S.abort = 0;
    S.issued = 0;
    S.tails = S.tail_last = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2 && lane == 0) prefetch_map(&map_a), prefetch_map(&map_b);
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  scan_groups<WEIGHTS>(P, S);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // (barriers of both blocks exist)
  tc_fence_after();
  const unsigned tmem = S.tmem;
  const int all = WEIGHTS ? P.groups : P.groups + 2;
  const long long units = (long long)S.first[all] * P.n_tiles * (WEIGHTS ? P.m_tiles : 1);
  const long long pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  constexpr int kPerStage = F8 ? 2 * kStageRows : kStageRows;
  auto steps_of = [&](const Unit &u) { return WEIGHTS ? (u.rows + kStageRows - 1) / kStageRows : u.group < P.groups ? (P.k + kPerStage - 1) / kPerStage : 0; };
  auto width_of = [&](const Unit &u) { return min(kPairN, (P.n - u.n0 + 31) / 32 * 32); };  // columns of the instruction
  auto boxes_of = [&](const Unit &u, int r) { return WEIGHTS ? 2 : u.rows > r * kTileM; };  // copies of the left operand

  // ==== copies ====
  if (warp == 0) {
    const bool lead = elect_one();
    const unsigned full0 = in_block(&S.full[0], 0), ring0 = smem_u32(ring);
    int step = 0, st = 0;
    unsigned lap = 1;    // (a new barrier counts as past its phase of parity 1)
    unsigned tails = 0;  // a bit per stage, the other way round after each sum that ended there
    bool ok = true;
    Walk<WEIGHTS, kPairN> walk(P, S);
    for (long long i = pair; i < units && ok; i += pairs) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u), n0 = u.n0 + (int)rank * (width_of(u) / 2), boxes = boxes_of(u, rank);
      constexpr unsigned kBox = WEIGHTS ? kStageRows * kRow : kTileM * kRow;
      const unsigned mine = boxes * kBox + kBBytes, both = (boxes_of(u, 0) + boxes_of(u, 1)) * kBox + 2 * kBBytes;
      for (int k = 0; k < steps; ++k, ++step) {
        if (!wait_pair(&S.empty[st], lap, abort)) {
          ok = false;
          break;
        }
        // a sum that ends inside a stage: each block sees its own copies land, to overwrite what lies behind the last row
        const bool tail = WEIGHTS && (k + 1) * kStageRows > u.rows;
        if (lead) {
          const unsigned a = ring0 + st * kStage, b = a + kABytes, bar = tail ? in_block(&S.tail[st], rank) : full0 + st * 8;
          if (tail) {
            mbar_expect_tx(&S.tail[st], mine);
            if (rank == 0) mbar_arrive(&S.full[st]);
            S.tails |= 1u << st, S.tail_last = (S.tail_last & ~(1u << st)) | (tails & (1u << st));
          } else if (rank == 0) {
            mbar_expect_tx(&S.full[st], both);
          }
          if (WEIGHTS) {
            for (int j = 0; j < 2; ++j) load_tile_pair(a + j * kStageRows * kRow, &map_a, u.m0 + (int)rank * kTileM + 64 * j, u.row + k * kStageRows, 0, 0, bar);
            for (int j = 0; j < 2; ++j) load_tile_pair(b + j * kStageRows * kRow, &map_b, n0 + 64 * j, u.row + k * kStageRows, 0, 0, bar);
          } else {
            if (boxes) load_tile_pair(a, &map_a, k * kPerStage, u.row + (int)rank * kTileM, 0, 0, bar);
            if (B_ROWS)
              for (int j = 0; j < 2; ++j) load_tile_pair(b + j * kStageRows * kRow, &map_b, n0 + 64 * j, k * kStageRows, u.group, 0, bar);
            else
              load_tile_pair(b, &map_b, k * kPerStage, n0, u.group, 0, bar);
          }
          S.issued = step + 1;
        }
        if (tail) tails ^= 1u << st;
        if (++st == kStages) st = 0, lap ^= 1;
        __syncwarp();
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== instructions ====
  else if (warp == 1) {
    const unsigned lead = elect_one(), ring0 = smem_u32(ring);
    int step = 0, turn = 0, st = 0;
    unsigned lap = 0, tails = 0;
    bool ok = true;
    Walk<WEIGHTS, kPairN> walk(P, S);
    for (long long i = pair; i < units && ok; i += pairs) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u);
      const unsigned idesc = P.idesc | (unsigned)(width_of(u) >> 3) << 17;
      const int behind = WEIGHTS ? u.rows % kStageRows : 0;
      for (int first = 0; first < steps && ok; first += SUMS ? P.drain : steps) {  // what is summed in one accumulator
        const int upto = SUMS ? min(steps, first + P.drain) : steps;
        if (rank == 0 && turn >= 2 && !wait_pair(&S.taken[turn & 1], ((turn >> 1) - 1) & 1, abort)) {
          ok = false;
          break;
        }
        const unsigned d = tmem + (turn & 1) * kColumns;
        for (int k = first; k < upto; ++k, ++step, lap ^= st == kStages - 1, st = st == kStages - 1 ? 0 : st + 1) {
          int instructions = 4;
          if (WEIGHTS && behind && k == steps - 1) {
            instructions = (behind + 15) / 16;
            if (!wait_pair(&S.tail[st], tails >> st & 1, abort)) {
              ok = false;
              break;
            }
            const int gap = (instructions * 16 - behind) * 8;
            for (int q = lane; q < gap * 4; q += 32)
              *reinterpret_cast<uint4 *>(ring + st * kStage + q / gap * (kStageRows * kRow) + behind * kRow + q % gap * 16) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive_at(in_block(&S.zeroed[st], 0));
            if (rank == 0 && !wait_pair(&S.zeroed[st], tails >> st & 1, abort)) {
              ok = false;
              break;
            }
            tails ^= 1u << st;
          }
          if (rank != 0) continue;
          if (!wait_pair(&S.full[st], lap, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const unsigned a = ring0 + st * kStage, b = a + kABytes;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= instructions) break;
            const unsigned pa = a + j * (WEIGHTS ? 16 * kRow : 32), pb = b + j * (WEIGHTS || B_ROWS ? 16 * kRow : 32);
            mma_pair_if<F8>(lead, d, desc_lo(pa, WEIGHTS ? kStageRows * kRow : 16), kDescHi, desc_lo(pb, WEIGHTS || B_ROWS ? kStageRows * kRow : 16), kDescHi,
                            idesc, k > first || j > 0);
          }
          if (!(P.drop && blockIdx.x == 0 && step == 0)) commit_pair_if(lead, &S.empty[st]);
          if (k == upto - 1) commit_pair_if(lead, &S.ready[turn & 1]);
          __syncwarp();
        }
        ++turn;
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== results ====
  else {
    const int quarter = warp % 4, half = (warp - 2) / 4;
    constexpr int kMine = kPairN / 2;
    const int lane_row = (int)rank * kTileM + quarter * 32 + lane;
    int turn = 0;
    bool ok = true;
    Walk<WEIGHTS, kPairN> walk(P, S);
    for (long long i = pair; i < units && ok; i += pairs) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u), columns = min(P.n - u.n0 - half * kMine, kMine);
      const bool summed = steps > 0;
      Terms<kMine, WEIGHTS, F8> terms;
      terms.read(P, u, u.n0 + half * kMine, lane_row, lane);
      if (SUMS && steps > P.drain) {  // a long sum: its parts into registers
        float sum[SUMS ? kMine : 1];
#pragma unroll
        for (int c = 0; c < (SUMS ? kMine : 1); ++c) sum[c] = 0.f;
        for (int t = (steps - 1) / P.drain; t >= 0; --t, ++turn) {
          if (!wait_pair(&S.ready[turn & 1], (turn >> 1) & 1, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kMine; c += 16) {
            if (c >= columns) break;
            float v[16];
            tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + (turn & 1) * kColumns + half * kMine + c, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[SUMS ? c + e : 0] += v[e];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(in_block(&S.taken[turn & 1], 0));
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kMine; c += 32) {
          if (c >= columns) break;
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = sum[SUMS ? c + e : 0];
          finish32(P, u, terms, c / 32, lane_row, u.n0 + half * kMine + c, S.columns[warp - 2], v);
        }
        continue;
      }
      if (summed && !wait_pair(&S.ready[turn & 1], (turn >> 1) & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const unsigned from = tmem + ((unsigned)(quarter * 32) << 16) + (turn & 1) * kColumns + half * kMine;
#pragma unroll
      for (int c = 0; c < kMine; c += 32) {
        if (c >= columns) break;
        float v[32];
        if (summed) {
          tmem_ld32(from + c, v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        }
        finish32(P, u, terms, c / 32, lane_row, u.n0 + half * kMine + c, S.columns[warp - 2], v);
      }
      if (summed) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(in_block(&S.taken[turn & 1], 0));
        ++turn;
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (S.abort) {  // own copies land before the block ends; those of full steps are counted by the leader
    if (tid == 0) {
      gave_up(P);
      if (rank == 0)
        for (int s = 0; s < kStages; ++s)
          if (S.issued > s) mbar_wait(&S.full[s], ((S.issued - 1 - s) / kStages) & 1);
      for (int s = 0; s < kStages; ++s)
        if (S.tails >> s & 1) mbar_wait(&S.tail[s], S.tail_last >> s & 1);
    }
  }
  __syncthreads();
  cluster_sync();  // (nothing of the other block is under way into this one's barriers or out of its operands)
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// 8 fp32 values as PARTS times 8 bf16 values: x = h + m + l, each part rounded to nearest of what the ones before leave.
// `plain`: no value is above bf16's largest (it would round to an infinity).
template <int PARTS>
__device__ __forceinline__ void split8(const float (&v)[8], bool plain, unsigned (&w)[3][4]) {
  if (plain) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        w[p][j] = pair(a, b, __nv_bfloat16());
        a -= __uint_as_float(w[p][j] << 16), b -= __uint_as_float(w[p][j] & 0xFFFF0000u);
      }
    }
  } else {  // such a value is cut off instead; an infinity or a NaN has no further parts
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float rest = v[j];
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        unsigned b = __bfloat16_as_ushort(__float2bfloat16_rn(rest));
        if (PARTS > 1 && (b & 0x7FFF) == 0x7F80 && isfinite(rest)) b = __float_as_uint(rest) >> 16;
        w[p][j / 2] = j % 2 ? w[p][j / 2] | b << 16 : b;
        rest = isfinite(rest) ? rest - __uint_as_float(b << 16) : 0.f;
      }
    }
  }
}
__device__ __forceinline__ bool all_plain(const float (&v)[8]) {  // (a NaN may take either way: all its parts are NaN)
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[j]));
  return __float_as_uint(most) < 0x7F7F8000u;
}

// Rows of a matrix as `parts` matrices of 16-bit values (or 8-bit ones, copied), planes padded with zeros to whole 16 bytes:
// what the copies above need where the operand is fp32 or its rows do not lie on 16 bytes.  One thread per 16 bytes of
// a part.  Bound by HBM: 4 bytes in, 2 per part out.
template <typename T, int PARTS>
__global__ void __launch_bounds__(256)
k_group_parts(const T *__restrict__ src, long long stride, int planes, long long n_pieces, int per_row, long long part_bytes,
              unsigned char *__restrict__ dst) {
  SCN_GRID_WAIT();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_pieces) return;
  constexpr int N = sizeof(T) == 1 ? 16 : 8;
  const long long row = i / per_row;
  const int c = (int)(i - row * per_row) * N;
  const T *from = src + row * stride + c;
  unsigned w[3][4] = {};
  if (sizeof(T) == 4) {
    float v[8];
    if (c + 8 <= planes && ((uintptr_t)from & 15) == 0) {
      const float4 p = __ldg((const float4 *)from), q = __ldg((const float4 *)from + 1);
      v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < planes ? __ldg((const float *)from + j) : 0.f;
    }
    split8<PARTS>(v, PARTS == 1 || all_plain(v), w);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const unsigned v = c + j < planes ? (sizeof(T) == 2 ? (unsigned)__ldg((const unsigned short *)from + j) : (unsigned)__ldg((const unsigned char *)from + j)) : 0u;
      w[0][j * (int)sizeof(T) / 4] |= v << (j * (int)sizeof(T) % 4 * 8);
    }
  }
#pragma unroll
  for (int p = 0; p < PARTS; ++p) *reinterpret_cast<uint4 *>(dst + p * part_bytes + i * 16) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// ---- fp32 operands, split on their way --------------------------------------------------------------------------------------
// The products of fp32 rows for layers of few planes, where a tile is a few steps long and the rows' bytes are what it costs:
// sixteen more warps read the fp32 rows, split them and write the parts into the operands' places, so that the parts are never
// in memory (4 bytes a value in instead of 4 in, 6 out and 6 in again).  A sum is at most kSplitSteps steps long, so that it
// needs no hand-over between: rows of up to 256 planes, units of 256 rows for the weights' gradient, whose partial sums are
// added by k_group_sum.  Where the results' rows (planes of x) leave a row of the last tile free, a plane of ones in x makes
// that row the bias sums.
constexpr int kSplitSteps = 4, kSplitWarps = 16, kSplitLoaders = kSplitWarps * 32, kSplitThreads = kThreads + kSplitWarps * 32;

struct Cursor {  // a step of a unit
  long long i;
  Unit u;
  int k, steps, step;
  bool live;
};

// PIECES pieces (8 values, 16 bytes of each part) of an operand's step, one thread's share: rows of WIDE pieces
struct Side {
  const float *p;
  long long stride;
  int quads, limit, col0, rows, first;  // limit: planes; rows: below it rows are real; first: the step's first row
};
template <int WIDE, int PIECES>
__device__ __forceinline__ void fetch(const Side &S, int t, float (&v)[PIECES][8]) {
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int row = (i * kSplitLoaders + t) / WIDE, col = S.col0 + t % WIDE * 8;
    const float *p = S.p + (S.first + row) * S.stride + col;
    const bool in = row < S.rows;
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (S.quads) {
        if (in && col + j < S.limit) q = __ldg((const float4 *)(p + j));
      } else if (in) {
        if (col + j < S.limit) q.x = __ldg(p + j);
        if (col + j + 1 < S.limit) q.y = __ldg(p + j + 1);
        if (col + j + 2 < S.limit) q.z = __ldg(p + j + 2);
        if (col + j + 3 < S.limit) q.w = __ldg(p + j + 3);
      }
      v[i][j] = q.x, v[i][j + 1] = q.y, v[i][j + 2] = q.z, v[i][j + 3] = q.w;
    }
  }
}
// `ones`: the plane that is one in every real row, -1: none.  Rows (K-major) or planes (M- / N-major) that no result needs keep
// what is there; rows behind a sum's last are needed, as zeros.
template <int PARTS, int WIDE, int PIECES, bool K_MAJOR>
__device__ __forceinline__ void put(const Side &S, int t, int limit, int ones, unsigned char *to, int part_bytes, float (&v)[PIECES][8]) {
  const int chunk = t % WIDE, col = S.col0 + chunk * 8;
  bool plain = true;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    if (!K_MAJOR && ones >= 0 && (ones >> 3) == (col >> 3)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j == ones) v[i][j] = (i * kSplitLoaders + t) / WIDE < S.rows ? 1.f : 0.f;
    }
    plain = plain && (PARTS == 1 || all_plain(v[i]));
  }
  if (!K_MAJOR && col >= limit) return;
  auto pieces = [&](bool quick) {  // (one branch for all: their chains of roundings and differences overlap)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int row = (i * kSplitLoaders + t) / WIDE;
      unsigned w[3][4];
      split8<PARTS>(v[i], quick, w);
      unsigned char *at = to + (K_MAJOR ? 0 : chunk / 8 * (kStageRows * kRow)) + row * kRow + ((chunk % 8) ^ (row & 7)) * 16;
      if (!K_MAJOR || row < S.rows) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p) *reinterpret_cast<uint4 *>(at + p * part_bytes) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
      }
    }
  };
  if (plain)
    pieces(true);
  else
    pieces(false);
}

template <int PARTS, int TN, bool WEIGHTS, bool B_ROWS>
__global__ void __launch_bounds__(kSplitThreads, 1)
k_group_split(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GroupParams P) {
  SCN_GRID_WAIT();
  constexpr int kABytes = kTileM * kRow, kBBytes = TN * kRow, kStage = PARTS * (kABytes + kBBytes);
  constexpr int kStages = kRing / kStage < kMostStages ? kRing / kStage : kMostStages, kAccs = PARTS > 1 ? 2 : 1, kColumns = 256;
  static_assert(kAccs * TN <= kColumns && kStages >= 2, "shape");
  extern __shared__ unsigned char raw[];
  unsigned char *ring = raw + (1024 - smem_u32(raw) % 1024) % 1024;
  __shared__ Shared S;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  volatile int *abort = &S.abort;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&S.full[i], kSplitWarps + !WEIGHTS), mbar_init(&S.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&S.ready[i], 1), mbar_init(&S.taken[i], kEpilogueWarps);
    S.abort = 0;
    S.issued = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (!WEIGHTS && warp == 2 && lane == 0) prefetch_map(&map_b);
  if (warp == 1) tmem_alloc(&S.tmem, 512);
  scan_groups<WEIGHTS>(P, S);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = S.tmem;
  const int all = WEIGHTS ? P.groups : P.groups + 2;
  const long long units = (long long)S.first[all] * P.n_tiles * (WEIGHTS ? P.m_tiles : 1);
  auto steps_of = [&](const Unit &u) { return ((WEIGHTS ? u.rows : u.group < P.groups ? P.k : 0) + kStageRows - 1) / kStageRows; };

  // ==== weights ====
  if (warp == 0) {
    const bool lead = elect_one();
    int step = 0;
    bool ok = true;
    // what a stage's place for weights holds: tiles of the same group and columns come one after the other, and with no more
    // steps than stages each finds its slice where the last one left it
    int held[kStages][3];
#pragma unroll
    for (int i = 0; i < kStages; ++i) held[i][0] = held[i][1] = held[i][2] = -1;
    Walk<WEIGHTS, TN> walk(P, S);
    for (long long i = blockIdx.x; i < units && ok; i += gridDim.x) {
      const Unit u = walk.at(i);
      const int steps = WEIGHTS ? 0 : steps_of(u);
      for (int k = 0; k < steps; ++k, ++step) {
        const int st = step % kStages;
        if (step >= kStages && !mbar_wait_warp(&S.empty[st], (step / kStages - 1) & 1, abort)) {
          ok = false;
          break;
        }
        bool here = false;
#pragma unroll
        for (int i = 0; i < kStages; ++i)
          if (i == st) {
            here = held[i][0] == u.group && held[i][1] == u.n0 && held[i][2] == k;
            held[i][0] = u.group, held[i][1] = u.n0, held[i][2] = k;
          }
        if (here) {
          if (lead) mbar_arrive(&S.full[st]);
        } else if (lead) {
          const unsigned b = smem_u32(ring) + st * kStage + PARTS * kABytes;
          mbar_expect_tx(&S.full[st], PARTS * kBBytes);
          for (int p = 0; p < PARTS; ++p) {
            if (B_ROWS)
              for (int j = 0; j < TN / 64; ++j) load_tile(b + p * kBBytes + j * kStageRows * kRow, &map_b, u.n0 + 64 * j, k * kStageRows, u.group, p, &S.full[st]);
            else
              load_tile(b + p * kBBytes, &map_b, k * kStageRows, u.n0, u.group, p, &S.full[st]);
          }
          S.issued = step + 1;
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== instructions ====
  else if (warp == 1) {
    const unsigned lead = elect_one();
    int step = 0, turn = 0;
    bool ok = true;
    Walk<WEIGHTS, TN> walk(P, S);
    for (long long i = blockIdx.x; i < units && ok; i += gridDim.x) {
      const Unit u = walk.at(i);
      const int steps = steps_of(u);
      if (!steps) continue;
      const unsigned idesc = P.idesc | (unsigned)(min(TN, (P.n - u.n0 + 15) / 16 * 16) >> 3) << 17;
      if (turn >= 2 && !mbar_wait_warp(&S.taken[turn & 1], ((turn >> 1) - 1) & 1, abort)) ok = false;
      for (int k = 0; k < steps && ok; ++k, ++step) {
        const int st = step % kStages;
        if (!mbar_wait_warp(&S.full[st], (step / kStages) & 1, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const unsigned a = smem_u32(ring) + st * kStage, b = a + PARTS * kABytes, d = tmem + (turn & 1) * kColumns;
        const int instructions = ((WEIGHTS ? min(kStageRows, u.rows - k * kStageRows) : min(kStageRows, P.k - k * kStageRows)) + 15) / 16;
        for (int j = 0; j < instructions; ++j) {
#pragma unroll
          for (int q = 0; q < Products<PARTS>::N; ++q) {
            const unsigned pa = a + part_a(q) * kABytes + j * (WEIGHTS ? 16 * kRow : 32), pb = b + part_b(q) * kBBytes + j * (WEIGHTS || B_ROWS ? 16 * kRow : 32);
            const unsigned fresh = k == 0 && j == 0 && (q == 0 || q == 1);
            mma_if<false>(lead, d + (q ? TN : 0), desc_lo(pa, WEIGHTS ? kStageRows * kRow : 16), kDescHi, desc_lo(pb, WEIGHTS || B_ROWS ? kStageRows * kRow : 16),
                          kDescHi, idesc, !fresh);
          }
        }
        if (!(P.drop && blockIdx.x == 0 && step == 0)) tc_commit_if(lead, &S.empty[st]);
        if (k == steps - 1) tc_commit_if(lead, &S.ready[turn & 1]);
        __syncwarp();
      }
      ++turn;
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== results ====
  else if (warp < 2 + kEpilogueWarps) {
    const int quarter = warp % 4, half = (warp - 2) / 4;
    constexpr int kMine = TN / 2;
    const int lane_row = quarter * 32 + lane;
    int turn = 0;
    bool ok = true;
    Walk<WEIGHTS, TN> walk(P, S);
    for (long long i = blockIdx.x; i < units && ok; i += gridDim.x) {
      const Unit u = walk.at(i);
      const int columns = min(P.n - u.n0 - half * kMine, kMine);
      const bool summed = steps_of(u) > 0;
      Terms<kMine, WEIGHTS, false> terms;
      terms.read(P, u, u.n0 + half * kMine, lane_row, lane);
      if (summed && !mbar_wait_warp(&S.ready[turn & 1], (turn >> 1) & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const unsigned from = tmem + ((unsigned)(quarter * 32) << 16) + (turn & 1) * kColumns + half * kMine;
#pragma unroll
      for (int c = 0; c < kMine; c += 32) {
        if (c >= columns) break;
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.f;
        if (summed) {
          tmem_ld32(from + c, v);
          if (kAccs == 2) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              float low[16];
              tmem_ld16(from + TN + c + e, low);
#pragma unroll
              for (int f = 0; f < 16; ++f) v[e + f] += low[f];
            }
          }
        }
        finish32(P, u, terms, c / 32, lane_row, u.n0 + half * kMine + c, S.columns[warp - 2], v);
      }
      if (summed) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.taken[turn & 1]);
        ++turn;
      }
    }
    if (!ok && lane == 0) *abort = 1;
  }
  // ==== rows ====
  else {
    const int t = tid - kThreads;
    constexpr int kLeft = kTileM * 8 / kSplitLoaders, kRight = TN * 8 / kSplitLoaders, kRightWide = TN / 8;  // pieces of a thread
    bool ok = true;
    Walk<WEIGHTS, TN> walk(P, S);
    Cursor next;
    next.i = blockIdx.x, next.k = next.step = 0;
    auto settle = [&] {  // on to a unit that has steps
      for (next.live = false; next.i < units; next.i += gridDim.x) {
        next.u = walk.at(next.i);
        next.steps = steps_of(next.u);
        if (next.steps) {
          next.live = true;
          break;
        }
      }
    };
    auto advance = [&] {
      ++next.step;
      if (++next.k < next.steps) return;
      next.k = 0;
      next.i += gridDim.x;
      settle();
    };
    auto left = [&](const Cursor &c) {
      return WEIGHTS ? Side{P.a, P.a_stride, P.a_quads, P.m, c.u.m0, c.u.rows - c.k * kStageRows, c.u.row + c.k * kStageRows}
                     : Side{P.a, P.a_stride, P.a_quads, P.k, c.k * kStageRows, c.u.rows, c.u.row};
    };
    auto right = [&](const Cursor &c) { return Side{P.b, P.b_stride, P.b_quads, P.n, c.u.n0, c.u.rows - c.k * kStageRows, c.u.row + c.k * kStageRows}; };
    // The next step's values are on their way while the present one's are split: rows by two sets of registers in turn, for the
    // weights' gradient the left operand's while the right one's are split and the other way round.
    float va[kLeft][8], vb[WEIGHTS ? kRight : kLeft][8];
    auto one = [&](auto &now, auto &then) {
      const Cursor c = next;
      unsigned char *to = ring + c.step % kStages * kStage;
      if constexpr (!WEIGHTS) {
        advance();
        if (next.live) fetch<8, kLeft>(left(next), t, then);
      }
      if (c.step >= kStages && !mbar_wait_warp(&S.empty[c.step % kStages], (c.step / kStages - 1) & 1, abort)) return false;
      if constexpr (!WEIGHTS) {
        put<PARTS, 8, kLeft, true>(left(c), t, 0, -1, to, kABytes, now);
      } else {
        put<PARTS, 16, kLeft, false>(left(c), t, P.m_rows, P.m_rows > P.m ? P.m : -1, to, kABytes, va);
        advance();
        if (next.live) fetch<16, kLeft>(left(next), t, va);
        put<PARTS, kRightWide, kRight, false>(right(c), t, P.n, -1, to + PARTS * kABytes, kBBytes, vb);
        if (next.live) fetch<kRightWide, kRight>(right(next), t, vb);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.full[c.step % kStages]);
      return true;
    };
    settle();
    if (next.live) {
      fetch<WEIGHTS ? 16 : 8, kLeft>(left(next), t, va);
      if constexpr (WEIGHTS) fetch<kRightWide, kRight>(right(next), t, vb);
    }
    while (next.live && ok) {
      ok = one(va, vb);
      if (!WEIGHTS && ok && next.live) ok = one(vb, va);
    }
    if (!ok && lane == 0) *abort = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (S.abort && tid == 0) {  // the weights' copies land before the block ends
    gave_up(P);
    // (a stage's barrier also counts the rows, which may not come any more: a bounded wait is long enough for a copy to land)
    for (int s = 0; s < kStages; ++s)
      if (S.issued > s) mbar_wait(&S.full[s], ((S.issued - 1 - s) / kStages) & 1);
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

__device__ __forceinline__ void put_value(void *out, int type, long long at, float v) {
  if (type == SCN_TYPE_FLOAT32)
    ((float *)out)[at] = v;
  else if (type == SCN_TYPE_BFLOAT16)
    ((__nv_bfloat16 *)out)[at] = __float2bfloat16_rn(v);
  else
    ((__half *)out)[at] = __float2half_rn(v);
}

// The gradients of the groups of several units: their partial sums, in an order that goes by the number of units alone.  Few
// units: a thread adds a result's sums, 256 results to a block.  Many (a group may have a hundred times the units of the
// next): 32 results to a block, 8 threads to a result, each adds every eighth unit, and their sums are added in order.  The
// blocks are dealt to the pieces of all such groups in turn.
constexpr int kManyUnits = 16;
__global__ void __launch_bounds__(256)
k_group_sum(const __grid_constant__ GroupParams P) {
  SCN_GRID_WAIT();
  __shared__ Shared S;
  __shared__ float slices[8][32];
  scan_groups<true>(P, S);
  const long long size = (long long)P.m_rows * P.n, weights = (long long)P.m * P.n;
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  auto store = [&](int g, long long i, float v) {
    if (i < weights)
      put_value(P.out, P.out_type, g * weights + i, v);
    else
      put_value(P.d_bias, P.out_type, (long long)g * P.n + i - weights, v);
  };
  long long turn = blockIdx.x;  // the first piece of the next such group that is this block's
  for (int g = 0; g < P.groups; ++g) {
    if (S.part[g] < 0) continue;
    const int units = S.first[g + 1] - S.first[g];
    const bool many = units >= kManyUnits;
    const int each = many ? 32 : 256;
    const long long pieces = (size + each - 1) >> (many ? 5 : 8);
    const float *from = P.partial + S.part[g] * size;
    for (; turn < pieces; turn += gridDim.x) {
      const long long i = turn * each + (many ? lane : threadIdx.x);
      const int step = many ? 8 : 1;
      float v = 0.f;
      if (i < size) {
        const long long stride = step * size;
        int u = many ? slice : 0;
        const float *p = from + u * size + i;
        for (; u + 3 * step < units; u += 4 * step, p += 4 * stride) {  // (added in order, asked for at once)
          const float x0 = __ldg(p), x1 = __ldg(p + stride), x2 = __ldg(p + 2 * stride), x3 = __ldg(p + 3 * stride);
          v += x0, v += x1, v += x2, v += x3;
        }
        for (; u < units; u += step, p += stride) v += __ldg(p);
      }
      if (!many) {
        if (i < size) store(g, i, v);
        continue;
      }
      slices[slice][lane] = v;
      __syncthreads();
      if (slice == 0 && i < size) {
#pragma unroll
        for (int j = 1; j < 8; ++j) v += slices[j][lane];
        store(g, i, v);
      }
      __syncthreads();
    }
    turn -= pieces;
  }
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// db[g] = sum of a group's rows: a block takes a unit of P.chunk rows and 32 planes, 8 rows at a time (m = 1)
template <typename T>
__global__ void __launch_bounds__(256)
k_group_bias(const __grid_constant__ GroupParams P, const T *__restrict__ d_out, long long stride) {
  SCN_GRID_WAIT();
  __shared__ Shared S;
  __shared__ float part[8][33];
  scan_groups<true>(P, S);
  const int lane = threadIdx.x % 32, along = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
  Walk<true, 64> walk(P, S);
  for (long long u = blockIdx.y; u < S.first[P.groups]; u += gridDim.y) {
    const Unit unit = walk.at(u);
    float v = 0.f;
    if (c < P.n) {
      int r = along;
      for (; r + 56 < unit.rows; r += 64) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = as_float(__ldg(d_out + (unit.row + r + 8 * j) * stride + c));
        v += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      }
      for (; r < unit.rows; r += 8) v += as_float(__ldg(d_out + (unit.row + r) * stride + c));
    }
    part[along][lane] = v;
    __syncthreads();
    if (along == 0 && c < P.n) {
#pragma unroll
      for (int j = 1; j < 8; ++j) v += part[j][lane];
      if (unit.part >= 0)
        P.partial[(long long)unit.part * P.n + c] = v;
      else
        put_value(P.out, P.out_type, (long long)unit.group * P.n + c, v);
    }
    __syncthreads();
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int encoder(EncodeTiled *out) {  // looked up through the runtime: the library loads on a machine without a driver
  static std::atomic<EncodeTiled> known{nullptr};
  *out = known.load();
  if (!*out) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    SCN_CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found));
    SCN_REQUIRE(fn && found == cudaDriverEntryPointSuccess, SCN_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    known.store(*out = (EncodeTiled)fn);
  }
  return SCN_OK;
}

// Where kernels of the current device say that they gave up: a word of pinned memory, so that the next call sees it without waiting.
int flag_of(int **word) {
  static std::mutex mu;
  static int *words = nullptr;
  int dev = 0;
  SCN_CUDA_CHECK(cudaGetDevice(&dev));
  SCN_REQUIRE(dev >= 0 && dev < 64, SCN_ERR_UNSUPPORTED, "device index %d unsupported", dev);
  std::lock_guard<std::mutex> lock(mu);
  if (!words) {  // (allowed while a stream of this thread is captured: nothing of it becomes part of the graph)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    SCN_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    void *p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, 64 * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    SCN_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    SCN_CUDA_CHECK(e);
    memset(p, 0, 64 * sizeof(int));
    words = (int *)p;
  }
  *word = words + dev;
  return SCN_OK;
}
// An error if a call before this one gave up, once
int look_at_flag(int *word) {
  SCN_REQUIRE(!__atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL), SCN_ERR_CUDA,
              "a wait inside an earlier grouped product ran out: its results are incomplete");
  return SCN_OK;
}

// An operand as the tensor maps need it
struct Operand {
  const void *p = nullptr;
  int bytes = 2;             // of a value
  long long stride = 0;      // bytes from row to row
  long long matrix = 0;      // bytes from group to group (weights)
  long long part = 0;        // bytes from part to part
};

int make_map(CUtensorMap *map, const Operand &o, int type, long long planes, long long rows, long long groups, int parts, int box_planes, int box_rows) {
  EncodeTiled encode;
  SCN_TRY(encoder(&encode));
  const long long matrix = o.matrix ? o.matrix : rows * o.stride, part = o.part ? o.part : groups * matrix;
  const cuuint64_t dims[4] = {(cuuint64_t)planes, (cuuint64_t)rows, (cuuint64_t)groups, (cuuint64_t)parts};
  const cuuint64_t strides[3] = {(cuuint64_t)o.stride, (cuuint64_t)matrix, (cuuint64_t)part};
  const cuuint32_t box[4] = {(cuuint32_t)box_planes, (cuuint32_t)box_rows, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t = type == SCN_TYPE_E4M3     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                : type == SCN_TYPE_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  auto make = [&] {
    return encode(map, t, 4, const_cast<void *>(o.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = make();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {  // a thread that has not launched anything yet (autograd's): the driver wants its context bound
    int dev = 0;
    SCN_CUDA_CHECK(cudaGetDevice(&dev));
    SCN_CUDA_CHECK(cudaSetDevice(dev));
    r = make();
  }
  SCN_REQUIRE(r == CUDA_SUCCESS, SCN_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return SCN_OK;
}

// The operand where it lies, or a copy in parts
int operand(const void *p, long long stride, int planes, long long rows, int type, int parts, Scratch &scratch, cudaStream_t stream, Operand *o) {
  const int size = type == SCN_TYPE_FLOAT32 ? 4 : type == SCN_TYPE_E4M3 ? 1 : 2;
  if (type != SCN_TYPE_FLOAT32 && (uintptr_t)p % 16 == 0 && stride * size % 16 == 0 && stride > 0 && stride * size < (1ll << 40)) {
    *o = Operand{p, size, stride * size, 0, 0};
    return SCN_OK;
  }
  const int held = size == 1 ? 1 : 2, per_row = (int)ceil_div((long long)planes * held, 16);
  const long long row_bytes = per_row * 16ll, part_bytes = rows * row_bytes, pieces = rows * per_row;
  unsigned char *to = nullptr;
  SCN_TRY(scratch.get(&to, (size_t)(parts * part_bytes)));
  const unsigned blocks = (unsigned)ceil_div(pieces, 256);
#define SCN_PARTS(T, N) SCN_LAUNCH((k_group_parts<T, N>), blocks, 256, 0, stream, (const T *)p, stride, planes, pieces, per_row, part_bytes, to)
  if (type == SCN_TYPE_FLOAT32) {
    if (parts == 3)
      SCN_PARTS(float, 3);
    else if (parts == 2)
      SCN_PARTS(float, 2);
    else
      SCN_PARTS(float, 1);
  } else if (size == 2) {
    SCN_PARTS(unsigned short, 1);
  } else {
    SCN_PARTS(unsigned char, 1);
  }
#undef SCN_PARTS
  SCN_CUDA_CHECK(cudaGetLastError());
  *o = Operand{to, held, row_bytes, 0, part_bytes};
  return SCN_OK;
}

constexpr int kSms = 148;

template <int PARTS, int TN, bool SUMS, bool WEIGHTS, bool B_ROWS, bool F8>
int launch(const CUtensorMap &a, const CUtensorMap &b, GroupParams P, long long most_units, cudaStream_t stream) {
  constexpr size_t smem = kRing + 1024;
  static std::atomic<bool> configured[64];
  int dev = 0;
  SCN_CUDA_CHECK(cudaGetDevice(&dev));
  SCN_REQUIRE(dev >= 0 && dev < 64, SCN_ERR_UNSUPPORTED, "device index %d unsupported", dev);
  constexpr auto kernel = k_group_product<PARTS, TN, SUMS, WEIGHTS, B_ROWS, F8>;
  if (!configured[dev].load()) {
    SCN_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured[dev].store(true);
  }
  int blocks = 0;
  SCN_TRY(resident_blocks<kernel>(kThreads, smem, &blocks));
  SCN_LAUNCH(kernel, (unsigned)std::min<long long>(blocks, most_units), kThreads, smem, stream, a, b, P);
  SCN_CUDA_CHECK(cudaGetLastError());
  return SCN_OK;
}

// Two blocks to a tile.  Worth it where the copies bound a tile: many rows to a group (a group ends in the middle of 256 rows
// instead of 128 on average) and tiles enough for all pairs.
bool paired(long long row_tiles_256, long long groups, int n) { return n > 128 && row_tiles_256 >= 2 * groups && row_tiles_256 * ceil_div(n, kPairN) >= kSms / 2; }

template <bool SUMS, bool WEIGHTS, bool B_ROWS, bool F8>
int launch_pair(const CUtensorMap &a, const CUtensorMap &b, const GroupParams &P, long long most_units, cudaStream_t stream) {
  constexpr size_t smem = kRing + 1024;
  static std::atomic<int> known[64];  // pairs that the device holds at once
  int dev = 0;
  SCN_CUDA_CHECK(cudaGetDevice(&dev));
  SCN_REQUIRE(dev >= 0 && dev < 64, SCN_ERR_UNSUPPORTED, "device index %d unsupported", dev);
  constexpr auto kernel = k_group_pair<SUMS, WEIGHTS, B_ROWS, F8>;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.blockDim = kThreads;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attr;
  int pairs = known[dev].load();
  if (!pairs) {
    SCN_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    config.gridDim = 2;
    config.attrs = attr + 1;
    config.numAttrs = 1;
    SCN_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&pairs, kernel, &config));
    SCN_REQUIRE(pairs > 0, SCN_ERR_CUDA, "no pair of blocks fits the device");
    known[dev].store(pairs);
    config.attrs = attr;
  }
  config.numAttrs = 1;  // (the cluster's size is the kernel's own)
  config.gridDim = (unsigned)(2 * std::min<long long>(pairs, most_units));
  note_launch();
  SCN_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a, b, P));
  return SCN_OK;
}

// Columns of a tile: as wide as the results are, but no wider than leaves every SM a tile.
int tile_columns(long long row_tiles, int n, int most) {
  int tn = most;
  while (tn > 64 && (n <= tn / 2 || row_tiles * ceil_div(n, tn) < kSms)) tn /= 2;
  return tn;
}

unsigned idesc_of(int type, bool a_rows, bool b_rows, int m) {  // fp32 sums; types: bf16 1, f16 0, e4m3 0
  const unsigned t = type == SCN_TYPE_FLOAT16 || type == SCN_TYPE_E4M3 ? 0 : 1;
  return (1u << 4) | (t << 7) | (t << 10) | ((unsigned)a_rows << 15) | ((unsigned)b_rows << 16) | ((unsigned)(m >> 4) << 24);
}

struct Groups {
  const void *offsets;
  int off64;
  long long n_rows;
  int groups;
  int *flag;
};

// y = x W: `b_rows`: the weights' n lie next to each other ([k][n]), else their k ([n][k])
int rows_product(const Groups &G, const Operand &x, const Operand &w, bool b_rows, int parts, int type, int k, int n, void *out, int out_type,
                 const void *bias, int bias_type, const float *row_scale, const float *col_scale, int drop, cudaStream_t stream) {
  const int per = type == SCN_TYPE_E4M3 ? 128 : 64;  // values of k in a step
  const bool f8 = type == SCN_TYPE_E4M3, fine = !f8 && (parts > 1 || out_type == SCN_TYPE_FLOAT32), sums = fine || ceil_div(k, per) > kLong;
  const long long row_tiles = G.n_rows / kTileM + std::min<long long>(G.groups + 2, G.n_rows);
  const long long pair_tiles = G.n_rows / (2 * kTileM) + std::min<long long>(G.groups + 2, G.n_rows);
  const bool pair = !fine && paired(pair_tiles, G.groups, n);
  const int tn = pair ? kPairN : tile_columns(row_tiles, n, fine ? 128 : 256);
  GroupParams P{};
  P.offsets = G.offsets, P.off64 = G.off64, P.groups = G.groups, P.n_rows = (int)G.n_rows, P.flag = G.flag;
  P.tile = pair ? 2 * kTileM : kTileM;
  P.k = k, P.n = n, P.n_tiles = (int)ceil_div(n, tn);
  P.idesc = idesc_of(type, false, b_rows, P.tile);
  const int out_size = out_type == SCN_TYPE_FLOAT32 ? 4 : 2;
  P.out = out, P.out_type = out_type, P.aligned = aligned_to((uintptr_t)out, n, out_size), P.part_aligned = aligned_to(0, n, 4);
  P.bias = bias, P.bias_type = bias_type, P.row_scale = row_scale, P.col_scale = col_scale, P.drop = drop;
  P.drain = fine ? kDrain : kLongDrain;
  CUtensorMap a, b;
  SCN_TRY(make_map(&a, x, type, k, G.n_rows, parts, 1, per, pair ? kTileM : kBoxRows));  // (parts lie where groups would)
  SCN_TRY(b_rows ? make_map(&b, w, type, n, k, G.groups, parts, 64, 64) : make_map(&b, w, type, k, n, G.groups, parts, per, pair ? tn / 2 : tn));
  const long long most = (pair ? pair_tiles : row_tiles) * P.n_tiles;
#define SCN_PAIR(SUMS)                                                                                        \
  (f8 ? launch_pair<SUMS, false, false, true>(a, b, P, most, stream)                                          \
   : b_rows ? launch_pair<SUMS, false, true, false>(a, b, P, most, stream) : launch_pair<SUMS, false, false, false>(a, b, P, most, stream))
  if (pair) return sums ? SCN_PAIR(true) : SCN_PAIR(false);
#undef SCN_PAIR
#define SCN_TN(PARTS, SUMS, B_ROWS, F8)                                                                       \
  (tn == 64 ? launch<PARTS, 64, SUMS, false, B_ROWS, F8>(a, b, P, most, stream)                               \
   : tn == 128 ? launch<PARTS, 128, SUMS, false, B_ROWS, F8>(a, b, P, most, stream)                           \
               : launch<PARTS, (PARTS > 1) ? 128 : 256, SUMS, false, B_ROWS, F8>(a, b, P, most, stream))
#define SCN_MAJOR(PARTS, SUMS) (b_rows ? SCN_TN(PARTS, SUMS, true, false) : SCN_TN(PARTS, SUMS, false, false))
  if (f8) return sums ? SCN_TN(1, true, false, true) : SCN_TN(1, false, false, true);
  if (!sums) return SCN_MAJOR(1, false);
  return parts == 1 ? SCN_MAJOR(1, true) : parts == 2 ? SCN_MAJOR(2, true) : SCN_MAJOR(3, true);
#undef SCN_MAJOR
#undef SCN_TN
}

// Rows of a unit of a sum over rows, such that a group that has all of them still gives most SMs some: where there are fewer
// than half as many tiles of the result as SMs, twice as many units as SMs.
int chunk_of(long long n_rows, long long tiles) {
  const long long wanted = tiles * 2 >= kSms ? 1 : 2 * kSms / tiles;
  return (int)std::max<long long>(512, ceil_div(ceil_div(n_rows, wanted), 64) * 64);
}

// The most units that groups of several units can have together: such a group has more than `chunk` rows, so there are at most K of
// them, and each rounds its rows / chunk up by less than one.
long long most_parts(const Groups &G, long long chunk) {
  const long long K = std::min<long long>(G.groups, G.n_rows / (chunk + 1));
  return (G.n_rows + K * (chunk - 1)) / chunk;
}

int sum_parts(GroupParams P, cudaStream_t stream) {
  const long long items = ceil_div((long long)P.m_rows * P.n, 32) * P.groups;
  SCN_LAUNCH(k_group_sum, (unsigned)std::min<long long>(items, 8 * kSms), 256, 0, stream, P);
  SCN_CUDA_CHECK(cudaGetLastError());
  return SCN_OK;
}

// dW = x^T dy by groups
int weights_product(const Groups &G, const Operand &x, const Operand &dy, int parts, int type, int m, int n, void *out, int out_type,
                    Scratch &scratch, cudaStream_t stream) {
  // (pairs: tiles of 256 x 256 of the result; a sum that ends inside a stage costs a pair 2 us, so not for sums of a few rows)
  const bool pair = parts == 1 && m > kTileM && n > 128 && G.n_rows >= 256ll * G.groups &&
                    ceil_div(m, 2 * kTileM) * ceil_div(n, kPairN) * std::max<long long>(G.groups, G.n_rows / 512) >= kSms / 2;
  const long long m_tiles = ceil_div(m, pair ? 2 * kTileM : kTileM);
  const int tn = pair ? kPairN : tile_columns(m_tiles * std::max<long long>(G.groups, G.n_rows / 512), n, parts > 1 ? 128 : 256);
  GroupParams P{};
  P.offsets = G.offsets, P.off64 = G.off64, P.groups = G.groups, P.n_rows = (int)G.n_rows, P.flag = G.flag;
  P.tile = pair ? 2 * kTileM : kTileM;
  P.m = P.m_rows = m, P.n = n, P.m_tiles = (int)m_tiles, P.n_tiles = (int)ceil_div(n, tn);
  P.chunk = chunk_of(G.n_rows, (long long)P.m_tiles * P.n_tiles);
  P.idesc = idesc_of(type, true, true, P.tile);
  const int out_size = out_type == SCN_TYPE_FLOAT32 ? 4 : 2;
  P.out = out, P.out_type = out_type, P.aligned = aligned_to((uintptr_t)out, n, out_size), P.part_aligned = aligned_to(0, n, 4);
  const bool split = G.n_rows > P.chunk;
  if (split) SCN_TRY(scratch.get(&P.partial, sizeof(float) * (size_t)most_parts(G, P.chunk) * m * n));
  CUtensorMap a, b;
  SCN_TRY(make_map(&a, x, type, m, G.n_rows, parts, 1, 64, kStageRows));
  SCN_TRY(make_map(&b, dy, type, n, G.n_rows, parts, 1, 64, kStageRows));
  const long long most = (ceil_div(G.n_rows, P.chunk) + G.groups) * P.m_tiles * P.n_tiles;
#define SCN_TN(PARTS, SUMS)                                                                 \
  (tn == 64 ? launch<PARTS, 64, SUMS, true, true, false>(a, b, P, most, stream)             \
   : tn == 128 ? launch<PARTS, 128, SUMS, true, true, false>(a, b, P, most, stream)         \
               : launch<PARTS, (PARTS > 1) ? 128 : 256, SUMS, true, true, false>(a, b, P, most, stream))
  // Groups of more rows than an accumulator takes (kLong): a launch of their own, whose epilogue keeps 128 sums a lane.  With its
  // registers, short groups took 12% longer (65536 rows of 64 groups, 4096 -> 4096); a launch that finds none takes 4 us.
  const bool long_sums = parts == 1 && P.chunk > kLong * kStageRows;
  P.drain = parts > 1 ? kDrain : kLongDrain;
  if (long_sums) {
    P.pick = G.groups > 1 ? 2 : 0;
    SCN_TRY((pair ? launch_pair<true, true, true, false>(a, b, P, most, stream) : SCN_TN(1, true)));
    P.pick = 1;
  }
  if (!long_sums || G.groups > 1)
    SCN_TRY((pair ? launch_pair<false, true, true, false>(a, b, P, most, stream) : parts > 1 ? SCN_TN(3, true) : SCN_TN(1, false)));
  P.pick = 0;
#undef SCN_TN
  return split ? sum_parts(P, stream) : SCN_OK;
}

template <int PARTS, int TN, bool WEIGHTS, bool B_ROWS>
int launch_split(const CUtensorMap &b, const GroupParams &P, long long most_units, cudaStream_t stream) {
  constexpr size_t smem = kRing + 1024;
  static std::atomic<int> known[64];
  int dev = 0;
  SCN_CUDA_CHECK(cudaGetDevice(&dev));
  SCN_REQUIRE(dev >= 0 && dev < 64, SCN_ERR_UNSUPPORTED, "device index %d unsupported", dev);
  constexpr auto kernel = k_group_split<PARTS, TN, WEIGHTS, B_ROWS>;
  int blocks = known[dev].load();
  if (!blocks) {
    SCN_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    SCN_CUDA_CHECK(cudaDeviceGetAttribute(&blocks, cudaDevAttrMultiProcessorCount, dev));
    known[dev].store(blocks);
  }
  SCN_LAUNCH(kernel, (unsigned)std::min<long long>(blocks, most_units), kSplitThreads, smem, stream, b, P);
  SCN_CUDA_CHECK(cudaGetLastError());
  return SCN_OK;
}

int quads_of(const void *p, long long stride, int planes) { return (uintptr_t)p % 16 == 0 && stride % 4 == 0 && planes % 4 == 0; }

// rows_product of fp32 rows, split in the kernel: sums of at most kSplitSteps steps
bool splits_rows(int type, int k) { return type == SCN_TYPE_FLOAT32 && k <= kSplitSteps * kStageRows; }
int rows_product_split(const Groups &G, const void *x, long long stride, const Operand &w, bool b_rows, int parts, int k, int n, void *out,
                       int out_type, const void *bias, int bias_type, int drop, cudaStream_t stream) {
  const long long row_tiles = G.n_rows / kTileM + std::min<long long>(G.groups + 2, G.n_rows);
  const int tn = tile_columns(row_tiles, n, 128);
  GroupParams P{};
  P.offsets = G.offsets, P.off64 = G.off64, P.groups = G.groups, P.n_rows = (int)G.n_rows, P.flag = G.flag;
  P.tile = kTileM;
  P.k = k, P.n = n, P.n_tiles = (int)ceil_div(n, tn);
  P.idesc = idesc_of(SCN_TYPE_BFLOAT16, false, b_rows, kTileM);
  P.out = out, P.out_type = out_type, P.aligned = aligned_to((uintptr_t)out, n, out_type == SCN_TYPE_FLOAT32 ? 4 : 2);
  P.bias = bias, P.bias_type = bias_type, P.drop = drop;
  P.a = (const float *)x, P.a_stride = stride, P.a_quads = quads_of(x, stride, k);
  CUtensorMap b;
  SCN_TRY(b_rows ? make_map(&b, w, SCN_TYPE_BFLOAT16, n, k, G.groups, parts, 64, 64) : make_map(&b, w, SCN_TYPE_BFLOAT16, k, n, G.groups, parts, 64, tn));
  const long long most = row_tiles * P.n_tiles;
#define SCN_TN(PARTS, B_ROWS) (tn == 64 ? launch_split<PARTS, 64, false, B_ROWS>(b, P, most, stream) : launch_split<PARTS, 128, false, B_ROWS>(b, P, most, stream))
#define SCN_MAJOR(PARTS) (b_rows ? SCN_TN(PARTS, true) : SCN_TN(PARTS, false))
  return parts == 1 ? SCN_MAJOR(1) : parts == 2 ? SCN_MAJOR(2) : SCN_MAJOR(3);
#undef SCN_MAJOR
#undef SCN_TN
}

// weights_product of fp32 rows, split in the kernel, with the bias sums where they fit (*bias_done).  Its units are short, and 256
// rows of m + n values bring m n partial sums: at most a third as many, for 128 x 256.  (Parts in memory would be one and a half
// times the rows.)
bool splits_weights(int type, int m, int n) { return type == SCN_TYPE_FLOAT32 && m <= 128 && n <= 256; }
int weights_product_split(const Groups &G, const void *x, long long x_stride, const void *dy, long long dy_stride, int m, int n, void *out,
                          void *d_bias, bool *bias_done, Scratch &scratch, cudaStream_t stream) {
  const int tn = n <= 64 ? 64 : 128;
  GroupParams P{};
  P.offsets = G.offsets, P.off64 = G.off64, P.groups = G.groups, P.n_rows = (int)G.n_rows, P.flag = G.flag;
  P.tile = kTileM;
  *bias_done = d_bias && m % kTileM != 0;
  P.m = m, P.m_rows = m + *bias_done, P.n = n, P.m_tiles = (int)ceil_div(m, kTileM), P.n_tiles = (int)ceil_div(n, tn);
  P.chunk = kSplitSteps * kStageRows;
  P.idesc = idesc_of(SCN_TYPE_BFLOAT16, true, true, kTileM);
  P.out = out, P.out_type = SCN_TYPE_FLOAT32, P.aligned = aligned_to((uintptr_t)out, n, 4), P.part_aligned = aligned_to(0, n, 4);
  P.d_bias = *bias_done ? d_bias : nullptr;
  if (*bias_done) P.aligned = std::min(P.aligned, aligned_to((uintptr_t)d_bias, n, 4));
  P.a = (const float *)x, P.a_stride = x_stride, P.a_quads = quads_of(x, x_stride, m);
  P.b = (const float *)dy, P.b_stride = dy_stride, P.b_quads = quads_of(dy, dy_stride, n);
  const bool split = G.n_rows > P.chunk;
  if (split) SCN_TRY(scratch.get(&P.partial, sizeof(float) * (size_t)most_parts(G, P.chunk) * P.m_rows * n));
  const long long most = (ceil_div(G.n_rows, P.chunk) + G.groups) * P.m_tiles * P.n_tiles;
  const CUtensorMap none{};
  SCN_TRY((tn == 64 ? launch_split<3, 64, true, true>(none, P, most, stream) : launch_split<3, 128, true, true>(none, P, most, stream)));
  return split ? sum_parts(P, stream) : SCN_OK;
}

int bias_sums(const Groups &G, const void *dy, long long stride, int type, int n, void *out, int out_type, Scratch &scratch, cudaStream_t stream) {
  GroupParams P{};
  P.offsets = G.offsets, P.off64 = G.off64, P.groups = G.groups, P.n_rows = (int)G.n_rows, P.flag = G.flag;
  P.m = P.m_rows = 1, P.n = n, P.m_tiles = P.n_tiles = 1;
  P.chunk = chunk_of(G.n_rows, std::max<long long>(1, ceil_div(n, 32) / 4));
  P.out = out, P.out_type = out_type;
  const bool split = G.n_rows > P.chunk;
  if (split) SCN_TRY(scratch.get(&P.partial, sizeof(float) * (size_t)most_parts(G, P.chunk) * n));
  const long long units = ceil_div(G.n_rows, P.chunk) + G.groups;
  const dim3 grid((unsigned)ceil_div(n, 32), (unsigned)std::min<long long>(units, 1024));
  if (type == SCN_TYPE_FLOAT32)
    SCN_LAUNCH(k_group_bias<float>, grid, 256, 0, stream, P, (const float *)dy, stride);
  else if (type == SCN_TYPE_BFLOAT16)
    SCN_LAUNCH(k_group_bias<__nv_bfloat16>, grid, 256, 0, stream, P, (const __nv_bfloat16 *)dy, stride);
  else
    SCN_LAUNCH(k_group_bias<__half>, grid, 256, 0, stream, P, (const __half *)dy, stride);
  SCN_CUDA_CHECK(cudaGetLastError());
  return split ? sum_parts(P, stream) : SCN_OK;
}

int parts_of(int type, int precision) {
  return type != SCN_TYPE_FLOAT32 ? 1 : precision == SCN_PRECISION_FP32 ? 3 : precision == SCN_PRECISION_BF16 ? 1 : 2;
}
bool is_type(int t) { return t == SCN_TYPE_FLOAT32 || t == SCN_TYPE_BFLOAT16 || t == SCN_TYPE_FLOAT16; }

int check_sizes(const void *offsets, int64_t n_rows, int n_groups, int n_in, int n_out) {
  SCN_REQUIRE(n_rows >= 0 && n_in >= 1 && n_out >= 1, SCN_ERR_BAD_ARG, "grouped_product: bad sizes");
  SCN_REQUIRE(n_groups >= 1 && n_groups <= kMostGroups, SCN_ERR_UNSUPPORTED, "grouped_product: 1 to %d groups", kMostGroups);
  SCN_REQUIRE(n_rows < (1ll << 31) - 65536, SCN_ERR_UNSUPPORTED, "grouped_product: too many rows");
  SCN_REQUIRE(n_in <= (1 << 20) && n_out <= (1 << 20), SCN_ERR_UNSUPPORTED, "grouped_product: too many planes");
  SCN_REQUIRE(n_rows == 0 || offsets, SCN_ERR_BAD_ARG, "grouped_product: null argument");
  return SCN_OK;
}

}  // namespace

extern thread_local int g_drop_arrival;  // test hook (conv_tc.cu)

}  // namespace scn

using namespace scn;

extern "C" {

int scn_grouped_product_forward(const void *x, int64_t x_stride, int type, const void *weight, const void *bias, int bias_type,
                                const void *offsets, int offsets_64, int64_t n_rows, int n_groups, int n_in, int n_out, int precision,
                                void *out, int out_type, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  SCN_REQUIRE(is_type(type) && is_type(out_type) && (!bias || is_type(bias_type)), SCN_ERR_BAD_ARG, "grouped_product: unknown type");
  SCN_REQUIRE(precision >= SCN_PRECISION_FP32 && precision <= SCN_PRECISION_TF32X3, SCN_ERR_BAD_ARG, "grouped_product: unknown precision");
  SCN_TRY(check_sizes(offsets, n_rows, n_groups, n_in, n_out));
  if (n_rows == 0) return SCN_OK;
  SCN_REQUIRE(x && weight && out, SCN_ERR_BAD_ARG, "grouped_product: null argument");
  int *flag = nullptr;
  SCN_TRY(flag_of(&flag));
  SCN_TRY(look_at_flag(flag));
  const Groups G{offsets, offsets_64, n_rows, n_groups, flag};
  const int parts = parts_of(type, precision), held = type == SCN_TYPE_FLOAT32 ? SCN_TYPE_BFLOAT16 : type;
  const int drop = g_drop_arrival;
  g_drop_arrival = 0;
  Scratch scratch(stream);
  Operand a, b;
  SCN_TRY(operand(weight, n_out, n_out, (long long)n_groups * n_in, type, parts, scratch, stream, &b));
  b.matrix = b.stride * n_in;
  if (splits_rows(type, n_in)) return rows_product_split(G, x, x_stride, b, true, parts, n_in, n_out, out, out_type, bias, bias_type, drop, stream);
  SCN_TRY(operand(x, x_stride, n_in, n_rows, type, parts, scratch, stream, &a));
  return rows_product(G, a, b, true, parts, held, n_in, n_out, out, out_type, bias, bias_type, nullptr, nullptr, drop, stream);
}

int scn_grouped_product_backward(const void *x, int64_t x_stride, int type, const void *weight, const void *d_out, int64_t d_out_stride,
                                 const void *offsets, int offsets_64, int64_t n_rows, int n_groups, int n_in, int n_out, int precision,
                                 void *d_x, void *d_weight, void *d_bias, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  SCN_REQUIRE(is_type(type), SCN_ERR_BAD_ARG, "grouped_product: unknown type");
  SCN_REQUIRE(precision >= SCN_PRECISION_FP32 && precision <= SCN_PRECISION_TF32X3, SCN_ERR_BAD_ARG, "grouped_product: unknown precision");
  SCN_TRY(check_sizes(offsets, n_rows, n_groups, n_in, n_out));
  if (n_rows == 0) {
    const size_t size = type == SCN_TYPE_FLOAT32 ? 4 : 2;
    if (d_weight) SCN_CUDA_CHECK(cudaMemsetAsync(d_weight, 0, size * n_groups * n_in * n_out, stream));
    if (d_bias) SCN_CUDA_CHECK(cudaMemsetAsync(d_bias, 0, size * n_groups * n_out, stream));
    return SCN_OK;
  }
  SCN_REQUIRE(d_out && (!d_x || weight) && (!d_weight || x), SCN_ERR_BAD_ARG, "grouped_product: null argument");
  int *flag = nullptr;
  SCN_TRY(flag_of(&flag));
  SCN_TRY(look_at_flag(flag));
  const Groups G{offsets, offsets_64, n_rows, n_groups, flag};
  const int held = type == SCN_TYPE_FLOAT32 ? SCN_TYPE_BFLOAT16 : type;
  // the input's gradient at the precision asked for, the weights' always as fp32
  const int dx_parts = parts_of(type, precision), dw_parts = parts_of(type, SCN_PRECISION_FP32);
  Scratch scratch(stream);
  const bool split_x = d_x && splits_rows(type, n_out), split_w = d_weight && splits_weights(type, n_in, n_out);
  Operand dy;
  if ((d_x && !split_x) || (d_weight && !split_w))
    SCN_TRY(operand(d_out, d_out_stride, n_out, n_rows, type, d_weight && !split_w ? dw_parts : dx_parts, scratch, stream, &dy));
  if (d_x) {
    Operand w;
    SCN_TRY(operand(weight, n_out, n_out, (long long)n_groups * n_in, type, dx_parts, scratch, stream, &w));
    w.matrix = w.stride * n_in;
    SCN_TRY(split_x ? rows_product_split(G, d_out, d_out_stride, w, false, dx_parts, n_out, n_in, d_x, type, nullptr, 0, 0, stream)
                    : rows_product(G, dy, w, false, dx_parts, held, n_out, n_in, d_x, type, nullptr, 0, nullptr, nullptr, 0, stream));
  }
  bool bias_done = false;
  if (split_w) {
    SCN_TRY(weights_product_split(G, x, x_stride, d_out, d_out_stride, n_in, n_out, d_weight, d_bias, &bias_done, scratch, stream));
  } else if (d_weight) {
    Operand a;
    SCN_TRY(operand(x, x_stride, n_in, n_rows, type, dw_parts, scratch, stream, &a));
    SCN_TRY(weights_product(G, a, dy, dw_parts, held, n_in, n_out, d_weight, type, scratch, stream));
  }
  return d_bias && !bias_done ? bias_sums(G, d_out, d_out_stride, type, n_out, d_bias, type, scratch, stream) : SCN_OK;
}

int scn_grouped_product_quantized(const void *q, int64_t q_stride, const float *scale, const void *weight, const float *weight_scale,
                                  const void *bias, int bias_type, const void *offsets, int offsets_64, int64_t n_rows, int n_groups,
                                  int n_in, int n_out, void *out, int out_type, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  SCN_REQUIRE(is_type(out_type) && (!bias || is_type(bias_type)), SCN_ERR_BAD_ARG, "grouped_product: unknown type");
  SCN_TRY(check_sizes(offsets, n_rows, n_groups, n_in, n_out));
  if (n_rows == 0) return SCN_OK;
  SCN_REQUIRE(q && scale && weight && weight_scale && out, SCN_ERR_BAD_ARG, "grouped_product: null argument");
  int *flag = nullptr;
  SCN_TRY(flag_of(&flag));
  SCN_TRY(look_at_flag(flag));
  const Groups G{offsets, offsets_64, n_rows, n_groups, flag};
  Scratch scratch(stream);
  Operand a, b;
  SCN_TRY(operand(q, q_stride, n_in, n_rows, SCN_TYPE_E4M3, 1, scratch, stream, &a));
  SCN_TRY(operand(weight, n_in, n_in, (long long)n_groups * n_out, SCN_TYPE_E4M3, 1, scratch, stream, &b));
  b.matrix = b.stride * n_out;
  return rows_product(G, a, b, false, 1, SCN_TYPE_E4M3, n_in, n_out, out, out_type, bias, bias_type, scale, weight_scale, 0, stream);
}

int scn_rows_poll_errors(void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  int *flag = nullptr;
  SCN_TRY(flag_of(&flag));
  note_host_wait();
  SCN_CUDA_CHECK(cudaStreamSynchronize(stream));
  return look_at_flag(flag);
}

}  // extern "C"

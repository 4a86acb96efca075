// Root-mean-square norm of rows with the residual's addition in front of it, and its gradients.
//
//     s = round(x + r)     k = 1 / sqrt(mean(s s) + eps)     y = s k w        (r, w: may be absent)
//     8 bits:  a = max(max |y|, 1e-30)     scale = a / 448     q = e4m3(y * (448 / a))
//     backward, h = s k, t = dy w:   dx = dr = k (t - h mean(t h)) + ds     dw = sum over the rows of dy h
//
// s is rounded to the rows' type before the norm, so that forward and backward pass work on the values that are kept.
// All sums, the norm and the products are fp32; one rounding to the type of each result.
//
// Bound by HBM: every row is read once and written once.  16381 x 4096 bf16 with residual: forward 80 us (6.7 TB/s), backward 94
// (5.7); 267011 x 96 fp32: 63 us (6.6) and 70 (5.8); 32768 x 4096 bf16 to 8 bits 145 us (6.5 TB/s; a copy measures 6.55).  The
// backward pass is short of that by what its registers leave in flight (three operands and the weights' sums).  A row lies in the registers of `lanes` threads, 8 values (16 or 32
// bytes) to a chunk and 1 to 4 chunks to a thread: with fewer lanes a warp holds several rows and the sums need shuffles
// only, with more the warps of a row meet at one barrier per sum.  Blocks stay for the whole launch; a thread's weights are
// read once, and the next row is asked for before the present one is summed.
#include <algorithm>
#include <atomic>

#include "rows.cuh"

namespace scn {
namespace {

constexpr int kThreads = 256;
constexpr int kMostLanes = 512;  // of 4 chunks: rows of up to 16 384 planes in registers
constexpr float kSmallest = 1e-30f, kE4m3Most = 448.f;

struct NormParams {
  const void *x, *r;  // r: may be null
  const float *w;     // may be null
  void *sum, *out;    // sum: null without r
  float *scale, *inv_rms;
  long long n_rows, x_stride, r_stride;
  int planes, out_type, lanes;
  float eps;
};

struct NormBackParams {
  const void *s, *dy, *ds;  // ds: may be null
  const float *w, *inv_rms;
  void *dx;
  float *partial;  // [blocks][planes], null when the weights' gradient is not wanted
  long long n_rows, s_stride;
  int planes, dy_type, lanes;
};

// max(a, |b|); a NaN is above all numbers
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("{.reg .f32 t; abs.f32 t, %2; max.NaN.f32 %0, %1, t;}" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// `sum`, and with MAX `most`, over the `lanes` threads of a row.  `turn` alternates between two buffers, so that one barrier is
// enough.
template <bool MAX>
__device__ __forceinline__ void over_row(float &sum, float &most, int lanes, float2 *shared, int &turn) {
  const unsigned full = 0xffffffffu;
  const int within = lanes < 32 ? lanes : 32;
  for (int d = within >> 1; d; d >>= 1) {
    sum += __shfl_xor_sync(full, sum, d);
    if (MAX) most = larger(most, __shfl_xor_sync(full, most, d));
  }
  if (lanes <= 32) return;
  float2 *buf = shared + (turn ^= 1) * (kMostLanes / 32);
  const int warp = threadIdx.x / 32, per_row = lanes / 32;
  if (threadIdx.x % 32 == 0) buf[warp] = make_float2(sum, most);
  __syncthreads();
  const float2 *mine = buf + warp / per_row * per_row;
  sum = mine[0].x, most = mine[0].y;
  for (int i = 1; i < per_row; ++i) {
    const float2 v = mine[i];
    sum += v.x;
    if (MAX) most = larger(most, v.y);
  }
}

template <int V, bool QUANT>
__device__ __forceinline__ void store_out(void *out, int type, long long row, int planes, int chunk, int lanes, int lane, const float (&y)[8]) {
  const long long at = row * planes;
  if (QUANT) {
    store8_e4m3<V>((unsigned char *)out + at, planes, chunk, lanes, lane, y);
  } else if (type == SCN_TYPE_BFLOAT16) {
    unsigned w[4];
    pack8(y, w, __nv_bfloat16());
    store8<__nv_bfloat16, V>((__nv_bfloat16 *)out + at, planes, chunk, lanes, lane, w);
  } else if (type == SCN_TYPE_FLOAT32) {
    unsigned w[8];
    pack8(y, w, 0.f);
    store8<float, V>((float *)out + at, planes, chunk, lanes, lane, w);
  } else {
    unsigned w[4];
    pack8(y, w, __half());
    store8<__half, V>((__half *)out + at, planes, chunk, lanes, lane, w);
  }
}

template <int V>
__device__ __forceinline__ void load_weights(const float *w, int planes, int chunk, int lanes, int lane, float (&v)[8]) {
  if (V == 8) {
    const int c = place<8>(chunk, 0, lanes, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = w || c >= planes ? 0.f : 1.f;
    if (w && c < planes) {
      const float4 p = __ldg((const float4 *)(w + c)), q = __ldg((const float4 *)(w + c) + 1);
      v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8 / V; ++j) {
    const int c = place<V>(chunk, j, lanes, lane);
#pragma unroll
    for (int i = 0; i < V; ++i) v[j * V + i] = c < planes ? (w ? __ldg(w + c + i) : 1.f) : 0.f;
  }
}

template <typename T, int V, int CH, bool QUANT>
__global__ void __launch_bounds__(kMostLanes)
k_rms_norm(const NormParams P) {
  SCN_GRID_WAIT();
  __shared__ float2 shared[2 * (kMostLanes / 32)];
  const int lanes = P.lanes, lane = threadIdx.x % lanes, per_block = blockDim.x / lanes;
  const long long step = (long long)gridDim.x * per_block;
  long long row = (long long)blockIdx.x * per_block + threadIdx.x / lanes;
  int turn = 0;
  float w[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) load_weights<V>(P.w, P.planes, i, lanes, lane, w[i]);
  unsigned x[CH][Words<T>::N], r[CH][Words<T>::N];
  auto ask = [&](long long at) {
    const int n = at < P.n_rows ? P.planes : 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      load8<T, V>((const T *)P.x + at * P.x_stride, n, i, lanes, lane, x[i]);
      if (P.r) load8<T, V>((const T *)P.r + at * P.r_stride, n, i, lanes, lane, r[i]);
    }
  };
  ask(row);
  for (long long first = (long long)blockIdx.x * per_block; first < P.n_rows; first += step, row += step) {
    const bool real = row < P.n_rows;
    float s[CH][8], squares = 0.f, most = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      unpack8(x[i], s[i], T());
      if (P.r) {
        float v[8];
        unpack8(r[i], v, T());
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += s[i][j];
        unsigned sw[Words<T>::N];
        pack8(v, sw, T());
        unpack8(sw, s[i], T());
        if (real) store8<T, V>((T *)P.sum + row * P.planes, P.planes, i, lanes, lane, sw);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        squares = fmaf(s[i][j], s[i][j], squares);
        s[i][j] *= w[i][j];
        if (QUANT) most = larger(most, s[i][j]);
      }
    }
    ask(row + step);
    over_row<QUANT>(squares, most, lanes, shared, turn);
    float k = __frsqrt_rn(squares / (float)P.planes + P.eps);
    if (P.inv_rms && lane == 0 && real) P.inv_rms[row] = k;
    if (QUANT) {  // the largest |s w| k is the largest |y|: one pass over the row for both sums
      most = larger(kSmallest, most * k);
      if (lane == 0 && real) P.scale[row] = most / kE4m3Most;
    }
    const float per = QUANT ? kE4m3Most / most : 1.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = s[i][j] * k * per;
    if (real) {
#pragma unroll
      for (int i = 0; i < CH; ++i) store_out<V, QUANT>(P.out, P.out_type, row, P.planes, i, lanes, lane, s[i]);
    }
  }
}

template <int V>
__device__ __forceinline__ void load_any(const void *p, int type, long long row, int planes, int n, int chunk, int lanes, int lane, float (&v)[8]) {
  const long long at = row * planes;
  if (type == SCN_TYPE_BFLOAT16) {
    unsigned w[4];
    load8<__nv_bfloat16, V>((const __nv_bfloat16 *)p + at, n, chunk, lanes, lane, w);
    unpack8(w, v, __nv_bfloat16());
  } else if (type == SCN_TYPE_FLOAT32) {
    unsigned w[8];
    load8<float, V>((const float *)p + at, n, chunk, lanes, lane, w);
    unpack8(w, v, 0.f);
  } else {
    unsigned w[4];
    load8<__half, V>((const __half *)p + at, n, chunk, lanes, lane, w);
    unpack8(w, v, __half());
  }
}

// The weights' gradient: a thread keeps the sums of its planes over all rows of its block, the rows' groups of a block are
// added in shared memory, the blocks' sums by k_add_blocks: a fixed order.
template <typename T, int V, int CH, bool SAME>
__global__ void __launch_bounds__(kMostLanes)
k_rms_norm_back(const NormBackParams P) {
  SCN_GRID_WAIT();
  __shared__ float2 shared[2 * (kMostLanes / 32)];
  extern __shared__ float sums[];  // [rows of a block][planes]
  const int lanes = P.lanes, lane = threadIdx.x % lanes, per_block = blockDim.x / lanes;
  const long long step = (long long)gridDim.x * per_block;
  long long row = (long long)blockIdx.x * per_block + threadIdx.x / lanes;
  int turn = 0;
  float dw[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  // the next row on its way (a gradient of another type than the rows' is read when it is needed)
  unsigned sw[CH][Words<T>::N], dyw[CH][Words<T>::N], dsw[CH][Words<T>::N];
  float k_next = 0.f;
  auto ask = [&](long long at) {
    const int n = at < P.n_rows ? P.planes : 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      load8<T, V>((const T *)P.s + at * P.s_stride, n, i, lanes, lane, sw[i]);
      if (SAME) load8<T, V>((const T *)P.dy + at * P.planes, n, i, lanes, lane, dyw[i]);
      if (P.ds) load8<T, V>((const T *)P.ds + at * P.planes, n, i, lanes, lane, dsw[i]);
    }
    k_next = n ? __ldg(P.inv_rms + at) : 0.f;
  };
  ask(row);
  for (long long first = (long long)blockIdx.x * per_block; first < P.n_rows; first += step, row += step) {
    const bool real = row < P.n_rows;
    const float k = k_next;
    float h[CH][8], d[CH][8], o[CH][8], along = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float w[8];
      load_weights<V>(P.w, P.planes, i, lanes, lane, w);
      unpack8(sw[i], h[i], T());
      if (SAME)
        unpack8(dyw[i], d[i], T());
      else
        load_any<V>(P.dy, P.dy_type, row, P.planes, real ? P.planes : 0, i, lanes, lane, d[i]);
      if (P.ds) unpack8(dsw[i], o[i], T());
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] *= k;
        dw[i][j] = fmaf(d[i][j], h[i][j], dw[i][j]);
        d[i][j] *= w[j];
        along = fmaf(d[i][j], h[i][j], along);
      }
    }
    ask(row + step);
    over_row<false>(along, none, lanes, shared, turn);
    along /= (float)P.planes;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] = k * (d[i][j] - h[i][j] * along);
        if (P.ds) h[i][j] += o[i][j];
      }
      unsigned q[Words<T>::N];
      pack8(h[i], q, T());
      if (real) store8<T, V>((T *)P.dx + row * P.planes, P.planes, i, lanes, lane, q);
    }
  }
  if (!P.partial) return;
  float *mine = sums + (size_t)(threadIdx.x / lanes) * P.planes;
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) {
      const int c = place<V>(i, j, lanes, lane);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c < P.planes) mine[c + e] = dw[i][j * V + e];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < P.planes; c += blockDim.x) {
    float v = 0.f;
    for (int g = 0; g < per_block; ++g) v += sums[(size_t)g * P.planes + c];
    P.partial[(long long)blockIdx.x * P.planes + c] = v;
  }
}

// out[c] = sum of partial[b][c] over b, in a fixed order: 32 columns to a block, 8 or 32 threads along b
__global__ void __launch_bounds__(1024)
k_add_blocks(const float *__restrict__ partial, long long blocks, int planes, float *__restrict__ out) {
  SCN_GRID_WAIT();
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < planes)
    for (long long b = threadIdx.y; b < blocks; b += blockDim.y) v += __ldg(partial + b * planes + c);
  part[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < planes) {
    for (int i = 1; i < (int)blockDim.y; ++i) v += part[i][threadIdx.x];
    out[c] = v;
  }
}

// Rows of more planes than the registers of a block hold: the row is read again for every sum (from L2).
__device__ __forceinline__ float any_value(const void *p, int type, long long at) {
  return type == SCN_TYPE_FLOAT32 ? ((const float *)p)[at]
         : type == SCN_TYPE_BFLOAT16 ? __bfloat162float(((const __nv_bfloat16 *)p)[at])
                                     : __half2float(((const __half *)p)[at]);
}
__device__ __forceinline__ void store_value(void *p, int type, long long at, float v) {
  if (type == SCN_TYPE_FLOAT32)
    ((float *)p)[at] = v;
  else if (type == SCN_TYPE_BFLOAT16)
    ((__nv_bfloat16 *)p)[at] = __float2bfloat16_rn(v);
  else if (type == SCN_TYPE_FLOAT16)
    ((__half *)p)[at] = __float2half_rn(v);
  else
    ((unsigned char *)p)[at] = (unsigned char)e4m3_pair(v, 0.f);
}
__device__ __forceinline__ float rounded(float v, int type) {
  return type == SCN_TYPE_FLOAT32 ? v
         : type == SCN_TYPE_BFLOAT16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}

__global__ void __launch_bounds__(kMostLanes)
k_rms_norm_long(const NormParams P, int type) {
  SCN_GRID_WAIT();
  __shared__ float2 shared[2 * (kMostLanes / 32)];
  int turn = 0;
  for (long long row = blockIdx.x; row < P.n_rows; row += gridDim.x) {
    auto value = [&](int c) {
      const float v = any_value(P.x, type, row * P.x_stride + c);
      return P.r ? rounded(v + any_value(P.r, type, row * P.r_stride + c), type) : v;
    };
    float squares = 0.f, most = 0.f;
    for (int c = threadIdx.x; c < P.planes; c += kMostLanes) {
      const float s = value(c);
      squares = fmaf(s, s, squares);
      most = larger(most, s * (P.w ? __ldg(P.w + c) : 1.f));
    }
    over_row<true>(squares, most, kMostLanes, shared, turn);
    const float k = __frsqrt_rn(squares / (float)P.planes + P.eps);
    if (P.inv_rms && threadIdx.x == 0) P.inv_rms[row] = k;
    float per = 1.f;
    if (P.out_type == SCN_TYPE_E4M3) {
      most = larger(kSmallest, most * k);
      if (threadIdx.x == 0) P.scale[row] = most / kE4m3Most;
      per = kE4m3Most / most;
    }
    for (int c = threadIdx.x; c < P.planes; c += kMostLanes) {
      const float s = value(c);
      if (P.r) store_value(P.sum, type, row * P.planes + c, s);
      store_value(P.out, P.out_type, row * P.planes + c, s * (P.w ? __ldg(P.w + c) : 1.f) * k * per);
    }
  }
}

__global__ void __launch_bounds__(kMostLanes)
k_rms_norm_back_long(const NormBackParams P, int type) {
  SCN_GRID_WAIT();
  __shared__ float2 shared[2 * (kMostLanes / 32)];
  int turn = 0;
  for (long long row = blockIdx.x; row < P.n_rows; row += gridDim.x) {
    const float k = __ldg(P.inv_rms + row);
    float along = 0.f;
    for (int c = threadIdx.x; c < P.planes; c += kMostLanes)
      along = fmaf(any_value(P.dy, P.dy_type, row * P.planes + c) * (P.w ? __ldg(P.w + c) : 1.f),
                   any_value(P.s, type, row * P.s_stride + c) * k, along);
    float none = 0.f;
    over_row<false>(along, none, kMostLanes, shared, turn);
    along /= (float)P.planes;
    for (int c = threadIdx.x; c < P.planes; c += kMostLanes) {
      const float t = any_value(P.dy, P.dy_type, row * P.planes + c) * (P.w ? __ldg(P.w + c) : 1.f);
      float v = k * (t - any_value(P.s, type, row * P.s_stride + c) * k * along);
      if (P.ds) v += any_value(P.ds, type, row * P.planes + c);
      store_value(P.dx, type, row * P.planes + c, v);
    }
  }
}

// partial[y][c]: the weights' gradient over every gridDim.y-th row, a thread per plane
__global__ void __launch_bounds__(kThreads)
k_rms_norm_weights_long(const NormBackParams P, int type) {
  SCN_GRID_WAIT();
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= P.planes) return;
  float v = 0.f;
  for (long long row = blockIdx.y; row < P.n_rows; row += gridDim.y)
    v = fmaf(any_value(P.dy, P.dy_type, row * P.planes + c), any_value(P.s, type, row * P.s_stride + c) * __ldg(P.inv_rms + row), v);
  P.partial[(long long)blockIdx.y * P.planes + c] = v;
}

// How a row lies in registers: `lanes` threads of `chunks` times 8 values with the fewest places left over, and among equals
// by what measured best (GB/s of 6548, forward 16384 x 4096 bf16: 4 chunks 6230, 2 5520, 1 5490; in 8 bits 6230, 5190, 4450; of
// 400000 x 32: 4700, 5510, 6010; 8192 x 4096 fp32: 2 chunks 5810, 1 5620, 4 5600; backward 16384 x 4096 bf16: 2 chunks 4180, 1
// 3250, 4 2000 (spills); 8192 x 4096 fp32: 1 chunk 5960, 2 5310; 267011 x 96
// fp32: 1 chunk 5860, 3 4180).  Rows of a few chunks are spread, so that a warp's loads are
// dense; long rows are held by as few threads as their registers allow, because each row costs all its threads a barrier.
bool shape_of(int planes, int type, bool backward, int *lanes, int *chunks) {
  const int need = (int)ceil_div(planes, 8);
  const bool wide = type == SCN_TYPE_FLOAT32;
  static const int orders[5][4] = {{1, 2, 3, 4}, {2, 1, 3, 4}, {4, 3, 2, 1}, {1, 2, 3, 4}, {2, 1, 3, 4}};
  const int *order = orders[backward ? (wide ? 3 : 4) : need <= 8 ? 0 : wide ? 1 : 2];
  int best = 0;
  for (int i = 0; i < 4; ++i) {
    if (backward && best && i == 2) break;  // 3 and 4 chunks spill there: rows of over 8192 planes only
    const int ch = order[i], l = (int)next_pow2((unsigned long long)ceil_div(need, ch));
    if (l > kMostLanes) continue;
    if (!best || l * ch < best) best = l * ch, *lanes = l, *chunks = ch;
  }
  return best > 0;
}

bool is_type(int t) { return t == SCN_TYPE_FLOAT32 || t == SCN_TYPE_BFLOAT16 || t == SCN_TYPE_FLOAT16; }
int size_of(int t) { return t == SCN_TYPE_FLOAT32 ? 4 : t == SCN_TYPE_E4M3 ? 1 : 2; }

// Values per vector: the widest that every address of every row allows.
struct Vectors {
  int v = 8;
  void add(const void *p, int type, long long stride, int planes) {
    if (!p) return;
    const int size = size_of(type);
    auto fits = [&](int n) {
      const uintptr_t bytes = (uintptr_t)(n * size);
      return (uintptr_t)p % bytes == 0 && (uintptr_t)(stride * size) % bytes == 0 && planes % n == 0;
    };
    if (v == 8 && !fits(8)) v = 2;
    if (v == 2 && !fits(2)) v = 1;
  }
};

template <typename T, int V>
int launch_forward(const NormParams &P, int chunks, cudaStream_t stream) {
  const int threads = std::max(kThreads, P.lanes);
  const long long need = ceil_div(P.n_rows, threads / P.lanes);
#define SCN_NORM(CH, Q)                                                                                       \
  case CH * 2 + Q: {                                                                                          \
    int most = 0;                                                                                             \
    SCN_TRY((resident_blocks<k_rms_norm<T, V, CH, Q>>(threads, 0, &most)));                                   \
    SCN_LAUNCH((k_rms_norm<T, V, CH, Q>), (unsigned)std::min<long long>(need, most), threads, 0, stream, P);  \
    break;                                                                                                    \
  }
  switch (chunks * 2 + (P.out_type == SCN_TYPE_E4M3)) {
    SCN_NORM(1, false) SCN_NORM(2, false) SCN_NORM(3, false) SCN_NORM(4, false)
    SCN_NORM(1, true) SCN_NORM(2, true) SCN_NORM(3, true) SCN_NORM(4, true)
  }
#undef SCN_NORM
  SCN_CUDA_CHECK(cudaGetLastError());
  return SCN_OK;
}

int add_blocks(const float *partial, long long blocks, int planes, float *out, cudaStream_t stream) {
  SCN_LAUNCH(k_add_blocks, (unsigned)ceil_div(planes, 32), dim3(32, blocks > 64 ? 32 : 8), 0, stream, partial, blocks, planes, out);
  SCN_CUDA_CHECK(cudaGetLastError());
  return SCN_OK;
}

// The shared memory that a block of `kernel` may have, for its weights' sums at most.  (Without it a block has 48 KB, what the
// kernel declares by itself included.)  It belongs to the kernel, not to a call:
// set once per device, so that two threads' calls of different widths do not take each other's away.
template <auto kernel>
int allow_shared() {
  static std::atomic<bool> configured[64];
  int dev = 0;
  SCN_CUDA_CHECK(cudaGetDevice(&dev));
  SCN_REQUIRE(dev >= 0 && dev < 64, SCN_ERR_UNSUPPORTED, "device index %d unsupported", dev);
  if (!configured[dev].load()) {
    SCN_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(float) * kMostLanes * 4 * 8)));
    configured[dev].store(true);
  }
  return SCN_OK;
}

template <typename T, int V, bool SAME>
int launch_back(NormBackParams P, int chunks, float *d_weight, cudaStream_t stream) {
  const int threads = std::max(kThreads, P.lanes);
  const long long need = ceil_div(P.n_rows, threads / P.lanes);
  const size_t smem = d_weight ? sizeof(float) * (size_t)(threads / P.lanes) * P.planes : 0;
  Scratch scratch(stream);
  long long blocks = 0;
#define SCN_NORM(CH)                                                                                           \
  case CH: {                                                                                                   \
    int most = 0;                                                                                              \
    if (smem > 32 * 1024) SCN_TRY((allow_shared<k_rms_norm_back<T, V, CH, SAME>>()));                          \
    SCN_TRY((resident_blocks<k_rms_norm_back<T, V, CH, SAME>>(threads, 0, &most)));                                  \
    blocks = std::min<long long>(need, most);                                                                  \
    if (d_weight) SCN_TRY(scratch.get(&P.partial, sizeof(float) * (size_t)blocks * P.planes));                 \
    SCN_LAUNCH((k_rms_norm_back<T, V, CH, SAME>), (unsigned)blocks, threads, smem, stream, P);                       \
    break;                                                                                                     \
  }
  switch (chunks) {
    SCN_NORM(1) SCN_NORM(2) SCN_NORM(3) SCN_NORM(4)
  }
#undef SCN_NORM
  SCN_CUDA_CHECK(cudaGetLastError());
  return d_weight ? add_blocks(P.partial, blocks, P.planes, d_weight, stream) : SCN_OK;
}

// (a gradient of another type than the rows' takes the form for any alignment)
template <typename T, int V>
int launch_backward(const NormBackParams &P, int chunks, float *d_weight, bool same, cudaStream_t stream) {
  return same ? launch_back<T, V, true>(P, chunks, d_weight, stream) : launch_back<T, 1, false>(P, chunks, d_weight, stream);
}

#define SCN_BY_TYPE(call, type, v, ...)                                                                        \
  (type == SCN_TYPE_FLOAT32                                                                                    \
       ? (v == 8 ? call<float, 8>(__VA_ARGS__) : v == 2 ? call<float, 2>(__VA_ARGS__) : call<float, 1>(__VA_ARGS__)) \
   : type == SCN_TYPE_BFLOAT16                                                                                 \
       ? (v == 8   ? call<__nv_bfloat16, 8>(__VA_ARGS__)                                                       \
          : v == 2 ? call<__nv_bfloat16, 2>(__VA_ARGS__)                                                       \
                   : call<__nv_bfloat16, 1>(__VA_ARGS__))                                                      \
       : (v == 8 ? call<__half, 8>(__VA_ARGS__) : v == 2 ? call<__half, 2>(__VA_ARGS__) : call<__half, 1>(__VA_ARGS__)))

}  // namespace
}  // namespace scn

using namespace scn;

extern "C" {

int scn_rms_norm_forward(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, int type,
                         const float *weight, int64_t n_rows, int n_planes, double eps, void *sum, void *out, int out_type,
                         float *scale, float *inv_rms, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  SCN_REQUIRE(is_type(type) && (is_type(out_type) || out_type == SCN_TYPE_E4M3), SCN_ERR_BAD_ARG, "rms_norm: unknown type");
  SCN_REQUIRE(n_rows >= 0 && n_planes >= 1, SCN_ERR_BAD_ARG, "rms_norm: bad sizes");
  SCN_REQUIRE(eps >= 0, SCN_ERR_BAD_ARG, "rms_norm: eps must not be negative");
  if (n_rows == 0) return SCN_OK;
  SCN_REQUIRE(x && out, SCN_ERR_BAD_ARG, "rms_norm: null argument");
  SCN_REQUIRE((residual != nullptr) == (sum != nullptr), SCN_ERR_BAD_ARG, "rms_norm: the sum is written with a residual, and only then");
  SCN_REQUIRE((out_type == SCN_TYPE_E4M3) == (scale != nullptr), SCN_ERR_BAD_ARG, "rms_norm: scales belong to 8-bit results");
  NormParams P{x, residual, weight, sum, out, scale, inv_rms, n_rows, x_stride, residual_stride, n_planes, out_type, 0, (float)eps};
  int chunks = 0;
  if (!shape_of(n_planes, type, false, &P.lanes, &chunks)) {
    int most = 0;
    SCN_TRY(resident_blocks<k_rms_norm_long>(kMostLanes, 0, &most));
    SCN_LAUNCH(k_rms_norm_long, (unsigned)std::min<long long>(n_rows, most), kMostLanes, 0, stream, P, type);
    SCN_CUDA_CHECK(cudaGetLastError());
    return SCN_OK;
  }
  Vectors vec;
  vec.add(x, type, x_stride, n_planes);
  vec.add(residual, type, residual_stride, n_planes);
  vec.add(sum, type, n_planes, n_planes);
  vec.add(out, out_type, n_planes, n_planes);
  vec.add(weight, SCN_TYPE_FLOAT32, n_planes, n_planes);
  return SCN_BY_TYPE(launch_forward, type, vec.v, P, chunks, stream);
}

int scn_rms_norm_backward(const void *s, int64_t s_stride, int type, const float *weight, const float *inv_rms, const void *d_out,
                          int d_out_type, const void *d_sum, int64_t n_rows, int n_planes, void *d_x, float *d_weight,
                          void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  SCN_REQUIRE(is_type(type) && is_type(d_out_type), SCN_ERR_BAD_ARG, "rms_norm: unknown type");
  SCN_REQUIRE(n_rows >= 0 && n_planes >= 1, SCN_ERR_BAD_ARG, "rms_norm: bad sizes");
  if (n_rows == 0) {
    if (d_weight) SCN_CUDA_CHECK(cudaMemsetAsync(d_weight, 0, sizeof(float) * (size_t)n_planes, stream));
    return SCN_OK;
  }
  SCN_REQUIRE(s && inv_rms && d_out && d_x, SCN_ERR_BAD_ARG, "rms_norm: null argument");
  NormBackParams P{s, d_out, d_sum, weight, inv_rms, d_x, nullptr, n_rows, s_stride, n_planes, d_out_type, 0};
  int chunks = 0;
  if (!shape_of(n_planes, type, true, &P.lanes, &chunks)) {
    int most = 0;
    SCN_TRY(resident_blocks<k_rms_norm_back_long>(kMostLanes, 0, &most));
    SCN_LAUNCH(k_rms_norm_back_long, (unsigned)std::min<long long>(n_rows, most), kMostLanes, 0, stream, P, type);
    SCN_CUDA_CHECK(cudaGetLastError());
    if (!d_weight) return SCN_OK;
    Scratch scratch(stream);
    const unsigned across = (unsigned)std::min<long long>(n_rows, 32);
    SCN_TRY(scratch.get(&P.partial, sizeof(float) * (size_t)across * n_planes));
    SCN_LAUNCH(k_rms_norm_weights_long, dim3((unsigned)ceil_div(n_planes, kThreads), across), kThreads, 0, stream, P, type);
    SCN_CUDA_CHECK(cudaGetLastError());
    return add_blocks(P.partial, across, n_planes, d_weight, stream);
  }
  Vectors vec;
  vec.add(s, type, s_stride, n_planes);
  vec.add(d_out, d_out_type, n_planes, n_planes);
  vec.add(d_sum, type, n_planes, n_planes);
  vec.add(d_x, type, n_planes, n_planes);
  vec.add(weight, SCN_TYPE_FLOAT32, n_planes, n_planes);
  return SCN_BY_TYPE(launch_backward, type, vec.v, P, chunks, d_weight, type == d_out_type, stream);
}

}  // extern "C"

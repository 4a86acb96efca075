// One step of AdamW over all tensors of a list, with moments in 32 bits or in 8.
//
//     t = steps done + 1     m = b1 m + (1 - b1) g     v = b2 v + (1 - b2) g g
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: m and r = sqrt(v) as e4m3 with one scale for 256 values (the block's largest / 448); r rather than v, because its
// range is half as wide in powers of two.  A decay of 0.1% is far below half a step of 8 bits, so rounding to nearest would
// leave a moment where it is for good: it is rounded up or down by chance, in proportion to the distance, which keeps its
// mean.  The bits come from a hash of seed, step and position: the same call gives the same bits.  A positive r is never
// rounded to zero (its value would be divided by eps then).  The step itself uses m and r as computed, in fp32.
//
// Bound by HBM: 28 bytes for a value in 32 bits, 16 in 8 (fp32 parameters and gradients).  17 M values in 119 tensors: 73 us in
// 32 bits (6.6 TB/s, what a copy measures), 66 in 8 (4.2 TB/s): there the 80-odd instructions a value, a fifth of them the
// hash, fill two thirds of the issue slots (the bytes alone take 42 us).  The list's pointers travel as
// kernel arguments (no copy to the device, nothing to keep alive for a graph).  A warp takes whole blocks of 256 values, 8 to
// a lane, and looks for a block's tensor from the one before on; a block's maximum is one reduction over the warp.
// The count of steps lives on the device, so that a replayed graph counts on: the last block to end adds one to it, and
// which block that is, is counted in the upper bits of the same word.
#include <math.h>

#include <algorithm>

#include "rows.cuh"

namespace scn {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kBlock = 256;  // values of a block
constexpr int kTicketShift = 40;
constexpr float kSmallest = 1e-30f, kE4m3Most = 448.f, kE4m3Least = 1.f / 512.f;

struct Entry {
  void *p, *m, *v, *copy;
  const void *g;
  float *m_scale, *v_scale;
  long long n, first;  // values; number of the tensor's first block in the list (lowest bit of `aligned` apart)
};
template <int CAP>
struct Table {
  Entry e[CAP];
};
struct Step {
  unsigned long long *word;  // steps done; blocks that have ended above bit 40
  const float *lr_dev;       // may be null
  double log_b1, log_b2;
  float lr, b1, b2, one_minus_b1, one_minus_b2, eps, wd, one;
  unsigned seed;
  int grad_type, copy_type;  // copy_type -1: none
  int count;                 // tensors of this launch
  int last;                  // of the list's launches: counts the step
  long long first, blocks;   // this launch's blocks of the list
};

__device__ __forceinline__ unsigned mixed(unsigned v) {  // the 32-bit finaliser of MurmurHash3
  v = (v ^ (v >> 16)) * 0x85EBCA6Bu;
  v = (v ^ (v >> 13)) * 0xC2B2AE35u;
  return v ^ (v >> 16);
}

// Two floats in a pair of registers: the FMA pipe takes both in one instruction.
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ void apart(Two t, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v)); }
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two add2_down(Two a, Two b) {
  Two r;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// The 16 bits of two hashes, lower or upper halves, as numbers 0 .. 65535
template <bool UPPER>
__device__ __forceinline__ Two chances(unsigned a, unsigned b) {  // (2^23 + bits) - 2^23
  const unsigned pick = UPPER ? 0x7632u : 0x7610u;
  return two(__uint_as_float(__byte_perm(a, 0x4B000000u, pick)), __uint_as_float(__byte_perm(b, 0x4B000000u, pick))) + two(-8388608.f);
}

// |y| <= 448 (and what rounding adds) to the multiples of their binades' steps below |y| + chance / 65536 steps: one of the two
// neighbours among the values of e4m3.  The addition of 2^23 steps, rounded down, drops what lies below a step.
__device__ __forceinline__ Two to_neighbours(float a, float b, Two chance) {
  const float ea = fmaxf(__uint_as_float(__float_as_uint(a) & 0x7F800000u), 0x1p-6f), eb = fmaxf(__uint_as_float(__float_as_uint(b) & 0x7F800000u), 0x1p-6f);
  const Two e = two(ea, eb), steps = e * two(0x1p20f);
  const Two sum = fma2(chance, e * two(0x1p-19f), two(fabsf(a), fabsf(b)));
  return add2_down(sum, steps) + steps * two(-1.f);
}

__device__ __forceinline__ float larger(float a, float b) {  // max(a, |b|); a NaN is above all numbers
  float r;
  asm("{.reg .f32 t; abs.f32 t, %2; max.NaN.f32 %0, %1, t;}" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float largest(float v) {  // over the warp, v >= 0 or NaN
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

__device__ __forceinline__ void from_e4m3(const uint2 q, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((i < 2 ? q.x : q.y) >> (i % 2 * 16)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    apart(two(f.x, f.y) * two(scale), v[2 * i], v[2 * i + 1]);
  }
}

template <typename T>
__device__ __forceinline__ float one(const void *p, long long i);
template <>
__device__ __forceinline__ float one<float>(const void *p, long long i) { return ((const float *)p)[i]; }
template <>
__device__ __forceinline__ float one<__nv_bfloat16>(const void *p, long long i) { return __bfloat162float(((const __nv_bfloat16 *)p)[i]); }
template <>
__device__ __forceinline__ float one<__half>(const void *p, long long i) { return __half2float(((const __half *)p)[i]); }
__device__ __forceinline__ void put(float *p, long long i, float v) { p[i] = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, long long i, float v) { p[i] = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half *p, long long i, float v) { p[i] = __float2half_rn(v); }

// The values at + 32 j that lie below n; 8 values from `at` on (vectors) where a block is whole
template <typename T>
__device__ __forceinline__ void get8(const void *p, long long at, long long n, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = at + 32 * j < n ? one<T>(p, at + 32 * j) : 0.f;
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void put8(void *p, long long at, long long n, const float (&v)[8]) {
  if (WHOLE) {
    unsigned w[Words<T>::N];
    pack8(v, w, T());
    store_words((T *)p + at, w);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + 32 * j < n) put((T *)p, at + 32 * j, v[j]);
  }
}
__device__ __forceinline__ void get8_e4m3(const void *p, long long at, long long n, float scale, float (&v)[8]) {
  const unsigned char *b = (const unsigned char *)p;
  unsigned c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = at + 32 * j < n ? b[at + 32 * j] : 0u;
  from_e4m3(make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24), scale, v);
}
template <bool WHOLE>
__device__ __forceinline__ void put8_e4m3(void *p, long long at, long long n, const float (&v)[8]) {
  unsigned char *b = (unsigned char *)p;
  const uint2 q = make_uint2(e4m3_pair(v[0], v[1]) | e4m3_pair(v[2], v[3]) << 16, e4m3_pair(v[4], v[5]) | e4m3_pair(v[6], v[7]) << 16);
  if (WHOLE) {
    __stcs(reinterpret_cast<uint2 *>(b + at), q);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + 32 * j < n) b[at + 32 * j] = (unsigned char)((j < 4 ? q.x : q.y) >> (j % 4 * 8));
  }
}

// What a warp reads of a block: asked for one block ahead where the block is whole (lane l has values 8 l to 8 l + 7).
template <typename P, int BITS>
struct Ahead {
  unsigned p[Words<P>::N], g[8], m[BITS == 8 ? 2 : 8], v[BITS == 8 ? 2 : 8];
  float m_scale, v_scale;
  __device__ __forceinline__ void ask(const Entry &E, const Step &A, long long at, int lane) {
    const long long first = at * kBlock + lane * 8;
    load_words((const P *)E.p + first, p);
    if (A.grad_type == SCN_TYPE_FLOAT32) {
      load_words((const float *)E.g + first, g);
    } else {
      unsigned w[4];
      load_words((const unsigned short *)E.g + first, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = w[i];
    }
    if constexpr (BITS == 8) {
      load_words((const unsigned char *)E.m + first, m);
      load_words((const unsigned char *)E.v + first, v);
      m_scale = __ldg(E.m_scale + at), v_scale = __ldg(E.v_scale + at);
    } else {
      load_words((const float *)E.m + first, m);
      load_words((const float *)E.v + first, v);
    }
  }
  __device__ __forceinline__ void take(const Step &A, float (&pf)[8], float (&gf)[8], float (&mf)[8], float (&rf)[8]) const {
    unpack8(p, pf, P());
    if (A.grad_type == SCN_TYPE_FLOAT32) {
      unpack8(g, gf, 0.f);
    } else {
      const unsigned w[4] = {g[0], g[1], g[2], g[3]};
      if (A.grad_type == SCN_TYPE_BFLOAT16)
        unpack8(w, gf, __nv_bfloat16());
      else
        unpack8(w, gf, __half());
    }
    if constexpr (BITS == 8) {
      from_e4m3(make_uint2(m[0], m[1]), m_scale, mf);
      from_e4m3(make_uint2(v[0], v[1]), v_scale, rf);
    } else {
      unpack8(m, mf, 0.f);
      unpack8(v, rf, 0.f);
    }
  }
};

// A block that ends early, or whose tensors lie on odd addresses: lane l has values l, l + 32 ..
template <typename P, int BITS>
__device__ __forceinline__ void read_block(const Entry &E, const Step &A, long long at, int lane, float (&p)[8], float (&g)[8], float (&m)[8],
                                           float (&r)[8]) {
  const long long first = at * kBlock + lane;
  get8<P>(E.p, first, E.n, p);
  if (A.grad_type == SCN_TYPE_FLOAT32)
    get8<float>(E.g, first, E.n, g);
  else if (A.grad_type == SCN_TYPE_BFLOAT16)
    get8<__nv_bfloat16>(E.g, first, E.n, g);
  else
    get8<__half>(E.g, first, E.n, g);
  if (BITS == 8) {
    get8_e4m3(E.m, first, E.n, E.m_scale[at], m);
    get8_e4m3(E.v, first, E.n, E.v_scale[at], r);
  } else {
    get8<float>(E.m, first, E.n, m);
    get8<float>(E.v, first, E.n, r);
  }
}

// One block of 256 values: block `number` of the list, `at` of its tensor
template <typename P, int BITS, bool WHOLE>
__device__ __forceinline__ void one_block(const Entry &E, const Step &A, long long at, long long number, unsigned key, float rate,
                                          float per_root, int lane, float (&p)[8], float (&g)[8], float (&m)[8], float (&r)[8]) {
  const long long first = at * kBlock + (WHOLE ? lane * 8 : lane);
  const Two b1 = two(A.b1), b2 = two(A.b2), c1 = two(A.one_minus_b1), c2 = two(A.one_minus_b2), keep = two(1.f - A.wd);
  // The roundings of the formula as it is written: a sum of products that came out one unit apart would be rounded to the
  // other neighbour now and then.  Pairs' mul.rn and add.rn do get contracted; times one, which the compiler cannot see, not.
  const Two one = two(A.one);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const Two gg = two(g[j], g[j + 1]), rr = two(r[j], r[j + 1]);
    const Two mm = fma2(two(m[j], m[j + 1]) * b1, one, gg * c1);
    const Two vv = fma2((BITS == 8 ? rr * rr : rr) * b2, one, (gg * gg) * c2);
    float v0, v1, x0, x1;
    apart(vv, v0, v1);
    apart(mm, m[j], m[j + 1]);
    const float r0 = __fsqrt_rn(v0), r1 = __fsqrt_rn(v1);
    apart(fma2(two(r0, r1), two(per_root), two(A.eps)), x0, x1);
    // (1 / x to a unit in the last place; eps keeps x above the subnormal numbers)
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x1));
    apart(fma2(mm * two(-rate), two(x0, x1), two(p[j], p[j + 1]) * keep), p[j], p[j + 1]);
    r[j] = BITS == 8 ? r0 : v0, r[j + 1] = BITS == 8 ? r1 : v1;
  }
  put8<P, WHOLE>(E.p, first, E.n, p);
  if (A.copy_type == SCN_TYPE_BFLOAT16)
    put8<__nv_bfloat16, WHOLE>(E.copy, first, E.n, p);
  else if (A.copy_type == SCN_TYPE_FLOAT16)
    put8<__half, WHOLE>(E.copy, first, E.n, p);
  if (BITS == 32) {
    put8<float, WHOLE>(E.m, first, E.n, m);
    put8<float, WHOLE>(E.v, first, E.n, r);
    return;
  }
  float most_m = 0.f, most_r = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    most_m = larger(most_m, m[j]);
    most_r = larger(most_r, r[j]);
  }
  most_m = __uint_as_float(max(__float_as_uint(largest(most_m)), __float_as_uint(kSmallest)));
  most_r = __uint_as_float(max(__float_as_uint(largest(most_r)), __float_as_uint(kSmallest)));
  if (lane == 0) {
    E.m_scale[at] = __fmul_rn(most_m, 1.f / kE4m3Most);
    E.v_scale[at] = __fmul_rn(most_r, 1.f / kE4m3Most);
  }
  const float per_m = __fmul_rn(__frcp_rn(most_m), kE4m3Most), per_r = __fmul_rn(__frcp_rn(most_r), kE4m3Most);
  const unsigned low = (unsigned)(number * kBlock) + (WHOLE ? lane * 8 : lane), high = (unsigned)(number * kBlock >> 32);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const unsigned h0 = mixed(mixed((low + (WHOLE ? j : 32 * j)) ^ key) ^ high), h1 = mixed(mixed((low + (WHOLE ? j + 1 : 32 * j + 32)) ^ key) ^ high);
    float a, b, c, d;
    apart(two(m[j], m[j + 1]) * two(per_m), a, b);
    apart(two(r[j], r[j + 1]) * two(per_r), c, d);
    apart(to_neighbours(a, b, chances<false>(h0, h1)), m[j], m[j + 1]);
    apart(to_neighbours(c, d, chances<true>(h0, h1)), r[j], r[j + 1]);
    m[j] = copysignf(m[j], a), m[j + 1] = copysignf(m[j + 1], b);
    if (c > 0.f) r[j] = larger(kE4m3Least, r[j]);
    if (d > 0.f) r[j + 1] = larger(kE4m3Least, r[j + 1]);
  }
  put8_e4m3<WHOLE>(E.m, first, E.n, m);
  put8_e4m3<WHOLE>(E.v, first, E.n, r);
}

template <typename P, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads)
k_adamw(const __grid_constant__ Table<CAP> T, const __grid_constant__ Step A) {
  SCN_GRID_WAIT();
  const int lane = threadIdx.x % 32;
  const unsigned long long mask = (1ull << kTicketShift) - 1;
  const unsigned long long done = *(volatile unsigned long long *)A.word & mask;
  const double t = (double)(done + 1);
  // 1 - b^t by expm1 of its logarithm: exact to fp32 for the first steps and for b near one alike
  const float bc1 = -expm1f((float)(t * A.log_b1)), bc2 = -expm1f((float)(t * A.log_b2));
  const float lr = A.lr_dev ? *A.lr_dev : A.lr;
  const float rate = lr / bc1, per_root = 1.f / sqrtf(bc2);
  const unsigned key = mixed((unsigned)(done + 1) * 0x9E3779B1u + A.seed);
  const long long warps = (long long)gridDim.x * kWarps, warp = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  // Neighbouring blocks go to neighbouring warps at the same time: DRAM sees seven streams, not seven for every warp.
  long long b = A.first + warp;
  const long long end = A.first + A.blocks;
  Step B = A;
  B.wd = lr * A.wd;
  if (b < end) {
    int lo = 0, hi = A.count - 1;  // the last tensor that begins at or before b and is not empty there
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (T.e[mid].first >> 1 <= b)
        lo = mid;
      else
        hi = mid - 1;
    }
    long long at;
    bool whole;
    Ahead<P, BITS> ahead;
    auto find = [&] {  // block b's tensor, and what it needs on its way
      while (lo + 1 < A.count && T.e[lo + 1].first >> 1 <= b) ++lo;
      const Entry &E = T.e[lo];
      at = b - (E.first >> 1);
      whole = (E.first & 1) && (at + 1) * kBlock <= E.n;
      if (whole) ahead.ask(E, A, at, lane);
    };
    for (find(); b < end;) {
      const Entry &E = T.e[lo];
      const long long number = b, mine = at;
      float p[8], g[8], m[8], r[8];
      if (whole) {
        ahead.take(A, p, g, m, r);
        b += warps;
        if (b < end) find();
        one_block<P, BITS, true>(E, B, mine, number, key, rate, per_root, lane, p, g, m, r);
      } else {
        read_block<P, BITS>(E, A, mine, lane, p, g, m, r);
        b += warps;
        if (b < end) find();
        one_block<P, BITS, false>(E, B, mine, number, key, rate, per_root, lane, p, g, m, r);
      }
    }
  }
  if (!A.last) return;
  __syncthreads();  // (every warp has read the word)
  if (threadIdx.x == 0) {
    const unsigned long long was = atomicAdd(A.word, 1ull << kTicketShift);
    if (was >> kTicketShift == gridDim.x - 1) atomicAdd(A.word, 1ull - ((unsigned long long)gridDim.x << kTicketShift));
  }
}

template <typename P, int BITS, int CAP>
int launch(const scn_adamw_tensor *tensors, int64_t n, Step A, cudaStream_t stream) {
  auto blocks_of = [](int64_t values) { return ceil_div(values, kBlock); };
  long long first = 0;
  int64_t i = 0;
  do {
    Table<CAP> T;
    A.count = 0;
    A.first = first;
    for (; i < n && A.count < CAP; ++i) {
      const scn_adamw_tensor &t = tensors[i];
      if (t.n == 0) continue;
      bool aligned = true;
      for (const void *p : {(const void *)t.param, t.grad, (const void *)t.exp_avg, (const void *)t.exp_avg_sq, (const void *)t.copy})
        aligned = aligned && (uintptr_t)p % 32 == 0;
      T.e[A.count++] = {t.param, t.exp_avg, t.exp_avg_sq, t.copy, t.grad, t.exp_avg_scale, t.exp_avg_sq_scale, t.n, first * 2 + aligned};
      first += blocks_of(t.n);
    }
    A.blocks = first - A.first;
    A.last = i == n;
    int most = 0;
    SCN_TRY((resident_blocks<k_adamw<P, BITS, CAP>>(kThreads, 0, &most)));
    const unsigned grid = (unsigned)std::max<long long>(1, std::min<long long>(most, ceil_div(A.blocks, kWarps)));
    SCN_LAUNCH((k_adamw<P, BITS, CAP>), grid, kThreads, 0, stream, T, A);
    SCN_CUDA_CHECK(cudaGetLastError());
  } while (i < n);
  return SCN_OK;
}

// Few tensors take a short table: 32 KB of arguments cost the launch some microseconds.
constexpr int kFew = 48, kMany = 440;
template <typename P, int BITS>
int launch_list(const scn_adamw_tensor *tensors, int64_t n, const Step &A, cudaStream_t stream) {
  return n <= kFew ? launch<P, BITS, kFew>(tensors, n, A, stream) : launch<P, BITS, kMany>(tensors, n, A, stream);
}

}  // namespace
}  // namespace scn

using namespace scn;

extern "C" int scn_adamw_step(const scn_adamw_tensor *tensors, int64_t n_tensors, int param_type, int grad_type, int state_bits,
                              int copy_type, int64_t *step, double lr, const float *lr_dev, double beta1, double beta2, double eps,
                              double weight_decay, uint32_t seed, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  auto is_type = [](int t) { return t == SCN_TYPE_FLOAT32 || t == SCN_TYPE_BFLOAT16 || t == SCN_TYPE_FLOAT16; };
  SCN_REQUIRE(is_type(param_type) && is_type(grad_type), SCN_ERR_BAD_ARG, "adamw_step: unknown type");
  SCN_REQUIRE(copy_type == -1 || copy_type == SCN_TYPE_BFLOAT16 || copy_type == SCN_TYPE_FLOAT16, SCN_ERR_BAD_ARG,
              "adamw_step: copies are bfloat16 or float16");
  SCN_REQUIRE(state_bits == 8 || state_bits == 32, SCN_ERR_BAD_ARG, "adamw_step: states have 8 or 32 bits");
  SCN_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, SCN_ERR_BAD_ARG, "adamw_step: betas must lie in [0, 1)");
  SCN_REQUIRE(eps >= 0 && weight_decay >= 0 && (lr_dev || lr >= 0), SCN_ERR_BAD_ARG,
              "adamw_step: lr, eps and weight_decay must not be negative");
  SCN_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || tensors) && step, SCN_ERR_BAD_ARG, "adamw_step: null argument");
  for (int64_t i = 0; i < n_tensors; ++i) {
    const scn_adamw_tensor &t = tensors[i];
    SCN_REQUIRE(t.n >= 0, SCN_ERR_BAD_ARG, "adamw_step: bad size");
    if (t.n == 0) continue;
    SCN_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq && (state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale)) &&
                    (copy_type == -1) == (t.copy == nullptr),
                SCN_ERR_BAD_ARG, "adamw_step: null argument");
  }
  Step A{};
  A.word = (unsigned long long *)step;
  A.lr_dev = lr_dev;
  // (b = 0 has no logarithm: 1 - 0^t = 1, which expm1 of a large negative number is too)
  A.log_b1 = beta1 > 0 ? log(beta1) : -1e4;
  A.log_b2 = beta2 > 0 ? log(beta2) : -1e4;
  A.lr = (float)lr, A.b1 = (float)beta1, A.b2 = (float)beta2;
  A.one_minus_b1 = (float)(1 - beta1), A.one_minus_b2 = (float)(1 - beta2);
  A.eps = (float)eps, A.wd = (float)weight_decay, A.one = 1.f;
  A.seed = seed, A.grad_type = grad_type, A.copy_type = copy_type;
#define SCN_BY_BITS(P) (state_bits == 8 ? launch_list<P, 8>(tensors, n_tensors, A, stream) : launch_list<P, 32>(tensors, n_tensors, A, stream))
  return param_type == SCN_TYPE_FLOAT32 ? SCN_BY_BITS(float) : param_type == SCN_TYPE_BFLOAT16 ? SCN_BY_BITS(__nv_bfloat16) : SCN_BY_BITS(__half);
#undef SCN_BY_BITS
}

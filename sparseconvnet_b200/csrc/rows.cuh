// Rows of 32- or 16-bit values in registers: what the row norms and the optimiser's step load, convert and store.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace scn {

template <typename T>
struct Words {
  static constexpr int N = 4;  // 32-bit words of 8 values
};
template <>
struct Words<float> {
  static constexpr int N = 8;
};

__device__ __forceinline__ void unpack8(const unsigned (&w)[8], float (&v)[8], float) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void unpack8(const unsigned (&w)[4], float (&v)[8], __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack8(const unsigned (&w)[4], float (&v)[8], __half) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ unsigned pair(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&p);
}
__device__ __forceinline__ unsigned pair(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&p);
}
template <typename T>
__device__ __forceinline__ void pack8(const float (&v)[8], unsigned (&w)[4], T t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pair(v[2 * i], v[2 * i + 1], t);
}
__device__ __forceinline__ void pack8(const float (&v)[8], unsigned (&w)[8], float) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
}

// N words of a stream that is read or written once, past L1.  8 words are one access of 32 bytes, a whole sector: as two of
// 16 bytes the neighbouring lanes' accesses lie 32 bytes apart, and every sector is asked for twice.  The 32-byte store belongs into
// code that is inlined: in a __noinline__ function nvcc 12.9 stored other registers in place of all but the first word.
__device__ __forceinline__ void load_words(const void *p, unsigned (&w)[4]) {
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}
__device__ __forceinline__ void load_words(const void *p, unsigned (&w)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void load_words(const void *p, unsigned (&w)[2]) {
  asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
}
__device__ __forceinline__ void store_words(void *p, const unsigned (&w)[4]) {
  __stcs(reinterpret_cast<uint4 *>(p), make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void store_words(void *p, const unsigned (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
               "r"(w[6]), "r"(w[7])
               : "memory");
}

// 8 values of a row as words, in vectors of V.  Vector j of thread `lane` of `lanes` holds the values from `at(j)` on, so
// that the threads of a row read neighbouring vectors; values past `n` are zero.
template <int V>
__device__ __forceinline__ int place(int chunk, int j, int lanes, int lane) {
  return ((chunk * (8 / V) + j) * lanes + lane) * V;
}
template <typename T, int V>
__device__ __forceinline__ void load8(const T *__restrict__ row, int n, int chunk, int lanes, int lane, unsigned (&w)[Words<T>::N]) {
  if (V == 8) {
    const int c = place<8>(chunk, 0, lanes, lane);
#pragma unroll
    for (int i = 0; i < Words<T>::N; ++i) w[i] = 0;
    if (c < n) load_words(row + c, w);
  } else {
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) {
      const int c = place<V>(chunk, j, lanes, lane);
      const bool in = c < n;  // (V divides n)
      if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[(j * V + i) % Words<T>::N] = in ? __ldg((const unsigned *)row + c + i) : 0u;
      } else if (V == 2) {
        w[j % Words<T>::N] = in ? __ldg((const unsigned *)(row + c)) : 0u;
      } else {
        const unsigned h = in ? (unsigned)__ldg((const unsigned short *)row + c) : 0u;
        w[j / 2 % Words<T>::N] = j % 2 ? w[j / 2 % Words<T>::N] | h << 16 : h;
      }
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store8(T *row, int n, int chunk, int lanes, int lane, const unsigned (&w)[Words<T>::N]) {
  if (V == 8) {
    const int c = place<8>(chunk, 0, lanes, lane);
    if (c < n) store_words(row + c, w);
  } else {
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) {
      const int c = place<V>(chunk, j, lanes, lane);
      if (c >= n) continue;
      if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) ((unsigned *)row)[c + i] = w[(j * V + i) % Words<T>::N];
      } else if (V == 2) {
        *(unsigned *)(row + c) = w[j % Words<T>::N];
      } else {
        ((unsigned short *)row)[c] = (unsigned short)(w[j / 2 % Words<T>::N] >> (j % 2 * 16));
      }
    }
  }
}

__device__ __forceinline__ unsigned e4m3_pair(float a, float b) {
  return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// 8 values as e4m3, saturated
template <int V>
__device__ __forceinline__ void store8_e4m3(unsigned char *row, int n, int chunk, int lanes, int lane, const float (&v)[8]) {
  if (V == 8) {
    const int c = place<8>(chunk, 0, lanes, lane);
    if (c < n)
      __stcs(reinterpret_cast<uint2 *>(row + c), make_uint2(e4m3_pair(v[0], v[1]) | e4m3_pair(v[2], v[3]) << 16,
                                                            e4m3_pair(v[4], v[5]) | e4m3_pair(v[6], v[7]) << 16));
  } else {
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) {
      const int c = place<V>(chunk, j, lanes, lane);
      if (c >= n) continue;
      const unsigned q = e4m3_pair(v[j * V], V == 2 ? v[j * V + 1] : 0.f);
      if (V == 2)
        *(unsigned short *)(row + c) = (unsigned short)q;
      else
        row[c] = (unsigned char)q;
    }
  }
}

// The number of blocks of `kernel` that the current device holds at once, asked for once per kernel and device.
template <auto kernel>
int resident_blocks(int threads, size_t smem, int *blocks) {
  static int known[64][11] = {};  // (0: not asked yet; two threads that ask store the same)
  int dev = 0, per_sm = 0, sms = 0;
  SCN_CUDA_CHECK(cudaGetDevice(&dev));
  const int slot = bit_length((unsigned long long)threads) - 1;  // powers of two up to 1024
  int *const at = dev < 64 && slot <= 10 ? &known[dev][slot] : nullptr;
  if (at && *at) {
    *blocks = *at;
    return SCN_OK;
  }
  SCN_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
  SCN_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  SCN_REQUIRE(per_sm > 0, SCN_ERR_CUDA, "a kernel does not fit an SM");
  *blocks = per_sm * sms;
  if (at) *at = *blocks;
  return SCN_OK;
}

}  // namespace scn

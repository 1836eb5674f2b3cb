// What the kernels of the model operators share: 16-bit types, rows by strides, gates in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tb200 {

struct RowsOf {  // an array of rows: strides in elements
  char* data;
  uint64_t row, seq;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const char* base, uint64_t element) {  // read once
  using P = Pack<T, V>;
  P p;
  const void* at = base + element * sizeof(T);
  if constexpr (sizeof(P) == 16) {
    const uint4 w = __ldcs(static_cast<const uint4*>(at));
    p = *reinterpret_cast<const P*>(&w);
  } else if constexpr (sizeof(P) == 8) {
    const uint2 w = __ldcs(static_cast<const uint2*>(at));
    p = *reinterpret_cast<const P*>(&w);
  } else if constexpr (sizeof(P) == 4) {
    const unsigned w = __ldcs(static_cast<const unsigned*>(at));
    p = *reinterpret_cast<const P*>(&w);
  } else {
    const unsigned short w = __ldcs(static_cast<const unsigned short*>(at));
    p = *reinterpret_cast<const P*>(&w);
  }
  return p;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack_of(const float (&f)[V]) {
  Pack<T, V> p;
#pragma unroll
  for (int i = 0; i < V; ++i) p.v[i] = from_f32<T>(f[i]);
  return p;
}

template <typename T, int V>
__device__ __forceinline__ void store_floats(char* base, uint64_t element, const float (&f)[V]) {
  const Pack<T, V> p = pack_of<T, V>(f);
  const uint64_t at = __cvta_generic_to_global(base + element * sizeof(T));
  if constexpr (sizeof(p) == 16) {
    const uint4 w = *reinterpret_cast<const uint4*>(&p);
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
  } else if constexpr (sizeof(p) == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(&p);
    asm volatile("st.global.v2.b32 [%0], {%1, %2};" ::"l"(at), "r"(w.x), "r"(w.y) : "memory");
  } else if constexpr (sizeof(p) == 4) {
    asm volatile("st.global.b32 [%0], %1;" ::"l"(at), "r"(*reinterpret_cast<const unsigned*>(&p)) : "memory");
  } else {
    asm volatile("st.global.b16 [%0], %1;" ::"l"(at), "h"(*reinterpret_cast<const unsigned short*>(&p)) : "memory");
  }
}

// 2^x, off by 2^-22 of the value; denormal results count as zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}
constexpr float kLog2e = 1.4426950408889634f;

// Two channels at once: the packed 32-bit instructions of this architecture do two in the issue slot of one.
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
template <int N>
__device__ __forceinline__ void fma_n(float (&d)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) fma2(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = fmaf(a[i], b[i], c[i]);
  }
}
template <int N>
__device__ __forceinline__ void mul_n(float (&d)[N], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) mul2(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = a[i] * b[i];
  }
}
template <int N>
__device__ __forceinline__ void add_n(float (&d)[N], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) add2(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = a[i] + b[i];
  }
}
template <int N>
__device__ __forceinline__ void fill_n(float (&d)[N], float v) {
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = v;
}

// exp(g) - 1 for g in [-0.3, 0]: its power series up to g^7 (the next term is 5e-9 of the value).
__device__ __forceinline__ float exp_minus_1(float g) {
  float p = 1.0f / 5040;
  p = fmaf(p, g, 1.0f / 720);
  p = fmaf(p, g, 1.0f / 120);
  p = fmaf(p, g, 1.0f / 24);
  p = fmaf(p, g, 1.0f / 6);
  p = fmaf(p, g, 0.5f);
  p = fmaf(p, g, 1.0f);
  return p * g;
}
constexpr float kNear = -0.3f;  // log gates from here to 0 are held as a - 1

// A gate in registers. Plain: a itself. Log: a - 1 with the sign bit set where the gate is near one, else a. Away from one
// the fast exponential will do: its error, 2 + 1.2 |g| units of 2^-23 of a, is kept for 1 / (1 - a) rows, fewer than four.
__device__ __forceinline__ float hold_gate(float g, bool log_gate) {
  if (!log_gate) return g;
  const bool near = g >= kNear && g <= 0.0f;
  const float m = __uint_as_float(__float_as_uint(exp_minus_1(g)) | 0x80000000u);
  return near ? m : __expf(g);
}
__device__ __forceinline__ bool held_near(float c, bool log_gate) { return log_gate && (__float_as_uint(c) >> 31); }
// a * h + x
__device__ __forceinline__ float advance(float c, bool near, float h, float x) {
  const float u = fmaf(c, h, x);
  return near ? h + u : u;
}

inline bool good_rows(const tb200_rows* r, int bytes) {
  return r != nullptr && r->data != nullptr && reinterpret_cast<uintptr_t>(r->data) % bytes == 0;
}
inline RowsOf rows_of(const tb200_rows* r, bool packed) {
  return RowsOf{static_cast<char*>(r->data), r->row_stride, packed ? 0 : r->sequence_stride};
}
// every row begins on a boundary of `bytes`
inline bool rows_on(const RowsOf& r, int elem, int bytes) {
  return (reinterpret_cast<uintptr_t>(r.data) | (r.row * elem) | (r.seq * elem)) % bytes == 0;
}
// The status of a call on packed sequences that has no rows or no sequences, and so no kernel that looks at its offsets.
template <typename O>
__global__ void __launch_bounds__(256) offsets_kernel(TempHeader* hdr, const O* offsets, uint64_t sequences, uint64_t rows) {
  bool bad = false;
  for (uint64_t i = threadIdx.x; i <= sequences; i += 256) {
    const int64_t v = offsets[i];
    bad = bad || v < 0 || (uint64_t)v > rows || (i == 0 ? v != 0 : v < (int64_t)offsets[i - 1]);
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) hdr->status = bad ? TB200_ERR_INVALID_ARGUMENT : TB200_OK;
}
inline int status_without_rows(void* d_temp, const void* offsets, int offset_bytes, uint64_t sequences, uint64_t rows,
                               cudaStream_t stream) {
  TempHeader* hdr = static_cast<TempHeader*>(d_temp);
  if (offset_bytes == 0) return (int)cudaMemsetAsync(hdr, 0, kHeaderBytes, stream);
  if (offset_bytes == 4) offsets_kernel<<<1, 256, 0, stream>>>(hdr, static_cast<const int32_t*>(offsets), sequences, rows);
  else offsets_kernel<<<1, 256, 0, stream>>>(hdr, static_cast<const int64_t*>(offsets), sequences, rows);
  trace_mark(stream);
  return (int)cudaGetLastError();
}
inline int model_bytes(int dtype) { return dtype == TB200_F32 ? 4 : dtype == TB200_F16 || dtype == TB200_BF16 ? 2 : 0; }

}  // namespace tb200

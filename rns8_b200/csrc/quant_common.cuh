// Shared by the 8-bit operators (row quantisation, scaled product, residual
// norms): element types, rows held in registers, block reductions and the
// quantisation rule.
//
// A row kernel gives every thread NV vectors of 8 elements. With ALIGNED rows
// (whole vectors, base and leading dimension on 16-byte boundaries) vector v of
// thread t covers elements 8 * (v * threads + t) .. + 7 and moves as 16-byte
// words, as do rows that start anywhere, shifted into place; where rows go
// element by element its e-th is (8 v + e) * threads + t, so that a warp's
// accesses are contiguous. Elements past the row read as
// zero. No kernel holds both forms: short calls wait for their code to arrive
// as much as for their data.
#pragma once

#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace rns8cuda {

// ---- element conversions -------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Vectors of 8 a thread of a row kernel holds. Few rows are a matter of latency:
// one vector a thread. With rows for every SM, blocks of at most 256 threads
// let the loads of one row run under the reductions of the others.
inline int row_vectors(int64_t rows, int vecs) {
  if (vecs > 1024) return 4;
  if (rows < 256 || vecs <= 256) return 1;
  return vecs <= 512 ? 2 : 4;
}

// Index of element (v, e) of this thread's part of a row.
template <bool ALIGNED>
__device__ __forceinline__ int row_index(int v, int e, int threads, int tid) {
  return ALIGNED ? (v * threads + tid) * 8 + e : (v * 8 + e) * threads + tid;
}

// ---- pairs of 32-bit floats ---------------------------------------------------------
// sm_100 multiplies and adds two floats an instruction; the row kernels are as
// much bound by issue as by HBM.
struct F2 {
  float2 v;
};
__device__ __forceinline__ F2 f2(float a, float b) { return F2{make_float2(a, b)}; }
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ uint64_t bits(F2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v.x), "f"(a.v.y));
  return r;
}
__device__ __forceinline__ F2 from_bits(uint64_t r) {
  F2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.v.x), "=f"(a.v.y) : "l"(r));
  return a;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return from_bits(r);
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return from_bits(r);
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return from_bits(r);
}
__device__ __forceinline__ float both(F2 a) { return a.v.x + a.v.y; }

// Two elements of a 16-bit type in a word, as floats and back.
template <typename T>
__device__ __forceinline__ F2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ F2 unpack2<__nv_bfloat16>(uint32_t w) {
  return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ F2 unpack2<__half>(uint32_t w) {
  return F2{__half22float2(*reinterpret_cast<const __half2*>(&w))};
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(F2 a);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(F2 a) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a.v.x, a.v.y);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(F2 a) {
  const __half2 r = __floats2half2_rn(a.v.x, a.v.y);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight elements as they lie in memory: the words of an aligned vector.
template <typename T>
struct Raw8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p, bool in) {
    w = in ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ F2 pair(int i) const {
    return unpack2<T>(i == 0 ? w.x : (i == 1 ? w.y : (i == 2 ? w.z : w.w)));
  }
  __device__ __forceinline__ void set(const F2 (&v)[4]) {
    w = make_uint4(pack2<T>(v[0]), pack2<T>(v[1]), pack2<T>(v[2]), pack2<T>(v[3]));
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
};
template <>
struct Raw8<float> {
  float4 lo, hi;
  __device__ __forceinline__ void load(const float* p, bool in) {
    lo = in ? reinterpret_cast<const float4*>(p)[0] : make_float4(0, 0, 0, 0);
    hi = in ? reinterpret_cast<const float4*>(p)[1] : make_float4(0, 0, 0, 0);
  }
  __device__ __forceinline__ F2 pair(int i) const {
    return i == 0 ? f2(lo.x, lo.y) : (i == 1 ? f2(lo.z, lo.w) : (i == 2 ? f2(hi.x, hi.y) : f2(hi.z, hi.w)));
  }
  __device__ __forceinline__ void set(const F2 (&v)[4]) {
    lo = make_float4(v[0].v.x, v[0].v.y, v[1].v.x, v[1].v.y);
    hi = make_float4(v[2].v.x, v[2].v.y, v[3].v.x, v[3].v.y);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = lo;
    reinterpret_cast<float4*>(p)[1] = hi;
  }
};

// Vector v of this thread's part of a row; elements at or past `cols` are zero.
template <bool ALIGNED, typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int cols, int v, int threads, int tid, F2 (&out)[4]) {
  if (ALIGNED) {
    const int i = (v * threads + tid) * 8;
    Raw8<T> raw;
    raw.load(row + i, i < cols);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = raw.pair(e);
  } else {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = row_index<ALIGNED>(v, e, threads, tid);
      x[e] = i < cols ? to_f32(row[i]) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = f2(x[2 * e], x[2 * e + 1]);
  }
}
template <bool ALIGNED, typename T>
__device__ __forceinline__ void store8(T* __restrict__ row, int cols, int v, int threads, int tid, const F2 (&in)[4]) {
  if (ALIGNED) {
    const int i = (v * threads + tid) * 8;
    Raw8<T> raw;
    raw.set(in);
    if (i < cols) raw.store(row + i);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = row_index<ALIGNED>(v, e, threads, tid);
      if (i < cols) row[i] = from_f32<T>(e % 2 ? in[e / 2].v.y : in[e / 2].v.x);
    }
  }
}

// ---- rows that start anywhere ---------------------------------------------------------
// Vectors as in aligned rows (element i of a row starts one, i a multiple of 8),
// read and written as the 16-byte words they straddle: a vector's own bytes are
// the words' shifted down by the row's offset, the same for all its vectors.
template <typename T>
constexpr int kVectorWords = 2 * static_cast<int>(sizeof(T));  // of 32 bits

// The vector that starts `bytes` (whole elements, below 16, the same in all
// lanes) into w. Selects, not branches: 8000 x 5001 f32 171 and 193 us.
template <typename T>
__device__ __forceinline__ void shift_down(const uint32_t (&w)[kVectorWords<T> + 4], uint32_t bytes,
                                           uint32_t (&out)[kVectorWords<T>]) {
  constexpr int W = kVectorWords<T>;
  uint32_t a[W + 2], b[W + 1];
#pragma unroll
  for (int k = 0; k < W + 2; ++k) a[k] = bytes & 8 ? w[k + 2] : w[k];
#pragma unroll
  for (int k = 0; k < W + 1; ++k) b[k] = bytes & 4 ? a[k + 1] : a[k];
#pragma unroll
  for (int k = 0; k < W; ++k) out[k] = sizeof(T) == 2 ? __funnelshift_r(b[k], b[k + 1], (bytes & 2) * 8) : b[k];
}
template <typename T>
__device__ __forceinline__ void get_words(const Raw8<T>& v, uint32_t* w) {
  if constexpr (sizeof(T) == 2) {
    w[0] = v.w.x, w[1] = v.w.y, w[2] = v.w.z, w[3] = v.w.w;
  } else {
    w[0] = __float_as_uint(v.lo.x), w[1] = __float_as_uint(v.lo.y), w[2] = __float_as_uint(v.lo.z);
    w[3] = __float_as_uint(v.lo.w), w[4] = __float_as_uint(v.hi.x), w[5] = __float_as_uint(v.hi.y);
    w[6] = __float_as_uint(v.hi.z), w[7] = __float_as_uint(v.hi.w);
  }
}
template <typename T>
__device__ __forceinline__ Raw8<T> from_words(const uint32_t* w) {
  Raw8<T> v;
  if constexpr (sizeof(T) == 2) {
    v.w = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    v.lo = make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
    v.hi = make_float4(__uint_as_float(w[4]), __uint_as_float(w[5]), __uint_as_float(w[6]), __uint_as_float(w[7]));
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void load_straddled(const uint8_t* from, uint32_t (&w)[kVectorWords<T> + 4]) {
#pragma unroll
  for (int k = 0; k < kVectorWords<T> + 4; k += 4) {
    const uint4 word = *reinterpret_cast<const uint4*>(from + 4 * k);
    w[k] = word.x, w[k + 1] = word.y, w[k + 2] = word.z, w[k + 3] = word.w;
  }
}
// From global memory: words that reach outside the row are read by elements.
template <typename T>
__device__ __forceinline__ Raw8<T> load_shifted(const T* row, int cols, int i) {
  uint32_t out[kVectorWords<T>] = {};
  const T* at = row + i;
  const uint32_t off = reinterpret_cast<uintptr_t>(at) % 16;
  const int before = static_cast<int>(off / sizeof(T)), reach = off ? 8 + static_cast<int>(16 / sizeof(T)) : 8;
  if (i >= before && i - before + reach <= cols) {
    if (off == 0) {
      Raw8<T> v;
      v.load(at, true);
      return v;
    }
    uint32_t w[kVectorWords<T> + 4];
    load_straddled<T>(reinterpret_cast<const uint8_t*>(at) - off, w);
    shift_down<T>(w, off, out);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < cols) {
        if constexpr (sizeof(T) == 2)
          out[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[e]) << (e % 2 * 16);
        else
          out[e] = reinterpret_cast<const uint32_t*>(at)[e];
      }
  }
  return from_words<T>(out);
}
// The warp's 32 consecutive vectors to global memory: a lane stores the words
// that its vector ends, with what the lane before has of the first. The warp's
// outermost elements, together one word, go one a lane; the vectors around the
// row's end by elements.
template <typename T>
__device__ __forceinline__ void store_shifted(T* row, int cols, int i, const Raw8<T>& v) {
  constexpr int W = kVectorWords<T>, PER_WORD = 16 / sizeof(T);
  const int lane = threadIdx.x % 32, first = i - 8 * lane;  // the warp's first element
  T* at = row + i;
  const uint32_t off = reinterpret_cast<uintptr_t>(at) % 16;  // the same in all lanes
  const int before = static_cast<int>(off / sizeof(T));
  if (first + 8 * 32 <= cols) {
    if (off == 0) return v.store(at);
    uint32_t w[W + 4], out[W];
    get_words<T>(v, w + 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __shfl_up_sync(0xFFFFFFFFu, w[W + k], 1);
    shift_down<T>(w, 16 - off, out);
#pragma unroll
    for (int h = 0; h < W / 4; ++h)
      if (h > 0 || lane > 0)
        reinterpret_cast<uint4*>(at - before)[h] = make_uint4(out[4 * h], out[4 * h + 1], out[4 * h + 2], out[4 * h + 3]);
    // Lane k: element k of the first word that is the warp's, or of the word past its last whole one.
    const bool front = lane + before < PER_WORD;
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t word = __shfl_sync(0xFFFFFFFFu, lane == 0 ? w[4 + k] : w[W + k], front ? 0 : 31);
      if (lane * sizeof(T) / 4 == k) mine = word;
    }
    if (lane < PER_WORD) {
      T* to = row + first + (front ? lane : 256 - PER_WORD + lane);
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(mine >> (lane % 2 * 16));
      else
        *reinterpret_cast<uint32_t*>(to) = mine;
    }
  } else {
    uint32_t own[W];
    get_words<T>(v, own);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < cols) {
        if constexpr (sizeof(T) == 2)
          reinterpret_cast<uint16_t*>(at)[e] = static_cast<uint16_t>(own[e / 2] >> (e % 2 * 16));
        else
          reinterpret_cast<uint32_t*>(at)[e] = own[e];
      }
  }
}

// ---- rows on 16-byte boundaries -------------------------------------------------------
// dst rows (ld_dst a multiple of 16) from int8 src rows of any alignment, 16
// bytes a thread: the five aligned words around them, shifted into place (1001
// x 2040 byte by byte: 3.7 us, this 2.0). Bytes past cols are zero; where a word
// would reach outside the matrix the bytes are read one by one.
struct AlignRows {
  const int8_t* src;
  int8_t* dst;
  int64_t rows, cols, ld, ld_dst;
};
__device__ __forceinline__ void align_rows(const AlignRows& j, int64_t first, int64_t step) {
  const int64_t per_row = j.ld_dst / 16, total = j.rows * per_row;
  const int8_t* end = j.src + (j.rows - 1) * j.ld + j.cols;
  for (int64_t i = first; i < total; i += step) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 16;
    const int8_t* from = j.src + r * j.ld + c;
    const uint32_t shift = reinterpret_cast<uintptr_t>(from) % 4 * 8;
    const int8_t* base = from - shift / 8;
    uint32_t w[4] = {0, 0, 0, 0};
    if (c + 16 <= j.cols && base >= j.src && base + 20 <= end) {
      uint32_t v[5];
#pragma unroll
      for (int k = 0; k < 5; ++k) v[k] = reinterpret_cast<const uint32_t*>(base)[k];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(v[k], v[k + 1], shift);
    } else {
#pragma unroll
      for (int b = 0; b < 16; ++b)
        if (c + b < j.cols) w[b / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(from[b])) << (8 * (b % 4));
    }
    *reinterpret_cast<uint4*>(j.dst + r * j.ld_dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- quantisation rule ------------------------------------------------------------
// Magnitudes are compared by their bits: for non-negative floats the unsigned
// order of the bits is the numeric order, and a NaN is above everything, so a
// row's maximum is NaN when it holds one.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

struct RowScale {
  float scale, inv;
};
// scale = a / 127 and its inverse 127 / a. Below 127 * 2^-126 the scale would
// be subnormal and 127 / a could overflow: such rows count as zero rows. For a
// non-finite a the scale is a and every q is zero.
__device__ __forceinline__ RowScale make_row_scale(uint32_t max_bits) {
  const float a = __uint_as_float(max_bits);
  RowScale r;
  if (max_bits >= 0x7F800000u) {
    r.scale = a;
    r.inv = 0.0f;
  } else if (a < 127.0f * FLT_MIN) {
    r.scale = 0.0f;
    r.inv = 0.0f;
  } else {
    r.scale = __fdiv_rn(a, 127.0f);
    r.inv = __fdiv_rn(127.0f, a);
  }
  return r;
}
// |x * inv| <= 127 (1 + 2^-22), which rounds to at most 127. With inv = 0 the
// product of an infinity or a NaN is a NaN, which converts to 0.
__device__ __forceinline__ int quantize_one(float x, float inv) { return __float2int_rn(x * inv); }

__device__ __forceinline__ uint32_t magnitude_bits(const F2 (&v)[4]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, max(magnitude_bits(v[e].v.x), magnitude_bits(v[e].v.y)));
  return top;
}

template <bool ALIGNED>
__device__ __forceinline__ void store_q8(int8_t* __restrict__ row, int cols, int v, int threads, int tid,
                                         const F2 (&in)[4], float inv) {
  uint32_t q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = static_cast<uint32_t>(quantize_one(e % 2 ? in[e / 2].v.y : in[e / 2].v.x, inv));
  if (ALIGNED) {
    const int i = (v * threads + tid) * 8;
    if (i < cols)
      *reinterpret_cast<uint2*>(row + i) =
          make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                     __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = row_index<ALIGNED>(v, e, threads, tid);
      if (i < cols) row[i] = static_cast<int8_t>(q[e]);
    }
  }
}

// ---- block reductions ---------------------------------------------------------------
// One barrier each: every warp leaves its part in `slots` and then joins all the
// parts itself, four at a time. Two reductions that follow one another use
// different slots; slots of warps that the block does not have are zero
// (clear_slots, before the first one).
//
// Sums of N values over a warp: while two lanes hold 2^k values each they swap
// halves instead of adding all of them twice, so that 8 values take 9 shuffles,
// not 40. Lane l ends with the total of value l / (32 / N2), N2 the power of
// two from N up.
template <int N>
constexpr int pow2_of() {
  return N <= 1 ? 1 : 2 * pow2_of<(N + 1) / 2>();
}
template <int N2>
__device__ __forceinline__ float warp_sum_spread(float (&v)[N2], int lane) {
#pragma unroll
  for (int half = N2 / 2, o = 16; o; o >>= 1) {
    if (half) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float send = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
        v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, o);
      }
      half >>= 1;
    } else {
      v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
    }
  }
  return v[0];
}

template <int N>
struct SumSlots {
  static constexpr int N2 = pow2_of<N>();
  float4 part[N2][8];  // [value][warp / 4], .xyzw by warp % 4
};
template <int N>
__device__ __forceinline__ void clear_slots(SumSlots<N>& s) {
  for (int i = threadIdx.x; i < SumSlots<N>::N2 * 32; i += blockDim.x) reinterpret_cast<float*>(s.part)[i] = 0.0f;
}

template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], SumSlots<N>& slots) {
  constexpr int N2 = SumSlots<N>::N2, SHARE = 32 / N2;  // lanes of a warp for each value
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  float w[N2];
#pragma unroll
  for (int n = 0; n < N2; ++n) w[n] = n < N ? v[n < N ? n : 0] : 0.0f;
  float total = warp_sum_spread(w, lane);
  if (warps > 1) {
    if (lane % SHARE == 0) reinterpret_cast<float*>(slots.part[lane / SHARE])[warp] = total;
    __syncthreads();
    // Four warps' parts a lane; 8 / (lanes a value has) rounds for up to 32 warps.
    total = 0.0f;
#pragma unroll
    for (int q = lane % SHARE; q < 8; q += SHARE) {
      if (q * 4 >= warps) break;
      const float4 f = slots.part[lane / SHARE][q];
      total += (f.x + f.y) + (f.z + f.w);
    }
    // The lanes past the eighth of a value have nothing: the sum stays whole.
#pragma unroll
    for (int o = (SHARE < 8 ? SHARE : 8) / 2; o; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
    if (SHARE > 8) total = __shfl_sync(0xFFFFFFFFu, total, lane / SHARE * SHARE);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = N2 == 1 ? total : __shfl_sync(0xFFFFFFFFu, total, n * SHARE);
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* slots) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if (warps == 1) return v;
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xFFFFFFFFu, lane < warps ? slots[lane] : 0u);
}

}  // namespace rns8cuda

// adjust_logits.hip - penalties for repeated tokens, biases and grammar masks on
// the logits of a denoising step, before the draw.
//
// For logit x of token v in a row of sequence b, c = count of v among
// tokens[b][0 .. lengths[b]):
//   c > 0: x = x > 0 ? x / repetition : x * repetition, then x -= frequency * c + presence
//   x += bias[v];   x = fill where the mask's bit of v is 0
// in fp32, rounded once to the logits' type. fill is finite, so a row whose mask
// leaves nothing holds it everywhere; and a finite logit stays finite, as the draw
// wants it: what a penalty or bias takes past the type's range (the type's lowest value
// times a repetition) becomes its largest of that sign.
//
// A workgroup takes 2048 tokens of the vocabulary for some of a sequence's rows:
// it counts its tokens among the history in LDS (integer adds: the order does
// not matter), keeps what depends on the token alone in registers (8 tokens a
// thread) and walks the rows, one 16-byte read and write a thread and row, four
// rows in flight. With no row loop's reads in flight and the bias and history
// requested one after another the same took 61 us instead of 46 (32 x 32 rows of
// 50258 bf16 logits; 41.3 now, 5.0 TB/s, a large copy's rate) and 13.5 instead of 10
// (64 fp32 rows, a bias and a mask each; 10.2 now).
#include "bd3_device.h"
#include "bd3_launch.h"

namespace bd3 {
namespace {

constexpr int kCols = 8;                    // tokens per thread
constexpr int kSlice = kLogitSlice;         // tokens per workgroup
constexpr int kThreads = kSlice / kCols;
static_assert(kThreads == 256, "one pass over a slice");

// |x| as an integer. Behind an empty asm: this code is built without honour to NaNs, and
// the compiler takes comparisons of plain bits back to such ones of floats, which a
// NaN passes.
__device__ __forceinline__ uint32_t magnitude(float x) {
  uint32_t u = __float_as_uint(x);
  asm("" : "+v"(u));
  return u & 0x7fffffffu;
}

constexpr uint32_t kInf = 0x7f800000u;  // magnitude of an infinite one; a NaN's is larger

// x, a result of a and b, or the largest number of its sign where x is infinite
// and a and b are finite.
__device__ __forceinline__ float finite(float x, float a, float b) {
  const bool over = magnitude(x) == kInf && magnitude(a) < kInf && magnitude(b) < kInf;
  return over ? __uint_as_float((__float_as_uint(x) & 0x80000000u) | (kInf - 1)) : x;
}

// Rows start at any element: 16-byte accesses of element alignment.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Eight logits of a row as they lie in memory: loads of several rows are in flight
// before the first is unpacked. bf16 logits are read once, non-temporally: their
// reads are not to push the result, which the draw reads next, out of the caches
// (32 x 32 rows of 50258: 46.2 us with plain reads, 40.8 so; 45.5 with non-temporal
// writes too). fp32 ones take two reads of a cache line, so plain ones (64 rows 10.0
// us, non-temporal 10.7).
template <typename T>
struct Row8;
template <>
struct Row8<uint16_t> {
  u32x4 w;
  __device__ __forceinline__ void load(const uint16_t* p, int left) {
    if (left >= kCols) {
      w = (u32x4)__builtin_nontemporal_load(reinterpret_cast<const u32x4_a2*>(p));
    } else {
      w = u32x4{};
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < left) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    }
  }
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&x)[kCols]) {
    w = __builtin_bit_cast(u32x4, to_bf16x8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]));
  }
  // Is any of them infinite (or NaN)?
  __device__ __forceinline__ bool infinite() const {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    return ((__builtin_bit_cast(uint32_t, m) + 0x00800080u) & 0x80008000u) != 0;
  }
  // The type's lowest or highest value for those that became infinite from finite ones.
  __device__ __forceinline__ void limit(const Row8& x, const float (&add)[kCols]) {
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const uint32_t u = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
      const bool over = (u & 0x7fffu) == 0x7f80u && magnitude(x.get(i)) < kInf && magnitude(add[i]) < kInf;
      w[i >> 1] -= over ? 1u << (16 * (i & 1)) : 0u;
    }
  }
  __device__ __forceinline__ void store(uint16_t* p, int left) const {
    if (left >= kCols) {
      *reinterpret_cast<u32x4_a2*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < left) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
};
template <>
struct Row8<float> {
  f32x4 w[2];
  __device__ __forceinline__ void load(const float* p, int left) {
    if (left >= kCols) {
      w[0] = (f32x4)*reinterpret_cast<const f32x4_a4*>(p);
      w[1] = (f32x4)*reinterpret_cast<const f32x4_a4*>(p + 4);
    } else {
      w[0] = w[1] = f32x4{};
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < left) w[i >> 2][i & 3] = p[i];
    }
  }
  __device__ __forceinline__ float get(int i) const { return w[i >> 2][i & 3]; }
  __device__ __forceinline__ void set(const float (&x)[kCols]) {
#pragma unroll
    for (int i = 0; i < kCols; ++i) w[i >> 2][i & 3] = x[i];
  }
  __device__ __forceinline__ bool infinite() const {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kCols; ++i) top = fmaxf(top, fabsf(get(i)));
    return magnitude(top) >= kInf;
  }
  __device__ __forceinline__ void limit(const Row8& x, const float (&add)[kCols]) {
#pragma unroll
    for (int i = 0; i < kCols; ++i) w[i >> 2][i & 3] = finite(get(i), x.get(i), add[i]);
  }
  __device__ __forceinline__ void store(float* p, int left) const {
    if (left >= kCols) {
      *reinterpret_cast<f32x4_a4*>(p) = w[0];
      *reinterpret_cast<f32x4_a4*>(p + 4) = w[1];
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < left) p[i] = w[i >> 2][i & 3];
    }
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(LogitArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t count[kSlice];
  const int tid = wi_x();
  const int slice = wg_x() % a.slices;
  const int part = wg_x() / a.slices % a.row_parts;
  const int b = wg_x() / a.slices / a.row_parts;
  const int v0 = slice * kSlice;
  const int col = v0 + tid * kCols;
  const int left = a.vocab - col;  // tokens from col on

  // Rows in flight: the first ones are requested before the history is counted.
  constexpr int kRows = sizeof(T) == 2 ? 4 : 2;
  const int row0 = part * a.part_rows;
  const int row_end = row0 + a.part_rows < a.rows ? row0 + a.part_rows : a.rows;
  const T* in = static_cast<const T*>(a.logits) + (int64_t)b * a.in_b + col;
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.out_b + col;
  const uint8_t* bits =  // of 8 tokens from a multiple of 8 on: one byte of the words
      a.allowed == nullptr ? nullptr
                           : reinterpret_cast<const uint8_t*>(a.allowed + (int64_t)b * a.allowed_b) + (col >> 3);
  Row8<T> v[kRows];
  uint32_t yes[kRows];
  auto load = [&](int r0) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      yes[k] = 0xff;
      if (r0 + k < row_end && left > 0) {
        v[k].load(in + (int64_t)(r0 + k) * a.in_r, left);
        if (bits != nullptr) yes[k] = bits[4 * (int64_t)(r0 + k) * a.allowed_r];
      }
    }
  };
  load(row0);
  // Everything else a thread waits for is requested beside them: the bias, the first
  // of the history (before its length is known), the penalties.
  // x becomes x * (x > 0 ? up : down) + add.
  float up[kCols], down[kCols], add[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    up[i] = down[i] = 1.f;
    add[i] = 0.f;
  }
  if (a.bias != nullptr && left > 0) {
    const float* bp = a.bias + (int64_t)b * a.bias_s + col;
    if (left >= kCols) {
#pragma unroll
      for (int i = 0; i < kCols; i += 4) {
        const f32x4 w = *reinterpret_cast<const f32x4_a4*>(bp + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) add[i + k] = w[k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < left) add[i] = bp[i];
    }
  }
  if (a.tokens != nullptr) {
    constexpr int kFlight = 8;  // tokens requested by a thread before the first is counted
    const int64_t* hist = a.tokens + (int64_t)b * a.tokens_s;
    int64_t t[kFlight];
    auto request = [&](int i0) {
#pragma unroll
      for (int k = 0; k < kFlight; ++k) t[k] = i0 + k * kThreads < a.history ? hist[i0 + k * kThreads] : -1;
    };
    request(tid);
    int n = a.history;
    if (a.lengths != nullptr) {
      const int len = a.lengths[b];
      n = len < 0 ? 0 : (len < n ? len : n);
    }
    const float f = a.frequency_p != nullptr ? a.frequency_p[b] : a.frequency;
    const float g = a.presence_p != nullptr ? a.presence_p[b] : a.presence;
    const float rep = a.repetition_p != nullptr ? a.repetition_p[b] : a.repetition;
#pragma unroll
    for (int i = 0; i < kCols; i += 4) *reinterpret_cast<u32x4*>(&count[tid * kCols + i]) = u32x4{};
    __syncthreads();
    for (int i0 = tid; i0 < n; i0 += kFlight * kThreads) {
      if (i0 > tid) request(i0);
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const uint64_t at = (uint64_t)t[k] - (uint64_t)v0;
        if (at < (uint64_t)kSlice && t[k] >= 0 && i0 + k * kThreads < n) atomicAdd(&count[at], 1u);
      }
    }
    __syncthreads();
    const float inv = 1.f / rep;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const uint32_t c = count[tid * kCols + i];
      if (c > 0) {
        up[i] = inv;
        down[i] = rep;
        const float pen = finite(fmaf(f, (float)c, g), f, g);
        add[i] = finite(add[i] - pen, add[i], pen);
      }
    }
  }
  if (left <= 0) return;

  for (int r0 = row0; r0 < row_end; r0 += kRows) {
    if (r0 > row0) load(r0);
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (r0 + k >= row_end) break;
      float x[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        x[i] = v[k].get(i);
        x[i] = fmaf(x[i], x[i] > 0.f ? up[i] : down[i], add[i]);
        x[i] = (yes[k] >> i) & 1 ? x[i] : a.fill;
      }
      // A row is looked at for infinite ones as a whole, 41.3 us; value by value, all of
      // them always, 43.4.
      Row8<T> y;
      y.set(x);
      if (__builtin_expect(__ballot(y.infinite()) != 0, 0)) {
        // bf16: read again (the result may lie over it, but is not written yet), so that the
        // row's registers are free before; with them kept there is a wave fewer per SIMD.
        if constexpr (sizeof(T) == 2) v[k].load(in + (int64_t)(r0 + k) * a.in_r, left);
        y.limit(v[k], add);
      }
      y.store(out + (int64_t)(r0 + k) * a.out_r, left);
    }
  }
}

}  // namespace

hipError_t launch_adjust_logits(const LogitArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.row_parts * a.slices));
  if (a.fp32)
    hipLaunchKernelGGL(adjust_logits_kernel<float>, grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(adjust_logits_kernel<uint16_t>, grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bd3

// adjust_logits.hip - penalties for repeated tokens, biases and grammar masks on
// the logits of a denoising step, before the draw.
//
// For logit x of token v in a row of sequence b, c = count of v among
// tokens[b][0 .. lengths[b]):
//   c > 0: x = x > 0 ? x / repetition : x * repetition, then x -= frequency * c + presence
//   x += bias[v];   x = fill where the mask's bit of v is 0
// in fp32, rounded once to the logits' type. fill is finite, so a row whose mask
// leaves nothing holds it everywhere.
//
// A workgroup takes 2048 tokens of the vocabulary for some of a sequence's rows:
// it counts its tokens among the history in LDS (integer adds: the order does
// not matter), keeps what depends on the token alone in registers (8 tokens a
// thread) and walks the rows, one 16-byte read and write a thread and row.
#include "bd3_device.h"
#include "bd3_launch.h"

namespace bd3 {
namespace {

constexpr int kCols = 8;                    // tokens per thread
constexpr int kSlice = kLogitSlice;         // tokens per workgroup
constexpr int kThreads = kSlice / kCols;
static_assert(kThreads == 256, "one pass over a slice");

// Rows start at any element: 16-byte accesses of element alignment.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

template <typename T>
struct Row8 {
  float x[kCols];
  __device__ __forceinline__ void load(const T* p, int left) {
    if (left >= kCols) {
      if constexpr (sizeof(T) == 2) {
        const bf16x8 v = __builtin_bit_cast(bf16x8, (u32x4)*reinterpret_cast<const u32x4_a2*>(p));
#pragma unroll
        for (int i = 0; i < kCols; ++i) x[i] = (float)v[i];
      } else {
#pragma unroll
        for (int i = 0; i < kCols; i += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4_a4*>(p + i);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[i + k] = v[k];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        if (i < left) {
          if constexpr (sizeof(T) == 2)
            x[i] = (float)__builtin_bit_cast(__bf16, p[i]);
          else
            x[i] = p[i];
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int left) const {
    if (left >= kCols) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4_a2*>(p) =
            __builtin_bit_cast(u32x4, to_bf16x8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]));
      } else {
#pragma unroll
        for (int i = 0; i < kCols; i += 4)
          *reinterpret_cast<f32x4_a4*>(p + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        if (i < left) {
          if constexpr (sizeof(T) == 2)
            p[i] = __builtin_bit_cast(uint16_t, (__bf16)x[i]);
          else
            p[i] = x[i];
        }
      }
    }
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(LogitArgs a) {
  __shared__ uint32_t count[kSlice];
  const int tid = wi_x();
  const int slice = wg_x() % a.slices;
  const int part = wg_x() / a.slices % a.row_parts;
  const int b = wg_x() / a.slices / a.row_parts;
  const int v0 = slice * kSlice;
  const int col = v0 + tid * kCols;
  const int left = a.vocab - col;  // tokens from col on

  float add[kCols] = {};
  uint32_t hit = 0;
  if (a.tokens != nullptr) {
#pragma unroll
    for (int i = 0; i < kCols; i += 4) *reinterpret_cast<u32x4*>(&count[tid * kCols + i]) = u32x4{};
    __syncthreads();
    const int64_t* hist = a.tokens + (int64_t)b * a.tokens_s;
    int n = a.history;
    if (a.lengths != nullptr) {
      const int len = a.lengths[b];
      n = len < 0 ? 0 : (len < n ? len : n);
    }
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t at = (uint64_t)(hist[i] - v0);
      if (at < (uint64_t)kSlice) atomicAdd(&count[at], 1u);
    }
    __syncthreads();
    const float f = a.frequency_p != nullptr ? a.frequency_p[b] : a.frequency;
    const float g = a.presence_p != nullptr ? a.presence_p[b] : a.presence;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const uint32_t n_i = count[tid * kCols + i];
      if (n_i > 0) {
        hit |= 1u << i;
        add[i] = -(f * (float)n_i + g);
      }
    }
  }
  if (left <= 0) return;
  if (a.bias != nullptr) {
    const float* bp = a.bias + (int64_t)b * a.bias_s + col;
#pragma unroll
    for (int i = 0; i < kCols; ++i)
      if (i < left) add[i] += bp[i];
  }
  const float rep = a.repetition_p != nullptr ? a.repetition_p[b] : a.repetition;

  const int row_end = (part + 1) * a.part_rows < a.rows ? (part + 1) * a.part_rows : a.rows;
  for (int r = part * a.part_rows; r < row_end; ++r) {
    Row8<T> v;
    v.load(static_cast<const T*>(a.logits) + (int64_t)b * a.in_b + (int64_t)r * a.in_r + col, left);
    uint32_t yes = 0xff;
    if (a.allowed != nullptr)  // the bits of 8 tokens from a multiple of 8 on: one byte of the words
      yes = reinterpret_cast<const uint8_t*>(a.allowed + (int64_t)b * a.allowed_b + (int64_t)r * a.allowed_r)[col >> 3];
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      float x = v.x[i];
      if ((hit >> i) & 1) x = x > 0.f ? x / rep : x * rep;
      x += add[i];
      v.x[i] = (yes >> i) & 1 ? x : a.fill;
    }
    v.store(static_cast<T*>(a.out) + (int64_t)b * a.out_b + (int64_t)r * a.out_r + col, left);
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

// Rotary positions of a step's queries and keys, with the K and V rows put into
// their cache pages: the rows vc_kv_commit later hashes in place.
//
// For a token at position p and rotated pair i, a = p * inv_freq[i] and
//   y1 = x1 * cos a - x2 * sin a,   y2 = x2 * cos a + x1 * sin a
// with both cos and sin times `factor` (1, or a long-context scaling's).  The
// angle and its cos/sin are taken in f64 (an f32 angle at position 10^5 is off
// by 2^-8 rad), rounded once to f32; the rotation runs in f32 FMAs and is
// rounded once to the row's type.
//
// Bound by memory: every element is read and written once.  One CTA handles one
// token (a share of its heads when there are few tokens), so the rotary_dim / 2
// f64 sincos are paid once per CTA and shared through shared memory by all its
// heads.  A unit of work is one 16-byte chunk of the first half of a head and its
// partner of the second half (neighbouring pairs: one chunk), or one chunk of
// the unrotated rest; narrower chunks where alignment or an odd rotary_dim asks
// for them.
//
// Measured: 8192 tokens of 64 + 8 + 8 heads of 128 in bf16 (336 MB moved) 57.7 us, 5.8
// TB/s; 256 tokens 6.3 us, one token 4.3 us (the launch, then positions, angles and rows
// one behind the other).  128 threads a CTA gave 3 % over 256; loading four units a
// thread ahead of the angles halved the CTAs an SM holds and took 181 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vc_internal.h"

namespace vc {
namespace {

constexpr int kThreads = 128;

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <typename T, int N, bool kLoose>
struct alignas(kLoose ? sizeof(T) : sizeof(T) * N) Vec {   // kLoose: only element-aligned
  T v[N];
};

// One token's units: rotated ones of a head first, then its unrotated chunks.
// V = elements of a chunk; a rotated unit covers V pairs (halves) or V / 2
// pairs (neighbours; V >= 2).
template <typename T, int V, bool kNeighbours, bool kLoose>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(RopeArgs a) {
  extern __shared__ float2 cs[];
  const int tok = blockIdx.x;
  const int half = a.rotary_dim >> 1;
  const int p = a.positions[tok];
  const int seq = a.seq_ids ? a.seq_ids[tok] : tok;
  if (p >= 0) {
    for (int i = threadIdx.x; i < half; i += kThreads) {
      double s, c;
      sincos(double(p) * a.inv_freq[i], &s, &c);
      cs[i] = make_float2(float(c * a.factor), float(s * a.factor));
    }
  }
  // Where the token's K and V rows go; -1: nowhere (padding, or a bad sequence or page).
  int64_t row = -1;
  if (p >= 0) {
    const int block = p / a.block_size;
    if (seq >= 0 && seq < a.n_seqs && block < a.max_blocks) {
      const int32_t page = a.block_tables[int64_t(seq) * a.max_blocks + block];
      const int64_t off = int64_t(page) * a.stride_page + int64_t(p - block * a.block_size) * a.stride_row;
      if (page >= 0 && off + a.row_span <= a.cache_elems) row = off;
    }
    if (row < 0 && threadIdx.x == 0) *a.err = 1;
  }
  __syncthreads();

  const int rot_units = kNeighbours ? a.rotary_dim / V : half / V;
  const int rest_units = (a.head_dim - a.rotary_dim) / V;
  const int head_units = rot_units + rest_units;
  const int v_units = a.head_dim / V;
  const int qk_units = (a.n_heads + a.n_kv_heads) * head_units;
  const int units = qk_units + a.n_kv_heads * v_units;
  using C = Vec<T, V, kLoose>;
  for (int u = blockIdx.y * kThreads + threadIdx.x; u < units; u += gridDim.y * kThreads) {
    if (u >= qk_units) {
      const int h = (u - qk_units) / v_units, j = (u - qk_units) - h * v_units;
      if (row >= 0)
        *reinterpret_cast<C*>(static_cast<T*>(a.v_cache) + row + h * a.stride_head + j * V) =
            *reinterpret_cast<const C*>(static_cast<const T*>(a.v) + tok * a.v_tok + h * a.v_head + j * V);
      continue;
    }
    const int h = u / head_units, j = u - h * head_units;
    const bool is_q = h < a.n_heads;
    if (!is_q && row < 0) continue;
    const int hk = h - a.n_heads;
    const T* src = is_q ? static_cast<const T*>(a.q) + tok * a.q_tok + h * a.q_head
                        : static_cast<const T*>(a.k) + tok * a.k_tok + hk * a.k_head;
    T* dst = is_q ? static_cast<T*>(a.q_out) + tok * a.qo_tok + h * a.qo_head
                  : static_cast<T*>(a.k_cache) + row + hk * a.stride_head;
    if (j >= rot_units || p < 0) {
      // the unrotated rest, or a padding token's query: copied
      if (j >= rot_units) {
        const int e = a.rotary_dim + (j - rot_units) * V;
        *reinterpret_cast<C*>(dst + e) = *reinterpret_cast<const C*>(src + e);
      } else {
        const C x = *reinterpret_cast<const C*>(src + j * V);
        if constexpr (!kNeighbours) {
          const C y = *reinterpret_cast<const C*>(src + half + j * V);
          *reinterpret_cast<C*>(dst + half + j * V) = y;
        }
        *reinterpret_cast<C*>(dst + j * V) = x;
      }
      continue;
    }
    C x = *reinterpret_cast<const C*>(src + j * V);
    if constexpr (kNeighbours) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 t = cs[j * (V / 2) + i];
        const float x1 = to_f32(x.v[2 * i]), x2 = to_f32(x.v[2 * i + 1]);
        x.v[2 * i] = from_f32<T>(fmaf(x1, t.x, -x2 * t.y));
        x.v[2 * i + 1] = from_f32<T>(fmaf(x2, t.x, x1 * t.y));
      }
    } else {
      C y = *reinterpret_cast<const C*>(src + half + j * V);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 t = cs[j * V + i];
        const float x1 = to_f32(x.v[i]), x2 = to_f32(y.v[i]);
        x.v[i] = from_f32<T>(fmaf(x1, t.x, -x2 * t.y));
        y.v[i] = from_f32<T>(fmaf(x2, t.x, x1 * t.y));
      }
      *reinterpret_cast<C*>(dst + half + j * V) = y;
    }
    *reinterpret_cast<C*>(dst + j * V) = x;
  }
}

template <typename T, int V>
cudaError_t launch_v(const RopeArgs& a, dim3 grid, cudaStream_t s) {
  const size_t smem = size_t(a.rotary_dim / 2) * sizeof(float2);
  if (a.neighbours)
    rope_append_kernel<T, V < 2 ? 2 : V, true, V < 2><<<grid, kThreads, smem, s>>>(a);
  else
    rope_append_kernel<T, V, false, false><<<grid, kThreads, smem, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const RopeArgs& a, int width, dim3 grid, cudaStream_t s) {
  switch (width) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_v<T, 8>(a, grid, s);
      return cudaErrorInvalidValue;
    case 4: return launch_v<T, 4>(a, grid, s);
    case 2: return launch_v<T, 2>(a, grid, s);
    default: return launch_v<T, 1>(a, grid, s);
  }
}

}  // namespace

// The widest chunk (elements) that divides every row part, stride and address.
int rope_chunk_width(const RopeArgs& a, int esz) {
  const int part = a.neighbours ? a.rotary_dim : a.rotary_dim / 2;
  for (int w = 16 / esz; w > 1; w >>= 1) {
    bool ok = part % w == 0 && a.head_dim % w == 0 && (a.head_dim - a.rotary_dim) % w == 0;
    const int64_t strides[] = {a.q_tok, a.q_head, a.qo_tok, a.qo_head, a.k_tok, a.k_head, a.v_tok, a.v_head,
                               a.stride_page, a.stride_row, a.stride_head};
    for (int64_t st : strides) ok = ok && st % w == 0;
    const void* ptrs[] = {a.q, a.q_out, a.k, a.v, a.k_cache, a.v_cache};
    for (const void* q : ptrs) ok = ok && reinterpret_cast<uintptr_t>(q) % (w * esz) == 0;
    if (ok) return w;
  }
  return 1;
}

cudaError_t launch_rope_append(const RopeArgs& a, int dtype, int width, int n_sm, cudaStream_t s) {
  // Few tokens: a token's heads over several CTAs, until the GPU has about two a SM.
  const int head_units = a.neighbours ? a.head_dim / width : (a.head_dim - a.rotary_dim / 2) / width;
  const int64_t units = int64_t(a.n_heads + a.n_kv_heads) * head_units + int64_t(a.n_kv_heads) * (a.head_dim / width);
  const int64_t most = (units + kThreads - 1) / kThreads;
  int64_t y = (2 * int64_t(n_sm) + a.n_tokens - 1) / a.n_tokens;
  if (y > most) y = most;
  if (y > 65535) y = 65535;
  if (y < 1) y = 1;
  const dim3 grid(unsigned(a.n_tokens), unsigned(y));
  switch (dtype) {
    case 0: return launch_t<__nv_bfloat16>(a, width, grid, s);
    case 1: return launch_t<float>(a, width, grid, s);
    default: return launch_t<__half>(a, width, grid, s);
  }
}

}  // namespace vc

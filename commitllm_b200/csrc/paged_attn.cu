// Attention of each sequence's newest tokens over its paged K/V cache.
//
// For sequence s of n = seq_lens[s] cached rows and new token j of n_new, token
// j sees rows p < n - n_new + 1 + j:
//   out = sum_p softmax_p(scale * q . k_p) v_p,   lse = log sum_p exp(scale * q . k_p)
// (no visible row: out = 0, lse = -inf).  Bound by memory: every K and V row is
// read once, for 4 * n_new * group operations per element (group = query heads
// of one KV head), far under the tensor cores' rate for a few new tokens.
//
// Work split.  A unit is (sequence, KV head, tile of up to R query rows); its
// rows' keys come in tiles of 64.  All units' tiles are laid end to end and cut
// into equal contiguous ranges, one per worker CTA (a fixed number of CTAs that
// are all resident), so a ragged batch and a single long sequence both spread
// evenly without the host knowing the lengths.  A unit that one worker holds
// whole is written by it; the others' parts (running maximum, sum and
// unnormalised output, f32) go to the workspace and a second, dependent kernel
// joins them.  Parts are joined in a fixed order, so results do not depend on
// timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "vc_internal.h"

namespace vc {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 64;          // keys of a tile: 16 per warp
constexpr int kJoinThreads = 128;

// ------------------------------------------------------------- common parts

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }

// Cached rows of sequence s, held to what its block table can address.
__device__ __forceinline__ int64_t seq_len(const AttnArgs& a, int s) {
  const int64_t n = a.seq_lens[s];
  const int64_t cap = int64_t(a.max_blocks) * a.block_size;
  return n < 0 ? 0 : (n > cap ? cap : n);
}

__device__ __forceinline__ int64_t seq_tiles(const AttnArgs& a, int s) {
  return (seq_len(a, s) + kTile - 1) / kTile;
}

// Inclusive sum of v over the block's 128 threads.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) v += warp_sum[w];
  return v;
}

struct Place {        // where a worker's first tile lies
  int seq;
  int64_t seq_base;   // first tile of that sequence
  int64_t total;      // tiles in all
};

__device__ __forceinline__ int64_t chunk_of(int64_t total, int n_workers) {
  return (total + n_workers - 1) / n_workers;
}

// The sequence that holds tile `worker * chunk`, found by the whole block.
__device__ Place locate(const AttnArgs& a, int units, int worker) {
  __shared__ int64_t warp_sum[kWarps];
  __shared__ int64_t found_base, found_total;
  __shared__ int found_seq;
  int64_t v0 = 0, incl0 = 0, base = 0;
  for (int c = 0; c < a.n_seqs; c += kThreads) {
    const int s = c + threadIdx.x;
    const int64_t v = s < a.n_seqs ? seq_tiles(a, s) * units : 0;
    const int64_t incl = base + block_scan(v, warp_sum);
    if (c == 0) v0 = v, incl0 = incl;
    if (threadIdx.x == kThreads - 1) found_total = incl;
    __syncthreads();
    base = found_total;
  }
  const int64_t total = base;
  const int64_t begin = int64_t(worker) * chunk_of(total, a.n_workers);
  Place pl{0, 0, total};
  if (begin >= total) return pl;
  base = 0;
  for (int c = 0; c < a.n_seqs; c += kThreads) {
    int64_t v = v0, incl = incl0;
    if (c) {
      const int s = c + threadIdx.x;
      v = s < a.n_seqs ? seq_tiles(a, s) * units : 0;
      incl = base + block_scan(v, warp_sum);
    }
    if (incl - v <= begin && begin < incl) {
      found_seq = c + threadIdx.x;
      found_base = incl - v;
    }
    if (c + kThreads < a.n_seqs) {
      if (threadIdx.x == kThreads - 1) found_total = incl;
      __syncthreads();
      base = found_total;
      __syncthreads();
    }
  }
  __syncthreads();
  pl.seq = found_seq;
  pl.seq_base = found_base;
  return pl;
}

// Element offset of the row of key p, or -1 (a bad page, reported through err).
__device__ __forceinline__ int64_t row_of(const AttnArgs& a, int seq, int p) {
  const int block = unsigned(p) / unsigned(a.block_size);
  const int32_t page = __ldg(a.block_tables + int64_t(seq) * a.max_blocks + block);
  const int64_t off = int64_t(page) * a.stride_page + int64_t(p - block * a.block_size) * a.stride_row;
  if (page < 0 || off + a.row_span > a.cache_elems) {
    *a.err = 1;
    return -1;
  }
  return off;
}

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

// Row r of a KV head's query rows is new token r / group, head r % group of the group.
struct RowAt {
  int64_t q;       // element offset in q
  int64_t out;     // row index in out / lse
  int tok;
};
__device__ __forceinline__ RowAt row_at(const AttnArgs& a, int seq, int kvh, int r) {
  const int group = a.n_heads / a.n_kv_heads;
  const int tok = r / group, h = kvh * group + (r - tok * group);
  return {seq * a.q_seq + tok * a.q_tok + h * a.q_head, (int64_t(seq) * a.n_new + tok) * a.n_heads + h, tok};
}

// A part in the workspace: R rows of DP outputs, then R x (maximum, sum).
template <int R, int DP> constexpr int64_t part_floats() { return int64_t(R) * DP + 2 * R; }

// Shared memory of a unit's end: each warp's outputs, maxima (base-2 exponents) and sums.
template <int R, int DP>
struct Merge {
  float o[kWarps][R][DP];
  float m[kWarps][R];
  float l[kWarps][R];
};

// The warps' results of one unit (or part of one), joined and written.
template <typename T, int R, int DP>
__device__ __forceinline__ void emit(const AttnArgs& a, Merge<R, DP>& mg, int seq, int kvh, int row0, bool whole,
                                     float* part) {
  __syncthreads();
  constexpr int kPer = R * DP / 4;     // float4 groups
  for (int i = threadIdx.x; i < kPer; i += kThreads) {
    const int r = i / (DP / 4), d = (i - r * (DP / 4)) * 4;
    float top = mg.m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, mg.m[w][r]);
    const float ref = top == ninf() ? 0.f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(mg.m[w][r] - ref);
      l += f * mg.l[w][r];
      const float4 x = *reinterpret_cast<const float4*>(&mg.o[w][r][d]);
      o.x += f * x.x;
      o.y += f * x.y;
      o.z += f * x.z;
      o.w += f * x.w;
    }
    if (!whole) {
      *reinterpret_cast<float4*>(part + r * DP + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(part + R * DP + 2 * r) = make_float2(top, l);
      continue;
    }
    if (row0 + r >= a.rows || d >= a.head_dim) continue;
    const RowAt at = row_at(a, seq, kvh, row0 + r);
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);     // a NaN sum stays NaN
    T* out = static_cast<T*>(a.out) + at.out * a.head_dim + d;
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < a.head_dim) out[e] = from_f32<T>(y[e]);
    if (d == 0 && a.lse) a.lse[at.out] = l == 0.f ? ninf() : (top + log2f(l)) * 0.6931471805599453f;
  }
  __syncthreads();
}

// ------------------------------------------- 16-bit rows: tensor-core variant

template <typename T> struct Bits;
template <> struct Bits<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7F80;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Bits<__half> {
  static constexpr uint32_t kExp = 0x7C00;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// One warp's running state over the keys it is given, 16 at a time.  No shared
// memory: K and V go from global memory straight into tensor-core fragments.
//
// Scores S = Q K^T (m16n8k16, rows = query rows, columns = keys).  The products'
// inner index may be any order of the head's elements as long as Q and K agree,
// so lane (n, c) = (lane / 4, lane % 4) takes the 16-byte chunks 4i + c of key
// row n: its 8 elements are the B fragment of two inner steps, and the same
// chunk of Q's row n is their A fragment.  With R = 8 the fragment's rows 8..15
// are zeros.
//
// Outputs O^T = V^T P^T (rows = head elements, columns = query rows): the scores'
// accumulators, rounded, are P^T's B fragment without any exchange.  V^T's A
// fragment wants two keys' values of one element in a register: lane (r, c) loads
// chunk 8e + r of keys 2c, 2c+1, 2c+8, 2c+9 and pairs them with byte permutes.
//
// P is rounded to 16 bits twice (its value, then what that left over), so the
// products see 16 (bf16) or more bits of it; the row sums are taken in f32.  The
// loop waits on memory, and the second product of 8 is free.
template <typename T, int R, int DP>
struct TensorCore {
  static constexpr int kRows = R, kDP = DP;
  static constexpr int KS = DP / 32;      // 16-byte chunks a lane holds of a K row
  static constexpr int VS = DP / 64;      // ... and of each of its V rows
  static constexpr int RT = R / 8;        // column tiles of P^T
  using B = Bits<T>;

  uint32_t q[RT][KS][4];
  float o[RT][VS * 4][4];
  float m[RT], l[RT];
  int lim[RT];                 // rows seen: key < lim
  uint4 kf[2][KS];             // K rows n and n + 8 of the tile to come
  uint4 vf[4][VS];             // V rows of the four keys
  int64_t off;                 // lane i < 16: row offset of key i of the loaded tile, -1: none

  __device__ __forceinline__ void begin(const AttnArgs& a, int seq, int kvh, int row0, int len) {
    const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = row0 + t * 8 + n;
      const bool real = r < a.rows;
      const RowAt at = row_at(a, seq, kvh, real ? r : 0);
      lim[t] = real ? len - a.n_new + 1 + at.tok : 0;
      const T* src = static_cast<const T*>(a.q) + at.q;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int e = (i * 4 + c) * 8;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (real && e < a.head_dim) x = *reinterpret_cast<const uint4*>(src + e);
        q[t][i][0] = x.x, q[t][i][1] = x.y, q[t][i][2] = x.z, q[t][i][3] = x.w;
      }
      m[t] = ninf();
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < VS * 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][i][j] = 0.f;
    }
  }

  // Row offsets of the 16 keys from p0 (lane i < 16 holds key i's).
  __device__ __forceinline__ void find(const AttnArgs& a, int seq, int kvh, int p0, int len) {
    const int lane = threadIdx.x & 31;
    off = -1;
    if (lane < 16 && p0 + lane < len) {
      off = row_of(a, seq, p0 + lane);
      if (off >= 0) off += kvh * a.stride_head;
    }
  }

  __device__ __forceinline__ void load_k(const AttnArgs& a) {
    const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int64_t at = __shfl_sync(~0u, off, n + 8 * x);
      const T* src = static_cast<const T*>(a.k) + at;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int e = (i * 4 + c) * 8;
        kf[x][i] = make_uint4(0, 0, 0, 0);
        if (at >= 0 && e < a.head_dim) kf[x][i] = ldg16(src + e);
      }
    }
  }

  __device__ __forceinline__ void load_v(const AttnArgs& a) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int64_t at = __shfl_sync(~0u, off, 2 * c + (x & 1) + (x >> 1) * 8);
      const T* src = static_cast<const T*>(a.v) + at;
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const int e = (i * 8 + r) * 8;
        vf[x][i] = make_uint4(0, 0, 0, 0);
        if (at >= 0 && e < a.head_dim) vf[x][i] = ldg16(src + e);
      }
    }
  }

  static __device__ __forceinline__ uint32_t word(const uint4& v, int f) {
    return f == 0 ? v.x : f == 1 ? v.y : f == 2 ? v.z : v.w;
  }

  // acc += V^T P^T of the 16 keys for one column tile; key x of the lane's four dropped where `keep` says so.
  __device__ __forceinline__ void pv(float (&acc)[VS * 4][4], const uint32_t (&hi)[2], const uint32_t (&lo)[2],
                                     unsigned keep = 15u) {
#pragma unroll
    for (int i = 0; i < VS; ++i)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = (keep >> x) & 1 ? word(vf[x][i], f) : 0u;
        const uint32_t a0 = __byte_perm(w[0], w[1], 0x5410), a1 = __byte_perm(w[0], w[1], 0x7632);
        const uint32_t a2 = __byte_perm(w[2], w[3], 0x5410), a3 = __byte_perm(w[2], w[3], 0x7632);
        B::mma(acc[i * 4 + f], a0, a1, a2, a3, hi[0], hi[1]);
        B::mma(acc[i * 4 + f], a0, a1, a2, a3, lo[0], lo[1]);
      }
  }

  __device__ __forceinline__ bool wild() const {       // an infinity or NaN among the lane's V values
    bool bad = false;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < VS; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const uint32_t w = word(vf[x][i], f);
          bad = bad || (w & B::kExp) == B::kExp || ((w >> 16) & B::kExp) == B::kExp;
        }
    return bad;
  }

  // The 16 keys from p0, whose K rows are in kf; next_k then issues the next loads of K.
  template <typename NextK>
  __device__ __forceinline__ void keys(const AttnArgs& a, int p0, int len, int row0, NextK next_k) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    float s[RT][2][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[t][x][j] = 0.f;
    // with two column tiles, rows 8..15 of the fragment are the second one
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t r1a = RT == 2 ? q[RT - 1][i][0] : 0u, r1b = RT == 2 ? q[RT - 1][i][1] : 0u;
        const uint32_t r1c = RT == 2 ? q[RT - 1][i][2] : 0u, r1d = RT == 2 ? q[RT - 1][i][3] : 0u;
        B::mma(s[0][x], q[0][i][0], r1a, q[0][i][1], r1b, kf[x][i].x, kf[x][i].y);
        B::mma(s[0][x], q[0][i][2], r1c, q[0][i][3], r1d, kf[x][i].z, kf[x][i].w);
      }
    if constexpr (RT == 2) {
#pragma unroll
      for (int x = 0; x < 2; ++x) s[1][x][0] = s[0][x][2], s[1][x][1] = s[0][x][3];
    }
    next_k();
    uint32_t hi[RT][2], lo[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float top = ninf();
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int p = p0 + 8 * x + 2 * c + j;
          s[t][x][j] = p < lim[t] ? s[t][x][j] * a.scale_log2 : ninf();
          top = fmaxf(top, s[t][x][j]);
        }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      top = fmaxf(top, m[t]);
      if (__any_sync(~0u, top > m[t])) {
        // the maximum grew: what is summed so far shrinks (rarely after the first tiles)
        const float f = m[t] == ninf() ? 0.f : exp2f(m[t] - top);
        l[t] *= f;
        const float f0 = __shfl_sync(~0u, f, c * 8), f1 = __shfl_sync(~0u, f, c * 8 + 4);
#pragma unroll
        for (int i = 0; i < VS * 4; ++i) {
          o[t][i][0] *= f0, o[t][i][2] *= f0;
          o[t][i][1] *= f1, o[t][i][3] *= f1;
        }
        m[t] = top;
      }
      const float ref = m[t] == ninf() ? 0.f : m[t];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float e0 = exp2f(s[t][x][0] - ref), e1 = exp2f(s[t][x][1] - ref);
        l[t] += e0 + e1;
        hi[t][x] = B::pack(e0, e1);
        const float2 h = B::unpack(hi[t][x]);
        lo[t][x] = B::pack(e0 - h.x, e1 - h.y);
      }
    }
    // Rows that differ in what they see share this tile: 0 * infinity of a value that
    // only later tokens see must not reach an earlier token's row.
    const bool mixed = p0 + 16 > len - a.n_new + 1 && a.n_new > 1;
    if (mixed && __any_sync(~0u, wild())) {
      const int group = a.n_heads / a.n_kv_heads;
#pragma unroll 1
      for (int tok = row0 / group; tok < a.n_new && tok * group < row0 + R; ++tok) {
        unsigned keep = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (p0 + 2 * c + (x & 1) + (x >> 1) * 8 < len - a.n_new + 1 + tok) keep |= 1u << x;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          float acc[VS * 4][4] = {};
          pv(acc, hi[t], lo[t], keep);
          const int r = row0 + t * 8 + 2 * c;
          const bool c0 = r / group == tok, c1 = (r + 1) / group == tok;
#pragma unroll
          for (int i = 0; i < VS * 4; ++i) {
            if (c0) o[t][i][0] += acc[i][0], o[t][i][2] += acc[i][2];
            if (c1) o[t][i][1] += acc[i][1], o[t][i][3] += acc[i][3];
          }
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < RT; ++t) pv(o[t], hi[t], lo[t]);
    }
  }

  // Tiles [t0, t1) of the unit: this warp's 16 keys of each.
  __device__ __forceinline__ void run(const AttnArgs& a, int seq, int kvh, int row0, int len, int t0, int t1) {
    const int warp = threadIdx.x >> 5;
    int p0 = t0 * kTile + warp * 16;
    find(a, seq, kvh, p0, len);
    load_k(a);
    load_v(a);
    begin(a, seq, kvh, row0, len);
#pragma unroll 1
    for (int t = t0; t < t1; ++t, p0 += kTile) {
      const bool more = t + 1 < t1;
      keys(a, p0, len, row0, [&] {
        if (more) {
          find(a, seq, kvh, p0 + kTile, len);
          load_k(a);
        }
      });
      if (more) load_v(a);
    }
  }

  __device__ __forceinline__ void store(Merge<R, DP>& mg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      l[t] += __shfl_xor_sync(~0u, l[t], 1);
      l[t] += __shfl_xor_sync(~0u, l[t], 2);
      if (c == 0) mg.m[warp][t * 8 + r] = m[t], mg.l[warp][t * 8 + r] = l[t];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < VS; ++i) {
          float* dst = &mg.o[warp][t * 8 + 2 * c + j][(i * 8 + r) * 8];
#pragma unroll
          for (int f = 0; f < 4; ++f) dst[2 * f] = o[t][i * 4 + f][j], dst[2 * f + 1] = o[t][i * 4 + f][2 + j];
        }
    }
  }
};

// ---------------------------- f32 rows, and 16-bit rows of any alignment: FMAs

// Eight lanes share a key (four keys at a time, 16 per warp and tile); each holds
// DP / 8 of its elements.  V elements a load; element (i, e) of lane g is
// (i * 8 + g) * V + e.  The query rows sit in shared memory as f32, scaled.
template <typename T, int V, int DP>
struct Fma {
  static constexpr int R = 4;
  static constexpr int kRows = R, kDP = DP;
  static constexpr int NL = DP / 8 / V;       // loads of a row
  float o[R][NL * V];
  float m[R], l[R];
  int lim[R];

  struct alignas(sizeof(T) * V) Chunk {
    T v[V];
  };

  __device__ __forceinline__ void load(float (&x)[NL * V], const T* src, bool real, int dim) {
    const int g = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int e = (i * 8 + g) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) x[i * V + j] = 0.f;
      if (real && e < dim) {
        const Chunk ch = *reinterpret_cast<const Chunk*>(src + e);
#pragma unroll
        for (int j = 0; j < V; ++j) x[i * V + j] = to_f32(ch.v[j]);
      }
    }
  }

  __device__ __forceinline__ void run(const AttnArgs& a, int seq, int kvh, int row0, int len, int t0, int t1,
                                      float (*qs)[DP]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & 7;
    for (int i = threadIdx.x; i < R * DP; i += kThreads) {
      const int r = i / DP, d = i - r * DP;
      float x = 0.f;
      if (row0 + r < a.rows && d < a.head_dim)
        x = to_f32(static_cast<const T*>(a.q)[row_at(a, seq, kvh, row0 + r).q + d]);
      qs[r][d] = x;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool real = row0 + r < a.rows;
      lim[r] = real ? len - a.n_new + 1 + row_at(a, seq, kvh, row0 + r).tok : 0;
      m[r] = ninf();
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NL * V; ++i) o[r][i] = 0.f;
    }
    __syncthreads();
    const T* kb = static_cast<const T*>(a.k) + kvh * a.stride_head;
    const T* vb = static_cast<const T*>(a.v) + kvh * a.stride_head;
    const int n = (t1 - t0) * 4;               // steps of four keys
    float kx[NL * V], vx[NL * V];
    int p = t0 * kTile + warp * 16 + (lane >> 3);
    int64_t off = p < len ? row_of(a, seq, p) : -1;
    load(kx, kb + off, off >= 0, a.head_dim);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      load(vx, vb + off, off >= 0, a.head_dim);
      float s[R];
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] = 0.f;
#pragma unroll
      for (int e = 0; e < NL; ++e)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < V; ++j) s[r] = fmaf(qs[r][(e * 8 + g) * V + j], kx[e * V + j], s[r]);
      // the next four keys
      const int pn = (i & 3) == 3 ? p + kTile - 12 : p + 4;
      const int64_t offn = i + 1 < n && pn < len ? row_of(a, seq, pn) : -1;
      load(kx, kb + offn, offn >= 0, a.head_dim);
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) s[r] += __shfl_xor_sync(~0u, s[r], d);
        const bool seen = p < lim[r];
        const float x = seen ? s[r] * a.scale_log2 : ninf();
        // the eight lanes of a key keep their own maximum: keys of other lane groups join at the end
        const float top = fmaxf(m[r], x);
        const float ref = top == ninf() ? 0.f : top;
        const float f = exp2f(m[r] - ref);
        const float e = exp2f(x - ref);
        m[r] = top;
        l[r] = fmaf(l[r], f, e);
        if (seen) {
#pragma unroll
          for (int j = 0; j < NL * V; ++j) o[r][j] = fmaf(e, vx[j], o[r][j] * f);
        }
      }
      p = pn;
      off = offn;
    }
  }

  __device__ __forceinline__ void store(Merge<R, DP>& mg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & 7;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = fmaxf(m[r], __shfl_xor_sync(~0u, m[r], 8));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
      const float ref = top == ninf() ? 0.f : top;
      const float f = exp2f(m[r] - ref);
      float sum = l[r] * f;
      sum += __shfl_xor_sync(~0u, sum, 8);
      sum += __shfl_xor_sync(~0u, sum, 16);
      if (lane == 0) mg.m[warp][r] = top, mg.l[warp][r] = sum;
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float x = o[r][i * V + j] * f;
          x += __shfl_xor_sync(~0u, x, 8);
          x += __shfl_xor_sync(~0u, x, 16);
          if (lane < 8) mg.o[warp][r][(i * 8 + g) * V + j] = x;
        }
    }
  }
};

// ------------------------------------------------------------------ kernels

template <typename T, typename Core, bool kFma>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int R = Core::kRows, DP = Core::kDP;
  extern __shared__ __align__(16) char smem[];
  Merge<R, DP>& mg = *reinterpret_cast<Merge<R, DP>*>(smem);
  const int row_tiles = (a.rows + R - 1) / R;
  const int units = a.n_kv_heads * row_tiles;
  const Place pl = locate(a, units, blockIdx.x);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t chunk = chunk_of(pl.total, a.n_workers);
  int64_t cur = int64_t(blockIdx.x) * chunk;
  const int64_t end = cur + chunk < pl.total ? cur + chunk : pl.total;
  int seq = pl.seq;
  int64_t base = pl.seq_base;
  float* parts = a.parts + int64_t(blockIdx.x) * 2 * part_floats<R, DP>();
  while (cur < end) {
    const int64_t nt = seq_tiles(a, seq);
    if (cur >= base + nt * units) {
      base += nt * units;
      ++seq;
      continue;
    }
    const int unit = int((cur - base) / nt);
    const int t0 = int((cur - base) - unit * nt);
    const int t1 = nt - t0 < end - cur ? int(nt) : t0 + int(end - cur);
    const int kvh = unit / row_tiles, row0 = (unit - kvh * row_tiles) * R;
    const int len = int(seq_len(a, seq));
    Core core;
    if constexpr (kFma)
      core.run(a, seq, kvh, row0, len, t0, t1, mg.o[0]);      // the queries sit where the outputs will
    else
      core.run(a, seq, kvh, row0, len, t0, t1);
    if constexpr (kFma) __syncthreads();
    core.store(mg);
    // a part that begins its unit goes to slot 1, one that continues a unit to slot 0
    emit<T, R, DP>(a, mg, seq, kvh, row0, t0 == 0 && t1 == nt, parts + (t0 == 0 ? part_floats<R, DP>() : 0));
    cur += t1 - t0;
  }
}

// One query row: the parts of its unit joined in worker order; units that one
// worker held whole are done, units without a key get zeros.
template <typename T, int R, int DP>
__global__ void __launch_bounds__(kJoinThreads) paged_attn_join_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ int64_t warp_sum[kWarps];
  __shared__ float2 ml_all[kWarps];
  __shared__ float acc[kWarps][DP];
  const int row_tiles = (a.rows + R - 1) / R;
  const int units = a.n_kv_heads * row_tiles;
  const int seq = blockIdx.x / a.n_kv_heads, kvh = blockIdx.x - seq * a.n_kv_heads;
  const int row = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // tiles before this sequence, and in all
  int64_t before = 0, total = 0;
  for (int s = threadIdx.x; s < a.n_seqs; s += kJoinThreads) {
    const int64_t v = seq_tiles(a, s) * units;
    total += v;
    if (s < seq) before += v;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    total += __shfl_xor_sync(~0u, total, d);
    before += __shfl_xor_sync(~0u, before, d);
  }
  if (lane == 0) warp_sum[warp] = total;
  __syncthreads();
  total = warp_sum[0] + warp_sum[1] + warp_sum[2] + warp_sum[3];
  __syncthreads();
  if (lane == 0) warp_sum[warp] = before;
  __syncthreads();
  before = warp_sum[0] + warp_sum[1] + warp_sum[2] + warp_sum[3];
  const int64_t nt = seq_tiles(a, seq);
  const RowAt at = row_at(a, seq, kvh, row);
  T* out = static_cast<T*>(a.out) + at.out * a.head_dim;
  if (nt == 0) {
    for (int d = threadIdx.x; d < a.head_dim; d += kJoinThreads) out[d] = from_f32<T>(0.f);
    if (threadIdx.x == 0 && a.lse) a.lse[at.out] = ninf();
  }
  // every CTA waits for the first kernel, so that what follows this one does too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nt == 0) return;
  const int64_t chunk = chunk_of(total, a.n_workers);
  const int64_t first = before + int64_t(kvh * row_tiles + row / R) * nt;
  const int64_t wa = first / chunk, wb = (first + nt - 1) / chunk;
  if (wa == wb) return;
  const int r = row % R;
  constexpr int64_t kPart = part_floats<R, DP>();
  auto part = [&](int64_t w) { return a.parts + (w * 2 + (w == wa ? 1 : 0)) * kPart; };
  float top = ninf();
  for (int64_t w = wa + threadIdx.x; w <= wb; w += kJoinThreads) top = fmaxf(top, __ldcg(part(w) + R * DP + 2 * r));
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (lane == 0) ml_all[warp].x = top;
  __syncthreads();
  top = fmaxf(fmaxf(ml_all[0].x, ml_all[1].x), fmaxf(ml_all[2].x, ml_all[3].x));
  const float ref = top == ninf() ? 0.f : top;
  constexpr int kQ = DP / 4 / 32 ? DP / 4 / 32 : 1;      // float4 a lane
  float4 o[kQ] = {};
  float l = 0.f;
#pragma unroll 4
  for (int64_t w = wa + warp; w <= wb; w += kWarps) {
    const float* src = part(w);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + R * DP + 2 * r));
    const float f = exp2f(ml.x - ref);
    l += f * ml.y;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int d = (i * 32 + lane) * 4;
      if (d < DP) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(src + r * DP + d));
        o[i].x += f * x.x, o[i].y += f * x.y, o[i].z += f * x.z, o[i].w += f * x.w;
      }
    }
  }
  if (lane == 0) ml_all[warp].y = l;
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const int d = (i * 32 + lane) * 4;
    if (d < DP) *reinterpret_cast<float4*>(&acc[warp][d]) = o[i];
  }
  __syncthreads();
  l = ml_all[0].y + ml_all[1].y + ml_all[2].y + ml_all[3].y;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  for (int d = threadIdx.x; d < a.head_dim; d += kJoinThreads)
    out[d] = from_f32<T>((acc[0][d] + acc[1][d] + acc[2][d] + acc[3][d]) * inv);
  if (threadIdx.x == 0 && a.lse) a.lse[at.out] = l == 0.f ? ninf() : (top + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ variants

struct Variant {
  const void* main;
  const void* join;
  int rows, dp;
  size_t smem, part;
};

template <typename T, typename Core, bool kFma>
Variant variant() {
  constexpr int R = Core::kRows, DP = Core::kDP;
  return {reinterpret_cast<const void*>(&paged_attn_kernel<T, Core, kFma>),
          reinterpret_cast<const void*>(&paged_attn_join_kernel<T, R, DP>), R, DP, sizeof(Merge<R, DP>),
          size_t(part_floats<R, DP>()) * sizeof(float)};
}

constexpr int kVariants = 18;
const Variant& variant_at(int i) {
  using bf = __nv_bfloat16;
  using hf = __half;
  static const Variant v[kVariants] = {
      variant<bf, TensorCore<bf, 8, 64>, false>(),  variant<bf, TensorCore<bf, 8, 128>, false>(),
      variant<bf, TensorCore<bf, 8, 256>, false>(), variant<bf, TensorCore<bf, 16, 64>, false>(),
      variant<bf, TensorCore<bf, 16, 128>, false>(), variant<hf, TensorCore<hf, 8, 64>, false>(),
      variant<hf, TensorCore<hf, 8, 128>, false>(), variant<hf, TensorCore<hf, 8, 256>, false>(),
      variant<hf, TensorCore<hf, 16, 64>, false>(), variant<hf, TensorCore<hf, 16, 128>, false>(),
      variant<float, Fma<float, 4, 128>, true>(),   variant<float, Fma<float, 4, 256>, true>(),
      variant<float, Fma<float, 1, 128>, true>(),   variant<float, Fma<float, 1, 256>, true>(),
      variant<bf, Fma<bf, 1, 128>, true>(),         variant<bf, Fma<bf, 1, 256>, true>(),
      variant<hf, Fma<hf, 1, 128>, true>(),         variant<hf, Fma<hf, 1, 256>, true>(),
  };
  return v[i];
}

}  // namespace

namespace {

cudaError_t plan_variant(int v, int n_sm, AttnPlan* plan) {
  const Variant& k = variant_at(v);
  static int resident[kVariants];      // CTAs an SM holds; the same on every B200
  int n = __atomic_load_n(&resident[v], __ATOMIC_RELAXED);
  if (n == 0) {
    cudaError_t e = cudaSuccess;
    if (k.smem > 48 * 1024)
      e = cudaFuncSetAttribute(k.main, cudaFuncAttributeMaxDynamicSharedMemorySize, int(k.smem));
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k.main, kThreads, k.smem);
    if (e != cudaSuccess) return e;
    if (n < 1) return cudaErrorInvalidConfiguration;
    __atomic_store_n(&resident[v], n, __ATOMIC_RELAXED);
  }
  plan->variant = v;
  plan->n_workers = n * n_sm;
  plan->workspace = size_t(plan->n_workers) * 2 * k.part;
  return cudaSuccess;
}

// dtype: VC_DTYPE_BF16 / F32 / F16 (0 / 1 / 3); wide: 16-byte chunks everywhere.
int variant_for(const AttnArgs& a, int dtype, bool wide) {
  if (dtype != 1 && wide) {
    const int size = a.head_dim <= 64 ? 0 : a.head_dim <= 128 ? 1 : 2;
    return (dtype == 0 ? 0 : 5) + (a.rows > 8 && size < 2 ? 3 + size : size);
  }
  return (dtype == 1 ? (wide ? 10 : 12) : dtype == 0 ? 14 : 16) + (a.head_dim <= 128 ? 0 : 1);
}

}  // namespace

cudaError_t paged_attn_workspace(const AttnArgs& a, int dtype, int n_sm, size_t* bytes) {
  *bytes = 0;
  for (int wide = 0; wide < 2; ++wide) {
    AttnPlan p;
    const cudaError_t e = plan_variant(variant_for(a, dtype, wide != 0), n_sm, &p);
    if (e != cudaSuccess) return e;
    if (p.workspace > *bytes) *bytes = p.workspace;
  }
  return cudaSuccess;
}

cudaError_t plan_paged_attn(const AttnArgs& a, int dtype, int n_sm, AttnPlan* plan) {
  const int esz = dtype == 1 ? 4 : 2;
  const int64_t strides[] = {a.q_seq, a.q_tok, a.q_head, a.stride_page, a.stride_row, a.stride_head, a.head_dim};
  const void* ptrs[] = {a.q, a.k, a.v};
  bool wide = true;
  for (int64_t s : strides) wide = wide && s * esz % 16 == 0;
  for (const void* p : ptrs) wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  return plan_variant(variant_for(a, dtype, wide), n_sm, plan);
}

cudaError_t launch_paged_attn(const AttnArgs& args, const AttnPlan& plan, cudaStream_t s) {
  const Variant& k = variant_at(plan.variant);
  AttnArgs a = args;
  void* params[] = {&a};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.n_workers));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = k.smem;
  cfg.stream = s;
  cudaError_t e = cudaLaunchKernelExC(&cfg, k.main, params);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(a.n_seqs) * unsigned(a.n_kv_heads), unsigned(a.rows));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, k.join, params);
}

}  // namespace vc

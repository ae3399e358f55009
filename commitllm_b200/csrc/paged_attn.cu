// Attention of each sequence's newest tokens over its paged K/V cache.
//
// For sequence s of n = seq_lens[s] cached rows and new token j of n_new, token
// j sees rows p < n - n_new + 1 + j:
//   out = sum_p softmax_p(scale * q . k_p) v_p,   lse = log sum_p exp(scale * q . k_p)
// (no visible row: out = 0, lse = -inf).  Bound by memory: every K and V row is
// read once, for 4 * n_new * group operations per element (group = query heads
// of one KV head), far under the tensor cores' rate for a few new tokens.
//
// Work split.  All sequences' keys, in tiles of 64 (and what starting a sequence costs,
// counted as tiles), are laid end to end and cut into equal contiguous ranges; a worker
// CTA takes one range for one unit (KV head, tile of up to R query rows).  The number
// of ranges is set so that the workers are all resident at once, so a ragged batch and
// a single long sequence both spread evenly without the host knowing the lengths.  The units of a range
// are neighbouring CTAs: they read the heads of the same cache rows, which lie
// side by side in memory, at about the same time.  A sequence that lies in one
// range is written by its worker; the others' parts (running maximum, sum and
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

// Cached rows of sequence s, held to what its block table can address (a longer one is
// reported through err).
__device__ __forceinline__ int64_t seq_len(const AttnArgs& a, int s) {
  const int64_t n = a.seq_lens[s];
  const int64_t cap = int64_t(a.max_blocks) * a.block_size;
  if (n > cap) *a.err = 1;
  return n < 0 ? 0 : (n > cap ? cap : n);
}

__device__ __forceinline__ int64_t key_tiles(const AttnArgs& a, int s) {
  return (seq_len(a, s) + kTile - 1) / kTile;
}

// What a sequence counts for when the ranges are cut: kStart tiles for starting it
// (queries to read, a result to write: about two tiles' time; counting it took 1024-token
// drafts from 31 to 27 us) and its keys' tiles behind them.
constexpr int kStart = 2;
__device__ __forceinline__ int64_t seq_tiles(const AttnArgs& a, int s) {
  const int64_t n = key_tiles(a, s);
  return n ? n + kStart : 0;
}

// Inclusive sum of v over the block's W warps.
template <int W>
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
  for (int w = 0; w < W; ++w)
    if (w < warp) v += warp_sum[w];
  return v;
}

struct Place {        // where a range's first tile lies
  int seq;
  int64_t seq_base;   // first tile of that sequence
  int64_t total;      // tiles in all
};

__device__ __forceinline__ int64_t chunk_of(int64_t total, int n_ranges) {
  return (total + n_ranges - 1) / n_ranges;
}

// The sequence that holds tile `range * chunk`, found by the whole block.  The second
// pass has its own running sum: a warp may still be reading the first pass's total.
template <int W>
__device__ Place locate(const AttnArgs& a, int range) {
  __shared__ int64_t warp_sum[W];
  __shared__ int64_t found_base, found_total, passed;
  __shared__ int found_seq;
  int64_t v0 = 0, incl0 = 0, base = 0;
  for (int c = 0; c < a.n_seqs; c += (W * 32)) {
    const int s = c + threadIdx.x;
    const int64_t v = s < a.n_seqs ? seq_tiles(a, s) : 0;
    const int64_t incl = base + block_scan<W>(v, warp_sum);
    if (c == 0) v0 = v, incl0 = incl;
    if (threadIdx.x == (W * 32) - 1) found_total = incl;
    __syncthreads();
    base = found_total;
  }
  const int64_t total = base;
  const int64_t begin = int64_t(range) * chunk_of(total, a.n_ranges);
  Place pl{0, 0, total};
  if (begin >= total) return pl;
  base = 0;
  for (int c = 0; c < a.n_seqs; c += (W * 32)) {
    int64_t v = v0, incl = incl0;
    if (c) {
      const int s = c + threadIdx.x;
      v = s < a.n_seqs ? seq_tiles(a, s) : 0;
      incl = base + block_scan<W>(v, warp_sum);
    }
    if (incl - v <= begin && begin < incl) {
      found_seq = c + threadIdx.x;
      found_base = incl - v;
    }
    if (c + (W * 32) < a.n_seqs) {
      if (threadIdx.x == (W * 32) - 1) passed = incl;
      __syncthreads();
      base = passed;
      __syncthreads();
    }
  }
  __syncthreads();
  pl.seq = found_seq;
  pl.seq_base = found_base;
  return pl;
}

// The sequence that holds a tile, and what a warp needs of it.
// Tiles are counted from the range's first one (the 32-bit registers are needed).
struct Cursor {
  int seq, len, nt;
  int base;           // its first tile of keys
  __device__ __forceinline__ void at(const AttnArgs& a, int s, int b) {
    seq = s, base = b;
    len = int(seq_len(a, s));
    nt = (len + kTile - 1) / kTile;
    if (nt) base += kStart;
  }
  // The first tile of keys from `tile` on, if it is before `end`; else end.
  __device__ __forceinline__ int advance(const AttnArgs& a, int tile, int end) {
    while (tile < end && tile >= base + nt) at(a, seq + 1, base + nt);
    if (tile < base) tile = base;
    return tile < end ? tile : end;
  }
};

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

// 2^x for x <= 0, within 2^-22 of itself; nothing below 2^-126.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ln(2^m * l).  The power of two in l goes to m first: a reference far below the maximum
// makes both large, and their sum is not.
__device__ __forceinline__ float log_sum(float m, float l) {
  int k;
  const float f = frexpf(l, &k);
  return ((m + float(k)) + log2f(f)) * 0.6931471805599453f;
}

// Weights are taken relative to a reference that is at most 2^8 below the largest one
// seen: it follows the maximum only when that has grown by more, so the sums so far are
// seldom rescaled (a maximum of random scores grows in half of the first 30 tiles) and
// no weight passes 2^8, which f16 holds too.
constexpr float kSlack = 8.f;

// Shared memory of a unit's end: the outputs of R rows from W warps that saw different
// keys, D elements at a time, with their maxima (base-2 exponents) and sums.  Rows are
// padded by 16 bytes: a warp's stores then fall into different banks.
template <int W, int R, int D>
struct Merge {
  float o[W][R][D + 4];
  float m[W][R];       // then the factors of the warps' outputs
  float l[W][R];
  int64_t at[R];       // where the row goes (elements of out or of the part), -1: nowhere
};

// Where a unit's rows go: the outputs, or (part not null) a part of DP-element rows
// whose maxima and sums follow at ml.
struct Target {
  int seq, kvh, row0;
  float* part;
  float* ml;
};

// The W warps' results, joined and written, elements d0.. of each row; `first`: the
// maxima and sums are new.  Buffer row b is query row row0 + (b / 8) * step + b % 8.
// One copy of the code for all its uses: it runs once a unit, and code that runs once
// costs its fetching (inlined and unrolled it made a short call microseconds longer).
template <typename T, int W, int R, int D, int DP>
__device__ __noinline__ void emit(const AttnArgs& a, Merge<W, R, D>& mg, Target to, int step, bool first, int d0) {
  __syncthreads();
  if (first) {
    const int b = threadIdx.x;
    if (b < R) {
      const int r = (b >> 3) * step + (b & 7);
      float top = mg.m[0][b];
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, mg.m[w][b]);
      const float ref = top == ninf() ? 0.f : top;
      float f[W], l = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        f[w] = ex2(mg.m[w][b] - ref);
        l += f[w] * mg.l[w][b];
      }
      float inv = 1.f;
      int64_t at = -1;
      if (to.part) {
        *reinterpret_cast<float2*>(to.ml + 2 * r) = make_float2(top, l);
        at = int64_t(r) * DP;
      } else {
        inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);     // a NaN sum stays NaN
        if (to.row0 + r < a.rows) {
          const RowAt ra = row_at(a, to.seq, to.kvh, to.row0 + r);
          at = ra.out * a.head_dim;
          if (a.lse) a.lse[ra.out] = l == 0.f ? ninf() : log_sum(top, l);
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) mg.m[w][b] = f[w] * inv;
      mg.at[b] = at;
    }
    __syncthreads();
  }
#pragma unroll 2
  for (int i = threadIdx.x; i < R * D / 4; i += blockDim.x) {
    const int b = i / (D / 4), e = (i - b * (D / 4)) * 4, d = d0 + e;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = mg.m[w][b];
      const float4 x = *reinterpret_cast<const float4*>(&mg.o[w][b][e]);
      o.x += f * x.x;
      o.y += f * x.y;
      o.z += f * x.z;
      o.w += f * x.w;
    }
    const int64_t at = mg.at[b];
    if (to.part) {
      *reinterpret_cast<float4*>(to.part + at + d) = o;
    } else if (at >= 0 && d < a.head_dim) {
      T* out = static_cast<T*>(a.out) + at + d;
      const float y[4] = {o.x, o.y, o.z, o.w};
      if (d + 4 <= a.head_dim && a.wide_out) {
        struct alignas(4 * sizeof(T)) Four {
          T v[4];
        } four = {{from_f32<T>(y[0]), from_f32<T>(y[1]), from_f32<T>(y[2]), from_f32<T>(y[3])}};
        *reinterpret_cast<Four*>(out) = four;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < a.head_dim) out[j] = from_f32<T>(y[j]);
      }
    }
  }
  __syncthreads();
}

// ------------------------------------------- 16-bit rows: tensor-core variant

// kLift: weights reach 2^(kLift + kSlack), and a reference comes down again where a row's
// tile lies below 2^-kLift of it (weigh; 0: it only rises).
template <typename T> struct Bits;
template <> struct Bits<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7F80;
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Bits<__half> {
  static constexpr uint32_t kExp = 0x7C00;
  static constexpr float kLift = 7.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// 16 bytes from global to shared memory without a register; zeros where size is 0.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// What one worker keeps in shared memory: a ring of stages a warp (16 keys' K rows,
// then their V rows), then what the end of a unit needs.
template <int R, int DP>
struct TcShape {
  static constexpr int kStage = 16 * DP * 2 * 2;
  static constexpr int kStages = DP == 64 ? 6 : 3;      // 96 KB a CTA (DP = 256: 192 KB)
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr size_t kSmem = kRing + sizeof(Merge<kWarps, 8, DP>);
};

// Whether n 16-byte chunks of shared memory hold an infinity or a NaN (by the whole warp).
template <typename B>
__device__ __noinline__ bool not_finite(uint32_t addr, int n) {
  bool bad = false;
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr + i * 16));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    for (int j = 0; j < 4; ++j) bad = bad || (w[j] & B::kExp) == B::kExp || ((w[j] >> 16) & B::kExp) == B::kExp;
  }
  return __any_sync(~0u, bad);
}

// The halves of a V^T register (keys p and p + 1) that a row which sees keys below lim keeps.
__device__ __forceinline__ uint32_t seen_pair(int p, int lim) {
  return (p < lim ? 0xFFFFu : 0u) | (p + 1 < lim ? 0xFFFF0000u : 0u);
}

// o += V^T P^T in the columns (query rows) that belong to one token.
template <typename B>
__device__ __forceinline__ void pv_of_token(float (&o)[4], const uint32_t (&vf)[4], const uint32_t (&hi)[2],
                                            const uint32_t (&lo)[2], bool c0, bool c1) {
  float y[4] = {o[0], o[1], o[2], o[3]};
  B::mma(y, vf[0], vf[1], vf[2], vf[3], hi[0], hi[1]);
  B::mma(y, vf[0], vf[1], vf[2], vf[3], lo[0], lo[1]);
  if (c0) o[0] = y[0], o[2] = y[2];
  if (c1) o[1] = y[1], o[3] = y[3];
}

// Scores to weights for one column tile of 8 query rows (the lane's: lane / 4) and NB
// blocks of 16 keys (the lane's of block b: 16b + 2c + {0, 1, 8, 9}; those from `left`
// after 2c on are not seen): the running reference and sum, the sums so far where the
// reference moves, and the weights in two 16-bit parts.  A lane compares only its own
// scores with the reference; the row's maximum is exchanged where one of them passes
// it.  scale is not negative.
//
// A 16-bit number has 11 bits only down to 2^-14 in f16, and nothing below 2^-24.  Next to
// a key that takes almost all of the softmax, the others' weights would be lost from the
// products while the f32 sum still counted them: with a value of zero at that key
// they are the whole output.  So f16 weights are taken relative to 2^-kLift of the
// largest (2^15 is then the most that occurs), and where a row's scores of the tile all lie
// another 2^kLift lower the reference follows them down: every tile's largest weight is
// at least 2^-7 and its two parts' error, 2^-25 at most, 2^-18 of it.  The sums are
// f32 and may grow with that: to 2^kRoom for a row's weights, 2^96 for its outputs.  The
// test costs 1 % where instructions bound (35 rows over 159 MB: 62.2 -> 62.9 us).
constexpr float kRoom = 80.f;
template <typename B, int NB, int KS>
__device__ __forceinline__ void weigh(float (&s)[NB][2][2], float scale, bool all_seen, int left, int c, float& m, float& l,
                                      float (&o)[KS][4], uint32_t (&hi)[NB][2], uint32_t (&lo)[NB][2]) {
  if (!all_seen) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (16 * b + 8 * i + j >= left) s[b][i][j] = ninf();
  }
  float top = ninf();
#pragma unroll
  for (int b = 0; b < NB; ++b) top = fmaxf(top, fmaxf(fmaxf(s[b][0][0], s[b][0][1]), fmaxf(s[b][1][0], s[b][1][1])));
  top = top == ninf() ? top : top * scale;       // (-infinity * 0)
  bool move = __any_sync(~0u, top > m + (kSlack + B::kLift));
  if constexpr (B::kLift > 0) {
    unsigned low = __ballot_sync(~0u, top < m - B::kLift);      // by lane; then of a row's four
    low &= low >> 1;
    low &= low >> 2;
    move = move || (low & 0x11111111u);
  }
  if (move) {
    // what is summed so far shrinks to the new maximum, or grows
    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
    top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
    float to = fmaxf(top - B::kLift, m);
    if constexpr (B::kLift > 0) {
      float sum = l + __shfl_xor_sync(~0u, l, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      // (the sum's exponent, rounded up)
      const float least = m + (float((__float_as_int(sum) >> 23) - 126) - kRoom);
      if (top < m - B::kLift && top > ninf()) to = fminf(fmaxf(top - B::kLift, least), m);
    }
    const float f = m == ninf() ? 0.f : ex2(m - to);
    l *= f;
    const float f0 = __shfl_sync(~0u, f, c * 8), f1 = __shfl_sync(~0u, f, c * 8 + 4);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      o[i][0] *= f0, o[i][2] *= f0;
      o[i][1] *= f1, o[i][3] *= f1;
    }
    m = to;
  }
  const float ref = m == ninf() ? 0.f : m;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float e[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        e[j] = ex2(fmaf(s[b][i][j], scale, -ref));
        if (!all_seen && 16 * b + 8 * i + j >= left) e[j] = 0.f;
      }
      l += e[0] + e[1];
      hi[b][i] = B::pack(e[0], e[1]);
      const float2 h = B::unpack(hi[b][i]);
      lo[b][i] = B::pack(e[0] - h.x, e[1] - h.y);
    }
}

// Attention of up to R query rows on the tensor cores, K and V rows of 16-bit types.
//
// What bounds it is how many bytes are on their way: 6.5 TB/s at some 2 us of loaded
// latency needs 13 MB, 90 KB an SM.  Registers cannot hold that next to the
// accumulators (a first version did, and read at 4.9 TB/s), so every warp has its own
// ring of stages that cp.async fills two stages ahead, across sequence boundaries too;
// no warp waits for another but at a unit's end.  A copy instruction covers whole
// rows (requests for half lines measured 5.1 against 6.0 TB/s), rows are swizzled so that ldmatrix
// reads without bank conflicts, and block-table entries are read one stage early.
//
// Scores S = Q K^T (rows = query rows, columns = keys).  Outputs O^T = V^T P^T (rows =
// head elements, columns = query rows): the scores' accumulators, rounded, are P^T's
// fragment without any exchange, and ldmatrix.trans gives V^T.
//
// P is rounded to 16 bits twice (its value, then what that left over), so the
// products see 16 (bf16) or more bits of it (f16: see weigh) and the output keeps the
// error of its own rounding; the row sums are taken in f32.
//
// Measured: 1.34 GB (64 sequences of up to 8192 rows, 8 KV heads of 128) in 198 us and
// 1.07 GB (2 of 131072) in 164 us, 6.6 - 6.8 TB/s; DRAM 81 %, tensor pipe 21 % busy.
template <typename T, int R, int DP>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : 2) paged_attn_tc_kernel(const __grid_constant__ AttnArgs a) {
  using B = Bits<T>;
  using Shape = TcShape<R, DP>;
  constexpr int KS = DP / 16;          // inner steps of Q K^T, row tiles of O^T
  constexpr int NT = R / 8;            // column tiles of P^T
  constexpr int kStages = Shape::kStages;
  constexpr int kCols = DP / 8;        // 16-byte chunks of a row
  constexpr int kRowsPerCopy = 32 / kCols > 0 ? 32 / kCols : 1;
  extern __shared__ __align__(128) char smem[];
  using Mg = Merge<kWarps, 8, DP>;
  Mg& mg = *reinterpret_cast<Mg*>(smem + Shape::kRing);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_addr(smem) + warp * (kStages * Shape::kStage);
  const int row_tiles = (a.rows + R - 1) / R;
  const int units = a.n_kv_heads * row_tiles;
  const int range = blockIdx.x / units, unit = blockIdx.x - range * units;
  const int rt = unit / a.n_kv_heads, kvh = unit - rt * a.n_kv_heads, row0 = rt * R;
  const int group = a.n_heads / a.n_kv_heads;
  const Place pl = locate<kWarps>(a, range);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t chunk = chunk_of(pl.total, a.n_ranges), first = int64_t(range) * chunk;
  if (first >= pl.total) return;
  const int end = int(pl.total - first < chunk ? pl.total - first : chunk);

  // ---- loading: lane i < 16 finds key i's row, one stage before it is copied
  Cursor ahead;
  ahead.at(a, pl.seq, int(pl.seq_base - first));
  int next = 0;                // tile the registers below describe
  int page = 0, slot = -1;             // -1: the lane has no row
  auto look = [&]() {
    slot = -1;
    next = ahead.advance(a, next, end);
    if (next < end) {
      const int p = (next - ahead.base) * kTile + warp * 16 + lane;
      if (lane < 16 && p < ahead.len) {
        const int block = unsigned(p) / unsigned(a.block_size);
        page = __ldg(a.block_tables + int64_t(ahead.seq) * a.max_blocks + block);
        slot = p - block * a.block_size;
      }
    }
  };
  int fill = 0;                        // stage to fill
  auto issue = [&]() {
    if (next < end) {
      int64_t off = -1;
      if (slot >= 0) {
        off = int64_t(page) * a.stride_page + int64_t(slot) * a.stride_row;
        if (page < 0 || off + a.row_span > a.cache_elems) {
          *a.err = 1;
          off = -1;
        } else {
          off += kvh * a.stride_head;
        }
      }
      ++next;
      look();
      const uint32_t dst = ring + fill * Shape::kStage;
#pragma unroll
      for (int j = 0; j < 16; j += kRowsPerCopy) {
        const int row = j + (kCols < 32 ? lane / kCols : 0), col = lane % kCols;
        const int64_t o = __shfl_sync(~0u, off, row);
        const int size = o >= 0 && col * 8 < a.head_dim ? 16 : 0;
        const int64_t at = size ? o + col * 8 : 0;
        const uint32_t d = dst + row * (DP * 2) + ((col ^ (row & 7)) << 4);
        copy16(d, static_cast<const T*>(a.k) + at, size);
        copy16(d + 16 * DP * 2, static_cast<const T*>(a.v) + at, size);
      }
    }
    fill = fill + 1 == kStages ? 0 : fill + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look();
  for (int i = 0; i < kStages - 1; ++i) issue();

  // ---- one sequence's part of the range after the other
  // lane's row and half of the four 8x8 blocks that a ldmatrix reads
  const int key = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1, flip = lane & 7;
  uint32_t q[KS][4];
  float o[NT][KS][4];
  float m[NT], l[NT];
  int lim[NT];
  int use = 0;                         // stage to use
  Cursor now;
  now.at(a, pl.seq, int(pl.seq_base - first));
  int cur = 0;
  while ((cur = now.advance(a, cur, end)) < end) {
    const int seq = now.seq, len = now.len;
    const int t0 = cur - now.base;
    const int t1 = now.nt - t0 < end - cur ? now.nt : t0 + (end - cur);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + h * 8 + n;
        const bool has = h * 8 < R && r < a.rows;
        const T* src = static_cast<const T*>(a.q) + row_at(a, seq, kvh, has ? r : 0).q;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int e = ks * 16 + x * 8 + 2 * c;
            q[ks][h + 2 * x] = has && e < a.head_dim ? *reinterpret_cast<const uint32_t*>(src + e) ^ a.q_sign : 0u;
          }
      }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = row0 + t * 8 + n;
      lim[t] = r < a.rows ? len - a.n_new + 1 + r / group : 0;
      m[t] = ninf();
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][i][j] = 0.f;
    }
#pragma unroll 1
    for (int p0 = t0 * kTile + warp * 16; p0 < t1 * kTile; p0 += kTile) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();                    // the stage has landed for all lanes, and the one before is free
      issue();
      const uint32_t kst = ring + use * Shape::kStage, vst = kst + 16 * DP * 2;
      use = use + 1 == kStages ? 0 : use + 1;
      float s[2][4] = {};
      // fragments are read one step ahead of the products that use them
      uint32_t kf[2][4];
      ldsm(kst + key * (DP * 2) + ((half ^ flip) << 4), kf[0]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + 1 < KS) ldsm(kst + key * (DP * 2) + ((((ks + 1) * 2 + half) ^ flip) << 4), kf[(ks + 1) & 1]);
        const uint32_t(&k)[4] = kf[ks & 1];
        B::mma(s[0], q[ks][0], q[ks][1], q[ks][2], q[ks][3], k[0], k[1]);
        B::mma(s[1], q[ks][0], q[ks][1], q[ks][2], q[ks][3], k[2], k[3]);
      }
      const int sure = len - a.n_new + 1;        // every row sees the keys before it
      const bool all_seen = p0 + 16 <= sure;
      uint32_t hi[NT][1][2], lo[NT][1][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[1][2][2] = {{{s[0][t * 2], s[0][t * 2 + 1]}, {s[1][t * 2], s[1][t * 2 + 1]}}};
        weigh<B, 1, KS>(x, a.scale_log2, all_seen, lim[t] - p0 - 2 * c, c, m[t], l[t], o[t], hi[t], lo[t]);
      }
      const uint32_t vrow = vst + key * (DP * 2);
      // Rows that see different keys share this tile: 0 * infinity of a value that only
      // later tokens see must not reach an earlier token's row.
      const bool wild = !all_seen && a.n_new > 1 && not_finite<B>(vst, 16 * kCols);
      if (!wild) {
        uint32_t vf[2][4];
        ldsm_t(vrow + ((half ^ flip) << 4), vf[0]);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          if (i + 1 < KS) ldsm_t(vrow + ((((i + 1) * 2 + half) ^ flip) << 4), vf[(i + 1) & 1]);
          const uint32_t(&v)[4] = vf[i & 1];
#pragma unroll
          for (int t = 0; t < NT; ++t) B::mma(o[t][i], v[0], v[1], v[2], v[3], hi[t][0][0], hi[t][0][1]);
#pragma unroll
          for (int t = 0; t < NT; ++t) B::mma(o[t][i], v[0], v[1], v[2], v[3], lo[t][0][0], lo[t][0][1]);
        }
      } else {
        // token by token: keys that it does not see become zeros, and only its columns are kept
#pragma unroll 1
        for (int tok = row0 / group; tok < a.n_new && tok * group < row0 + R; ++tok) {
          const uint32_t m0 = seen_pair(p0 + 2 * c, sure + tok), m1 = seen_pair(p0 + 2 * c + 8, sure + tok);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            uint32_t vf[4];
            ldsm_t(vrow + (((i * 2 + half) ^ flip) << 4), vf);
            vf[0] &= m0, vf[1] &= m0, vf[2] &= m1, vf[3] &= m1;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const int r = row0 + t * 8 + 2 * c;
              pv_of_token<B>(o[t][i], vf, hi[t][0], lo[t][0], r / group == tok, (r + 1) / group == tok);
            }
          }
        }
      }
    }
    // the four warps' results, eight rows at a time; a part that begins its sequence
    // goes to slot 1, one that continues it to slot 0
    const bool whole = t0 == 0 && t1 == now.nt;
    float* part = a.parts + (int64_t(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * part_floats<R, DP>();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float sum = l[t] + __shfl_xor_sync(~0u, l[t], 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      if (c == 0) mg.m[warp][n] = m[t], mg.l[warp][n] = sum;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mg.o[warp][2 * c + (j & 1)][i * 16 + (j >> 1) * 8 + n] = o[t][i][j];
      emit<T, kWarps, 8, DP, DP>(a, mg, {seq, kvh, row0 + t * 8, whole ? nullptr : part + t * 8 * DP, part + R * DP + t * 16}, 8,
                                 true, 0);
    }
    cur += t1 - t0;
  }
}

// More than 16 query rows (drafted tokens): the CTA's warps share each stage of 64 keys,
// WR row tiles of 16 query rows times two halves of the keys, one warp each.  A warp that
// held all rows would need 255 registers and leave two warps a scheduler; here it is
// three, with 92 B/clk of shared memory reads at the HBM's rate, of 128.  Bound by
// instruction latency, not by the bytes: 35 rows over 16 sequences of up to 8192 (159
// MB) take 63 us (68 with the queries in registers, which spilled), eight times longer
// ones 320 us where the bytes take 195 (21 rows: 234); tensor pipe 42 %, 0.41 instructions
// a cycle and scheduler, most stalls on fixed latencies.  Two blocks of 16 keys side by
// side gave 8 % over one.  Row tiles of 8, five warps a scheduler with 96 registers,
// spilled and took 91 us; leaving out the products of column tiles without a query row
// gave 4 % at 35 rows and cost 6 % at 21 and 42.
template <int WR, int DP>
struct RowsShape {
  static constexpr int kWarpsHere = WR * 2;
  static constexpr int kStage = kTile * DP * 2 * 2;
  static constexpr int kStages = DP == 64 ? 6 : 3;
  static constexpr int kRing = kStages * kStage;             // 96 KB
  using Mg = Merge<2, WR * 8, DP / 2>;      // 8 rows of each row tile, half of their elements
  // three row tiles leave 168 registers a thread: their queries stay in shared memory,
  // where the outputs will be
  static constexpr bool kQShared = WR > 2;
  static constexpr size_t kTail = kQShared && WR * 16 * DP * 2 > sizeof(Mg) ? WR * 16 * DP * 2 : sizeof(Mg);
  static constexpr size_t kSmem = kRing + kTail;
};

template <typename T, int WR, int DP>
__global__ void __launch_bounds__(WR * 64, 2) paged_attn_rows_kernel(const __grid_constant__ AttnArgs a) {
  using B = Bits<T>;
  using Shape = RowsShape<WR, DP>;
  constexpr int R = WR * 16;
  constexpr int KS = DP / 16;
  constexpr int kStages = Shape::kStages, kW = Shape::kWarpsHere;
  constexpr int kCols = DP / 8;                        // 16-byte chunks of a row
  constexpr int kRowsPerCopy = 32 / kCols;
  constexpr int kCopies = (kTile / kRowsPerCopy + kW - 1) / kW;      // a warp's, of K and of V
  extern __shared__ __align__(128) char smem[];
  typename Shape::Mg& mg = *reinterpret_cast<typename Shape::Mg*>(smem + Shape::kRing);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  const int wr = warp >> 1, kh = warp & 1;
  const uint32_t ring = smem_addr(smem);
  const int row_tiles = (a.rows + R - 1) / R;
  const int units = a.n_kv_heads * row_tiles;
  const int range = blockIdx.x / units, unit = blockIdx.x - range * units;
  const int rt = unit / a.n_kv_heads, kvh = unit - rt * a.n_kv_heads;
  const int row0 = rt * R, wrow0 = row0 + wr * 16;
  const int group = a.n_heads / a.n_kv_heads;
  const Place pl = locate<kW>(a, range);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t chunk = chunk_of(pl.total, a.n_ranges), first = int64_t(range) * chunk;
  if (first >= pl.total) return;
  const int end = int(pl.total - first < chunk ? pl.total - first : chunk);

  // ---- loading: a warp copies every kW-th group of kRowsPerCopy rows; lane i finds the i-th of its rows
  Cursor ahead;
  ahead.at(a, pl.seq, int(pl.seq_base - first));
  int next = 0;
  int page = 0, slot = -1;             // -1: the lane has no row
  const int my_group = warp + lane / kRowsPerCopy * kW, my_row = my_group * kRowsPerCopy + lane % kRowsPerCopy;
  auto look = [&]() {
    slot = -1;
    next = ahead.advance(a, next, end);
    if (next < end) {
      const int p = (next - ahead.base) * kTile + my_row;
      if (lane < kCopies * kRowsPerCopy && my_row < kTile && p < ahead.len) {
        const int block = unsigned(p) / unsigned(a.block_size);
        page = __ldg(a.block_tables + int64_t(ahead.seq) * a.max_blocks + block);
        slot = p - block * a.block_size;
      }
    }
  };
  int fill = 0;
  auto issue = [&]() {
    if (next < end) {
      int64_t off = -1;
      if (slot >= 0) {
        off = int64_t(page) * a.stride_page + int64_t(slot) * a.stride_row;
        if (page < 0 || off + a.row_span > a.cache_elems) {
          *a.err = 1;
          off = -1;
        } else {
          off += kvh * a.stride_head;
        }
      }
      ++next;
      look();
      const uint32_t dst = ring + fill * Shape::kStage;
#pragma unroll
      for (int j = 0; j < kCopies; ++j) {
        const int row = (warp + j * kW) * kRowsPerCopy + lane / kCols, col = lane % kCols;
        const int64_t o = __shfl_sync(~0u, off, j * kRowsPerCopy + lane / kCols);
        if (row < kTile) {
          const int size = o >= 0 && col * 8 < a.head_dim ? 16 : 0;
          const int64_t at = size ? o + col * 8 : 0;
          const uint32_t d = dst + row * (DP * 2) + ((col ^ (row & 7)) << 4);
          copy16(d, static_cast<const T*>(a.k) + at, size);
          copy16(d + kTile * DP * 2, static_cast<const T*>(a.v) + at, size);
        }
      }
    }
    fill = fill + 1 == kStages ? 0 : fill + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look();
  for (int i = 0; i < kStages - 1; ++i) issue();

  const int key = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1, flip = lane & 7;
  uint32_t q[Shape::kQShared ? 1 : KS][4];
  const int qrow = wr * 16 + half * 8 + (lane & 7);
  const uint32_t qs = smem_addr(smem + Shape::kRing) + qrow * (DP * 2);
  float o[2][KS][4];
  float m[2], l[2];
  int lim[2];
  int use = 0;
  Cursor now;
  now.at(a, pl.seq, int(pl.seq_base - first));
  int cur = 0;
  while ((cur = now.advance(a, cur, end)) < end) {
    const int seq = now.seq, len = now.len;
    const int t0 = cur - now.base;
    const int t1 = now.nt - t0 < end - cur ? now.nt : t0 + (end - cur);
    if constexpr (Shape::kQShared) {
      for (int i = threadIdx.x; i < R * kCols; i += WR * 64) {
        const int r = i / kCols, col = i - r * kCols;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row0 + r < a.rows && col * 8 < a.head_dim)
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + row_at(a, seq, kvh, row0 + r).q + col * 8);
        x.x ^= a.q_sign, x.y ^= a.q_sign, x.z ^= a.q_sign, x.w ^= a.q_sign;
        *reinterpret_cast<uint4*>(smem + Shape::kRing + r * (DP * 2) + ((col ^ (r & 7)) << 4)) = x;
      }
      __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = wrow0 + h * 8 + n;
      const bool has = r < a.rows;
      if constexpr (!Shape::kQShared) {
        const T* src = static_cast<const T*>(a.q) + row_at(a, seq, kvh, has ? r : 0).q;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int e = ks * 16 + x * 8 + 2 * c;
            q[ks][h + 2 * x] = has && e < a.head_dim ? *reinterpret_cast<const uint32_t*>(src + e) ^ a.q_sign : 0u;
          }
      }
      lim[h] = has ? len - a.n_new + 1 + r / group : 0;
      m[h] = ninf();
      l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[h][i][j] = 0.f;
    }
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncthreads();                 // the stage has landed for all warps, and the one before is free
      issue();
      const uint32_t kst = ring + use * Shape::kStage, vst = kst + kTile * DP * 2;
      use = use + 1 == kStages ? 0 : use + 1;
      const int sure = len - a.n_new + 1;
      // the warp's 32 keys as two blocks of 16 side by side: four independent chains of products
      const int at = kh * 32, p0 = t * kTile + at;     // rows of the stage
      const uint32_t krow = kst + (at + key) * (DP * 2), vrow = vst + (at + key) * (DP * 2);
      constexpr uint32_t kBlock = 16 * DP * 2;
      float s[2][2][4] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t f[4];
        if constexpr (Shape::kQShared) {
          // blocks of a Q fragment: rows 0-7 and 8-15 of the left half, then of the right
          ldsm(qs + (((ks * 2 + (lane >> 4)) ^ flip) << 4), f);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = q[ks][j];
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t k[4];
          ldsm(krow + b * kBlock + (((ks * 2 + half) ^ flip) << 4), k);
          B::mma(s[b][0], f[0], f[1], f[2], f[3], k[0], k[1]);
          B::mma(s[b][1], f[0], f[1], f[2], f[3], k[2], k[3]);
        }
      }
      const bool all_seen = p0 + 32 <= sure;
      uint32_t hi[2][2][2], lo[2][2][2];               // [column tile][block]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[2][2][2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 2; ++i) x[b][i][0] = s[b][i][h * 2], x[b][i][1] = s[b][i][h * 2 + 1];
        weigh<B, 2, KS>(x, a.scale_log2, all_seen, lim[h] - p0 - 2 * c, c, m[h], l[h], o[h], hi[h], lo[h]);
      }
      // rows that see different keys share this tile: see paged_attn_tc_kernel
      const bool wild = !all_seen && a.n_new > 1 && not_finite<B>(vst + at * (DP * 2), 32 * kCols);
      if (!wild) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            uint32_t v[4];
            ldsm_t(vrow + b * kBlock + (((i * 2 + half) ^ flip) << 4), v);
#pragma unroll
            for (int h = 0; h < 2; ++h) B::mma(o[h][i], v[0], v[1], v[2], v[3], hi[h][b][0], hi[h][b][1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) B::mma(o[h][i], v[0], v[1], v[2], v[3], lo[h][b][0], lo[h][b][1]);
          }
      } else {
#pragma unroll 1
        for (int tok = wrow0 / group; tok < a.n_new && tok * group < wrow0 + 16; ++tok) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int pb = p0 + 16 * b + 2 * c;
            const uint32_t m0 = seen_pair(pb, sure + tok), m1 = seen_pair(pb + 8, sure + tok);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              uint32_t vf[4];
              ldsm_t(vrow + b * kBlock + (((i * 2 + half) ^ flip) << 4), vf);
              vf[0] &= m0, vf[1] &= m0, vf[2] &= m1, vf[3] &= m1;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int r = wrow0 + h * 8 + 2 * c;
                pv_of_token<B>(o[h][i], vf, hi[h][b], lo[h][b], r / group == tok, (r + 1) / group == tok);
              }
            }
          }
        }
      }
    }
    // the key halves' results: query rows 0-7 or 8-15 of each row tile, and half of their
    // elements, at a time; buffer row 8 * wr + n is query row row0 + 16 * wr + 8 * h + n
    const bool whole = t0 == 0 && t1 == now.nt;
    if constexpr (Shape::kQShared) __syncthreads();      // the queries make place
    float* part = a.parts + (int64_t(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * part_floats<R, DP>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = l[h] + __shfl_xor_sync(~0u, l[h], 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      if (c == 0) mg.m[kh][wr * 8 + n] = m[h], mg.l[kh][wr * 8 + n] = sum;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
#pragma unroll
        for (int i = 0; i < KS / 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mg.o[kh][wr * 8 + 2 * c + (j & 1)][i * 16 + (j >> 1) * 8 + n] = o[h][z * (KS / 2) + i][j];
        emit<T, 2, WR * 8, DP / 2, DP>(a, mg, {seq, kvh, row0 + 8 * h, whole ? nullptr : part + 8 * h * DP, part + R * DP + 16 * h}, 16,
                                       z == 0, z * (DP / 2));
      }
    }
    cur += t1 - t0;
  }
}

// ----------------------------------------------- rows of any alignment: FMAs

// Eight lanes share a key (four keys at a time, 16 per warp and tile); each holds
// DP / 8 of its elements, one a load: number i of lane g is i * 8 + g.  The query rows
// sit in shared memory as f32.  Bound by the instructions of loads of one element:
// heads of 66 elements, 32 sequences of 4096 keys, 8 KV heads and 4 query rows take 418 us
// in bf16 (277 MB, 0.66 TB/s) and 243 in f32 (554 MB, 2.28 TB/s).
template <typename T, int DP>
struct Fma {
  static constexpr int R = 4;
  static constexpr int kRows = R, kDP = DP;
  static constexpr int NL = DP / 8;           // elements of a lane
  float o[R][NL];
  float m[R], l[R];
  int lim[R];

  __device__ __forceinline__ void load(float (&x)[NL], const T* src, bool real, int dim) {
    const int g = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < NL; ++i) x[i] = real && i * 8 + g < dim ? to_f32(src[i * 8 + g]) : 0.f;
  }

  __device__ __forceinline__ void run(const AttnArgs& a, int seq, int kvh, int row0, int len, int t0, int t1,
                                      float (*qs)[DP + 4]) {
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
      for (int i = 0; i < NL; ++i) o[r][i] = 0.f;
    }
    __syncthreads();
    const T* kb = static_cast<const T*>(a.k) + kvh * a.stride_head;
    const T* vb = static_cast<const T*>(a.v) + kvh * a.stride_head;
    const int n = (t1 - t0) * 4;               // steps of four keys
    float kx[NL], vx[NL];
    int p = t0 * kTile + warp * 16 + (lane >> 3);
    int64_t off = p < len ? row_of(a, seq, p) : -1;
    load(kx, kb + off, off >= 0, a.head_dim);
    load(vx, vb + off, off >= 0, a.head_dim);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      // the next four keys' rows are found now, and loaded as soon as this step's are used
      const int pn = (i & 3) == 3 ? p + kTile - 12 : p + 4;
      const int64_t offn = i + 1 < n && pn < len ? row_of(a, seq, pn) : -1;
      float s[R];
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] = 0.f;
#pragma unroll
      for (int e = 0; e < NL; ++e)
#pragma unroll
        for (int r = 0; r < R; ++r)
          s[r] = fmaf(qs[r][e * 8 + g], kx[e], s[r]);
      load(kx, kb + offn, offn >= 0, a.head_dim);
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) s[r] += __shfl_xor_sync(~0u, s[r], d);
        const bool seen = p < lim[r];
        const float x = seen ? s[r] * a.scale_log2 : ninf();
        // the eight lanes of a key keep their own reference: the other keys' lanes join at the end
        if (__any_sync(~0u, x > m[r] + kSlack)) {
          const float top = fmaxf(m[r], x);
          const float f = m[r] == ninf() ? 0.f : ex2(m[r] - top);
          l[r] *= f;
#pragma unroll
          for (int j = 0; j < NL; ++j) o[r][j] *= f;
          m[r] = top;
        }
        const float ref = m[r] == ninf() ? 0.f : m[r];
        const float e = ex2(x - ref);
        l[r] += e;
        if (seen) {
#pragma unroll
          for (int j = 0; j < NL; ++j) o[r][j] = fmaf(e, vx[j], o[r][j]);
        }
      }
      load(vx, vb + offn, offn >= 0, a.head_dim);
      p = pn;
      off = offn;
    }
  }

  __device__ __forceinline__ void store(Merge<kWarps, R, DP>& mg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & 7;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = fmaxf(m[r], __shfl_xor_sync(~0u, m[r], 8));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
      const float ref = top == ninf() ? 0.f : top;
      const float f = ex2(m[r] - ref);
      float sum = l[r] * f;
      sum += __shfl_xor_sync(~0u, sum, 8);
      sum += __shfl_xor_sync(~0u, sum, 16);
      if (lane == 0) mg.m[warp][r] = top, mg.l[warp][r] = sum;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        float x = o[r][i] * f;
        x += __shfl_xor_sync(~0u, x, 8);
        x += __shfl_xor_sync(~0u, x, 16);
        if (lane < 8) mg.o[warp][r][i * 8 + g] = x;
      }
    }
  }
};

// ------------------------------------------------------------------ kernels

template <typename T, typename Core>
__global__ void __launch_bounds__(kThreads) paged_attn_fma_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int R = Core::kRows, DP = Core::kDP;
  extern __shared__ __align__(128) char smem[];
  using Mg = Merge<kWarps, R, DP>;
  Mg& mg = *reinterpret_cast<Mg*>(smem);
  const int row_tiles = (a.rows + R - 1) / R;
  const int units = a.n_kv_heads * row_tiles;
  const int range = blockIdx.x / units, unit = blockIdx.x - range * units;
  const int rt = unit / a.n_kv_heads, kvh = unit - rt * a.n_kv_heads, row0 = rt * R;
  const Place pl = locate<kWarps>(a, range);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t chunk = chunk_of(pl.total, a.n_ranges), first = int64_t(range) * chunk;
  if (first >= pl.total) return;
  const int end = int(pl.total - first < chunk ? pl.total - first : chunk);
  int cur = 0;
  Cursor now;
  now.at(a, pl.seq, int(pl.seq_base - first));
  while ((cur = now.advance(a, cur, end)) < end) {
    const int seq = now.seq, len = now.len, nt = now.nt;
    const int t0 = cur - now.base;
    const int t1 = nt - t0 < end - cur ? nt : t0 + (end - cur);
    Core core;
    core.run(a, seq, kvh, row0, len, t0, t1, mg.o[0]);      // the queries sit where the outputs will
    __syncthreads();
    core.store(mg);
    // a part that begins its sequence goes to slot 1, one that continues it to slot 0
    float* part = a.parts + (int64_t(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * part_floats<R, DP>();
    emit<T, kWarps, R, DP, DP>(a, mg, {seq, kvh, row0, t0 == 0 && t1 == nt ? nullptr : part, part + R * DP}, 8, true, 0);
    cur += t1 - t0;
  }
}

// f32 rows on 16-byte boundaries: the ring of paged_attn_tc_kernel in stages of 8 keys,
// with the products in f32 FMAs (512 a lane for 8 keys and 8 query rows).  Eight lanes
// share a key, four keys at a time; a lane's elements of a row are chunks i * 8 + lane %
// 8 of four.  Measured on 318 MB: 4 query rows 62 us (5.2 TB/s; 79 with loads straight
// into registers, one step ahead), 7 rows 82 us, where the instructions bound it; a call
// of 20 MB and 6 rows takes 20.6 us, most of it starting up.  Packed pairs of FMAs
// measured no faster.
template <int R, int DP>
struct F32Shape {
  static constexpr int kKeys = 8;
  static constexpr int kStage = kKeys * DP * 4 * 2;
  static constexpr int kStages = DP == 64 ? 6 : 3;
  static constexpr int kRing = kWarps * kStages * kStage;
  using Mg = Merge<kWarps, R, DP>;
  static constexpr size_t kSmem = kRing + sizeof(Mg);
};

template <int R, int DP>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : 2) paged_attn_f32_kernel(const __grid_constant__ AttnArgs a) {
  using Shape = F32Shape<R, DP>;
  constexpr int NL = DP / 32;          // four-element chunks a lane has of a row
  constexpr int kStages = Shape::kStages;
  constexpr int kCols = DP / 4;        // 16-byte chunks of a row
  extern __shared__ __align__(128) char smem[];
  typename Shape::Mg& mg = *reinterpret_cast<typename Shape::Mg*>(smem + Shape::kRing);
  float(*qs)[DP + 4] = mg.o[0];        // the queries sit where the outputs will
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & 7, kq = lane >> 3;
  char* ring = smem + warp * (kStages * Shape::kStage);
  const uint32_t ring_s = smem_addr(ring);
  const int row_tiles = (a.rows + R - 1) / R;
  const int units = a.n_kv_heads * row_tiles;
  const int range = blockIdx.x / units, unit = blockIdx.x - range * units;
  const int rt = unit / a.n_kv_heads, kvh = unit - rt * a.n_kv_heads, row0 = rt * R;
  const Place pl = locate<kWarps>(a, range);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t chunk = chunk_of(pl.total, a.n_ranges), first = int64_t(range) * chunk;
  if (first >= pl.total) return;
  const int end = int(pl.total - first < chunk ? pl.total - first : chunk);

  // ---- loading: lane i < 8 finds key i's row, one stage before it is copied
  Cursor ahead;
  ahead.at(a, pl.seq, int(pl.seq_base - first));
  int next = 0;                // tile, and which 8 of the warp's 16 keys of it
  int next_half = 0;
  int page = 0, slot = -1;             // -1: the lane has no row
  auto look = [&]() {
    slot = -1;
    const int t = ahead.advance(a, next, end);
    if (t != next) next = t, next_half = 0;
    if (next < end) {
      const int p = (next - ahead.base) * kTile + warp * 16 + next_half * 8 + lane;
      if (lane < 8 && p < ahead.len) {
        const int block = unsigned(p) / unsigned(a.block_size);
        page = __ldg(a.block_tables + int64_t(ahead.seq) * a.max_blocks + block);
        slot = p - block * a.block_size;
      }
    }
  };
  int fill = 0;
  auto issue = [&]() {
    if (next < end) {
      int64_t off = -1;
      if (slot >= 0) {
        off = int64_t(page) * a.stride_page + int64_t(slot) * a.stride_row;
        if (page < 0 || off + a.row_span > a.cache_elems) {
          *a.err = 1;
          off = -1;
        } else {
          off += kvh * a.stride_head;
        }
      }
      if (next_half) ++next;
      next_half ^= 1;
      look();
      const uint32_t dst = ring_s + fill * Shape::kStage;
#pragma unroll
      for (int j = 0; j < 8 * kCols / 32; ++j) {
        const int row = (j * 32 + lane) / kCols, col = (j * 32 + lane) % kCols;
        const int64_t o = __shfl_sync(~0u, off, row);
        const int size = o >= 0 && col * 4 < a.head_dim ? 16 : 0;
        const int64_t at = size ? o + col * 4 : 0;
        const uint32_t d = dst + (row * kCols + col) * 16;
        copy16(d, static_cast<const float*>(a.k) + at, size);
        copy16(d + 8 * DP * 4, static_cast<const float*>(a.v) + at, size);
      }
    }
    fill = fill + 1 == kStages ? 0 : fill + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look();
  for (int i = 0; i < kStages - 1; ++i) issue();

  float4 o[R][NL];
  float m[R], l[R];
  int lim[R];
  int use = 0;
  Cursor now;
  now.at(a, pl.seq, int(pl.seq_base - first));
  int cur = 0;
  while ((cur = now.advance(a, cur, end)) < end) {
    const int seq = now.seq, len = now.len;
    const int t0 = cur - now.base;
    const int t1 = now.nt - t0 < end - cur ? now.nt : t0 + (end - cur);
    for (int i = threadIdx.x; i < R * kCols; i += kThreads) {
      const int r = i / kCols, d = (i - r * kCols) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row0 + r < a.rows && d < a.head_dim)
        x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + row_at(a, seq, kvh, row0 + r).q + d);
      *reinterpret_cast<float4*>(&qs[r][d]) = x;
    }
    const int group = a.n_heads / a.n_kv_heads;
    int tok = row0 / group, in_group = row0 - tok * group;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      lim[r] = row0 + r < a.rows ? len - a.n_new + 1 + tok : 0;
      if (++in_group == group) in_group = 0, ++tok;
      m[r] = ninf();
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NL; ++i) o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    const int sure = len - a.n_new + 1;
#pragma unroll 1
    for (int step = t0 * 2; step < t1 * 2; ++step) {
      const int p0 = (step >> 1) * kTile + warp * 16 + (step & 1) * 8;
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();                    // the stage has landed for all lanes, and the one before is free
      issue();
      const float4* kst = reinterpret_cast<const float4*>(ring + use * Shape::kStage);
      const float4* vst = kst + 8 * kCols;
      use = use + 1 == kStages ? 0 : use + 1;
      // the lane's keys: kq and kq + 4
      float s[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = 0.f;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const float4 k0 = kst[kq * kCols + i * 8 + g], k1 = kst[(kq + 4) * kCols + i * 8 + g];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 x = *reinterpret_cast<const float4*>(&qs[r][(i * 8 + g) * 4]);
          s[r][0] = fmaf(x.x, k0.x, fmaf(x.y, k0.y, fmaf(x.z, k0.z, fmaf(x.w, k0.w, s[r][0]))));
          s[r][1] = fmaf(x.x, k1.x, fmaf(x.y, k1.y, fmaf(x.z, k1.z, fmaf(x.w, k1.w, s[r][1]))));
        }
      }
      const bool all_seen = p0 + 8 <= sure;
      float e[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) s[r][x] += __shfl_xor_sync(~0u, s[r][x], d);
          s[r][x] = all_seen || p0 + kq + 4 * x < lim[r] ? s[r][x] * a.scale_log2 : ninf();
        }
        // the eight lanes of a key keep their own reference: the other lanes' join at the end
        const float top = fmaxf(s[r][0], s[r][1]);
        if (__any_sync(~0u, top > m[r] + kSlack)) {
          const float to = fmaxf(m[r], top);
          const float f = m[r] == ninf() ? 0.f : ex2(m[r] - to);
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < NL; ++i) o[r][i].x *= f, o[r][i].y *= f, o[r][i].z *= f, o[r][i].w *= f;
          m[r] = to;
        }
        const float ref = m[r] == ninf() ? 0.f : m[r];
        e[r][0] = ex2(s[r][0] - ref), e[r][1] = ex2(s[r][1] - ref);
        l[r] += e[r][0] + e[r][1];
      }
      // a value that a row does not see must not reach it, not even times 0
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const float4 v = vst[(kq + 4 * x) * kCols + i * 8 + g];
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (all_seen || p0 + kq + 4 * x < lim[r]) {
              o[r][i].x = fmaf(e[r][x], v.x, o[r][i].x);
              o[r][i].y = fmaf(e[r][x], v.y, o[r][i].y);
              o[r][i].z = fmaf(e[r][x], v.z, o[r][i].z);
              o[r][i].w = fmaf(e[r][x], v.w, o[r][i].w);
            }
        }
      }
    }
    __syncthreads();                   // the queries make place
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = fmaxf(m[r], __shfl_xor_sync(~0u, m[r], 8));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
      const float f = ex2(m[r] - (top == ninf() ? 0.f : top));
      float sum = l[r] * f;
      sum += __shfl_xor_sync(~0u, sum, 8);
      sum += __shfl_xor_sync(~0u, sum, 16);
      if (lane == 0) mg.m[warp][r] = top, mg.l[warp][r] = sum;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        float y[4] = {o[r][i].x * f, o[r][i].y * f, o[r][i].z * f, o[r][i].w * f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[j] += __shfl_xor_sync(~0u, y[j], 8);
          y[j] += __shfl_xor_sync(~0u, y[j], 16);
        }
        if (lane < 8) *reinterpret_cast<float4*>(&mg.o[warp][r][(i * 8 + g) * 4]) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
    float* part = a.parts + (int64_t(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * part_floats<R, DP>();
    emit<float, kWarps, R, DP, DP>(a, mg, {seq, kvh, row0, t0 == 0 && t1 == now.nt ? nullptr : part, part + R * DP}, 8, true, 0);
    cur += t1 - t0;
  }
}

// One query row: the parts of its sequence joined in the ranges' order; sequences
// in one range are done, those without a key get zeros.
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
    const int64_t v = seq_tiles(a, s);
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
  const int64_t nt = key_tiles(a, seq);
  const RowAt at = row_at(a, seq, kvh, row);
  T* out = static_cast<T*>(a.out) + at.out * a.head_dim;
  if (nt == 0) {
    for (int d = threadIdx.x; d < a.head_dim; d += kJoinThreads) out[d] = from_f32<T>(0.f);
    if (threadIdx.x == 0 && a.lse) a.lse[at.out] = ninf();
  }
  // every CTA waits for the first kernel, so that what follows this one does too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nt == 0) return;
  const int64_t chunk = chunk_of(total, a.n_ranges);
  before += kStart;
  const int64_t wa = before / chunk, wb = (before + nt - 1) / chunk;
  if (wa == wb) return;
  const int r = row % R;
  constexpr int64_t kPart = part_floats<R, DP>();
  const int unit = row / R * a.n_kv_heads + kvh;
  auto part = [&](int64_t w) { return a.parts + ((w * units + unit) * 2 + (w == wa ? 1 : 0)) * kPart; };
  // each warp takes every fourth part, relative to the largest maximum it has met
  constexpr int kQ = DP / 4 / 32 ? DP / 4 / 32 : 1;      // float4 a lane
  float4 o[kQ] = {};
  float m = ninf(), l = 0.f;
#pragma unroll 4
  for (int64_t w = wa + warp; w <= wb; w += kWarps) {
    const float* src = part(w);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + R * DP + 2 * r));
    const float top = fmaxf(m, ml.x), ref = top == ninf() ? 0.f : top;
    const float g = ex2(m - ref), f = ex2(ml.x - ref);
    m = top;
    l = l * g + f * ml.y;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int d = (i * 32 + lane) * 4;
      if (d < DP) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(src + r * DP + d));
        o[i].x = o[i].x * g + f * x.x, o[i].y = o[i].y * g + f * x.y;
        o[i].z = o[i].z * g + f * x.z, o[i].w = o[i].w * g + f * x.w;
      }
    }
  }
  if (lane == 0) ml_all[warp] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const int d = (i * 32 + lane) * 4;
    if (d < DP) *reinterpret_cast<float4*>(&acc[warp][d]) = o[i];
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(ml_all[0].x, ml_all[1].x), fmaxf(ml_all[2].x, ml_all[3].x));
  const float ref = top == ninf() ? 0.f : top;
  float f[kWarps];
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    f[w] = ex2(ml_all[w].x - ref);
    l += f[w] * ml_all[w].y;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  for (int d = threadIdx.x; d < a.head_dim; d += kJoinThreads)
    out[d] = from_f32<T>((f[0] * acc[0][d] + f[1] * acc[1][d] + f[2] * acc[2][d] + f[3] * acc[3][d]) * inv);
  if (threadIdx.x == 0 && a.lse) a.lse[at.out] = l == 0.f ? ninf() : log_sum(top, l);
}

// ------------------------------------------------------------------ variants

struct Variant {
  const void* main;
  const void* join;
  int rows, threads;
  bool tensor;
  size_t esz;
  size_t smem, part;
};

template <typename T, int R, int DP>
Variant tc() {
  return {reinterpret_cast<const void*>(&paged_attn_tc_kernel<T, R, DP>),
          reinterpret_cast<const void*>(&paged_attn_join_kernel<T, R, DP>), R, kThreads, true, sizeof(T),
          TcShape<R, DP>::kSmem,
          size_t(part_floats<R, DP>()) * sizeof(float)};
}

template <typename T, int WR, int DP>
Variant shared_rows() {
  return {reinterpret_cast<const void*>(&paged_attn_rows_kernel<T, WR, DP>),
          reinterpret_cast<const void*>(&paged_attn_join_kernel<T, WR * 16, DP>), WR * 16, WR * 64, true, sizeof(T),
          RowsShape<WR, DP>::kSmem, size_t(part_floats<WR * 16, DP>()) * sizeof(float)};
}

template <int R, int DP>
Variant f32_rows() {
  return {reinterpret_cast<const void*>(&paged_attn_f32_kernel<R, DP>),
          reinterpret_cast<const void*>(&paged_attn_join_kernel<float, R, DP>), R, kThreads, false, sizeof(float),
          F32Shape<R, DP>::kSmem, size_t(part_floats<R, DP>()) * sizeof(float)};
}

template <typename T, int DP>
Variant fma_rows() {
  using Core = Fma<T, DP>;
  return {reinterpret_cast<const void*>(&paged_attn_fma_kernel<T, Core>),
          reinterpret_cast<const void*>(&paged_attn_join_kernel<T, Core::kRows, DP>), Core::kRows, kThreads, false, sizeof(T),
          sizeof(Merge<kWarps, Core::kRows, DP>), size_t(part_floats<Core::kRows, DP>()) * sizeof(float)};
}

// [bf16, f16] x ([8, 16 query rows] x [64, 128, 256 elements], [32, 48 rows] x [64, 128
// elements]), then f32, and f32 and the 16-bit types of any alignment.
constexpr int kVariants = 31;
template <typename T>
struct TcVariants {
  static void fill(Variant* v) {
    v[0] = tc<T, 8, 64>(), v[1] = tc<T, 8, 128>(), v[2] = tc<T, 8, 256>();
    v[3] = tc<T, 16, 64>(), v[4] = tc<T, 16, 128>(), v[5] = tc<T, 16, 256>();
    v[6] = shared_rows<T, 2, 64>(), v[7] = shared_rows<T, 2, 128>();
    v[8] = shared_rows<T, 3, 64>(), v[9] = shared_rows<T, 3, 128>();
  }
};
struct Variants {
  Variant v[kVariants];
  Variants() {
    using bf = __nv_bfloat16;
    using hf = __half;
    TcVariants<bf>::fill(v);
    TcVariants<hf>::fill(v + 10);
    v[20] = f32_rows<4, 64>(), v[21] = f32_rows<4, 128>(), v[22] = f32_rows<4, 256>();
    v[23] = f32_rows<8, 64>(), v[24] = f32_rows<8, 128>();
    v[25] = fma_rows<float, 128>(), v[26] = fma_rows<float, 256>();
    v[27] = fma_rows<bf, 128>(), v[28] = fma_rows<bf, 256>();
    v[29] = fma_rows<hf, 128>(), v[30] = fma_rows<hf, 256>();
  }
};
const Variant& variant_at(int i) {
  static const Variants all;
  return all.v[i];
}

}  // namespace

namespace {

cudaError_t plan_variant(int v, int n_kv_heads, int rows, int n_sm, AttnPlan* plan) {
  const Variant& k = variant_at(v);
  // CTAs an SM holds, per device: the first use on a device also raises the kernel's
  // shared-memory limit there
  constexpr int kDevices = 16;
  static int resident[kDevices][kVariants];
  int dev = 0, n = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kDevices) n = __atomic_load_n(&resident[dev][v], __ATOMIC_RELAXED);
  if (n == 0) {
    if (k.smem > 48 * 1024)
      e = cudaFuncSetAttribute(k.main, cudaFuncAttributeMaxDynamicSharedMemorySize, int(k.smem));
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k.main, k.threads, k.smem);
    if (e != cudaSuccess) return e;
    if (n < 1) return cudaErrorInvalidConfiguration;
    if (dev < kDevices) __atomic_store_n(&resident[dev][v], n, __ATOMIC_RELAXED);
  }
  // Ranges: the workers just fill the GPU; where a range has so many units that this
  // would leave a fifth of it idle, at least four rounds of workers.
  const int64_t units = int64_t(n_kv_heads) * ((rows + k.rows - 1) / k.rows);
  const int64_t slots = int64_t(n) * n_sm;
  int64_t ranges = slots / units;
  if (ranges * units * 5 < slots * 4 || ranges < 1) ranges = (4 * slots + units - 1) / units;
  if (ranges * units > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  plan->variant = v;
  plan->n_ranges = int(ranges);
  plan->n_workers = int(ranges * units);
  plan->workspace = ranges > 1 ? size_t(plan->n_workers) * 2 * k.part : 16;      // one range splits nothing
  return cudaSuccess;
}

// dtype: VC_DTYPE_BF16 / F32 / F16 (0 / 1 / 3); wide: 16-byte chunks everywhere.
int variant_for(const AttnArgs& a, int dtype, bool wide) {
  const int size = a.head_dim <= 64 ? 0 : a.head_dim <= 128 ? 1 : 2;
  if (!wide) return (dtype == 1 ? 25 : dtype == 0 ? 27 : 29) + (size == 2 ? 1 : 0);
  if (dtype == 1) return a.rows > 4 && size < 2 ? 23 + size : 20 + size;
  const int first = dtype == 0 ? 0 : 10;
  if (a.rows <= 8) return first + size;
  if (a.rows <= 16 || size == 2) return first + 3 + size;
  // 32 or 48 rows a unit: whichever reads the keys in fewer units, then the smaller
  return first + ((a.rows + 31) / 32 <= (a.rows + 47) / 48 ? 6 : 8) + size;
}

}  // namespace

cudaError_t paged_attn_workspace(const AttnArgs& a, int dtype, int n_sm, size_t* bytes) {
  *bytes = 0;
  for (int wide = 0; wide < 2; ++wide) {
    AttnPlan p;
    const cudaError_t e = plan_variant(variant_for(a, dtype, wide != 0), a.n_kv_heads, a.rows, n_sm, &p);
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
  return plan_variant(variant_for(a, dtype, wide), a.n_kv_heads, a.rows, n_sm, plan);
}

cudaError_t launch_paged_attn(const AttnArgs& args, const AttnPlan& plan, cudaStream_t s) {
  const Variant& k = variant_at(plan.variant);
  AttnArgs a = args;
  // a negative scale turns the queries' signs (of two 16-bit elements) in the tensor-core variants
  const size_t esz = k.esz;
  a.wide_out = reinterpret_cast<uintptr_t>(a.out) % (4 * esz) == 0 && a.head_dim % 4 == 0;
  if (k.tensor && a.scale_log2 < 0) a.scale_log2 = -a.scale_log2, a.q_sign = 0x80008000u;
  void* params[] = {&a};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(plan.n_workers));
  a.n_ranges = plan.n_ranges;
  cfg.blockDim = dim3(unsigned(k.threads));
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

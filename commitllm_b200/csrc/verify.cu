// Verification of drafted tokens against the target's logits, from given
// uniform numbers.
//
// For sequence s and position i, p_i = softmax(logits_i / T) (T = 0: all on the
// lowest index of the largest logit).  With draft probabilities q, draft x_i is
// kept while u_i * q_i(x_i) < p_i(x_i); at the first refused one the token is drawn
// from max(p_i - q_i, 0), after the last kept one from p_i, both with u_last.
// Without them the token at i is the one p_i gives for u_i, and x_i is kept while
// it equals that token.  A draw for u from weights w is the lowest v with
// w_0 + .. + w_v > u * sum(w).
//
// Two launches.  The first reads every logits row once (what bounds the call): a
// CTA takes a slice of a row and leaves its maximum, the sum of exp2 over it in
// f32 (joined in f64), the lowest index of the maximum, and how much of the sum
// lies before x.  The second has one cluster of CTAs per sequence.  It walks the
// positions with those sums and then draws the one token that needs a whole row.
// A drawn token must not depend on rounding: with 10^5 weights a running sum off
// by 10^-7 moves one draw in a hundred to a neighbour, so the drawn row is summed
// in f64 from f64 exponentials (a part of 1 / (drafts + 1) of the elements), and a
// keep-or-refuse test that the f32 sums leave open is taken again in f64.
//
// Measured: 64 sequences of 4 drafts over 128256 f32 logits with draft probabilities 70
// us: the row sums read 164 MB in 33 (5.0 TB/s), the drawn rows, two f64 passes each, take
// 35 (f64 pipe 30 %, half of the issue slots: conversions, table look-ups and the f64
// chain).  32 sequences of 7 drafts over 152064 bf16 logits 37 us, one sequence 16.6 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cmath>

#include "vc_internal.h"

namespace cg = cooperative_groups;

namespace vc {
namespace {

constexpr int kStatThreads = 256;
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kMaxCluster = 8;
static_assert(32 * sizeof(VerifyPart) <= kVerifyRowBytes, "a row's slices fit its workspace");

// How far a keep-or-refuse quantity of the f32 sums may be from its exact value,
// relative to the row's sum: an exponent of at most 126 (smaller weights are
// nothing) is rounded four times by 2^-24 of itself (log2(e), its quotient by T, the
// difference of the logits, the product), exp2 is off by 2^-22 in it and at each of
// three joins (warp, block, row), a thread's sum of at most 2^7 rounded terms by
// 2^-17, and its at most 12 changes of the maximum by 2^-21 each; 126 * 4 * 2^-24 * ln
// 2 + 4 * 2^-22 + 2^-17 + 12 * 2^-21 < 3.6e-5.
constexpr double kOpen = 4e-5;
// That holds for temperatures in [1e-30, 1e30]: log2(e) / T is then a normal number, and
// a difference of two logits that passes f32 weighs nothing.  At any other temperature
// every test is open.
__device__ __forceinline__ double open_part(float t) { return t >= 1e-30f && t <= 1e30f ? kOpen : double(INFINITY); }

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }

// log2(e) / T, kept finite and above 0; 1 for a greedy sequence (T not above 0), whose sums nobody reads.
__device__ __forceinline__ float exponent_scale(float t) {
  return t > 0.f ? fmaxf(fminf(1.4426950408889634f / t, 3e38f), 1e-37f) : 1.f;
}

__device__ __forceinline__ float ex2(float x) {      // 2^x within 2^-22 of itself, nothing below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A thread's maximum, sum of exp2((l - m) * c), and the part of it before x.  A NaN
// or a +infinity leaves a NaN in s (inf - inf), which is how such a row is told.
template <bool kBefore>
struct Running {
  float m = ninf(), s = 0.f, b = 0.f;
  int best = 0x7fffffff;

  // N elements, of which l[e] is number at + (e / W) * step + e % W
  template <int N, int W>
  __device__ __forceinline__ void add(const float (&l)[N], int at, int step, float c, int x) {
    float top = l[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, l[i]);
    if (top > m) {
      const float f = m == ninf() ? 0.f : ex2((m - top) * c);
      s *= f;
      if (kBefore) b *= f;
      m = top;
      // the lowest index of the new maximum in this batch
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (l[i] == top) best = at + (i / W) * step + i % W;
    }
    const float ref = m == ninf() ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = ex2((l[i] - ref) * c);
      s += w;
      if (kBefore && at + (i / W) * step + i % W < x) b += w;
    }
  }
};

template <typename T, typename R>
__device__ __forceinline__ void stat_slice(const T* src, int lo, int hi, float c, int x, R& r) {
  constexpr int N = 16 / sizeof(T);
  constexpr int kBatch = 4;           // 16-byte loads a thread has under way
  struct alignas(16) Chunk {
    T v[N];
  };
  // single elements up to the first 16-byte boundary, chunks, single elements
  const int head = lo < hi ? min(int((16 - (reinterpret_cast<uintptr_t>(src + lo) & 15)) & 15) / int(sizeof(T)), hi - lo) : 0;
  const int body = lo < hi ? (hi - lo - head) / N : 0;
  const int tail = lo + head + body * N;
  if (int(threadIdx.x) < head) {
    const float l[1] = {to_f32(src[lo + threadIdx.x])};
    r.template add<1, 1>(l, lo + threadIdx.x, 0, c, x);
  }
  // a batch of chunks; of f32 ones, the next is on its way while one is summed (74.6 ->
  // 71.7 us for 320 rows; of 16-bit ones it costs too many registers: 39 -> 48 us)
  int j = threadIdx.x;
  constexpr bool kAhead = sizeof(T) == 4;
  constexpr int kStep = kBatch * kStatThreads;
  Chunk ch[kBatch];
  auto load = [&](int from) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      ch[k] = *reinterpret_cast<const Chunk*>(src + lo + head + (from + k * kStatThreads) * N);
  };
  bool full = j + kStep - kStatThreads < body;
  if (kAhead && full) load(j);
  while (full) {
    if (!kAhead) load(j);
    float l[kBatch * N];
#pragma unroll
    for (int e = 0; e < kBatch * N; ++e) l[e] = to_f32(ch[e / N].v[e % N]);
    const int at = lo + head + j * N;
    j += kStep;
    full = j + kStep - kStatThreads < body;
    if (kAhead && full) load(j);
    r.template add<kBatch * N, N>(l, at, kStatThreads * N, c, x);
  }
  for (; j < body; j += kStatThreads) {
    const int at = lo + head + j * N;
    const Chunk ch = *reinterpret_cast<const Chunk*>(src + at);
    float l[N];
#pragma unroll
    for (int e = 0; e < N; ++e) l[e] = to_f32(ch.v[e]);
    r.template add<N, N>(l, at, 0, c, x);
  }
  if (tail + int(threadIdx.x) < hi) {
    const float l[1] = {to_f32(src[tail + threadIdx.x])};
    r.template add<1, 1>(l, tail + threadIdx.x, 0, c, x);
  }
}

template <typename T, bool kBefore>
__global__ void __launch_bounds__(kStatThreads) verify_stat_kernel(const __grid_constant__ VerifyArgs a) {
  const int row = blockIdx.x, split = blockIdx.y;
  const int seq = row / (a.n_draft + 1), i = row - seq * (a.n_draft + 1);
  const T* src = static_cast<const T*>(a.logits) + seq * a.logits_seq + i * a.logits_tok;
  const int lo = split * a.slice;
  const int hi = min(lo + a.slice, a.vocab);
  const float c = exponent_scale(a.temperature[seq]);
  // without draft probabilities the part of the sum before the draft is wanted
  const int x = kBefore && i < a.n_draft ? a.drafts[int64_t(seq) * a.n_draft + i] : -1;
  // a slice behind x has none of that part, one before x all of it: only the slice
  // that holds x looks at each element
  Running<true> r;
  if (kBefore && lo < x && x < hi) {
    stat_slice<T>(src, lo, hi, c, x, r);
  } else {
    Running<false> rr;
    stat_slice<T>(src, lo, hi, c, x, rr);
    r.m = rr.m, r.s = rr.s, r.best = rr.best;
    r.b = kBefore && x >= hi ? rr.s : 0.f;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the block's
  __shared__ float sm[kStatThreads / 32];
  __shared__ double ss[kStatThreads / 32], sb[kStatThreads / 32];
  __shared__ int si[kStatThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = r.m;
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
  // a sum without a maximum is 0 or NaN, and a NaN stays one
  const float f = r.m == ninf() ? 1.f : ex2((r.m - m) * c);
  double s = double(r.s * f), b = double(r.b * f);
  int best = r.m == m ? r.best : 0x7fffffff;
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s += __shfl_xor_sync(~0u, s, d);
    if (kBefore) b += __shfl_xor_sync(~0u, b, d);
    best = min(best, __shfl_xor_sync(~0u, best, d));
  }
  if (lane == 0) sm[warp] = m, ss[warp] = s, sb[warp] = b, si[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    VerifyPart p{};
    p.m = ninf();
    for (int w = 0; w < kStatThreads / 32; ++w) p.m = fmaxf(p.m, sm[w]);
    p.best = 0x7fffffff;
    for (int w = 0; w < kStatThreads / 32; ++w) {
      const double g = sm[w] == ninf() ? 1.0 : double(ex2((sm[w] - p.m) * c));
      p.s += g * ss[w];
      p.b += g * sb[w];
      if (sm[w] == p.m) p.best = min(p.best, si[w]);
    }
    a.parts[int64_t(row) * a.splits + split] = p;
  }
}

// 2^(y / 1024) in f64 for y in [-2^31, 0], 2^-1000 or so below that: 2^(j / 1024) from a table (shared memory,
// made by exp2), the rest |r| <= 1/2 by the series of 2^(r / 1024) up to r^3 (what
// follows is below 2^-50).  Seven f64 operations and no branch: f64 arithmetic bounds
// the drawn row, and exp() takes about twenty.
constexpr int kTable = 1024;
__device__ __forceinline__ double pow2(double y, const double* table) {
  constexpr double kMagic = 6755399441055744.0;      // 1.5 * 2^52: rounds to a whole number
  const double z = y + kMagic;
  const int n = __double2loint(z);
  const double r = y - (z - kMagic);
  constexpr double l = 0.693147180559945309417 / kTable;      // ln 2 / 1024
  double p = fma(r, l * l * l / 6, l * l / 2);
  p = fma(r, p, l);
  const double v = table[n & (kTable - 1)];
  p = fma(r * p, v, v);
  return __hiloint2double(__double2hiint(p) + (max(n >> 10, -1000) << 20), __double2loint(p));
}

// One position: its row's joined sums, and the draft's weight and probability.
struct Row {
  double s, b;       // relative to m
  double wx;         // exact
  float m, qx;
  int best, x;
  bool usable, there;
};

// The weight of element v of a row: 2^((l - m) log2(e) / T), or what that over the
// row's sum has above the draft's probability.
template <typename T>
struct Weights {
  const T* l;
  const float* q;      // nullptr: plain weights
  const double* table;
  double m, c, scale;  // maximum, 1024 log2(e) / T, 1 / the row's sum
  float none;          // logits below it weigh nothing: exp would round to 0
  bool wide;           // rows on 16-byte boundaries
  // (a weight from there to 2^-1000 counts as about 2^-1000: enough to be drawn at
  // u = 0, nothing in a sum)
  __device__ __forceinline__ double plain(float x) const {
    const double w = pow2((double(x) - m) * c, table);
    return x < none ? 0.0 : w;
  }
  template <bool kOver>
  __device__ __forceinline__ double of(float x, float qv) const {
    const double w = plain(x);
    if (!kOver) return w;
    const double d = fma(w, scale, -double(qv));
    return d > 0.0 ? d : 0.0;
  }
  __device__ __forceinline__ double at(int v) const {
    return q ? of<true>(to_f32(l[v]), q[v]) : of<false>(to_f32(l[v]), 0.f);
  }
};

// This CTA's slice [lo, hi) of the vocabulary; its warps hold equal contiguous
// parts, a multiple of 8 elements but for the last.
struct Slice {
  int lo, hi, per_warp;
};

struct Box {
  double sum[2];                 // this CTA's sums, for the others: two calls' in turn
  double warp[kPickWarps];       // its warps'
  double warp2[kPickWarps];
  int token;
};

// Sum of the weights over a warp's part [b, e), by its lanes; kOver: over the draft's
// probabilities.
template <typename T, bool kOver>
__device__ __forceinline__ double part_sum(const Weights<T>& w, int b, int e) {
  constexpr int N = 16 / sizeof(T);
  constexpr int kBatch = sizeof(T) == 4 ? 2 : 1;      // chunks a lane has under way
  struct alignas(16) Chunk {
    T v[N];
  };
  const int lane = threadIdx.x & 31;
  double v = 0;
  int j = b;
  if (w.wide) {
    const int n = (e - b) / N;
    // chunks past the end are read again and not counted, so a batch has no branches
    Chunk ch[kBatch];
    float4 qv[kBatch * N / 4];
    auto load = [&](int k) {
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const int at = b + min(k + 32 * x, n - 1) * N;
        ch[x] = *reinterpret_cast<const Chunk*>(w.l + at);
        if (kOver) {
#pragma unroll
          for (int i = 0; i < N / 4; ++i) qv[x * (N / 4) + i] = *reinterpret_cast<const float4*>(w.q + at + 4 * i);
        }
      }
    };
    if (n > 0) load(lane);
    for (int k = lane; k - lane < n; k += 32 * kBatch) {
      float l[kBatch * N], q[kBatch * N];
#pragma unroll
      for (int x = 0; x < kBatch; ++x)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          l[x * N + i] = to_f32(ch[x].v[i]);
          const float4 f = qv[x * (N / 4) + i / 4];
          q[x * N + i] = !kOver ? 0.f : i % 4 == 0 ? f.x : i % 4 == 1 ? f.y : i % 4 == 2 ? f.z : f.w;
        }
      if (k - lane + 32 * kBatch < n) load(k + 32 * kBatch);      // while this batch is weighed
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        double t = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) t += w.template of<kOver>(l[x * N + i], q[x * N + i]);
        v += k + 32 * x < n ? t : 0.0;
      }
    }
    j = b + n * N;
  }
#pragma unroll 4
  for (j += lane; j < e; j += 32) v += w.template of<kOver>(to_f32(w.l[j]), kOver ? w.q[j] : 0.f);
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// Sum of the weights over the slice: all threads get the CTA's, box.warp keeps the parts.
template <typename T>
__device__ double slice_sum(const Weights<T>& w, const Slice& sl, Box& box) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = min(sl.lo + warp * sl.per_warp, sl.hi), e = min(b + sl.per_warp, sl.hi);
  const double v = w.q ? part_sum<T, true>(w, b, e) : part_sum<T, false>(w, b, e);
  __syncthreads();               // the last call's parts have been read
  if (lane == 0) box.warp[warp] = v;
  __syncthreads();
  double t = 0;
#pragma unroll
  for (int x = 0; x < kPickWarps; ++x) t += box.warp[x];
  return t;
}

// The first of n consecutive parts whose running sum passes goal, and the sum
// before it.  Parts' sums are rounded apart from the total that goal comes from, so
// a goal next to the total may be passed by none: then the last part that still
// adds to the running sum, not a negligible one behind it.
__device__ __forceinline__ int first_past(const double* part, int n, double goal, double& before) {
  double run = before;
  int at = 0;
  for (int x = 0; x < n; ++x) {
    const double next = run + part[x];
    if (next > run) at = x, before = run;
    run = next;
    if (run > goal) break;
  }
  return at;
}

// The lowest v whose running sum passes goal; all[]: the CTAs' sums.  The CTA that
// holds it calls done(v) from one thread.
template <typename T, typename Done>
__device__ void find(const Weights<T>& w, const Slice& sl, Box& box, const double (&all)[kMaxCluster], int n_cta, int me,
                     double goal, Done done) {
  double before = 0;
  if (first_past(all, n_cta, goal, before) != me) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wp = first_past(box.warp, kPickWarps, goal, before);
  // that warp's part, cut again over all warps
  const int b = min(sl.lo + wp * sl.per_warp, sl.hi), e = min(b + sl.per_warp, sl.hi);
  const int per = (e - b + kPickWarps - 1) / kPickWarps;
  const int b2 = min(b + warp * per, e), e2 = min(b2 + per, e);
  double v = 0;
#pragma unroll 2
  for (int j = b2 + lane; j < e2; j += 32) v += w.at(j);
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  if (lane == 0) box.warp2[warp] = v;
  __syncthreads();
  if (first_past(box.warp2, kPickWarps, goal, before) != warp) return;
  int token = -1, last = b2;
  for (int j = b2; j < e2 && token < 0; j += 32) {
    v = j + lane < e2 ? w.at(j + lane) : 0.0;
    double incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_up_sync(~0u, incl, d);
      if (lane >= d) incl += o;
    }
    const double run = before + incl;
    double prev = __shfl_up_sync(~0u, run, 1);
    if (lane == 0) prev = before;
    const unsigned hit = __ballot_sync(~0u, v > 0 && run > goal), adds = __ballot_sync(~0u, run > prev);
    if (hit) token = j + __ffs(hit) - 1;
    if (adds) last = j + 31 - __clz(adds);
    before = __shfl_sync(~0u, run, 31);
  }
  if (lane == 0) done(token < 0 ? last : token);
}

template <typename T>
__global__ void __launch_bounds__(kPickThreads, 1) verify_pick_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ Box box;
  __shared__ Row rows[kPickWarps];
  __shared__ double table[kTable];
  cg::cluster_group cl = cg::this_cluster();
  const int n_cta = int(cl.num_blocks()), me = int(cl.block_rank());
  const int seq = blockIdx.x / n_cta;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kTable; i += kPickThreads) table[i] = exp2(double(i) / kTable);
  Slice sl;
  const int per_cta = ((a.vocab + n_cta - 1) / n_cta + 7) / 8 * 8;
  sl.lo = min(me * per_cta, a.vocab);
  sl.hi = min(sl.lo + per_cta, a.vocab);
  sl.per_warp = ((per_cta + kPickWarps - 1) / kPickWarps + 7) / 8 * 8;
  const float temp = a.temperature[seq];
  const bool greedy = !(temp > 0.f);
  const double open = open_part(temp);
  const double* u = a.uniforms + int64_t(seq) * (a.n_draft + 1);
  const int32_t* drafts = a.drafts + int64_t(seq) * a.n_draft;
  int32_t* out = a.tokens + int64_t(seq) * (a.n_draft + 1);
  Weights<T> w;
  w.table = table;
  w.c = kTable * 1.4426950408889634074 / double(temp);
  w.q = nullptr;
  w.scale = 1.0;
  auto set_row = [&](int i, float m) {
    w.l = static_cast<const T*>(a.logits) + seq * a.logits_seq + i * a.logits_tok;
    w.m = double(m);
    // never above the lowest finite value: a row may consist of it, and only -infinity rules out
    w.none = fmaxf(__fadd_ru(m, __fmul_rn(temp, -744.44f)), -FLT_MAX);
  };
  auto probs_row = [&](int i) { return a.draft_probs + seq * a.probs_seq + i * a.probs_tok; };
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Rows of 16 positions at a time, one a warp, alike in every CTA of the cluster.
  auto load_rows = [&](int i0) {
    const int i = i0 + warp;
    if (i <= a.n_draft) {
      const float c = exponent_scale(temp);
      const VerifyPart* p = a.parts + (int64_t(seq) * (a.n_draft + 1) + i) * a.splits;
      VerifyPart v{};
      v.m = ninf();
      v.best = 0x7fffffff;
      if (lane < a.splits) v = p[lane];
      Row r;
      r.x = i < a.n_draft ? drafts[i] : -1;
      r.there = r.x >= 0 && r.x < a.vocab;
      const T* l = static_cast<const T*>(a.logits) + seq * a.logits_seq + i * a.logits_tok;
      const float lx = r.there ? to_f32(l[r.x]) : 0.f;
      r.qx = r.there && a.draft_probs ? probs_row(i)[r.x] : 0.f;
      float m = v.m;
#pragma unroll
      for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
      const double f = v.m == ninf() ? 1.0 : double(ex2((v.m - m) * c));
      double s = v.s * f, b = v.b * f;
      int best = v.m == m ? v.best : 0x7fffffff;
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        s += __shfl_xor_sync(~0u, s, d);
        b += __shfl_xor_sync(~0u, b, d);
        best = min(best, __shfl_xor_sync(~0u, best, d));
      }
      r.m = m, r.s = s, r.b = b, r.best = best;
      r.usable = m > ninf() && m < -ninf() && s == s;
      set_row(i, m);
      r.wx = r.there && r.usable ? w.plain(lx) : 0.0;
      if (lane == 0) rows[warp] = r;
    }
    __syncthreads();
  };
  double all[kMaxCluster];
  int turn = 0;
  auto total_of = [&]() {      // exact sum of w's row, by the cluster
    const double mine = slice_sum(w, sl, box);
    if (threadIdx.x == 0) box.sum[turn] = mine;
    cl.sync();
    double t = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      all[r] = r < n_cta ? *cl.map_shared_rank(&box.sum[turn], r) : 0.0;
      t += all[r];
    }
    turn ^= 1;
    return t;
  };

  int i = 0;
  bool drawn = false;          // the last token comes from find
  bool usable = true;
  int token = -1;
  load_rows(0);
  for (;; ++i) {
    if (i && i % kPickWarps == 0) {
      __syncthreads();
      load_rows(i);
    }
    const Row r = rows[i % kPickWarps];
    usable = r.usable;
    if (!usable) break;
    if (greedy) {
      token = r.best;
      if (r.there && r.x == token) continue;
      break;
    }
    set_row(i, r.m);
    w.q = nullptr;
    w.wide = a.wide_logits;
    if (!a.draft_probs) {
      const double goal = u[i] * r.s, edge = open * r.s;
      const bool in = goal > r.b + edge && goal < r.b + r.wx - edge;
      const bool off = goal < r.b - edge || goal > r.b + r.wx + edge;
      if (r.there && in) continue;                  // kept, whatever the rounding
      const double t = total_of();
      if (r.there && !off) {                        // open: the token drawn decides
        find(w, sl, box, all, n_cta, me, u[i] * t, [&](int v) {
          for (int k = 0; k < n_cta; ++k) *cl.map_shared_rank(&box.token, k) = v;
        });
        cl.sync();
        token = box.token;
        cl.sync();
        if (token == r.x) continue;
        break;
      }
      find(w, sl, box, all, n_cta, me, u[i] * t, [&](int v) { out[i] = v; });
      drawn = true;
      break;
    }
    double total = 0;
    bool have_total = false;
    if (r.there) {
      const double want = u[i] * double(r.qx), have = want * r.s;
      bool keep = have < r.wx;
      if (!(fabs(have - r.wx) > open * fmax(have, r.wx)) && have > 0.0) {
        total = total_of();
        have_total = true;
        keep = want < r.wx / total;
      }
      if (keep) continue;
    }
    if (!have_total) total = total_of();
    double sum = total;
    if (r.there) {
      w.q = probs_row(i);
      w.scale = 1.0 / total;
      w.wide = a.wide_logits && a.wide_probs;
      sum = total_of();
      if (!(sum > 0)) {
        w.q = nullptr;
        sum = total_of();
      }
    }
    find(w, sl, box, all, n_cta, me, u[a.n_draft] * sum, [&](int v) { out[i] = v; });
    drawn = true;
    break;
  }
  if (me == 0) {
    for (int j = threadIdx.x; j <= a.n_draft; j += kPickThreads)
      if (j != i || !drawn) out[j] = j < i ? drafts[j] : j == i && usable ? token : -1;
    if (threadIdx.x == 0) a.counts[seq] = i + (usable ? 1 : 0);
  }
  cl.sync();      // no CTA leaves while another may still read its shared memory
}

template <typename T>
cudaError_t launch_t(const VerifyArgs& args, int cluster, cudaStream_t s) {
  VerifyArgs a = args;
  a.wide_logits = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.logits_seq * int64_t(sizeof(T)) % 16 == 0 &&
                  a.logits_tok * int64_t(sizeof(T)) % 16 == 0;
  a.wide_probs = reinterpret_cast<uintptr_t>(a.draft_probs) % 16 == 0 && a.probs_seq % 4 == 0 && a.probs_tok % 4 == 0;
  const dim3 grid(unsigned(a.n_seqs) * unsigned(a.n_draft + 1), unsigned(a.splits));
  if (a.draft_probs)
    verify_stat_kernel<T, false><<<grid, kStatThreads, 0, s>>>(a);
  else
    verify_stat_kernel<T, true><<<grid, kStatThreads, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(a.n_seqs) * unsigned(cluster));
  cfg.blockDim = dim3(kPickThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  void* params[] = {&a};
  return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(&verify_pick_kernel<T>), params);
}

}  // namespace

// Slices of a row in the first launch: enough CTAs to fill the GPU a few times, of
// 2048 elements or more and 2^15 or less (128 a thread, which kOpen counts on), at
// most 32 (one a lane when they are joined; vocab is at most 2^20).
void plan_verify(VerifyArgs* a, int n_sm) {
  const int64_t rows = int64_t(a->n_seqs) * (a->n_draft + 1);
  int64_t n = (int64_t(n_sm) * 8 + rows - 1) / rows;
  if (n > 32) n = 32;
  const int64_t most = (int64_t(a->vocab) + 2047) / 2048;
  if (n > most) n = most;
  const int64_t least = (int64_t(a->vocab) + 32767) / 32768;
  if (n < least) n = least;
  int64_t slice = (int64_t(a->vocab) + n - 1) / n;
  slice = (slice + 7) / 8 * 8;
  a->slice = int32_t(slice);
  a->splits = int32_t((int64_t(a->vocab) + slice - 1) / slice);
}

cudaError_t launch_verify(const VerifyArgs& a, int dtype, int n_sm, cudaStream_t s) {
  // CTAs of a sequence's cluster: as many as stay resident at once (one an SM, whose
  // 128 registers a thread measured 3 % faster than two with 64), one for a short row
  int cluster = a.vocab > 4096 ? kMaxCluster : 1;
  while (cluster > 1 && int64_t(a.n_seqs) * cluster > n_sm) cluster /= 2;
  switch (dtype) {
    case 0: return launch_t<__nv_bfloat16>(a, cluster, s);
    case 1: return launch_t<float>(a, cluster, s);
    default: return launch_t<__half>(a, cluster, s);
  }
}

}  // namespace vc

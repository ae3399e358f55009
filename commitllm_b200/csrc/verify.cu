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
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vc_internal.h"

namespace cg = cooperative_groups;

namespace vc {
namespace {

constexpr int kStatThreads = 256;
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kMaxCluster = 8;

// How far a keep-or-refuse quantity of the f32 sums may be from its exact value,
// relative to the row's sum: an exponent of at most 126 (smaller weights are
// nothing) is rounded three times by 2^-24 of itself, exp2 is off by 2^-22, and
// a thread's sum of at most 2^7 rounded terms by 2^-17; 126 * 3 * 2^-24 * ln 2 +
// 2^-22 + 2^-17 < 2.4e-5.
constexpr double kOpen = 4e-5;

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }

// log2(e) / T, kept finite; 0 for a greedy sequence (T not above 0).
__device__ __forceinline__ float exponent_scale(float t) { return t > 0.f ? fminf(1.4426950408889634f / t, 3e38f) : 0.f; }

struct Running {
  float m = ninf(), s = 0.f, b = 0.f;   // maximum, sum of exp2((l - m) * c), the part of it before x
  int best = 0x7fffffff;
  bool bad = false;                     // a NaN

  template <int N>
  __device__ __forceinline__ void add(const float (&l)[N], int at, float c, int x) {
    float top = l[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, l[i]);
    if (top > m) {
      const float f = m == ninf() ? 0.f : exp2f((m - top) * c);
      s *= f;
      b *= f;
      m = top;
      // the lowest index of the new maximum in this chunk
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (l[i] == top) best = at + i;
    }
    const float ref = m == ninf() ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      bad = bad || l[i] != l[i];
      const float w = exp2f((l[i] - ref) * c);
      s += w;
      if (at + i < x) b += w;
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kStatThreads) verify_stat_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int N = 16 / sizeof(T);
  struct alignas(16) Chunk {
    T v[N];
  };
  const int row = blockIdx.x, split = blockIdx.y;
  const int seq = row / (a.n_draft + 1), i = row - seq * (a.n_draft + 1);
  const T* src = static_cast<const T*>(a.logits) + seq * a.logits_seq + i * a.logits_tok;
  const int lo = split * a.slice;
  const int hi = min(lo + a.slice, a.vocab);
  const float c = exponent_scale(a.temperature[seq]);
  // without draft probabilities the part of the sum before the draft is wanted
  const int x = a.draft_probs == nullptr && i < a.n_draft ? a.drafts[int64_t(seq) * a.n_draft + i] : -1;
  Running r;
  // single elements up to the first 16-byte boundary, chunks, single elements
  const int head = lo < hi ? min(int((16 - (reinterpret_cast<uintptr_t>(src + lo) & 15)) & 15) / int(sizeof(T)), hi - lo) : 0;
  const int body = lo < hi ? (hi - lo - head) / N : 0;
  const int tail = lo + head + body * N;
  if (int(threadIdx.x) < head) {
    const float l[1] = {to_f32(src[lo + threadIdx.x])};
    r.add(l, lo + threadIdx.x, c, x);
  }
#pragma unroll 4
  for (int j = threadIdx.x; j < body; j += kStatThreads) {
    const int at = lo + head + j * N;
    const Chunk ch = *reinterpret_cast<const Chunk*>(src + at);
    float l[N];
#pragma unroll
    for (int e = 0; e < N; ++e) l[e] = to_f32(ch.v[e]);
    r.add(l, at, c, x);
  }
  if (tail + int(threadIdx.x) < hi) {
    const float l[1] = {to_f32(src[tail + threadIdx.x])};
    r.add(l, tail + threadIdx.x, c, x);
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
  const float f = r.m == ninf() ? 0.f : exp2f((r.m - m) * c);
  double s = double(r.s * f), b = double(r.b * f);
  int best = r.m == m ? r.best : 0x7fffffff;
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s += __shfl_xor_sync(~0u, s, d);
    b += __shfl_xor_sync(~0u, b, d);
    best = min(best, __shfl_xor_sync(~0u, best, d));
  }
  if (lane == 0) sm[warp] = m, ss[warp] = s, sb[warp] = b, si[warp] = best;
  const int bad = __syncthreads_or(r.bad);
  if (threadIdx.x == 0) {
    VerifyPart p{};
    p.m = ninf();
    for (int w = 0; w < kStatThreads / 32; ++w) p.m = fmaxf(p.m, sm[w]);
    p.best = 0x7fffffff;
    for (int w = 0; w < kStatThreads / 32; ++w) {
      const double g = sm[w] == ninf() ? 0.0 : double(exp2f((sm[w] - p.m) * c));
      p.s += g * ss[w];
      p.b += g * sb[w];
      if (sm[w] == p.m) p.best = min(p.best, si[w]);
    }
    p.bad = bad;
    a.parts[int64_t(row) * a.splits + split] = p;
  }
}

// One position's joined sums.
struct Row {
  float m;
  double s, b;     // relative to m
  int best;
  bool usable;
};

struct Pick {
  const VerifyArgs& a;
  cg::cluster_group cl;
  int seq;
  double* box;          // this CTA's value for the others
  double* warp_box;     // [kPickWarps]
  int* int_box;
  Row* row_box;

  // Joined by warp 0 of every CTA alike.
  __device__ Row row(int i) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
      const float c = exponent_scale(a.temperature[seq]);
      const VerifyPart* p = a.parts + (int64_t(seq) * (a.n_draft + 1) + i) * a.splits;
      VerifyPart v{};
      v.m = ninf();
      v.best = 0x7fffffff;
      if (lane < a.splits) v = p[lane];
      float m = v.m;
#pragma unroll
      for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
      const double f = v.m == ninf() ? 0.0 : double(exp2f((v.m - m) * c));
      double s = v.s * f, b = v.b * f;
      int best = v.m == m ? v.best : 0x7fffffff;
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        s += __shfl_xor_sync(~0u, s, d);
        b += __shfl_xor_sync(~0u, b, d);
        best = min(best, __shfl_xor_sync(~0u, best, d));
      }
      const bool bad = __any_sync(~0u, v.bad != 0);
      if (lane == 0) *row_box = Row{m, s, b, best, !bad && m > ninf() && m < -ninf()};
    }
    __syncthreads();
    const Row r = *row_box;
    __syncthreads();
    return r;
  }

  // Every CTA's v, in rank order, into all[].
  __device__ void exchange(double v, double (&all)[kMaxCluster]) {
    if (threadIdx.x == 0) *box = v;
    cl.sync();
    for (unsigned r = 0; r < kMaxCluster; ++r) all[r] = r < cl.num_blocks() ? *cl.map_shared_rank(box, r) : 0.0;
    cl.sync();
  }
};

// The weight of element v of the drawn row: exp((l - m) / T), or what that over
// the row's sum has above the draft's probability.
template <typename T>
struct Weights {
  const T* l;
  double m, t;
  const float* q;      // nullptr: plain weights
  double total;
  __device__ __forceinline__ double plain(int v) const { return exp((double(to_f32(l[v])) - m) / t); }
  __device__ __forceinline__ double operator()(int v) const {
    const double w = plain(v);
    if (!q) return w;
    const double d = w / total - double(q[v]);
    return d > 0.0 ? d : 0.0;
  }
};

// This CTA's slice [lo, hi) of the vocabulary; its warps hold equal contiguous parts.
struct Slice {
  int lo, hi, per_warp;
};

template <typename T>
__device__ double slice_sum(Pick& k, const Weights<T>& w, const Slice& sl, double& warp_part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = min(sl.lo + warp * sl.per_warp, sl.hi), e = min(b + sl.per_warp, sl.hi);
  double v = 0;
#pragma unroll 4
  for (int j = b + lane; j < e; j += 32) v += w(j);
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  warp_part = v;
  if (lane == 0) k.warp_box[warp] = v;
  __syncthreads();
  double t = 0;
  for (int x = 0; x < kPickWarps; ++x) t += k.warp_box[x];
  return t;       // warp_box keeps the parts
}

// The lowest v whose running sum passes `goal`, by the whole cluster; sums is each
// CTA's total and warp_box each warp's.  Where rounding leaves none, the last
// element with a weight.
template <typename T>
__device__ int find(Pick& k, const Weights<T>& w, const Slice& sl, const double (&sums)[kMaxCluster], double goal) {
  const unsigned n = k.cl.num_blocks(), me = k.cl.block_rank();
  unsigned who = 0;
  double before = 0, run = 0;
  bool found = false;
  for (unsigned r = 0; r < n && !found; ++r) {
    if (sums[r] > 0) who = r, before = run;
    run += sums[r];
    found = run > goal;
  }
  if (me == who && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    double base = before;
    run = before;
    int wp = 0;
    found = false;
    for (int x = 0; x < kPickWarps && !found; ++x) {
      const double s = k.warp_box[x];
      if (s > 0) wp = x, base = run;
      run += s;
      found = run > goal;
    }
    const int b = min(sl.lo + wp * sl.per_warp, sl.hi), e = min(b + sl.per_warp, sl.hi);
    // a contiguous run of elements a lane
    const int per = (e - b + 31) / 32;
    const int lb = min(b + lane * per, e), le = min(lb + per, e);
    double v = 0;
    for (int j = lb; j < le; ++j) v += w(j);
    double incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_up_sync(~0u, incl, d);
      if (lane >= d) incl += o;
    }
    unsigned pass = __ballot_sync(~0u, v > 0 && base + incl > goal);
    if (!pass) {
      const unsigned any = __ballot_sync(~0u, v > 0);
      pass = any ? 1u << (31 - __clz(any)) : 1u;
    }
    const int ln = __ffs(pass) - 1;
    base += __shfl_sync(~0u, incl - v, ln);
    // that lane's elements, one a lane
    const int b2 = min(b + ln * per, e), e2 = min(b2 + per, e);
    int token = -1, last = -1;
    for (int j = b2; j < e2 && token < 0; j += 32) {
      v = j + lane < e2 ? w(j + lane) : 0.0;
      incl = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(~0u, incl, d);
        if (lane >= d) incl += o;
      }
      const unsigned hit = __ballot_sync(~0u, v > 0 && base + incl > goal), any = __ballot_sync(~0u, v > 0);
      if (hit) token = j + __ffs(hit) - 1;
      if (any) last = j + 31 - __clz(any);
      base += __shfl_sync(~0u, incl, 31);
    }
    if (token < 0) token = last < 0 ? b2 : last;
    if (lane == 0)
      for (unsigned r = 0; r < n; ++r) *k.cl.map_shared_rank(k.int_box, r) = token;
  }
  k.cl.sync();
  const int token = *k.int_box;
  k.cl.sync();
  return token;
}

template <typename T>
__global__ void __launch_bounds__(kPickThreads) verify_pick_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double box, warp_box[kPickWarps];
  __shared__ int int_box;
  __shared__ Row row_box;
  cg::cluster_group cl = cg::this_cluster();
  const int seq = blockIdx.x / cl.num_blocks();
  Pick k{a, cl, seq, &box, warp_box, &int_box, &row_box};
  const int per_cta = (a.vocab + int(cl.num_blocks()) - 1) / int(cl.num_blocks());
  Slice sl;
  sl.lo = min(int(cl.block_rank()) * per_cta, a.vocab);
  sl.hi = min(sl.lo + per_cta, a.vocab);
  sl.per_warp = (per_cta + kPickWarps - 1) / kPickWarps;
  const float temp = a.temperature[seq];
  const bool greedy = !(temp > 0.f);
  const double* u = a.uniforms + int64_t(seq) * (a.n_draft + 1);
  const int32_t* drafts = a.drafts + int64_t(seq) * a.n_draft;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  auto weights = [&](int i, const Row& r) {
    Weights<T> w;
    w.l = static_cast<const T*>(a.logits) + seq * a.logits_seq + i * a.logits_tok;
    w.m = double(r.m);
    w.t = double(temp);
    w.q = nullptr;
    w.total = 1.0;
    return w;
  };
  double all[kMaxCluster], warp_part;
  auto total_of = [&](const Weights<T>& w) {      // exact sum of the row; all[] and warp_box keep the parts
    k.exchange(slice_sum(k, w, sl, warp_part), all);
    double t = 0;
    for (unsigned r = 0; r < cl.num_blocks(); ++r) t += all[r];
    return t;
  };
  auto draw = [&](const Weights<T>& w, double at) {
    const double t = total_of(w);
    return find(k, w, sl, all, at * t);
  };

  int i = 0, token = -1;
  bool usable = true;
  for (;; ++i) {
    const Row r = k.row(i);
    usable = r.usable;
    const int x = i < a.n_draft ? drafts[i] : -1;
    const bool there = x >= 0 && x < a.vocab;
    if (!usable) break;
    if (greedy) {
      token = r.best;
      if (there && x == token) continue;
      break;
    }
    const Weights<T> w = weights(i, r);
    if (!a.draft_probs) {
      if (there) {
        const double goal = u[i] * r.s, wx = exp((double(to_f32(w.l[x])) - w.m) / w.t), edge = kOpen * r.s;
        if (goal > r.b + edge && goal < r.b + wx - edge) continue;      // kept, whatever the rounding
      }
      token = draw(w, u[i]);
      if (there && x == token) continue;
      break;
    }
    const float* q = a.draft_probs + seq * a.probs_seq + i * a.probs_tok;
    if (there) {
      const double have = u[i] * double(q[x]) * r.s, wx = w.plain(x);
      bool keep = have < wx;
      if (!(fabs(have - wx) > kOpen * fmax(have, wx)) && have > 0.0) keep = u[i] * double(q[x]) < wx / total_of(w);
      if (keep) continue;
    }
    Weights<T> wr = w;
    const double goal = u[a.n_draft];
    if (there) {
      wr.q = q;
      wr.total = total_of(w);
      const double over = total_of(wr);
      if (over > 0) {
        token = find(k, wr, sl, all, goal * over);
        break;
      }
    }
    token = draw(w, goal);
    break;
  }
  if (cl.block_rank() == 0) {
    int32_t* out = a.tokens + int64_t(seq) * (a.n_draft + 1);
    for (int j = threadIdx.x; j <= a.n_draft; j += kPickThreads)
      out[j] = j < i ? drafts[j] : j == i && usable ? token : -1;
    if (threadIdx.x == 0) a.counts[seq] = i + (usable ? 1 : 0);
  }
  cl.sync();      // no CTA leaves while another may still read its shared memory
}

template <typename T>
cudaError_t launch_t(const VerifyArgs& args, int cluster, cudaStream_t s) {
  VerifyArgs a = args;
  const dim3 grid(unsigned(a.n_seqs) * unsigned(a.n_draft + 1), unsigned(a.splits));
  verify_stat_kernel<T><<<grid, kStatThreads, 0, s>>>(a);
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

cudaError_t launch_verify(const VerifyArgs& a, int dtype, cudaStream_t s) {
  const int cluster = a.vocab > 4096 ? kMaxCluster : 1;
  switch (dtype) {
    case 0: return launch_t<__nv_bfloat16>(a, cluster, s);
    case 1: return launch_t<float>(a, cluster, s);
    default: return launch_t<__half>(a, cluster, s);
  }
}

}  // namespace vc

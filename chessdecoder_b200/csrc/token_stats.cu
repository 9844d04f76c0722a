// Statistics of given tokens under a row of logits: log-probability, entropy and
// the best alternatives, and the gradient of the first two (the log_softmax and
// gather of chessdecoder/rl/log_probs.py:58-101, with what a policy-gradient step
// with an entropy term and a scoring interface want beside it).
//
// With m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//   L = m + log s,  lp = x_target - L,  entropy = log s - t / s
//   dx_j = g (1[j = target] - p_j) - h p_j (log p_j + entropy)
// (m, s, t) of two parts of a row join as  a_i = e^(m_i - m):  s = sum a_i s_i,
// t = sum a_i (t_i + s_i (m_i - m)).
//
// Bound by HBM: the forward reads each logit once, the backward reads and writes
// it once.  The forward spends one ex2 and about eight other instructions per
// logit, a half (fp32) to all but a fifth (bf16) of what the SM issues in the
// time that HBM takes.
//
// Alternatives.  Each thread's largest logit comes with its running maximum.  T,
// the k-th largest of these (as a (value, index) rank), is a lower bound of the
// k-th best of the row, and only the k threads that reach T can hold one of the
// k best: their logits are read again (k of 32 or 256 threads' share, from L2),
// those that reach T are gathered in shared memory -- k and a few -- and sorted by
// a warp.  So the streaming pass has no work for the alternatives but to note
// in which of its chunks a thread's maximum lay.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "cdk.h"
#include "cdk_common.cuh"

using namespace cdk;

namespace {

constexpr int kMaxTop = 32;
constexpr int kUnroll = 4;             // 16-byte loads in flight per thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kFar = -1000.f;        // e^z is 0 in fp32 long before

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of the alternatives as one integer: larger value first, then smaller
// index.  The float's bits are mapped to an unsigned integer that orders like the
// value (-0 as +0, NaN above +inf); the index enters inverted.  0 is below every
// rank.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t j) {
  uint32_t u = __float_as_uint(x + 0.f);
  if (x != x) u = 0x7fffffffu;
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~j;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// ---------------------------------------------------------------------------
// A row as 16-byte vectors.  Vector v holds elements v * N - mis ... + N - 1, mis
// the row's distance from a 16-byte boundary, so that whole vectors are aligned
// whatever the pitch; the first and the last one may be partial.
// ---------------------------------------------------------------------------
template <bool BF16>
struct Row {
  static constexpr int N = BF16 ? 8 : 4;
  const char* base;  // address of element -mis
  int mis;
  int ncls;
  __device__ __forceinline__ Row(const void* logits, long long ldl, long long r, int n) : ncls(n) {
    const char* p = reinterpret_cast<const char*>(logits) + r * ldl * (BF16 ? 2 : 4);
    mis = (int)((reinterpret_cast<uintptr_t>(p) & 15) / (BF16 ? 2 : 4));
    base = p - mis * (BF16 ? 2 : 4);
  }
  __device__ __forceinline__ int vectors() const { return (ncls + mis + N - 1) / N; }
  __device__ __forceinline__ bool whole(int v) const { return v * N >= mis && v * N - mis + N <= ncls; }
  __device__ __forceinline__ float at(int j) const {
    if (BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[j + mis]);
    return reinterpret_cast<const float*>(base)[j + mis];
  }
  // The N elements of vector v; -inf where it reaches out of the row.
  __device__ __forceinline__ uint4 load(int v) const {
    if (whole(v)) return *reinterpret_cast<const uint4*>(base + (long long)v * 16);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (BF16) {
        const int e0 = v * N - mis + 2 * i;
        uint32_t lo = 0xff80u, hi = 0xff80u;
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base);
        if (e0 >= 0 && e0 < ncls) lo = p[e0 + mis];
        if (e0 + 1 >= 0 && e0 + 1 < ncls) hi = p[e0 + 1 + mis];
        w[i] = lo | (hi << 16);
      } else {
        const int e0 = v * N - mis + i;
        w[i] = e0 >= 0 && e0 < ncls ? reinterpret_cast<const uint32_t*>(base)[e0 + mis] : 0xff800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ void values(uint4 u, float (&x)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (BF16) {
        x[(2 * i) % N] = __uint_as_float(w[i] << 16);
        x[(2 * i + 1) % N] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        x[i % N] = __uint_as_float(w[i]);
      }
    }
  }
};

struct Stat {
  float m, s, t;  // m >= the lowest finite number, so x - m is never -inf - -inf
};

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  Stat c;
  c.m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - c.m, kFar), db = fmaxf(b.m - c.m, kFar);  // (inf - inf stays out: s is NaN then)
  const float fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
  c.s = a.s * fa + b.s * fb;
  c.t = fa * (a.t + a.s * da) + fb * (b.t + b.s * db);
  return c;
}

__device__ __forceinline__ Stat shfl_xor(const Stat& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
          __shfl_xor_sync(0xffffffffu, a.t, o)};
}

// One thread's share: vectors first, first + step, ... below last.  key: rank of its
// largest element (want_key), 0 if it has none.
template <bool BF16>
__device__ __forceinline__ Stat stream(const Row<BF16>& row, int first, int step, int last, bool want_t, bool want_key,
                                       uint64_t* key) {
  constexpr int N = Row<BF16>::N;
  Stat st{kLowest, 0.f, 0.f};
  float best = -INFINITY;  // this thread's largest element, in the chunk that begins at vector where
  int where = first;
  for (int v0 = first; v0 < last; v0 += kUnroll * step) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = v0 + u * step;
      const uint32_t none = BF16 ? 0xff80ff80u : 0xff800000u;
      raw[u] = v < last ? row.load(v) : make_uint4(none, none, none, none);
    }
    float cm = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[N];
      Row<BF16>::values(raw[u], x);
#pragma unroll
      for (int i = 0; i < N; ++i) cm = fmaxf(cm, x[i]);
    }
    if (cm > best) {
      best = cm;
      where = v0;
    }
    if (cm > st.m) {
      const float d = fmaxf(st.m - cm, kFar), f = ex2(d * kLog2e);
      st.t = f * (st.t + st.s * d);
      st.s *= f;
      st.m = cm;
    }
    float s2 = 0.f, t2 = 0.f;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[N];
      Row<BF16>::values(raw[u], x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = x[i] - st.m, e = ex2(z * kLog2e);
        s2 += e;
        if (want_t) t2 = fmaf(e, fmaxf(z, kFar), t2);
      }
    }
    st.s += s2;
    st.t += t2;
  }
  if (want_key) {
    // the first element that equals the maximum (a NaN makes s a NaN: ranked elsewhere)
    uint32_t j = 0xffffffffu;
    for (int u = kUnroll - 1; u >= 0; --u) {
      const int v = where + u * step;
      if (v >= last) continue;
      float x[N];
      Row<BF16>::values(row.load(v), x);
#pragma unroll
      for (int i = N - 1; i >= 0; --i) {
        const int e = v * N - row.mis + i;
        if (x[i] == best && e >= 0 && e < row.ncls) j = (uint32_t)e;
      }
    }
    *key = j == 0xffffffffu ? 0 : rank_key(best, j);
  }
  return st;
}

// ---------------------------------------------------------------------------
// Ranks in a warp: lane i holds one.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t exchange(uint64_t a, int o, bool keep_max) {
  const uint64_t b = __shfl_xor_sync(0xffffffffu, a, o);
  return (a > b) == keep_max ? a : b;
}
// bitonic sequence -> descending by lane
__device__ __forceinline__ uint64_t bitonic_merge(uint64_t a, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = exchange(a, o, (lane & o) == 0);
  return a;
}
__device__ __forceinline__ uint64_t sort32(uint64_t a, int lane) {
#pragma unroll
  for (int size = 2; size <= 16; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) a = exchange(a, o, ((lane & o) == 0) == ((lane & size) == 0));
  return bitonic_merge(a, lane);
}
// the 32 best of two descending lists, descending
__device__ __forceinline__ uint64_t best32(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  return bitonic_merge(a > r ? a : r, lane);
}

// Candidates: the elements of thread `owner`'s share (as in stream) whose rank
// reaches T, taken by threads i = 0 ... n - 1 together.
constexpr int kCandidates = 512;
template <bool BF16>
__device__ __forceinline__ void gather_share(const Row<BF16>& row, int v, uint64_t T, uint64_t* cand, int* count) {
  constexpr int N = Row<BF16>::N;
  float x[N];
  Row<BF16>::values(row.load(v), x);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = v * N - row.mis + i;
    if (e < 0 || e >= row.ncls) continue;
    const uint64_t key = rank_key(x[i], (uint32_t)e);
    if (key >= T) {
      const int at = atomicAdd(count, 1);
      if (at < kCandidates) cand[at] = key;
    }
  }
}

struct Args {
  const void* logits;
  long long ldl, rows;
  int ncls;
  const int32_t* target;
  float* lp;
  float* entropy;
  float* lse;
  int32_t* top_ids;
  float* top_lp;
  int k;
};

// Outputs of row r from its joined statistics (one thread), and its alternatives
// (one warp, lane i the i-th best rank).
template <bool BF16>
__device__ __forceinline__ void finish(const Args& a, const Row<BF16>& row, long long r, const Stat& st, int lane,
                                       uint64_t top) {
  const bool none = st.s == 0.f;  // every logit -inf
  const float ls = logf(st.s);
  if (lane == 0) {
    const int tg = a.target[r];
    a.lp[r] = (tg < 0 || tg >= a.ncls) ? 0.f : none ? -INFINITY : (row.at(tg) - st.m) - ls;
    if (a.entropy) a.entropy[r] = none ? 0.f : ls - st.t / st.s;
    if (a.lse) a.lse[r] = none ? -INFINITY : st.m + ls;
  }
  if (lane < a.k) {
    a.top_ids[r * a.k + lane] = (int32_t)~(uint32_t)top;
    a.top_lp[r * a.k + lane] = none ? -INFINITY : (key_value(top) - st.m) - ls;
  }
}

// The k best of vectors [v0, v1) by k passes of one warp: for rows with a NaN, and
// where more candidates reach T than there is room for (hundreds of the best
// logits in the share of k threads).
template <bool BF16>
__device__ __noinline__ uint64_t slow_top(const Row<BF16>& row, int v0, int v1, int k, int lane) {
  constexpr int N = Row<BF16>::N;
  uint64_t last = ~0ull, mine = 0;
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (int v = v0 + lane; v < v1; v += 32) {
      float x[N];
      Row<BF16>::values(row.load(v), x);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const int e = v * N - row.mis + c;
        const uint64_t key = e >= 0 && e < row.ncls ? rank_key(x[c], (uint32_t)e) : 0;
        if (key < last && key > best) best = key;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    last = best;
    if (lane == i) mine = best;
  }
  return mine;
}

// ---------------------------------------------------------------------------
// Short rows: a warp per row.
// ---------------------------------------------------------------------------
constexpr int kWarpsPerBlock = 8;

template <bool BF16>
__global__ void __launch_bounds__(kWarpsPerBlock * 32) token_stats_warp_kernel(const Args a) {
  __shared__ uint64_t cand_s[kWarpsPerBlock][kCandidates];
  __shared__ int count_s[kWarpsPerBlock];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r = (long long)blockIdx.x * kWarpsPerBlock + warp;
  if (r >= a.rows) return;
  const Row<BF16> row(a.logits, a.ldl, r, a.ncls);
  const int nv = row.vectors();
  uint64_t key = 0;
  Stat st = stream<BF16>(row, lane, 32, nv, a.entropy != nullptr, a.k > 0, &key);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st = join(st, shfl_xor(st, o));
  uint64_t top = 0;
  if (a.k > 0) {
    if (st.s != st.s) {
      top = slow_top<BF16>(row, 0, nv, a.k, lane);
    } else {
      const uint64_t T = __shfl_sync(0xffffffffu, sort32(key, lane), a.k - 1);
      uint32_t owners = __ballot_sync(0xffffffffu, key != 0 && key >= T);
      if (lane == 0) count_s[warp] = 0;
      __syncwarp();
      const int per = (nv + 31) / 32;  // vectors of a lane's share
      while (owners) {
        const int c = __ffs(owners) - 1;
        owners &= owners - 1;
        for (int i = lane; i < per; i += 32)
          if (c + 32 * i < nv) gather_share<BF16>(row, c + 32 * i, T, cand_s[warp], &count_s[warp]);
      }
      __syncwarp();
      const int n = count_s[warp];
      if (n > kCandidates) {
        top = slow_top<BF16>(row, 0, nv, a.k, lane);
      } else {
        top = sort32(lane < n ? cand_s[warp][lane] : 0, lane);
        for (int i = 32; i < n; i += 32) top = best32(top, sort32(i + lane < n ? cand_s[warp][i + lane] : 0, lane), lane);
      }
    }
  }
  finish<BF16>(a, row, r, st, lane, top);
}

// ---------------------------------------------------------------------------
// Long rows: a block of 256 threads per row, or a cluster of blocks that share
// the row's vectors when there are few rows; the blocks' (m, s, t) and best lists
// are joined by the first of them through distributed shared memory.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kRowWarps = kThreads / 32;

struct RowShared {
  uint64_t lists[kRowWarps][32];
  uint64_t cand[kCandidates];
  uint64_t best[32];  // this block's best, descending
  uint64_t T;
  int owners[32];
  int n_owners, count;
  Stat part[kRowWarps];
  Stat st;            // this block's
};

__device__ __forceinline__ const RowShared* remote(const RowShared* p, uint32_t rank) {
  uint64_t q;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<const RowShared*>(q);
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads) token_stats_block_kernel(const Args a, int blocks_per_row) {
  __shared__ RowShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x / blocks_per_row;
  const int rank = (int)(blockIdx.x % blocks_per_row);
  const Row<BF16> row(a.logits, a.ldl, r, a.ncls);
  const int nv = row.vectors();
  const int per_block = (nv + blocks_per_row - 1) / blocks_per_row;
  const int v0 = min(rank * per_block, nv), v1 = min(v0 + per_block, nv);
  uint64_t key = 0;
  Stat st = stream<BF16>(row, v0 + tid, kThreads, v1, a.entropy != nullptr, a.k > 0, &key);
  const uint64_t mine = key;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st = join(st, shfl_xor(st, o));
  if (lane == 0) sh.part[warp] = st;
  if (a.k > 0) sh.lists[warp][lane] = sort32(key, lane);
  if (tid == 0) sh.n_owners = sh.count = 0;
  __syncthreads();
  st = sh.part[0];
#pragma unroll
  for (int w = 1; w < kRowWarps; ++w) st = join(st, sh.part[w]);  // the same order in every thread
  const bool broken = st.s != st.s;
  if (a.k > 0 && !broken) {
    if (warp == 0) {
      uint64_t l = sh.lists[0][lane];
#pragma unroll 1
      for (int w = 1; w < kRowWarps; ++w) l = best32(l, sh.lists[w][lane], lane);
      if (lane == a.k - 1) sh.T = l;
    }
    __syncthreads();
    const uint64_t T = sh.T;
    if (mine != 0 && mine >= T) sh.owners[atomicAdd(&sh.n_owners, 1)] = tid;  // at most k of them
    __syncthreads();
    const int per = (v1 - v0 + kThreads - 1) / kThreads;
    for (int i = tid; i < sh.n_owners * per; i += kThreads) {
      const int v = v0 + sh.owners[i / per] + kThreads * (i % per);
      if (v < v1) gather_share<BF16>(row, v, T, sh.cand, &sh.count);
    }
    __syncthreads();
  }
  uint64_t top = 0;
  if (warp == 0 && a.k > 0) {
    const int n = sh.count;
    if (broken || n > kCandidates) {
      top = slow_top<BF16>(row, v0, v1, a.k, lane);
    } else {
      top = sort32(lane < n ? sh.cand[lane] : 0, lane);
      for (int i = 32; i < n; i += 32) top = best32(top, sort32(i + lane < n ? sh.cand[i + lane] : 0, lane), lane);
    }
  }
  if (blocks_per_row > 1) {
    if (warp == 0) sh.best[lane] = top;
    if (tid == 0) sh.st = st;
    cluster_sync();
    if (rank == 0 && warp == 0) {
      for (int c = 1; c < blocks_per_row; ++c) {
        const RowShared* o = remote(&sh, (uint32_t)c);
        st = join(st, Stat{o->st.m, o->st.s, o->st.t});
        if (a.k > 0) top = best32(top, o->best[lane], lane);
      }
    }
    cluster_sync();  // the others' shared memory stays until it has been read
    if (rank != 0) return;
  }
  if (warp == 0) finish<BF16>(a, row, r, st, lane, top);
}

// ---------------------------------------------------------------------------
// Backward: a warp per kUnroll * 32 vectors of a row.  logits and dlogits may be
// the same: every element is read by the thread that writes it.
// ---------------------------------------------------------------------------
template <bool BF16>
__global__ void __launch_bounds__(256)
    token_stats_bwd_kernel(const void* logits, long long ldl, long long rows, int ncls,
                           const int32_t* __restrict__ target, const float* __restrict__ lse,
                           const float* __restrict__ entropy, const float* __restrict__ dlp,
                           const float* __restrict__ dentropy, void* dlogits, long long ldd, int slabs) {
  constexpr int N = Row<BF16>::N;
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long r = unit / slabs;
  if (r >= rows) return;
  const int v0 = (int)(unit % slabs) * (32 * kUnroll) + lane;
  const Row<BF16> row(logits, ldl, r, ncls);
  const int nv = row.vectors();
  const int tg = target[r];
  const float g = dlp && tg >= 0 && tg < ncls ? dlp[r] : 0.f;
  const float h = dentropy ? dentropy[r] : 0.f;
  const float L = lse[r], H = dentropy ? entropy[r] : 0.f;
  const bool zero = L == -INFINITY || (g == 0.f && h == 0.f && L == L);  // nothing to read
  uint4 raw[kUnroll];
  if (!zero) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + 32 * u < nv) raw[u] = row.load(v0 + 32 * u);
  }
  char* out = reinterpret_cast<char*>(dlogits) + r * ldd * (BF16 ? 2 : 4);  // element 0
  const bool same = ((reinterpret_cast<uintptr_t>(out) & 15) / (BF16 ? 2 : 4)) == (uintptr_t)row.mis;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int v = v0 + 32 * u;
    if (v >= nv) break;
    const int e0 = v * N - row.mis;
    float d[N];
    if (zero) {
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = 0.f;
    } else {
      Row<BF16>::values(raw[u], d);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = d[i] - L, p = ex2(z * kLog2e);
        float y = -p * fmaf(h, z + H, g);
        if (p == 0.f) y = 0.f;
        if (e0 + i == tg) y += g;
        d[i] = y;
      }
    }
    if (same && row.whole(v)) {
      uint4 w;
      if (BF16)
        w = make_uint4(pack_bf16(d[0], d[1]), pack_bf16(d[2 % N], d[3 % N]), pack_bf16(d[4 % N], d[5 % N]),
                       pack_bf16(d[6 % N], d[7 % N]));
      else
        w = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2 % N]),
                       __float_as_uint(d[3 % N]));
      *reinterpret_cast<uint4*>(out + (long long)e0 * (BF16 ? 2 : 4)) = w;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = e0 + i;
        if (e < 0 || e >= ncls) continue;
        if (BF16) reinterpret_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(d[i]);
        else reinterpret_cast<float*>(out)[e] = d[i];
      }
    }
  }
}

inline bool al(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

template <bool BF16>
cudaError_t launch_fwd(const Args& a, cudaStream_t st) {
  const int n = BF16 ? 8 : 4;
  // A warp per row up to 4096 bytes per lane's four loads twice over; beyond that
  // (or with fewer rows than would fill the device) a block per row, and a cluster
  // of blocks per row while there are fewer blocks than two per SM.
  const long long vectors = (a.ncls + n - 1) / n;
  if (vectors <= 8 * 32 || (vectors <= 32 * 32 && a.rows >= 148 * 16)) {
    const long long blocks = (a.rows + kWarpsPerBlock - 1) / kWarpsPerBlock;
    token_stats_warp_kernel<BF16><<<(unsigned)blocks, kWarpsPerBlock * 32, 0, st>>>(a);
    return cudaGetLastError();
  }
  int c = 1;
  while (c < 8 && a.rows * c < 2 * 148 && vectors >= 2 * c * kThreads * kUnroll) c *= 2;
  if (a.rows * c > 0x7fffffffll) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * c));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, token_stats_block_kernel<BF16>, (const Args)a, c);
}

}  // namespace

extern "C" int cdk_token_logprobs(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                  const int32_t* target, float* lp, float* entropy, float* lse, int32_t* top_ids,
                                  float* top_lp, int64_t k, void* stream) {
  if (rows == 0) return 0;
  if (!logits || !target || !lp || rows < 0 || rows > 0x7fffffff) return -1;
  if (dtype != 0 && dtype != 1) return -2;
  if (ncls <= 0 || ncls >= 0x7fffffe0 || ldl < ncls) return -3;
  if (!al(logits, dtype ? 2 : 4)) return -4;
  if (!top_ids != !top_lp) return -5;
  if (!top_ids) k = 0;
  if (k < 0 || k > kMaxTop || k > ncls) return -6;
  const Args a{logits, ldl, rows, (int)ncls, target, lp, entropy, lse, top_ids, top_lp, (int)k};
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  return (int)(dtype ? launch_fwd<true>(a, st) : launch_fwd<false>(a, st));
}

extern "C" int cdk_token_logprobs_bwd(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                      const int32_t* target, const float* lse, const float* entropy, const float* dlp,
                                      const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  if (rows == 0) return 0;
  if (!logits || !target || !lse || !dlogits || rows < 0 || rows > 0x7fffffff) return -1;
  if (dtype != 0 && dtype != 1) return -2;
  if (ncls <= 0 || ncls >= 0x7fffffe0 || ldl < ncls || ldd < ncls) return -3;
  if (!al(logits, dtype ? 2 : 4) || !al(dlogits, dtype ? 2 : 4)) return -4;
  if (dentropy && !entropy) return -5;
  if (logits == dlogits && ldl != ldd) return -6;
  const int n = dtype ? 8 : 4;
  const long long slabs = ((ncls + n - 1) / n + 1 + 32 * kUnroll - 1) / (32 * kUnroll);  // + 1: a row that begins inside a vector
  const long long blocks = (rows * slabs + 7) / 8;
  if (blocks > 0x7fffffff) return -7;
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype)
    token_stats_bwd_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(logits, ldl, rows, (int)ncls, target, lse, entropy,
                                                                   dlp, dentropy, dlogits, ldd, (int)slabs);
  else
    token_stats_bwd_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(logits, ldl, rows, (int)ncls, target, lse, entropy,
                                                                    dlp, dentropy, dlogits, ldd, (int)slabs);
  return (int)cudaGetLastError();
}

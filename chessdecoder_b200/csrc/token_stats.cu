// Statistics of given tokens under a row of logits: log-probability, entropy and
// the best alternatives, and the gradient of the first two (the log_softmax and
// gather of chessdecoder/rl/log_probs.py:58-101, with what a policy-gradient step
// with an entropy term and a scoring interface want beside it).
//
// With m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//   L = m + log s,  lp = x_target - L,  entropy = log s - t / s
//   dx_j = g (1[j = target] - p_j) - h p_j (log p_j + entropy)
// L alone is off by half a step of it, which would be a relative error of every p_j of
// the row, so the gradient takes what its rounding lost as well.
// (m, s, t) of two parts of a row join as  a_i = e^(m_i - m):  s = sum a_i s_i,
// t = sum a_i (t_i + s_i (m_i - m)).
//
// Bound by HBM: the forward reads each logit once, the backward reads and writes
// it once.  The forward spends one ex2 and about eight other instructions per
// logit, half (fp32) to most (bf16) of what an SM issues in the time that HBM takes.
//
// Alternatives.  A thread notes the maximum of each of up to four parts of its vectors.
// T, the k-th largest of the threads' maxima (or parts' of them), is a lower bound of
// the k-th best logit, and only a share (of a thread and part) whose maximum reaches T
// can hold one of the k best: these few are read again, the logits that reach T are
// gathered in shared memory -- k and a few -- and sorted by a warp.  So the streaming
// pass has next to no work for the alternatives.
//
// Measured on one B200 (device time, share of the copy rate): 16384 x 1924 fp32
// forward 23 us (84%), with 5 alternatives 36 us (54%), gradient 41 us (95%); 8192 x 8000
// fp32 forward 46 us (88%), with 5 alternatives 53 us (77%); 509 x 131071 bf16 forward
// 32 us (65%), with 20 alternatives 36 us (58%: selecting takes each block about 3 us
// at its end, when its neighbours do the same), gradient 43 us (96%); 300 x 131071
// fp32 forward 29 us (84%).
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
// rank, ~0 above.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t j) {
  uint32_t u = __float_as_uint(x + 0.f);
  if (x != x) u = 0x7fc00000u;
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~j;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// ---------------------------------------------------------------------------
// A row as 16-byte vectors.  Vector v holds elements v * N - mis ... + N - 1, mis
// the row's distance from a 16-byte boundary, so that vectors are aligned whatever
// the pitch.  Those that lie in the row entirely are [begin, end); the elements
// before and behind them, fewer than N each, are the edges: lane i has edge i.
// ---------------------------------------------------------------------------
template <bool BF16>
struct Row {
  static constexpr int N = BF16 ? 8 : 4;
  static constexpr int kElt = BF16 ? 2 : 4;
  const char* base;  // address of element -mis
  int mis, ncls;
  __device__ __forceinline__ Row(const void* logits, long long ldl, long long r, int n) : ncls(n) {
    const char* p = reinterpret_cast<const char*>(logits) + r * ldl * kElt;
    mis = (int)((reinterpret_cast<uintptr_t>(p) & 15) / kElt);
    base = p - mis * kElt;
  }
  __device__ __forceinline__ int begin() const { return mis > 0 ? 1 : 0; }
  __device__ __forceinline__ int end() const { return max((ncls + mis) / N, begin()); }
  __device__ __forceinline__ float at(int j) const {
    if (BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[j + mis]);
    return reinterpret_cast<const float*>(base)[j + mis];
  }
  __device__ __forceinline__ uint4 load(int v) const {
    return *reinterpret_cast<const uint4*>(base + (long long)v * 16);
  }
  // Element of edge i < 32, -1 if there is none: the first ones, then the last ones.
  __device__ __forceinline__ int edge(int i) const {
    const int head = mis > 0 ? min(N - mis, ncls) : 0, tail0 = end() * N - mis;
    if (i < head) return i;
    const int j = max(tail0, head) + (i - head);
    return j < ncls && i < 2 * N ? j : -1;
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

// Largest element of a vector (NaN ignored).
template <bool BF16>
__device__ __forceinline__ float vector_max(uint4 u) {
  if (BF16) {
    const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}

struct Stat {
  float m, s, t;  // m >= the lowest finite number, so x - m is never -inf - -inf
  __device__ __forceinline__ void rise(float to) {  // a new maximum
    const float d = fmaxf(m - to, kFar), f = ex2(d * kLog2e);  // (inf - inf stays out: s is a NaN then)
    t = f * (t + s * d);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {
    if (x > m) rise(x);
    const float z = x - m, e = ex2(z * kLog2e);
    s += e;
    t = fmaf(e, fmaxf(z, kFar), t);
  }
};

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  a.rise(m);
  b.rise(m);
  return {m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ Stat join_warp(Stat a) {
  a.rise(warp_max(a.m));
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  return a;
}

// One thread's share of a row: vectors first + tid, first + tid + STEP, ... below
// last and the edge with index `edge` (or none: -1).  PARTS > 0: the largest of its
// vectors' elements in each part of [first, last), parts of `part` chunks (of kUnroll
// vectors a thread), goes to maxima[p * STEP + tid], and that of all to best.  PARTS *
// part is above the chunks that every thread has whole.
template <bool BF16, int STEP, int PARTS>
__device__ __forceinline__ Stat stream(const Row<BF16>& row, int first, int tid, int last, int edge, bool want_t,
                                       int part, float* maxima, float* best) {
  constexpr int N = Row<BF16>::N;
  Stat st{kLowest, 0.f, 0.f};
  float most = -INFINITY;  // in this part
  int p = 0, left = part;
  if (PARTS) *best = -INFINITY;
  auto rise = [&](float cm) {
    if (PARTS) most = fmaxf(most, cm);
    if (cm > st.m) st.rise(cm);
  };
  auto add = [&](uint4 raw, float (&s2)[2], float (&t2)[2]) {
    float x[N];
    Row<BF16>::values(raw, x);
    if (want_t) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = x[i] - st.m, e = ex2(z * kLog2e);
        s2[i & 1] += e;
        t2[i & 1] = fmaf(e, fmaxf(z, kFar), t2[i & 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) s2[i & 1] += ex2((x[i] - st.m) * kLog2e);
    }
  };
  uint4 raw[kUnroll];
  bool more = first + kUnroll * STEP <= last;  // a chunk that every thread has whole
  if (more) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = row.load(first + tid + u * STEP);
  }
#pragma unroll 1
  while (more) {
    first += kUnroll * STEP;
    more = first + kUnroll * STEP <= last;
    uint4 next[kUnroll];
    if (more) {  // the next chunk is on its way while this one is added up
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) next[u] = row.load(first + tid + u * STEP);
    }
    float cm = vector_max<BF16>(raw[0]);
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) cm = fmaxf(cm, vector_max<BF16>(raw[u]));
    rise(cm);
    float s2[2] = {0.f, 0.f}, t2[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) add(raw[u], s2, t2);
    st.s += s2[0] + s2[1];
    st.t += t2[0] + t2[1];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = next[u];
    if (PARTS && --left == 0) {
      maxima[p++ * STEP + tid] = most;
      *best = fmaxf(*best, most);
      most = -INFINITY;
      left = part;
    }
  }
  const int v = first + tid;
  if (v < last) {  // what is left: a vector at least
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * STEP < last) raw[u] = row.load(v + u * STEP);
    float cm = vector_max<BF16>(raw[0]);
#pragma unroll
    for (int u = 1; u < kUnroll; ++u)
      if (v + u * STEP < last) cm = fmaxf(cm, vector_max<BF16>(raw[u]));
    rise(cm);
    float s2[2] = {0.f, 0.f}, t2[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * STEP < last) add(raw[u], s2, t2);
    st.s += s2[0] + s2[1];
    st.t += t2[0] + t2[1];
  }
  const int e = edge >= 0 ? row.edge(edge) : -1;
  if (e >= 0) st.add(row.at(e));
  if (PARTS) {
    maxima[p * STEP + tid] = most;
    *best = fmaxf(*best, most);
  }
  return st;
}

// ---------------------------------------------------------------------------
// Ranks, or values, in a warp: lane i holds one.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t exchange(uint64_t a, int o, bool keep_max) {
  const uint64_t b = __shfl_xor_sync(0xffffffffu, a, o);
  return (a > b) == keep_max ? a : b;
}
__device__ __forceinline__ float exchange(float a, int o, bool keep_max) {
  const float b = __shfl_xor_sync(0xffffffffu, a, o);
  return keep_max ? fmaxf(a, b) : fminf(a, b);
}
// bitonic sequence -> descending by lane
template <typename T>
__device__ __forceinline__ T bitonic_merge(T a, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = exchange(a, o, (lane & o) == 0);
  return a;
}
template <typename T>
__device__ __forceinline__ T sort32(T a, int lane) {
#pragma unroll
  for (int size = 2; size <= 16; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) a = exchange(a, o, ((lane & o) == 0) == ((lane & size) == 0));
  return bitonic_merge(a, lane);
}
// the 32 best of two descending lists, descending
template <typename T>
__device__ __forceinline__ T best32(T a, T b, int lane) {
  const T r = __shfl_sync(0xffffffffu, b, 31 - lane);
  return bitonic_merge(a > r ? a : r, lane);
}

// Rank that bounds the k-th best from below, from the value of the k-th maximum.  Every
// element of the value reaches it; where that is -inf (fewer than k maxima are above:
// a masked row), only the first k elements, from index `first` on.
__device__ __forceinline__ uint64_t bound(float value, int first, int k) {
  return rank_key(value, value == -INFINITY ? (uint32_t)(first + k - 1) : 0xffffffffu);
}

// Whether a share whose vectors begin with element `first`, `best` the largest, may hold
// a rank that reaches T.
__device__ __forceinline__ bool owns(uint64_t T, float best, uint32_t first) {
  const float value = key_value(T);
  return best > value || (best == value && first <= ~(uint32_t)T);
}

// Elements whose rank reaches T join the candidates, until there is no room: count is
// above `most` then.  (Of a warp's 32 maxima the 32nd is a weak bound; in a row of equal
// logits every element reaches it.)  The k-th best of those that found room is a better
// bound, and the look is repeated with it, up to kLooks times.
constexpr int kCandidates = 512, kLooks = 4;
template <bool SHARED>  // by several warps: count is in shared memory; else it is the warp's own
struct Candidates {
  uint64_t* list;
  int* count;
  int most;
  uint64_t T;
  float value;  // T's
  __device__ __forceinline__ Candidates(uint64_t* l, int* c, int m, uint64_t T_)
      : list(l), count(c), most(m), T(T_), value(key_value(T_)) {}
  __device__ __forceinline__ bool full() const {  // the same in every lane of the warp
    return SHARED ? __any_sync(0xffffffffu, *const_cast<volatile int*>(count) > most) : *count > most;
  }
  // Elements e + i, x[i], of every lane that has them; each lane's one by one.  A warp on
  // its own counts by ballots (a shared atomic per candidate costs some 70 cycles each;
  // 4000 rows of 3934 bf16 with 24 alternatives: 37 us, 24 so); the warps of a block
  // have a few each.
  template <int N>
  __device__ __forceinline__ void take(const float (&x)[N], int e, bool have, int lane) const {
    uint32_t left = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) left |= x[i] < value ? 0u : 1u << i;
    if (!have) left = 0;
    while (SHARED ? left != 0 : __any_sync(0xffffffffu, left != 0)) {
      const int i = __ffs(left) - 1;
      float y = x[0];
#pragma unroll
      for (int c = 1; c < N; ++c) y = i == c ? x[c] : y;
      const uint64_t key = rank_key(y, (uint32_t)(e + i));
      const bool in = left != 0 && key >= T;
      left &= left - 1;
      int at = most;
      if (SHARED) {
        if (in && (at = atomicAdd(count, 1)) >= most) break;
      } else {
        const uint32_t mask = __ballot_sync(0xffffffffu, in);
        if (in) at = *count + __popc(mask & ((1u << lane) - 1));
        *count += __popc(mask);
      }
      if (at < most) list[at] = key;
    }
  }
  // Second look at n shares, owner o's being vectors o % STEP, + STEP, ... of part o / STEP
  // of [v0, v1), by THREADS threads: 2^lg of them, the least power of two that covers a share, per
  // owner.  Where all shares are owners, in the row's order: equal logits (a mask's) leave
  // no room then, and what found room has the low indices.
  template <bool BF16, int STEP, int THREADS>
  __device__ __forceinline__ void take_shares(const Row<BF16>& row, int v0, int v1, int part, const uint16_t* owners,
                                              int n, int shares, int tid) const {
    constexpr int N = Row<BF16>::N;
    const int per = (part + STEP - 1) / STEP, lg = per > 1 ? 32 - __clz(per - 1) : 0, lane = tid & 31;
    const bool all = n == shares;
    const int slots = all ? v1 - v0 : n << lg;
    for (int i0 = tid - lane; i0 < slots; i0 += 4 * THREADS) {
      if (full()) return;
      uint4 raw[4];
      int v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + lane + u * THREADS;
        v[u] = v1;
        if (i < slots && all) {
          v[u] = v0 + i;
        } else if (i < slots) {
          const int o = owners[i >> lg], at = o % STEP + STEP * (i & ((1 << lg) - 1));  // in its part
          if (at < part) v[u] = v0 + o / STEP * part + at;
        }
        raw[u] = v[u] < v1 ? row.load(v[u]) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool have = v[u] < v1 && !(vector_max<BF16>(raw[u]) < value);
        if (SHARED ? !have : !__any_sync(0xffffffffu, have)) continue;
        float x[N];
        Row<BF16>::values(raw[u], x);
        take(x, v[u] * N - row.mis, have, lane);
      }
    }
  }
};

struct Args {
  const void* logits;
  long long ldl, rows;
  int ncls;
  const int32_t* target;
  float* lp;
  float* entropy;
  float* lse;
  float* lse_low;
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
    const float L = none ? -INFINITY : st.m + ls;
    if (a.lse) a.lse[r] = L;
    if (a.lse_low) {  // the rest of the sum, exactly: the parts of m and log s that L holds taken from them
      const float of_m = L - ls, of_ls = L - of_m;
      a.lse_low[r] = none ? 0.f : (st.m - of_m) + (ls - of_ls);
    }
  }
  if (lane < a.k) {
    a.top_ids[r * a.k + lane] = (int32_t)~(uint32_t)top;
    a.top_lp[r * a.k + lane] = none ? -INFINITY : (key_value(top) - st.m) - ls;
  }
}

// The k best of vectors [v0, v1) and, if asked, the edges by k passes of one warp: for
// rows with a NaN, and where more candidates reach T than there is room for after
// kLooks looks (thousands of the best logits, ascending, in the share of k threads).
template <bool BF16>
__device__ __noinline__ uint64_t slow_top(const Row<BF16>& row, int v0, int v1, bool edges, int k, int lane) {
  constexpr int N = Row<BF16>::N;
  uint64_t last = ~0ull, mine = 0;
  const int e = edges ? row.edge(lane) : -1;
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    if (e >= 0) {
      const uint64_t key = rank_key(row.at(e), (uint32_t)e);
      if (key < last) best = key;
    }
    for (int v = v0 + lane; v < v1; v += 32) {
      float x[N];
      Row<BF16>::values(row.load(v), x);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const uint64_t key = rank_key(x[c], (uint32_t)(v * N - row.mis + c));
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

// The 32 best of n gathered candidates, descending by lane.
__device__ __forceinline__ uint64_t best_of(const uint64_t* cand, int n, int lane) {
  uint64_t top = sort32(lane < n ? cand[lane] : 0, lane);
#pragma unroll 1
  for (int i = 32; i < n; i += 32) top = best32(top, sort32(i + lane < n ? cand[i + lane] : 0, lane), lane);
  return top;
}

// ---------------------------------------------------------------------------
// Short rows: a warp per row.
// ---------------------------------------------------------------------------
constexpr int kWarpsPerBlock = 8;
constexpr int kWarpCandidates = 160;  // the slow way is short here, and shared memory is warps

// Parts of a row whose shares are looked at again apart: of 4 x 32 shares (or 4 x 256)
// those that can hold one of the best are little of the row.
constexpr int kParts = 4;
struct Parts {
  int chunks, vectors;  // of one
  int n;                // those that are not empty
  __device__ __forceinline__ Parts(int vectors_, int step) {
    const int whole = vectors_ / (step * kUnroll);
    chunks = whole / kParts + 1;
    vectors = chunks * step * kUnroll;
    n = whole / chunks + 1;
  }
};

template <bool BF16, bool TOP>
__global__ void __launch_bounds__(kWarpsPerBlock * 32, TOP ? 4 : 5) token_stats_warp_kernel(const Args a) {
  constexpr int N = Row<BF16>::N;
  __shared__ uint64_t cand_s[TOP ? kWarpsPerBlock : 1][TOP ? kWarpCandidates : 1];
  __shared__ float maxima_s[TOP ? kWarpsPerBlock : 1][TOP ? kParts * 32 : 1];
  __shared__ uint16_t owners_s[TOP ? kWarpsPerBlock : 1][TOP ? kParts * 32 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r = (long long)blockIdx.x * kWarpsPerBlock + warp;
  if (r >= a.rows) return;
  const Row<BF16> row(a.logits, a.ldl, r, a.ncls);
  const int v0 = row.begin(), v1 = row.end();
  const Parts parts(v1 - v0, 32);
  float* maxima = maxima_s[TOP ? warp : 0];
  uint16_t* owners = owners_s[TOP ? warp : 0];
  float best;  // of this lane
  const Stat st = join_warp(
      stream<BF16, 32, TOP ? kParts : 0>(row, v0, lane, v1, lane, a.entropy != nullptr, parts.chunks, maxima, &best));
  uint64_t top = 0;
  if (TOP) {
    bool slow = st.s != st.s;
    // the k-th of 32 maxima, or 64 or 128 where k is near that: the 32nd of 32 admits 130 of a row, of 128 37
    const int lists = min(a.k <= 12 ? 1 : a.k <= 24 ? 2 : 4, parts.n);
    float order = -INFINITY;
    if (lists == 1) {
      order = sort32(best, lane);
    } else {
#pragma unroll 1
      for (int i = 0; i < lists; ++i) {
        float x = -INFINITY;
        for (int p = i; p < parts.n; p += lists) x = fmaxf(x, maxima[p * 32 + lane]);
        order = best32(order, sort32(x, lane), lane);
      }
    }
    uint64_t T = bound(__shfl_sync(0xffffffffu, order, a.k - 1), 0, a.k);
#pragma unroll 1
    for (int look = 0; !slow; ++look) {
      int n_owners = 0;
#pragma unroll 1
      for (int p = 0; p < parts.n; ++p) {
        const bool owner = owns(T, maxima[p * 32 + lane], (uint32_t)(p * parts.vectors + lane) * N);
        const uint32_t mask = __ballot_sync(0xffffffffu, owner);
        if (owner) owners[n_owners + __popc(mask & ((1u << lane) - 1))] = (uint16_t)(p * 32 + lane);
        n_owners += __popc(mask);
      }
      __syncwarp();
      int n = 0;
      const Candidates<false> cand(cand_s[TOP ? warp : 0], &n, kWarpCandidates, T);
      const int e = row.edge(lane);
      const float xe[1] = {e >= 0 ? row.at(e) : 0.f};
      cand.take(xe, e, e >= 0, lane);
      cand.take_shares<BF16, 32, 32>(row, v0, v1, parts.vectors, owners, n_owners, 32 * parts.n, lane);
      __syncwarp();
      top = best_of(cand_s[TOP ? warp : 0], min(n, kWarpCandidates), lane);
      if (n <= kWarpCandidates) break;
      T = __shfl_sync(0xffffffffu, top, a.k - 1);
      slow = look == kLooks - 1;
      __syncwarp();  // every lane has read the list
    }
    if (slow) top = slow_top<BF16>(row, v0, v1, true, a.k, lane);
  }
  finish<BF16>(a, row, r, st, lane, top);
}

// ---------------------------------------------------------------------------
// Long rows: a block of 256 or 128 threads per row, or a cluster of blocks that share
// the row's vectors; the blocks' (m, s, t) and best lists are joined by the first
// of them through distributed shared memory.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;

template <bool TOP, int THREADS>
struct RowShared {
  uint64_t cand[TOP ? kCandidates : 1];
  uint64_t best[32];  // this block's best, descending
  uint64_t T;
  float maxima[64];   // of THREADS / 64 threads each
  float shares[TOP ? kParts * THREADS : 1];
  uint16_t owners[TOP ? kParts * THREADS : 1];
  int n_owners, count;
  Stat part[THREADS / 32];
  Stat st;            // this block's
};

template <typename T>
__device__ __forceinline__ const T* remote(const T* p, uint32_t rank) {
  uint64_t q;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<const T*>(q);
}

template <bool BF16, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, (TOP ? 4 : 5) * kThreads / THREADS) token_stats_block_kernel(const Args a, int blocks_per_row) {
  __shared__ RowShared<TOP, THREADS> sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x / blocks_per_row;
  const int rank = (int)(blockIdx.x % blocks_per_row);
  const Row<BF16> row(a.logits, a.ldl, r, a.ncls);
  const int begin = row.begin(), end = row.end();
  const int per_block = (end - begin + blocks_per_row - 1) / blocks_per_row;
  const int v0 = min(begin + rank * per_block, end), v1 = min(v0 + per_block, end);
  const int first = rank == 0 ? 0 : v0 * Row<BF16>::N - row.mis;  // element
  const int edge = rank == 0 && warp == 0 ? lane : -1;  // the first warp of the first block has the edges
  const Parts parts(v1 - v0, THREADS);
  float best;  // of this thread
  Stat st = stream<BF16, THREADS, TOP ? kParts : 0>(row, v0, tid, v1, edge, a.entropy != nullptr, parts.chunks,
                                                    sh.shares, &best);
  if (TOP) {
    constexpr int kGroup = THREADS / 64;
    float x = best;
#pragma unroll
    for (int o = 1; o < kGroup; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    if (lane % kGroup == 0) sh.maxima[tid / kGroup] = x;
  }
  st = join_warp(st);
  if (lane == 0) sh.part[warp] = st;
  if (tid == 0) sh.n_owners = sh.count = 0;
  __syncthreads();
  st = sh.part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) st = join(st, sh.part[w]);  // the same order in every thread
  uint64_t top = 0;
  if (TOP) {
    const bool broken = st.s != st.s;
    bool slow = broken;
    if (!broken) {
      const float m0 = sh.maxima[lane], m1 = sh.maxima[lane + 32];  // every warp for itself: no barrier
      const float order = a.k <= 16 ? sort32(fmaxf(m0, m1), lane) : best32(sort32(m0, lane), sort32(m1, lane), lane);
      uint64_t T = bound(__shfl_sync(0xffffffffu, order, a.k - 1), first, a.k);
#pragma unroll 1
      for (int look = 0;; ++look) {
        const Candidates<true> cand(sh.cand, &sh.count, kCandidates, T);
        if (__any_sync(0xffffffffu, best >= cand.value)) {
#pragma unroll 1
          for (int p = 0; p < parts.n; ++p) {
            const bool owner =
                owns(T, sh.shares[p * THREADS + tid], first + (uint32_t)(p * parts.vectors + tid) * Row<BF16>::N);
            const uint32_t owners = __ballot_sync(0xffffffffu, owner);
            if (owners == 0) continue;
            int at = 0;
            if (lane == 0) at = atomicAdd(&sh.n_owners, __popc(owners));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(owners & ((1u << lane) - 1));
            if (owner) sh.owners[at] = (uint16_t)(p * THREADS + tid);
          }
        }
        if (rank == 0 && warp == 0) {
          const int e = row.edge(lane);
          const float xe[1] = {e >= 0 ? row.at(e) : 0.f};
          cand.take(xe, e, e >= 0, lane);
        }
        __syncthreads();
        cand.take_shares<BF16, THREADS, THREADS>(row, v0, v1, parts.vectors, sh.owners, sh.n_owners,
                                                   THREADS * parts.n, tid);
        __syncthreads();
        const int n = sh.count;
        if (warp == 0) top = best_of(sh.cand, min(n, kCandidates), lane);
        slow = n > kCandidates;
        if (!slow || look == kLooks - 1) break;
        __syncthreads();  // every thread has read the count
        if (warp == 0 && lane == a.k - 1) sh.T = top;
        if (tid == 0) sh.n_owners = sh.count = 0;
        __syncthreads();
        T = sh.T;
      }
    }
    if (slow && warp == 0) top = slow_top<BF16>(row, v0, v1, rank == 0, a.k, lane);
  }
  if (blocks_per_row > 1) {
    if (TOP && warp == 0) sh.best[lane] = top;
    if (tid == 0) sh.st = st;
    cluster_sync();
    if (rank == 0 && warp == 0) {
      for (int c = 1; c < blocks_per_row; ++c) {
        const RowShared<TOP, THREADS>* o = remote(&sh, (uint32_t)c);
        st = join(st, Stat{o->st.m, o->st.s, o->st.t});
        if (TOP) top = best32(top, o->best[lane], lane);
      }
    }
    cluster_sync();  // the others' shared memory stays until it has been read
    if (rank != 0) return;
  }
  if (warp == 0) finish<BF16>(a, row, r, st, lane, top);
}

// ---------------------------------------------------------------------------
// Backward: a warp per kSlab vectors of a row.  logits and dlogits may be the same:
// every element is read by the thread that writes it.
// ---------------------------------------------------------------------------
constexpr int kSlab = 32 * kUnroll * 4;

template <bool BF16>
__global__ void __launch_bounds__(256)
    token_stats_bwd_kernel(const void* logits, long long ldl, int ncls, const int32_t* __restrict__ target,
                           const float* __restrict__ lse, const float* __restrict__ lse_low,
                           const float* __restrict__ entropy, const float* __restrict__ dlp, const float* __restrict__ dentropy, void* dlogits,
                           long long ldd, unsigned units, unsigned slabs) {
  constexpr int N = Row<BF16>::N, kElt = Row<BF16>::kElt;
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const unsigned r = unit / slabs, slab = unit - r * slabs;
  const Row<BF16> row(logits, ldl, r, ncls);
  const int tg = target[r];
  const float g = dlp && tg >= 0 && tg < ncls ? dlp[r] : 0.f;
  const float h = dentropy ? dentropy[r] : 0.f;
  const float L = lse[r], low = lse_low ? lse_low[r] : 0.f, H = dentropy ? entropy[r] : 0.f;
  const bool zero = L == -INFINITY || (g == 0.f && h == 0.f && L == L);  // nothing to read
  char* out = reinterpret_cast<char*>(dlogits) + (long long)r * ldd * kElt;
  // with z = x - L, log p = z - low:  -p (g + h (log p + H)) = p (nc + nh z)
  const float nh = -h, nc = -fmaf(h, H - low, g), l2 = -low * kLog2e;
  auto grad = [&](float x, int e) {
    if (zero) return 0.f;
    const float z = x - L, d = ex2(fmaf(z, kLog2e, l2)) * fmaf(nh, fmaxf(z, kFar), nc);
    return e == tg ? d + g : d;  // (a target outside the classes has g = 0)
  };
  auto put = [&](int e, float d) {
    if (BF16) reinterpret_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(d);
    else reinterpret_cast<float*>(out)[e] = d;
  };
  const int begin = row.begin(), end = row.end();
  if ((reinterpret_cast<uintptr_t>(out) & 15) != (uintptr_t)(row.mis * kElt)) {  // vectors do not line up
    const int e0 = slab * kSlab * N, e1 = slab + 1 == slabs ? ncls : min(e0 + kSlab * N, ncls);
    for (int e = e0 + lane; e < e1; e += 32) put(e, grad(row.at(e), e));
    return;
  }
  char* outv = out - row.mis * kElt;  // vector 0
  const int v1 = min(begin + (int)(slab + 1) * kSlab, end);
#pragma unroll 1
  for (int v0 = begin + (int)slab * kSlab + lane; v0 < v1; v0 += 32 * kUnroll) {
    uint4 raw[kUnroll];
    if (!zero) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (v0 + 32 * u < v1) raw[u] = row.load(v0 + 32 * u);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (v0 + 32 * u >= v1) break;
      const int e0 = (v0 + 32 * u) * N - row.mis;
      float d[N];
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = 0.f;
      if (!zero) {
        Row<BF16>::values(raw[u], d);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float z = d[i] - L;
          d[i] = ex2(fmaf(z, kLog2e, l2)) * fmaf(nh, fmaxf(z, kFar), nc);
        }
        if ((unsigned)(tg - e0) < (unsigned)N) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (e0 + i == tg) d[i] += g;
        }
      }
      uint4 w;
      if (BF16)
        w = make_uint4(pack_bf16(d[0], d[1]), pack_bf16(d[2 % N], d[3 % N]), pack_bf16(d[4 % N], d[5 % N]),
                       pack_bf16(d[6 % N], d[7 % N]));
      else
        w = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2 % N]),
                       __float_as_uint(d[3 % N]));
      *reinterpret_cast<uint4*>(outv + (long long)(v0 + 32 * u) * 16) = w;
    }
  }
  if (slab == 0) {
    const int e = row.edge(lane);
    if (e >= 0) put(e, grad(row.at(e), e));
  }
}

inline bool al(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

template <bool BF16, bool TOP>
cudaError_t launch_fwd(const Args& a, cudaStream_t st) {
  const int n = BF16 ? 8 : 4;
  // A warp per row up to 256 vectors, and up to 2048 where there are rows to fill the
  // device with warps (8192 x 8000 fp32 45 us, with 5 alternatives 53; a block per row 54
  // and 92: its parts wait for one another at each step of the selection; beyond, few
  // warps have rows that are too long: 2400 x 32003 bf16 43 us, 35); else a block per
  // row, or a cluster of up to 8 that share it (two chunks each at least) while there are
  // few blocks per SM: fewer than four (300 rows of 131071 fp32: 35 -> 29 us), or two with
  // alternatives, since every block then selects its own (509 rows of 131071 bf16, 20 of
  // them: 42 us, 49 with two blocks).
  const long long vectors = (a.ncls + n - 1) / n;
  if (vectors <= 8 * 32 || (vectors <= 64 * 32 && a.rows >= 148 * 16)) {
    const long long blocks = (a.rows + kWarpsPerBlock - 1) / kWarpsPerBlock;
    token_stats_warp_kernel<BF16, TOP><<<(unsigned)blocks, kWarpsPerBlock * 32, 0, st>>>(a);
    return cudaGetLastError();
  }
  int c = 1;
  while (c < 8 && a.rows * c < (TOP ? 2 : 4) * 148 && vectors >= 2 * (2 * c) * kThreads * kUnroll) c *= 2;
  if (a.rows * c > 0x7fffffffll) return cudaErrorInvalidValue;
  // Half the threads where rows are not very long and fill the device all the same: more
  // rows at a time on an SM, so that one selects while others stream (8192 x 32003 bf16
  // 102 -> 91 us, with 5 alternatives 150 -> 116; 1300 x 131071 with 20: 79, 90).
  const bool small = c == 1 && vectors <= 8192 && a.rows >= (vectors <= 2048 ? 2 : 4) * 148;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * c));
  cfg.blockDim = dim3(small ? kThreads / 2 : kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1 ? 1 : 0;
  return cudaLaunchKernelEx(
      &cfg, small ? token_stats_block_kernel<BF16, TOP, kThreads / 2> : token_stats_block_kernel<BF16, TOP, kThreads>,
      (const Args)a, c);
}

}  // namespace

extern "C" int cdk_token_logprobs_split(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                        const int32_t* target, float* lp, float* entropy, float* lse, float* lse_low,
                                        int32_t* top_ids, float* top_lp, int64_t k, void* stream) {
  if (rows == 0) return 0;
  if (!logits || !target || !lp || rows < 0 || rows > 0x7fffffff) return -1;
  if (dtype != 0 && dtype != 1) return -2;
  if (ncls <= 0 || ncls >= 0x7fffffe0 || ldl < ncls) return -3;
  if (!al(logits, dtype ? 2 : 4)) return -4;
  if (!top_ids != !top_lp) return -5;
  if (!top_ids) k = 0;
  if (k < 0 || k > kMaxTop || k > ncls) return -6;
  const Args a{logits, ldl, rows, (int)ncls, target, lp, entropy, lse, lse_low, top_ids, top_lp, (int)k};
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  if (k) return (int)(dtype ? launch_fwd<true, true>(a, st) : launch_fwd<false, true>(a, st));
  return (int)(dtype ? launch_fwd<true, false>(a, st) : launch_fwd<false, false>(a, st));
}

extern "C" int cdk_token_logprobs(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                  const int32_t* target, float* lp, float* entropy, float* lse, int32_t* top_ids,
                                  float* top_lp, int64_t k, void* stream) {
  return cdk_token_logprobs_split(logits, dtype, ldl, rows, ncls, target, lp, entropy, lse, nullptr, top_ids, top_lp, k,
                                  stream);
}

extern "C" int cdk_token_logprobs_bwd_split(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                            const int32_t* target, const float* lse, const float* lse_low,
                                            const float* entropy, const float* dlp, const float* dentropy,
                                            void* dlogits, int64_t ldd, void* stream) {
  if (rows == 0) return 0;
  if (!logits || !target || !lse || !dlogits || rows < 0 || rows > 0x7fffffff) return -1;
  if (dtype != 0 && dtype != 1) return -2;
  if (ncls <= 0 || ncls >= 0x7fffffe0 || ldl < ncls || ldd < ncls) return -3;
  if (!al(logits, dtype ? 2 : 4) || !al(dlogits, dtype ? 2 : 4)) return -4;
  if (dentropy && !entropy) return -5;
  if (logits == dlogits && ldl != ldd) return -6;
  const int n = dtype ? 8 : 4;
  const long long slabs = ((ncls + n - 1) / n + kSlab - 1) / kSlab;
  if (rows * slabs > 0xfffffff0ll) return -7;
  const unsigned units = (unsigned)(rows * slabs), blocks = (units + 7) / 8;
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype)
    token_stats_bwd_kernel<true><<<blocks, 256, 0, st>>>(logits, ldl, (int)ncls, target, lse, lse_low, entropy, dlp,
                                                         dentropy, dlogits, ldd, units, (unsigned)slabs);
  else
    token_stats_bwd_kernel<false><<<blocks, 256, 0, st>>>(logits, ldl, (int)ncls, target, lse, lse_low, entropy, dlp,
                                                          dentropy, dlogits, ldd, units, (unsigned)slabs);
  return (int)cudaGetLastError();
}

extern "C" int cdk_token_logprobs_bwd(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                      const int32_t* target, const float* lse, const float* entropy, const float* dlp,
                                      const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  return cdk_token_logprobs_bwd_split(logits, dtype, ldl, rows, ncls, target, lse, nullptr, entropy, dlp, dentropy,
                                      dlogits, ldd, stream);
}

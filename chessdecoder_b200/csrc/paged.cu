// Paged KV cache: rows written (rotated, optionally quantised), read back, and
// attended by one new token per sequence.
//
// Layout per layer, in HBM: k, v [num_pages][kv_heads][page_size][64] (bf16 or
// e4m3), so that the rows of one (page, head) are contiguous; for e4m3 one scale
// byte e per row (the row stands for code * 2^(e - 127)); a table of page
// numbers per sequence.  The reference keeps one dense cache with a common
// length (chessdecoder/cpp/decoder/batched_backbone.hpp:17-94); decode.cu is
// that form.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "cdk.h"
#include "cdk_common.cuh"

using namespace cdk;

namespace {

constexpr int kHD = 64;           // head dim, as everywhere in the library
constexpr int kMaxSeqs = 16384;   // sequences of one attention call
constexpr int kMaxGroup = 16;     // query heads per key / value head

__device__ __forceinline__ float2 bf2f(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Two e4m3 codes -> two fp32 values (exact).
__device__ __forceinline__ float2 e4m3x2_f(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Value of a scale byte: 2^(e - 127), as the upper 16 bits of an fp32.  Bytes 1..254 are
// exponent fields; byte 0 (never written here) is the subnormal 2^-127 and 255 a NaN, as
// in e8m0.
__device__ __forceinline__ uint32_t scale16_of(uint32_t e) { return e == 0 ? 0x0040u : e == 255 ? 0x7fc0u : e << 7; }
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(scale16_of(e) << 16); }

// The pages of one call, as the kernels see them.
struct Pages {
  char* k;
  char* v;
  uint8_t* ks;
  uint8_t* vs;
  const int32_t* table;
  long long ldt, width, num_pages;
  long long ld_page;   // bytes from page to page
  long long ld_scale;  // bytes from page to page of the scales
  int kv_heads;
  int log_page;        // log2(page_size)
};

// Byte-row index of row j of sequence b: page * ld_page + (head, offset) rows.
// Returns the page number or -1 (with the index error bit) where the table has
// no such row.
__device__ __forceinline__ int page_of(const Pages& p, long long b, long long j) {
  const long long c = j >> p.log_page;
  int page = -1;
  if (c >= 0 && c < p.width) page = p.table[b * p.ldt + c];
  if (page < 0 || page >= p.num_pages) {
    report_error(kErrIndex);
    return -1;
  }
  return page;
}

// ---------------------------------------------------------------------------
// Append.  A warp takes a token, or every `parts`-th group of four heads of it;
// eight lanes per row of 64, eight values each; key and value of a head together,
// since they go to the same place of two pools.  What belongs to the token --
// its sequence, place in the cache, position and rotation -- is found once.  The
// rotation is three separately rounded operations per value (no fused multiply-
// add), so that a quantised code does not depend on how a compiler contracts
// them.  Bound by HBM: one read of qkv, one write of each row.  Measured on one
// B200 (16 + 16 + 16 heads): 18,200 fp32 tokens rotated into bf16 pages 54 us, 97%
// of the copy rate, into e4m3 pages 49 us (95%); bf16 rows into e4m3 pages 23 us
// (74%, 57% of the issue slots: a warp loads its next heads after it has stored the
// present ones, and meanwhile has nothing in flight).  A lane per eight values with all
// indices its own took 70 us there; a warp per token whose row loads came after
// the place was looked up 35, before it 27; keys and values together 24, blocks of 128
// threads 23.
// ---------------------------------------------------------------------------
// Eight values of a row as loaded, and as numbers.
template <bool F32>
struct Raw8 {
  uint4 w[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const char* p) {
    w[0] = *reinterpret_cast<const uint4*>(p);
    if (F32) w[F32 ? 1 : 0] = reinterpret_cast<const uint4*>(p)[1];
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    const uint32_t a[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
    if (F32) {
      const uint4 c = w[F32 ? 1 : 0];
      const uint32_t d[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __uint_as_float(a[i]);
        x[4 + i] = __uint_as_float(d[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = bf2f(a[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

// cos and sin of a lane's four pairs.
struct Turn {
  float c[4], s[4];
  __device__ __forceinline__ void load(const float* p) {
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    c[0] = x.x, s[0] = x.y, c[1] = x.z, s[1] = x.w;
    c[2] = y.x, s[2] = y.y, c[3] = y.z, s[3] = y.w;
  }
  __device__ __forceinline__ void apply(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = x[2 * i], w = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(v, c[i]), __fmul_rn(w, s[i]));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(w, c[i]), __fmul_rn(v, s[i]));
    }
  }
};

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// e4m3 codes of this lane's eight of a row's 64 values; the row is on eight lanes in a
// row of a warp that is here as a whole.  byte: the scale's.
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], int* byte) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), as an exponent field: + 1 where the fraction is above 0x600000
  *byte = max((int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8, 1);
  const float inv = __uint_as_float((uint32_t)(254 - *byte) << 23);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_SATFINITE,
                                               __NV_E4M3)
            << 16);
  return make_uint2(w[0], w[1]);
}

template <bool F32, bool FP8>
__global__ void __launch_bounds__(128, 8)  // (a block's warps end at different times: 256 threads 2% longer)
    paged_append_kernel(const void* __restrict__ qkv, long long ldq, const int32_t* __restrict__ pos,
                        const float* __restrict__ rope, long long rope_len, unsigned S_new, int H, Pages pg,
                        const int32_t* __restrict__ start, const int32_t* __restrict__ num_new,
                        __nv_bfloat16* __restrict__ q_out, long long ldo, unsigned tokens, unsigned parts) {
  constexpr int kU = F32 ? 1 : 2;          // heads in flight per lane: 64 bytes of key and value rows
  constexpr int kE = FP8 ? 1 : 2;          // bytes per cached value
  constexpr int kIn = kHD * (F32 ? 4 : 2);  // bytes of a row of qkv
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const unsigned unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const unsigned t = unit / parts, part = unit - t * parts;
  if (t >= tokens) return;
  const unsigned b = t / S_new, s = t - b * S_new;
  if (num_new != nullptr && (int)s >= num_new[b]) return;  // padding
  const int kvn = pg.kv_heads, step = parts * 4, h0 = part * 4 + (lane >> 3);
  const char* src = reinterpret_cast<const char*>(qkv) + (long long)t * ldq * (F32 ? 4 : 2) + sub * (kIn / 8);
  const char* src_k = src + H * kIn;
  const int v_off = kvn * kIn;
  Raw8<F32> kr[kU], vr[kU];
  auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (h + u * step < kvn) {
        kr[u].load(src_k + (h + u * step) * kIn);
        vr[u].load(src_k + (h + u * step) * kIn + v_off);
      }
  };
  load(h0);  // before what follows, whose loads wait for one another
  Turn turn;
  if (rope != nullptr) {
    const long long p = pos[t];
    if (p < 0 || p >= rope_len) {
      if (lane == 0) report_error(kErrIndex);
      return;
    }
    turn.load(rope + (p * 32 + sub * 4) * 2);
  }
  const long long slot = (long long)start[b] + s;
  const int page = page_of(pg, b, slot);  // -1: reported, no row is written
  const unsigned off = (unsigned)(slot & ((1ll << pg.log_page) - 1));  // row in its page and head
  char* dst_k = pg.k + (long long)page * pg.ld_page + sub * (8 * kE);
  char* dst_v = pg.v + (long long)page * pg.ld_page + sub * (8 * kE);

  // (every lane of the warp runs the same number of rounds: the scale's exchange needs its row's eight lanes)
#pragma unroll 1
  for (int h = h0; h - (lane >> 3) < kvn; h += kU * step) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int hh = h + u * step;
      const bool live = hh < kvn && page >= 0;
      const unsigned row = ((unsigned)hh << pg.log_page) + off;  // below 2^24 where it is live
      float x[8];
      kr[u].values(x);
      if (rope != nullptr) turn.apply(x);
      int byte;
      if (FP8) {
        const uint2 w = quantise8(x, &byte);
        if (live) {
          *reinterpret_cast<uint2*>(dst_k + (size_t)row * (kHD * kE)) = w;
          if (sub == 0) pg.ks[(long long)page * pg.ld_scale + row] = (uint8_t)byte;
        }
      } else if (live) {
        *reinterpret_cast<uint4*>(dst_k + (size_t)row * (kHD * kE)) = pack8(x);
      }
      vr[u].values(x);
      if (FP8) {
        const uint2 w = quantise8(x, &byte);
        if (live) {
          *reinterpret_cast<uint2*>(dst_v + (size_t)row * (kHD * kE)) = w;
          if (sub == 0) pg.vs[(long long)page * pg.ld_scale + row] = (uint8_t)byte;
        }
      } else if (live) {
        *reinterpret_cast<uint4*>(dst_v + (size_t)row * (kHD * kE)) = pack8(x);
      }
    }
    load(h + kU * step);
  }

  if (q_out == nullptr) return;
  uint4* qo = reinterpret_cast<uint4*>(q_out + (long long)t * ldo) + sub;
  constexpr int kQ = 2 * kU;
#pragma unroll 1
  for (int h = h0; h < H; h += kQ * step) {
    Raw8<F32> qr[kQ];
#pragma unroll
    for (int u = 0; u < kQ; ++u)
      if (h + u * step < H) qr[u].load(src + (h + u * step) * kIn);
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
      if (h + u * step >= H) break;
      float x[8];
      qr[u].values(x);
      if (rope != nullptr) turn.apply(x);
      qo[(h + u * step) * 8] = pack8(x);
    }
  }
}

// ---------------------------------------------------------------------------
// Read back.  Grid (chunks of 128 rows, kv head, sequence); a lane takes 16 bytes of
// a key row and of its value row, of four (bf16) or two (e4m3) rows at a time.
// Bound by HBM: one read of the pages, one write of the rows.  Measured on one B200:
// 16 sequences of up to 8191 tokens, 16 heads: e4m3 67 us (95% of the copy rate; 81
// with 16 contiguous bytes of codes a lane, whose two stores each fill half a
// sector), bf16 86 us (98%).
// ---------------------------------------------------------------------------
constexpr int kGatherRows = 128;

template <bool FP8>
__global__ void __launch_bounds__(256)
    paged_gather_kernel(Pages pg, const int32_t* __restrict__ lens, __nv_bfloat16* __restrict__ k_out,
                        __nv_bfloat16* __restrict__ v_out, long long sb, long long sh, long long ss, long long S) {
  constexpr int kLanes = FP8 ? 4 : 8;        // lanes per row
  constexpr int kPass = 256 / kLanes;        // rows per block and pass
  constexpr int kU = kGatherRows / kPass;
  const long long b = blockIdx.z;
  const int h = blockIdx.y, sub = threadIdx.x % kLanes;
  long long len = lens[b];
  if (len > S) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && h == 0) report_error(kErrIndex);
    len = S;
  }
  const long long j0 = (long long)blockIdx.x * kGatherRows + threadIdx.x / kLanes;
  if ((long long)blockIdx.x * kGatherRows >= len) return;
  int page[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) page[u] = j0 + u * kPass < len ? page_of(pg, b, j0 + u * kPass) : -1;
  // e4m3: 8 bytes from each half of a row, so that the 16-byte stores of four lanes meet
  auto load16 = [&](const char* p) {
    if (!FP8) return *reinterpret_cast<const uint4*>(p);
    const uint2 x = *reinterpret_cast<const uint2*>(p), y = *reinterpret_cast<const uint2*>(p + 32);
    return make_uint4(x.x, x.y, y.x, y.y);
  };
  uint4 kw[kU], vw[kU];
  uint32_t ke[kU], ve[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const long long r = ((long long)h << pg.log_page) + ((j0 + u * kPass) & ((1ll << pg.log_page) - 1));
    if (page[u] >= 0) {
      const long long at = page[u] * pg.ld_page + r * (kHD * (FP8 ? 1 : 2)) + sub * (FP8 ? 8 : 16);
      kw[u] = load16(pg.k + at);
      vw[u] = load16(pg.v + at);
      if (FP8) {
        ke[u] = pg.ks[page[u] * pg.ld_scale + r];
        ve[u] = pg.vs[page[u] * pg.ld_scale + r];
      }
    }
  }
  auto store = [&](__nv_bfloat16* out, uint4 w, uint32_t e) {
    if (!FP8) {
      *reinterpret_cast<uint4*>(out + sub * 8) = w;
      return;
    }
    const float s = scale_of(e);
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = e4m3x2_f(in[i]), y = e4m3x2_f(in[i] >> 16);
      o[2 * i] = pack_bf16(x.x * s, x.y * s);
      o[2 * i + 1] = pack_bf16(y.x * s, y.y * s);
    }
    *reinterpret_cast<uint4*>(out + sub * 8) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(out + 32 + sub * 8) = make_uint4(o[4], o[5], o[6], o[7]);
  };
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (page[u] >= 0) {
      const long long o = b * sb + h * sh + (j0 + u * kPass) * ss;
      store(k_out + o, kw[u], ke[u]);
      store(v_out + o, vw[u], ve[u]);
    }
}

// ---------------------------------------------------------------------------
// One new token per sequence.
//
// o = sum_j w_j v_j / sum_j w_j with w_j = 2^(s_j - m), s = scale log2(e) q . k:
// one pass over the cached rows, which is what bounds it (HBM; the products are a
// few percent of the tensor pipe even for one query).  m is any common reference:
// it follows the maximum, but only when a score passes it by 8 (weights stay
// below 2^8), so that most tiles need no exchange between lanes and no rescaling.
//
// Work.  The keys of one (sequence, kv head) item are cut into tiles of 32.
// Where the tables hold few tiles per item (warps_per_item), a block takes an item, its
// warps a part of the tiles each, or a warp does.  Otherwise the tiles of all items,
// in the order (sequence, head, tile), are dealt to the grid's warps in equal
// contiguous runs, whatever the lengths; an item counts kSetup tiles more than it
// has, for what it costs a warp to begin one.  A warp that holds a whole item writes
// its output; a block inside one item adds up its warps in shared memory; what is
// shared beyond that is left as partial results (m, l, O) in the workspace and
// added up in a fixed order by paged_attn_join_kernel.  Warps never wait for other
// blocks.
//
// Tile.  Scores are taken transposed, S^T = K Q^T, with mma.sync m16n8k16: 16
// keys by 8 queries, so a group of up to 8 query heads costs what one costs.
// Operands come from HBM straight into registers: the sum over dims may run in
// any order, so a lane takes 16 contiguous bytes of a key row as its share of
// the k index (and of q alike).  O^T = V^T P^T takes 8 contiguous dims of a value
// row per lane; pairs of keys are interleaved by byte permutes, and P^T is
// turned from the accumulator's layout into the operand's by movmatrix.  No
// shared memory, no barrier in the loop: the loads of the next tile's keys are
// issued before this tile's softmax, those of its values after its products.
//
// bf16 pages: the weights are split into two bf16 (w = hi + lo, 2^-17 of w) so
// that they add no error beside the output's rounding.  e4m3 pages: codes are
// exact in fp16; q is scaled to fp16 by a power of two per head.  The products
// with the values take w_j 2^e_j, e_j the value row's scale, so that m has to
// follow s_j + e_j: weights then fit fp16 whatever the scales are, and are split
// like the others into two fp16 (2^-22 of w, and 2^-32 of the largest).  The sum
// of the w_j alone reaches 2^(15 - e_j); e_j below -88 counts as -88 for m (a row
// of zeros has the smallest scale), which only values below 448 * 2^-88 feel.
// Scores beyond 2^24 do not resolve s_j + e_j: such a weight may overflow.
//
// Measured on one B200 (16 heads, device time, join and all): bf16, 256 sequences of up to
// 4095 keys 319 us (2.15 GB: the copy rate; 334 by the deal), 64 of up to 2000 49 us
// (84%), 64 x 512 25 us (82%); e4m3, 256 x 2000 166 us (99%; 163 with weights in one
// fp16), 6 of up to 65536 with groups of 8 heads 27 us (61%: of the 11 us over the floor
// about 5 pass before the first rows arrive -- launch, lengths, table, rows -- and 2 in
// the join; the loop leaves half of the issue slots free, four warps to a scheduler
// waiting for their loads).  Pages of 16 rows: 256 sequences of up to 4000 keys 337 us
// bf16 (96%), 180 e4m3 (92%; 174).  Groups of 9 to 16 heads, 16 x 9001..20000 keys x 4 kv
// heads: 69 us bf16 (52%), 51 e4m3 (36%).
// ---------------------------------------------------------------------------
constexpr int kTK = 32;             // keys per tile
// 4 warps.  Groups of up to 8 heads: 128 registers, 4 blocks per SM (bf16 kernels spill 20 to
// 116 bytes, e4m3 none); on e4m3 pages with more than some 1700 sequences the deal's prefix
// beside the rings leaves shared memory for 3.  Larger groups: up to 168 registers, 3 blocks
// (bf16 spills up to 72 bytes).  The deal is cut for 4 all the same: where 3 fit, a quarter of
// its blocks start when others end.
constexpr int kAttnThreads = 128;
constexpr int kWarps = kAttnThreads / 32;
constexpr int kAttnBlocks = 148 * 4;
constexpr int kAttnWarps = kAttnBlocks * kWarps;
constexpr int kSlots = 2 * kAttnWarps;
constexpr float kNoScore = -3.0e38f;  // m before the first key
constexpr float kSlack = 8.f;
// e4m3 pages: how far below the largest s_j + e_j m is put, so that weights reach 2^15 at
// most, 2^7 at least, and their two fp16 parts leave 2^-32 of the largest.
constexpr float kLift = 7.f;
constexpr float kLowScale = -88.f;  // smallest e_j that m follows
// What beginning an item costs a warp, in tiles of the deal: its table, queries and
// first rows come one after the other.  (64 sequences of 0 .. 2000 keys: 72 us
// without, 59 with 1, 50 with 2, 51 with 3 -- a warp that is dealt fourteen items of
// one tile waits for fourteen such chains.)
constexpr int kSetup = 2;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint4 ld_once(const char* p) {  // read once: no place in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void e4m3x4_h(uint32_t w, uint32_t& lo, uint32_t& hi) {  // four codes -> fp16 (exact)
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct AttnArgs {
  const __nv_bfloat16* q;
  long long ldq;
  Pages pg;
  int B, group;
  const int32_t* lens;
  __nv_bfloat16* out;
  long long ldo;
  float scale_log2;
  int32_t* prefix;  // workspace: [B + 1] shares of the deal before each sequence, per kv head
  float2* stat;     // workspace: [kSlots][group] (m, l)
  float* part;      // workspace: [kSlots][group][64]
};

__device__ __forceinline__ int length_of(const AttnArgs& a, int b, bool report) {
  long long len = max(a.lens[b], 0);
  const long long cap = a.pg.width << a.pg.log_page;
  if (len > cap) {
    if (report) report_error(kErrIndex);
    len = cap;
  }
  return (int)len;
}

// Shares of the deal of one item: its tiles and kSetup, nothing for an empty one.
__device__ __forceinline__ int shares_of(int len) {
  return len > 0 ? (len + kTK - 1) / kTK + kSetup : 0;
}

// Writes 8 dims of the output of one (sequence, head).
__device__ __forceinline__ void store_out8(const AttnArgs& a, int b, int h, int d, const float (&o)[8], float f) {
  *reinterpret_cast<uint4*>(a.out + (long long)b * a.ldo + h * kHD + d) =
      make_uint4(pack_bf16(o[0] * f, o[1] * f), pack_bf16(o[2] * f, o[3] * f), pack_bf16(o[4] * f, o[5] * f),
                 pack_bf16(o[6] * f, o[7] * f));
}

// State of one warp and item.  Lane (g, t4) = (lane / 4, lane % 4) holds, for
// heads 8 n + 2 t4 + c of the group, dims 8 g ... 8 g + 7 of O.
template <int NT>
struct Acc {
  float o[NT][4][4];  // [dim pair i][c, 2 + c]: dims 8 g + 2 i and 8 g + 2 i + 1
  float m[NT][2], l[NT][2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      m[n][0] = m[n][1] = kNoScore;
      l[n][0] = l[n][1] = 0.f;
    }
  }
  __device__ __forceinline__ void sum_lanes() {  // l over the lanes of a column
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
  }
  __device__ __forceinline__ void dims(int n, int c, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = o[n][i][c];
      v[2 * i + 1] = o[n][i][2 + c];
    }
  }
};

// Pages of this lane's key of a tile (key tile * 32 + lane); -1 past the end.
__device__ __forceinline__ int page_of_key(const AttnArgs& a, const int32_t* trow, int tile, int tb, int len,
                                           int lane) {
  const int key = tile * kTK + lane;
  return tile < tb && key < len ? __ldg(trow + (key >> a.pg.log_page)) : -1;
}
// Which of a tile's keys count: inside the length, on a page that there is.
__device__ __forceinline__ uint32_t mask_of_tile(const AttnArgs& a, int tile, int page, int len, int lane) {
  const bool ok = (unsigned)page < (unsigned)a.pg.num_pages;
  const uint32_t mask = __ballot_sync(0xffffffffu, ok);
  if (mask != 0xffffffffu && !ok && tile * kTK + lane < len) report_error(kErrIndex);
  return mask;
}

// The reference follows the scores of a tile where one passes it, and stays `lift` below
// them; mx: this lane's largest per column.
template <int NT>
__device__ __forceinline__ void follow(Acc<NT>& acc, const float (&mx)[NT][2], float lift) {
  bool pass = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)  // (by the difference: m + kSlack rounds up where a step of m is 16)
    pass |= mx[n][0] - acc.m[n][0] > kSlack + lift || mx[n][1] - acc.m[n][1] > kSlack + lift;
  if (!__any_sync(0xffffffffu, pass)) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x = mx[n][c];
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
      x = fmaxf(x - lift, acc.m[n][c]);
      const float al = ex2(acc.m[n][c] - x);
      acc.m[n][c] = x;
      acc.l[n][c] *= al;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc.o[n][i][c] *= al;
        acc.o[n][i][2 + c] *= al;
      }
    }
}

// Tiles [ta, tb) of one item on bf16 pages: acc over its keys below len.  WIDE: pages
// hold tiles whole.
template <int NT, bool WIDE>
__device__ __forceinline__ void attend_bf16(const AttnArgs& a, int b, int kvh, int ta, int tb, int len, int lane,
                                            Acc<NT>& acc) {
  constexpr int kRow = 2 * kHD;  // bytes of a cached row
  const Pages& pg = a.pg;
  const int g = lane >> 2, t4 = lane & 3;
  const int32_t* trow = pg.table + (long long)b * pg.ldt;
  const int head_row = kvh << pg.log_page;
  const int pmask = (1 << pg.log_page) - 1;

  uint4 kr[4][2];  // rows g + 8 r, chunks t4 and 4 + t4
  uint4 vr[2][4];  // rows 16 jj + 2 t4 + {0, 1, 8, 9}, chunk g
  auto load_k = [&](int tile, int page, uint32_t mask) {
    const int t0 = tile * kTK;
    if (WIDE && mask == 0xffffffffu) {
      const long long p0 = __shfl_sync(0xffffffffu, page, 0);
      const char* base = pg.k + p0 * pg.ld_page + (long long)(head_row + (t0 & pmask) + g) * kRow + t4 * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c) kr[r][c] = ld_once(base + r * 8 * kRow + c * 64);
    } else if (!WIDE && pg.log_page == 4 && mask == 0xffffffffu) {  // 16 rows in a row in one page
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const long long p = __shfl_sync(0xffffffffu, page, 16 * x);
        const char* base =
            pg.k + p * pg.ld_page + (long long)(head_row + ((t0 + 16 * x) & pmask) + g) * kRow + t4 * 16;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) kr[2 * x + r][c] = ld_once(base + r * 8 * kRow + c * 64);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int y = g + 8 * r;
        const long long p = __shfl_sync(0xffffffffu, page, y);
        const char* base = pg.k + p * pg.ld_page + (long long)(head_row + ((t0 + y) & pmask)) * kRow + t4 * 16;
#pragma unroll
        for (int c = 0; c < 2; ++c) kr[r][c] = (mask >> y) & 1 ? ld_once(base + c * 64) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  auto load_v = [&](int tile, int page, uint32_t mask) {
    const int t0 = tile * kTK;
    if (WIDE && mask == 0xffffffffu) {
      const long long p0 = __shfl_sync(0xffffffffu, page, 0);
      const char* base = pg.v + p0 * pg.ld_page + (long long)(head_row + (t0 & pmask) + 2 * t4) * kRow + g * 16;
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[jj][i] = ld_once(base + (16 * jj + (i & 1) + (i >> 1) * 8) * kRow);
    } else if (!WIDE && pg.log_page == 4 && mask == 0xffffffffu) {
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const long long p = __shfl_sync(0xffffffffu, page, 16 * jj);
        const char* base =
            pg.v + p * pg.ld_page + (long long)(head_row + ((t0 + 16 * jj) & pmask) + 2 * t4) * kRow + g * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[jj][i] = ld_once(base + ((i & 1) + (i >> 1) * 8) * kRow);
      }
    } else {
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = 16 * jj + 2 * t4 + (i & 1) + (i >> 1) * 8;
          const long long p = __shfl_sync(0xffffffffu, page, y);
          const char* base = pg.v + p * pg.ld_page + (long long)(head_row + ((t0 + y) & pmask)) * kRow + g * 16;
          vr[jj][i] = (mask >> y) & 1 ? ld_once(base) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
  };

  int page = page_of_key(a, trow, ta, tb, len, lane);
  uint32_t mask = mask_of_tile(a, ta, page, len, lane);
  load_k(ta, page, mask);
  load_v(ta, page, mask);
  page = page_of_key(a, trow, ta + 1, tb, len, lane);

  // queries of the group as the B operand: head 8 n + g, its chunks t4 and 4 + t4
  uint32_t qf[NT][8];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int hq = n * 8 + g;
    const __nv_bfloat16* qrow = a.q + (long long)b * a.ldq + (kvh * a.group + hq) * kHD;
    uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
    if (hq < a.group) {
      x = *reinterpret_cast<const uint4*>(qrow + 8 * t4);
      y = *reinterpret_cast<const uint4*>(qrow + 32 + 8 * t4);
    }
    qf[n][0] = x.x, qf[n][1] = x.y, qf[n][2] = x.z, qf[n][3] = x.w;
    qf[n][4] = y.x, qf[n][5] = y.y, qf[n][6] = y.z, qf[n][7] = y.w;
  }

#pragma unroll 1
  for (int tile = ta; tile < tb; ++tile) {
    // the table two tiles ahead: there when the next tile's scores are done
    const int page2 = page_of_key(a, trow, tile + 2, tb, len, lane);
    // S^T: keys g + 8 r by heads 2 t4 + c -> s[n][r][c]
    float s[NT][4][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float d[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 u = kr[2 * i][c], w4 = kr[2 * i + 1][c];
        const uint32_t a0[4] = {u.x, w4.x, u.y, w4.y}, a1[4] = {u.z, w4.z, u.w, w4.w};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16_16816(d[n], a0, qf[n][4 * c], qf[n][4 * c + 1]);
          mma_bf16_16816(d[n], a1, qf[n][4 * c + 2], qf[n][4 * c + 3]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s[n][2 * i][c] = d[n][c] * a.scale_log2;
          s[n][2 * i + 1][c] = d[n][2 + c] * a.scale_log2;
        }
    }
    if (mask != 0xffffffffu) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!((mask >> (g + 8 * r)) & 1)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][r][0] = s[n][r][1] = -INFINITY;
        }
    }
    if (tile + 1 < tb) {
      mask = mask_of_tile(a, tile + 1, page, len, lane);
      load_k(tile + 1, page, mask);
    }
    float mx[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) mx[n][c] = fmaxf(fmaxf(s[n][0][c], s[n][1][c]), fmaxf(s[n][2][c], s[n][3][c]));
    follow<NT>(acc, mx, 0.f);

    // weights of keys (16 jj + g, + 8) for heads 2 t4, 2 t4 + 1, as the B operand: high and low parts
    uint32_t ph[NT][2][2], pl[NT][2][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p0 = ex2(s[n][r][0] - acc.m[n][0]), p1 = ex2(s[n][r][1] - acc.m[n][1]);
        acc.l[n][0] += p0;
        acc.l[n][1] += p1;
        const uint32_t hi = pack_bf16(p0, p1);
        const float2 back = bf2f(hi);
        ph[n][r >> 1][r & 1] = transpose8x8(hi);
        pl[n][r >> 1][r & 1] = transpose8x8(pack_bf16(p0 - back.x, p1 - back.y));
      }

    // O^T += V^T P^T: the A operand's rows g and g + 8 of product i are dims 8 g + 2 i and 8 g + 2 i + 1
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      const uint32_t w4[4][4] = {{vr[jj][0].x, vr[jj][0].y, vr[jj][0].z, vr[jj][0].w},
                                 {vr[jj][1].x, vr[jj][1].y, vr[jj][1].z, vr[jj][1].w},
                                 {vr[jj][2].x, vr[jj][2].y, vr[jj][2].z, vr[jj][2].w},
                                 {vr[jj][3].x, vr[jj][3].y, vr[jj][3].z, vr[jj][3].w}};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t af[4] = {__byte_perm(w4[0][i], w4[1][i], 0x5410), __byte_perm(w4[0][i], w4[1][i], 0x7632),
                                __byte_perm(w4[2][i], w4[3][i], 0x5410), __byte_perm(w4[2][i], w4[3][i], 0x7632)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16_16816(acc.o[n][i], af, ph[n][jj][0], ph[n][jj][1]);
          mma_bf16_16816(acc.o[n][i], af, pl[n][jj][0], pl[n][jj][1]);
        }
      }
    }
    if (tile + 1 < tb) {
      load_v(tile + 1, page, mask);
      page = page2;
    }
  }
}

// The same on e4m3 pages.  A tile is half the bytes, so its loads have to be twice
// as far ahead: they go through a ring of kStages tiles per warp in shared memory
// (cp.async, rows that do not count filled with zeros), two tiles ahead.  (Through
// registers, one tile ahead: 266 us against 176 for 256 x 2000 keys x 16 heads.)
//
// Stage: 32 key rows, then 32 value rows, of 64 bytes; two rows to a 128-byte
// line, whose 16-byte chunks are swapped around by twice the line's number, so
// that both the fragments' reads (8 key rows by one chunk; 4 value rows, every
// second one, by half a row) and the copies touch every bank once.
constexpr int kStages = 3;
constexpr int kStageBytes = 2 * kTK * kHD;

// Offset of chunk c of a row in its stage.  Rows 8 apart are 512 bytes apart.
__device__ __forceinline__ int chunk_at(int row, int c) {
  return (row >> 1) * 128 + (((((row & 1) << 2) | c) ^ (((row >> 1) & 3) << 1)) << 4);
}

template <int NT, bool WIDE>
__device__ __forceinline__ void attend_e4m3(const AttnArgs& a, int b, int kvh, int ta, int tb, int len, int lane,
                                            char* ring, Acc<NT>& acc) {
  const Pages& pg = a.pg;
  const int g = lane >> 2, t4 = lane & 3;
  const int32_t* trow = pg.table + (long long)b * pg.ldt;
  const int head_row = kvh << pg.log_page;
  const int pmask = (1 << pg.log_page) - 1;
  const int k_at = chunk_at(g, t4);  // this lane's chunk of key row g (rows g + 8 i: 512 i further)
  // its half chunk of value row 2 t4; row 2 t4 + 1 is in the same line, four chunks on or back
  const int v_at = kTK * kHD + chunk_at(2 * t4, g >> 1) + (g & 1) * 8;
  const uint32_t dst0 = smem_u32(ring) + k_at;

  // Starts the copies of a tile and loads its keys' scale bytes.
  auto fetch = [&](int tile, int page, int stage, uint32_t& mask, uint32_t& sk, uint32_t& sv) {
    mask = sk = sv = 0;
    if (tile < tb) {
      const int t0 = tile * kTK;
      mask = mask_of_tile(a, tile, page, len, lane);
      if ((mask >> lane) & 1) {
        const long long r = (long long)page * pg.ld_scale + head_row + ((t0 + lane) & pmask);
        sk = __ldg(pg.ks + r);
        sv = __ldg(pg.vs + r);
      }
      const uint32_t dst = dst0 + stage * kStageBytes;
      if (WIDE && mask == 0xffffffffu) {
        const long long p0 = __shfl_sync(0xffffffffu, page, 0);
        const long long at = p0 * pg.ld_page + (long long)(head_row + (t0 & pmask) + g) * kHD + t4 * 16;
        const char* ks = pg.k + at;
        const char* vs = pg.v + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          cp_async_16(dst + i * 512, ks + i * 8 * kHD);
          cp_async_16(dst + kTK * kHD + i * 512, vs + i * 8 * kHD);
        }
      } else if (!WIDE && pg.log_page == 4 && mask == 0xffffffffu) {  // 16 rows in a row in one page
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const long long p = __shfl_sync(0xffffffffu, page, 16 * x);
          const long long at = p * pg.ld_page + (long long)(head_row + ((t0 + 16 * x) & pmask) + g) * kHD + t4 * 16;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            cp_async_16(dst + (2 * x + i) * 512, pg.k + at + i * 8 * kHD);
            cp_async_16(dst + kTK * kHD + (2 * x + i) * 512, pg.v + at + i * 8 * kHD);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = g + 8 * i;
          const long long p = __shfl_sync(0xffffffffu, page, y);
          const bool ok = (mask >> y) & 1;
          const long long at = ok ? p * pg.ld_page + (long long)(head_row + ((t0 + y) & pmask)) * kHD + t4 * 16 : 0;
          cp_async_16_zfill(dst + i * 512, pg.k + at, ok);
          cp_async_16_zfill(dst + kTK * kHD + i * 512, pg.v + at, ok);
        }
      }
    }
    cp_async_commit();
  };

  __syncwarp();  // every lane is done with the ring
  uint32_t mask, mask1, mask2, sk, sv, sk1, sv1, sk2, sv2;
  {
    const int p0 = page_of_key(a, trow, ta, tb, len, lane), p1 = page_of_key(a, trow, ta + 1, tb, len, lane);
    fetch(ta, p0, 0, mask, sk, sv);
    fetch(ta + 1, p1, 1, mask1, sk1, sv1);
  }
  int page = page_of_key(a, trow, ta + 2, tb, len, lane);
  int stage = 0;
  uint32_t sc = scale16_of(sk) | (scale16_of(sv) << 16);  // scales of this tile, key and value

  // queries as the B operand: head 8 n + g, 16 dims from 16 t4, scaled to fp16
  uint32_t qf[NT][8];
  float qs[NT][2];  // factor of the scores of heads 8 n + 2 t4, + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int hq = n * 8 + g;
    const __nv_bfloat16* qrow = a.q + (long long)b * a.ldq + (kvh * a.group + hq) * kHD + 16 * t4;
    uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
    if (hq < a.group) {
      x = *reinterpret_cast<const uint4*>(qrow);
      y = *reinterpret_cast<const uint4*>(qrow + 8);
    }
    const uint32_t raw[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    uint32_t top = 0;  // the row's largest magnitude, as bf16 bits
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // largest in [2^14, 2^15): fp16 then holds all 8 bits of whatever is above 2^-31 of it
    const int e = max((int)(top >> 7), 15);  // exponent field, <= 255; the factor 2^(141 - e) is a normal number
    const float up = __uint_as_float((uint32_t)(127 + 141 - e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = bf2f(raw[i]);
      qf[n][i] = pack_f16(v.x * up, v.y * up);
    }
    // lanes (g, *) hold head g's factor; this lane's score columns are heads 2 t4, 2 t4 + 1
    qs[n][0] = a.scale_log2 / __shfl_sync(0xffffffffu, up, 8 * t4);
    qs[n][1] = a.scale_log2 / __shfl_sync(0xffffffffu, up, 8 * t4 + 4);
  }

#pragma unroll 1
  for (int tile = ta; tile < tb; ++tile) {
    cp_async_wait<1>();
    __syncwarp();  // the tile has landed, for every lane; the stage before it has been read by every lane
    const int page3 = page_of_key(a, trow, tile + 3, tb, len, lane);
    fetch(tile + 2, page, stage == 0 ? 2 : stage - 1, mask2, sk2, sv2);
    page = page3;
    const char* st = ring + stage * kStageBytes;

    // S^T: keys g + 8 r by heads 2 t4 + c -> s[n][r][c]
    float s[NT][4][2], vs[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float d[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
      const uint4 u = *reinterpret_cast<const uint4*>(st + k_at + i * 1024);
      const uint4 w = *reinterpret_cast<const uint4*>(st + k_at + i * 1024 + 512);
      const uint32_t lo[4] = {u.x, u.y, u.z, u.w}, hi[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t af[4];
        e4m3x4_h(lo[j], af[0], af[2]);
        e4m3x4_h(hi[j], af[1], af[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(d[n], af, qf[n][2 * j], qf[n][2 * j + 1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 2 * i + h;
        const uint32_t x = __shfl_sync(0xffffffffu, sc, g + 8 * r);
        const float ks = __uint_as_float(x << 16);
        vs[r] = __uint_as_float(x & 0xffff0000u);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) s[n][r][c] = d[n][2 * h + c] * (qs[n][c] * ks);
      }
    }
    if (mask != 0xffffffffu) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!((mask >> (g + 8 * r)) & 1)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][r][0] = s[n][r][1] = -INFINITY;
        }
    }
    float mx[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float e = fmaxf((float)((int)(__float_as_uint(vs[r]) >> 23) - 127), kLowScale);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mx[n][0] = fmaxf(mx[n][0], s[n][r][0] + e);
        mx[n][1] = fmaxf(mx[n][1], s[n][r][1] + e);
      }
    }
    follow<NT>(acc, mx, kLift);

    // weights with the value scales, as the B operand: high and low parts
    uint32_t ph[NT][2][2], pl[NT][2][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p0 = ex2(s[n][r][0] - acc.m[n][0]), p1 = ex2(s[n][r][1] - acc.m[n][1]);
        acc.l[n][0] += p0;
        acc.l[n][1] += p1;
        const float w0 = p0 * vs[r], w1 = p1 * vs[r];
        const uint32_t hi = pack_f16(w0, w1);
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        ph[n][r >> 1][r & 1] = transpose8x8(hi);
        pl[n][r >> 1][r & 1] = transpose8x8(pack_f16(w0 - back.x, w1 - back.y));
      }

    // O^T += V^T P^T; bytes of two keys interleaved first: one permute gives two dims of both
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      uint2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = *reinterpret_cast<const uint2*>(st + (v_at ^ ((i & 1) << 6)) + jj * 1024 + (i >> 1) * 512);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
        const uint32_t lo = i < 2 ? __byte_perm(v[0].x, v[1].x, sel) : __byte_perm(v[0].y, v[1].y, sel);
        const uint32_t hi = i < 2 ? __byte_perm(v[2].x, v[3].x, sel) : __byte_perm(v[2].y, v[3].y, sel);
        uint32_t af[4];
        e4m3x4_h(lo, af[0], af[1]);
        e4m3x4_h(hi, af[2], af[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16_16816(acc.o[n][i], af, ph[n][jj][0], ph[n][jj][1]);
          mma_f16_16816(acc.o[n][i], af, pl[n][jj][0], pl[n][jj][1]);
        }
      }
    }
    mask = mask1, mask1 = mask2;
    sc = scale16_of(sk1) | (scale16_of(sv1) << 16);  // loaded a tile ago
    sk1 = sk2, sv1 = sv2;
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
}

template <bool FP8, int NT, bool WIDE>
__device__ __forceinline__ void attend(const AttnArgs& a, int b, int kvh, int ta, int tb, int len, int lane, char* ring,
                                       Acc<NT>& acc) {
  if constexpr (FP8) attend_e4m3<NT, WIDE>(a, b, kvh, ta, tb, len, lane, ring, acc);
  else attend_bf16<NT, WIDE>(a, b, kvh, ta, tb, len, lane, acc);
}

// Shared memory of a block.  e4m3: a warp's results take the place of its ring,
// which it is done with.  bf16: sized by the group; what a block does not take
// stays L1, where the loads in flight land.
struct AttnShared {
  char* warps;   // a region per warp: o [group][64], stat [group] (m, l), or the ring, on a 128-byte line
  int region;    // its bytes
  int group;
  int* prefix;   // [B + 1]
  __device__ __forceinline__ AttnShared(char* p, int group_, bool fp8) : region(region_bytes(group_, fp8)), group(group_) {
    warps = p + ((128 - (smem_u32(p) & 127)) & 127);
    prefix = reinterpret_cast<int*>(warps + kWarps * region);
  }
  __device__ __forceinline__ char* of(int warp) const { return warps + warp * region; }
  __device__ __forceinline__ float* o(int warp, int hq) const { return reinterpret_cast<float*>(of(warp)) + hq * kHD; }
  __device__ __forceinline__ float2& stat(int warp, int hq) const {
    return reinterpret_cast<float2*>(of(warp) + group * kHD * 4)[hq];
  }
  static __host__ __device__ constexpr int region_bytes(int group, bool fp8) {
    const int results = (group * (kHD * 4 + 8) + 15) / 16 * 16;
    return fp8 && results < kStages * kStageBytes ? kStages * kStageBytes : results;
  }
  static __host__ __device__ constexpr int bytes(int group, bool fp8, int n_warps = kWarps) {
    return n_warps * region_bytes(group, fp8) + 112;
  }
};
static_assert(kMaxGroup * (kHD * 4 + 8) <= kStages * kStageBytes, "a warp's results fit its ring");

// The output of an item from the state of the warp that had all of it.
template <int NT>
__device__ __forceinline__ void store_item(const AttnArgs& a, const Acc<NT>& acc, int b, int kvh, int lane) {
  const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int hq = n * 8 + 2 * t4 + c;
      if (hq >= a.group) continue;
      float v[8];
      acc.dims(n, c, v);
      store_out8(a, b, kvh * a.group + hq, 8 * g, v, acc.l[n][c] == 0.f ? 0.f : 1.f / acc.l[n][c]);
    }
}

// A block whose warps all worked on one item (a warp without tiles has an empty
// state): their sum goes to the output, or to workspace slot `slot` when other
// blocks share the item.
template <int NT, int W>
__device__ __forceinline__ void merge_block(const AttnArgs& a, const AttnShared& sh, const Acc<NT>& acc, int b, int kvh,
                                            bool whole, int slot) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  __syncwarp();  // every lane is done with the ring
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int hq = n * 8 + 2 * t4 + c;
      if (hq >= a.group) continue;
      float v[8];
      acc.dims(n, c, v);
      float4* dst = reinterpret_cast<float4*>(sh.o(warp, hq) + 8 * g);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      if (g == 0) sh.stat(warp, hq) = make_float2(acc.m[n][c], acc.l[n][c]);
    }
  __syncthreads();
  for (int i = tid; i < a.group * (kHD / 8); i += W * 32) {
    const int hq = i / (kHD / 8), d = (i % (kHD / 8)) * 8;
    float m = kNoScore, l = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int w = 0; w < W; ++w) m = fmaxf(m, sh.stat(w, hq).x);
#pragma unroll 4
    for (int w = 0; w < W; ++w) {
      const float f = ex2(sh.stat(w, hq).x - m);
      l += sh.stat(w, hq).y * f;
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] += sh.o(w, hq)[d + x] * f;
    }
    if (whole) {
      store_out8(a, b, kvh * a.group + hq, d, v, l == 0.f ? 0.f : 1.f / l);
    } else {
      const int at = slot * a.group + hq;
      float4* dst = reinterpret_cast<float4*>(a.part + at * kHD + d);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) a.stat[at] = make_float2(m, l);
    }
  }
}

// SPLIT warps per (sequence, kv head): a block of them, or a warp of a block of four.
template <bool FP8, int NT, bool WIDE, int SPLIT>
__global__ void __launch_bounds__(SPLIT > 4 ? SPLIT * 32 : kAttnThreads, SPLIT > 4 ? 3 - NT : 5 - NT)
    paged_attn_item_kernel(const AttnArgs a) {
  extern __shared__ __align__(16) char smem[];
  const AttnShared sh(smem, a.group, FP8);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  char* ring = sh.of(warp);
  const int item = SPLIT == 1 ? (int)blockIdx.x * kWarps + warp : (int)blockIdx.x;
  if (SPLIT == 1 && item >= a.B * a.pg.kv_heads) return;
  const int b = item / a.pg.kv_heads, kvh = item - b * a.pg.kv_heads;
  const int len = length_of(a, b, kvh == 0 && (SPLIT == 1 ? lane : (int)threadIdx.x) == 0);
  const int tiles = (len + kTK - 1) / kTK, per = (tiles + SPLIT - 1) / SPLIT;
  const int ta = SPLIT == 1 ? 0 : min(warp * per, tiles), tb = min(ta + per, tiles);
  Acc<NT> acc;
  acc.clear();
  if (ta < tb) attend<FP8, NT, WIDE>(a, b, kvh, ta, tb, len, lane, ring, acc);
  acc.sum_lanes();
  if (SPLIT == 1) store_item<NT>(a, acc, b, kvh, lane);  // len 0: l = 0, zeros
  else merge_block<NT, SPLIT>(a, sh, acc, b, kvh, true, 0);
}

// Shares [f, f + chunk) of the deal for warp w = f / chunk; see the join for the slots.
template <bool FP8, int NT, bool WIDE>
__global__ void __launch_bounds__(kAttnThreads, NT == 1 ? 4 : 3) paged_attn_kernel(const AttnArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ int warp_tiles[kWarps];
  const AttnShared sh(smem, a.group, FP8);
  char* ring = sh.of(threadIdx.x >> 5);
  int* prefix = sh.prefix;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvn = a.pg.kv_heads;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may be set up; it waits for this grid
  {  // shares before each sequence: thread i takes a contiguous run of sequences
    const int per = (a.B + kAttnThreads - 1) / kAttnThreads;
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += shares_of(length_of(a, b, blockIdx.x == 0));
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) warp_tiles[warp] = scan;
    __syncthreads();
    int at = scan - sum;
    for (int w = 0; w < warp; ++w) at += warp_tiles[w];
    for (int b = b0; b < b1; ++b) {
      prefix[b] = at;
      if (blockIdx.x == 0) a.prefix[b] = at;
      at += b1 - b0 == 1 ? sum : shares_of(length_of(a, b, false));
    }
    if (tid == kAttnThreads - 1) {
      prefix[a.B] = at;
      if (blockIdx.x == 0) a.prefix[a.B] = at;
    }
    __syncthreads();
  }
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)  // sequences without keys
    if (prefix[b] == prefix[b + 1])
      for (int i = tid; i < kvn * a.group * (kHD / 8); i += kAttnThreads)
        *reinterpret_cast<uint4*>(a.out + (long long)b * a.ldo + i * 8) = make_uint4(0u, 0u, 0u, 0u);

  // shares, and w * chunk with them, fit 32 bits: total < 2^31 (checked on the host)
  const unsigned total = (unsigned)prefix[a.B] * kvn, n_warps = gridDim.x * kWarps;
  const unsigned chunk = (total + n_warps - 1) / n_warps;
  const unsigned w0 = blockIdx.x * kWarps, w = w0 + warp;
  const unsigned block_f = w0 * chunk, block_end = min(block_f + kWarps * chunk, total);
  if (block_f >= block_end) return;
  unsigned f = w * chunk;
  const unsigned f_end = min(f + chunk, total);

  struct Item {
    int b, kvh, n;   // n: its shares
    unsigned first;  // the first of them
  };
  auto item_of = [&](unsigned x) {  // of share x < total
    int lo = 0, hi = a.B;           // last b with prefix[b] * kv_heads <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((unsigned)prefix[mid] * kvn <= x) lo = mid;
      else hi = mid;
    }
    Item it;
    it.b = lo;
    it.n = prefix[lo + 1] - prefix[lo];
    const unsigned first = (unsigned)prefix[lo] * kvn;
    it.kvh = (int)((x - first) / (unsigned)it.n);
    it.first = first + it.kvh * it.n;
    return it;
  };
  const Item bi = item_of(block_f);
  if (block_end <= bi.first + bi.n) {  // the block is inside one item
    const int ta = max((int)(f - bi.first) - kSetup, 0), tb = (int)(f_end - bi.first) - kSetup;
    Acc<NT> acc;
    acc.clear();
    if (f < f_end && ta < tb) attend<FP8, NT, WIDE>(a, bi.b, bi.kvh, ta, tb, length_of(a, bi.b, false), lane, ring, acc);
    acc.sum_lanes();
    merge_block<NT, kWarps>(a, sh, acc, bi.b, bi.kvh, block_f == bi.first && block_end == bi.first + bi.n, 2 * (int)w0);
    return;
  }
  while (f < f_end) {
    const Item it = item_of(f);
    const unsigned last = min(it.first + it.n, f_end);
    const int ta = max((int)(f - it.first) - kSetup, 0), tb = (int)(last - it.first) - kSetup;
    f = last;
    if (ta >= tb) continue;  // nothing but the item's setup
    Acc<NT> acc;
    acc.clear();
    attend<FP8, NT, WIDE>(a, it.b, it.kvh, ta, tb, length_of(a, it.b, false), lane, ring, acc);
    acc.sum_lanes();
    if (ta == 0 && tb == it.n - kSetup) {
      store_item<NT>(a, acc, it.b, it.kvh, lane);
      continue;
    }
    const int slot = 2 * (int)w + (ta == 0 ? 1 : 0);
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int hq = n * 8 + 2 * t4 + c;
        if (hq >= a.group) continue;
        float v[8];
        acc.dims(n, c, v);
        const int at = slot * a.group + hq;
        float4* dst = reinterpret_cast<float4*>(a.part + at * kHD + 8 * g);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        if (g == 0) a.stat[at] = make_float2(acc.m[n][c], acc.l[n][c]);
      }
  }
}

// Adds up the partial results of the items that several warps shared, in the
// order of the deal.  A block inside an item left one result, in its first warp's
// slot 0; other warps left the item they end in slot 0, the one they begin in
// slot 1.  One block per (sequence, query head); eight lanes take a result, eight
// dims each, so a warp has eight results in flight (one sequence of 131072 keys with
// one kv head, 512 results for each of its 8 heads: 17 us, 32 with a result per warp).
constexpr int kJoinWarps = 16;  // at most

__global__ void __launch_bounds__(kJoinWarps * 32) paged_attn_join_kernel(const AttnArgs a, unsigned n_warps) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int heads = a.pg.kv_heads * a.group;
  const int b = blockIdx.x / heads, h = blockIdx.x - b * heads;
  const int kvh = h / a.group, hq = h - kvh * a.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int before = a.prefix[b], shares = a.prefix[b + 1] - before;
  if (shares == 0) return;
  const unsigned kvn = a.pg.kv_heads, total = (unsigned)a.prefix[a.B] * kvn;
  const unsigned chunk = (total + n_warps - 1) / n_warps, span = chunk * kWarps;
  const unsigned first = before * kvn + kvh * shares, end = first + shares;
  // warps with tiles of the item
  const int w0 = (int)((first + kSetup) / chunk), w1 = (int)((end - 1) / chunk);
  // blocks inside the item: [c0, c1); each has tiles of it, having more shares than kSetup
  static_assert(kWarps > kSetup, "a block inside an item is more than its setup");
  const int c0 = (int)((first + span - 1) / span), c1 = (int)((end == total ? end + span - 1 : end) / span);
  const int inside = max(c1 - c0, 0), cw = w0 / kWarps;
  if (w0 == w1 && !(cw >= c0 && cw < c1)) return;                                // written by that warp
  if (inside == 1 && c0 * span == first && min((c0 + 1) * span, total) == end) return;  // written by that block
  const int head = inside ? max(c0 * kWarps - w0, 0) : w1 - w0 + 1;  // warps before them (all, without them)
  const int tail = inside ? max(w1 + 1 - c1 * kWarps, 0) : 0;        // and after them
  const int n = head + inside + tail;
  const int sub = lane >> 3, d = (lane & 7) * 8, warps = blockDim.x >> 5;
  float m = kNoScore, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto add = [&](float pm, float pl, const float (&po)[8]) {
    const float nm = fmaxf(m, pm), f0 = ex2(m - nm), f1 = ex2(pm - nm);
    l = l * f0 + pl * f1;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * f0 + po[i] * f1;
    m = nm;
  };
  auto at_of = [&](int i) {
    const int w = i < head ? w0 + i : i < head + inside ? (c0 + i - head) * kWarps : c1 * kWarps + (i - head - inside);
    const bool begins = (i < head && i == 0);
    return (2 * w + (begins ? 1 : 0)) * a.group + hq;
  };
  for (int i = warp * 4 + sub; i - sub < n; i += 8 * warps) {
    float2 st[2];
    float v[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = i + u * 4 * warps;
      st[u] = make_float2(kNoScore, 0.f);
#pragma unroll
      for (int c = 0; c < 8; ++c) v[u][c] = 0.f;
      if (k < n) {
        const int at = at_of(k);
        st[u] = a.stat[at];
        const float4* p = reinterpret_cast<const float4*>(a.part + at * kHD + d);
        const float4 x = p[0], y = p[1];
        v[u][0] = x.x, v[u][1] = x.y, v[u][2] = x.z, v[u][3] = x.w;
        v[u][4] = y.x, v[u][5] = y.y, v[u][6] = y.z, v[u][7] = y.w;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) add(st[u].x, st[u].y, v[u]);
  }
#pragma unroll
  for (int x = 8; x < 32; x <<= 1) {  // the warp's four
    float po[8];
    const float pm = __shfl_xor_sync(0xffffffffu, m, x), pl = __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) po[i] = __shfl_xor_sync(0xffffffffu, o[i], x);
    add(pm, pl, po);
  }
  __shared__ float2 st_s[kJoinWarps];
  __shared__ float4 o_s[kJoinWarps][kHD / 4];
  if (sub == 0) {
    if (lane == 0) st_s[warp] = make_float2(m, l);
    o_s[warp][d / 4] = make_float4(o[0], o[1], o[2], o[3]);
    o_s[warp][d / 4 + 1] = make_float4(o[4], o[5], o[6], o[7]);
  }
  __syncthreads();
  if (warp || sub) return;
  for (int i = 1; i < warps; ++i) {
    const float4 x = o_s[i][d / 4], y = o_s[i][d / 4 + 1];
    const float po[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    add(st_s[i].x, st_s[i].y, po);
  }
  store_out8(a, b, h, d, o, l == 0.f ? 0.f : 1.f / l);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int take_pages(const CdkPagedCache* c, Pages* p) {
  if (!c || !c->k || !c->v || (!c->table && c->width != 0)) return -1;
  if (c->dtype != 0 && c->dtype != 1) return -2;
  if (c->dtype == 1 && (!c->k_scale || !c->v_scale)) return -3;
  if (c->kv_heads <= 0 || c->page_size <= 0 || (c->page_size & (c->page_size - 1)) || c->page_size > 65536 ||
      (int64_t)c->kv_heads * c->page_size > (1 << 24))
    return -4;
  if (c->num_pages <= 0 || c->num_pages > 0x7fffffff || c->width < 0 || c->width > 0x7fffffff || c->ldt < c->width)
    return -5;
  const int64_t rows = (int64_t)c->kv_heads * c->page_size;
  const int elt = c->dtype == 1 ? 1 : 2;
  if (c->ld_page < rows * kHD || (c->ld_page * elt) % 16 || (c->dtype == 1 && c->ld_scale < rows)) return -6;
  if (!al16(c->k) || !al16(c->v) || (reinterpret_cast<uintptr_t>(c->table) & 3)) return -7;
  p->k = static_cast<char*>(c->k);
  p->v = static_cast<char*>(c->v);
  p->ks = c->k_scale;
  p->vs = c->v_scale;
  p->table = c->table;
  p->ldt = c->ldt;
  p->width = c->width;
  p->num_pages = c->num_pages;
  p->ld_page = c->ld_page * elt;
  p->ld_scale = c->ld_scale;
  p->kv_heads = c->kv_heads;
  p->log_page = 0;
  while ((1 << p->log_page) < c->page_size) ++p->log_page;
  return 0;
}

inline int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : (int)e;
}

}  // namespace

extern "C" int cdk_paged_append(const void* qkv, int64_t ldq, int qkv_f32, const int32_t* pos, const float* rope,
                                int64_t rope_len, int64_t B, int64_t S_new, int64_t H, const CdkPagedCache* cache,
                                const int32_t* start, const int32_t* num_new, void* q_out, int64_t ldo,
                                void* stream) {
  if (B == 0 || S_new == 0) return 0;
  Pages pg;
  if (const int rc = take_pages(cache, &pg)) return rc;
  if (!qkv || !start || B < 0 || S_new < 0 || H < 0 || H > 65536) return -10;
  const int64_t heads = H + 2 * (int64_t)pg.kv_heads;
  if (ldq < heads * kHD || ldq % (qkv_f32 ? 4 : 8) || !al16(qkv)) return -11;
  if (rope && (!pos || rope_len <= 0 || !al16(rope))) return -12;
  if (q_out && (ldo < H * kHD || ldo % 8 || !al16(q_out))) return -13;
  if (B > 0x7fffffffll / S_new) return -14;
  // a warp per token; several, down to four heads each, while there are fewer than 16 warps per SM
  const long long tokens = B * S_new, most = q_out && H > pg.kv_heads ? H : pg.kv_heads;
  long long parts = (148 * 16 + tokens - 1) / tokens;
  if (parts > (most + 3) / 4) parts = (most + 3) / 4;
  if (tokens * parts > 0xfffffff0ll) parts = 1;
  const long long blocks = (tokens * parts + 3) / 4;
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  auto* qo = reinterpret_cast<__nv_bfloat16*>(q_out);
#define CDK_APPEND(F32, FP8)                                                                                     \
  paged_append_kernel<F32, FP8><<<(unsigned)blocks, 128, 0, st>>>(qkv, ldq, pos, rope, rope_len, (unsigned)S_new,   \
                                                                  (int)H, pg, start, num_new, qo, ldo,               \
                                                                  (unsigned)tokens, (unsigned)parts)
  if (cache->dtype == 1) {
    if (qkv_f32) CDK_APPEND(true, true);
    else CDK_APPEND(false, true);
  } else {
    if (qkv_f32) CDK_APPEND(true, false);
    else CDK_APPEND(false, false);
  }
#undef CDK_APPEND
  return launched();
}

extern "C" int cdk_paged_gather(const CdkPagedCache* cache, int64_t B, const int32_t* lens, void* k_out, void* v_out,
                                int64_t sb, int64_t sh, int64_t ss, int64_t S, void* stream) {
  if (B == 0 || S == 0) return 0;
  Pages pg;
  if (const int rc = take_pages(cache, &pg)) return rc;
  if (!lens || !k_out || !v_out || B < 0 || S < 0) return -10;
  if (sb % 8 || sh % 8 || ss % 8 || !al16(k_out) || !al16(v_out)) return -11;
  const long long chunks = (S + kGatherRows - 1) / kGatherRows;
  if (B > 65535 || pg.kv_heads > 65535 || chunks > 0x7fffffff) return -12;
  const dim3 grid((unsigned)chunks, (unsigned)pg.kv_heads, (unsigned)B);
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  auto* ko = reinterpret_cast<__nv_bfloat16*>(k_out);
  auto* vo = reinterpret_cast<__nv_bfloat16*>(v_out);
  if (cache->dtype == 1) paged_gather_kernel<true><<<grid, 256, 0, st>>>(pg, lens, ko, vo, sb, sh, ss, S);
  else paged_gather_kernel<false><<<grid, 256, 0, st>>>(pg, lens, ko, vo, sb, sh, ss, S);
  return launched();
}

namespace {
inline int64_t prefix_bytes(int64_t B) { return ((B + 1) * 4 + 15) / 16 * 16; }

// Warps that share an item of at most max_tiles tiles, or 0: the deal.  The deal's cost
// beside the keys -- its search, the partial results, the second launch -- is some 5 us
// and grows with the items; a block per item leaves SMs idle at the end while the
// longest is read.  So a block takes an item up to 32 tiles (300 x 1000 keys of 2 heads:
// 35 us both ways, 150 x 1000: 18 and 22), and longer ones where items are many and
// the end is little of the whole (1600 x 1 .. 4000 keys of 2 heads: 252 us, 270 by the
// deal; 64 x 1 .. 2000 of 16: 53, 49).  Eight warps while every block of that size is
// resident at once (72 x 1000 of 2 heads: 11.8 us, 14.4 with four, 16.0 by the deal); a
// warp of its own where blocks would be many and short (1600 x 32 of 2 heads: 9.9, 17.4).
// The tiles of bf16 pages below 32 rows take a warp twice as long, so that the end is
// more (256 x 1 .. 4000 keys of 16 heads on pages of 16: 361 us, 338 by the deal).
constexpr int kMany = 8;
constexpr int kWideLog = 5;  // pages of 32 rows and more hold a tile whole
inline int warps_per_item(long long items, long long max_tiles, int group, bool fp8, bool wide) {
  if (items > kAttnBlocks && max_tiles <= (items < 2 * kAttnBlocks ? 2 : fp8 ? 8 : 4)) return 1;
  if (items <= (group <= 8 ? 2 : 1) * 148 && max_tiles > 4 && max_tiles <= 32) return kMany;
  const long long most = fp8 || wide ? items / 18 : 0;
  return max_tiles <= (most < 32 ? 32 : most > 256 ? 256 : most) ? kWarps : 0;
}

template <bool FP8, int NT, bool WIDE>
cudaError_t launch_attn(const AttnArgs& a, long long max_tiles, cudaStream_t st) {
  const long long items = (long long)a.B * a.pg.kv_heads;
  const int smem = AttnShared::bytes(a.group, FP8);
  static bool done[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= 64) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
  if (!done[dev]) {
    auto allow = [&](const void* f, int bytes) {
      if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    allow((const void*)paged_attn_item_kernel<FP8, NT, WIDE, 1>, AttnShared::bytes(kMaxGroup, FP8));
    allow((const void*)paged_attn_item_kernel<FP8, NT, WIDE, kWarps>, AttnShared::bytes(kMaxGroup, FP8));
    allow((const void*)paged_attn_item_kernel<FP8, NT, WIDE, kMany>, AttnShared::bytes(kMaxGroup, FP8, kMany));
    allow((const void*)paged_attn_kernel<FP8, NT, WIDE>, (int)prefix_bytes(kMaxSeqs) + AttnShared::bytes(kMaxGroup, FP8));
    if (e != cudaSuccess) return e;
    done[dev] = true;
  }
  const int split = warps_per_item(items, max_tiles, a.group, FP8, WIDE);
  if (split == 1) {
    const unsigned blocks = (unsigned)((items + kWarps - 1) / kWarps);
    paged_attn_item_kernel<FP8, NT, WIDE, 1><<<blocks, kAttnThreads, smem, st>>>(a);
  } else if (split == kWarps) {
    paged_attn_item_kernel<FP8, NT, WIDE, kWarps><<<(unsigned)items, kAttnThreads, smem, st>>>(a);
  } else if (split == kMany) {
    paged_attn_item_kernel<FP8, NT, WIDE, kMany>
        <<<(unsigned)items, kMany * 32, AttnShared::bytes(a.group, FP8, kMany), st>>>(a);
  }
  if (split) return cudaGetLastError();
  // no more warps than tiles that the tables can hold: one tile is the smallest share
  const long long bound = max_tiles * items;
  const unsigned grid = (unsigned)(bound >= kAttnWarps ? kAttnBlocks : (bound + kWarps - 1) / kWarps);
  paged_attn_kernel<FP8, NT, WIDE><<<grid, kAttnThreads, (int)prefix_bytes(a.B) + smem, st>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * a.group));
  // eight results in flight per warp; an item has one from each block inside it, and of
  // the warps of the blocks at its ends (592 of one long item, 12 of 23 tiles)
  const long long results = (max_tiles < kAttnWarps ? max_tiles : kAttnWarps) / kWarps + 6;
  const long long warps = (results + 7) / 8, most = items >= 148 ? 4 : kJoinWarps;
  const int join = (int)(warps < most ? warps : most);
  cfg.blockDim = dim3(join * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];  // set up while the first kernel drains; it waits for it before its first load
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_join_kernel, (const AttnArgs)a, grid * (unsigned)kWarps);
}
}  // namespace

extern "C" int64_t cdk_paged_attn_workspace(int64_t B, int64_t H, int64_t kv_heads, int64_t max_keys) {
  if (B < 0 || B > kMaxSeqs || H <= 0 || H > 65536 || kv_heads <= 0 || H % kv_heads || H / kv_heads > kMaxGroup ||
      max_keys < 0)
    return -1;
  // whatever the pages are: the smaller set of those that need none
  if (max_keys < (1ll << 31) && warps_per_item(B * kv_heads, (max_keys + kTK - 1) / kTK, (int)(H / kv_heads), false, false))
    return 0;
  return prefix_bytes(B) + (int64_t)kSlots * (H / kv_heads) * (16 + kHD * 4);
}

extern "C" int cdk_paged_attn_launches(const CdkPagedCache* cache, int64_t B, int64_t H) {
  if (B == 0) return 0;
  Pages pg;
  if (const int rc = take_pages(cache, &pg)) return rc;
  if (B < 0 || B > kMaxSeqs || H <= 0 || H > 65536 || H % pg.kv_heads || H / pg.kv_heads > kMaxGroup) return -11;
  const int64_t tiles = ((pg.width << pg.log_page) + kTK - 1) / kTK;
  return warps_per_item(B * pg.kv_heads, tiles, (int)(H / pg.kv_heads), cache->dtype == 1, pg.log_page >= kWideLog) ? 1 : 2;
}

extern "C" int cdk_paged_attn(const void* q, int64_t ldq, const CdkPagedCache* cache, int64_t B, int64_t H,
                              const int32_t* lens, void* out, int64_t ldo, float scale, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (B == 0) return 0;
  AttnArgs a;
  if (const int rc = take_pages(cache, &a.pg)) return rc;
  if (!q || !lens || !out || B < 0 || H <= 0) return -10;
  const int64_t keys = a.pg.width << a.pg.log_page, tiles = (keys + kTK - 1) / kTK;  // per item, at most
  const int64_t need = cdk_paged_attn_workspace(B, H, a.pg.kv_heads, keys);
  if (need < 0) return -11;
  if (need > 0 && (!workspace || workspace_bytes < need || !al16(workspace))) return -12;
  if (ldq < H * kHD || ldq % 8 || ldo < H * kHD || ldo % 8 || !al16(q) || !al16(out)) return -13;
  if (!(scale == scale)) return -14;
  if (keys >= (1ll << 31) - 64 || (tiles + kSetup) * a.pg.kv_heads > ((1ll << 31) - 1) / B)
    return -15;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.ldq = ldq;
  a.B = (int)B;
  a.group = (int)(H / a.pg.kv_heads);
  a.lens = lens;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.ldo = ldo;
  a.scale_log2 = scale * 1.4426950408889634f;
  char* ws = static_cast<char*>(workspace);
  a.prefix = reinterpret_cast<int32_t*>(ws);
  a.stat = reinterpret_cast<float2*>(ws + prefix_bytes(B));
  a.part = reinterpret_cast<float*>(ws + prefix_bytes(B) + (int64_t)kSlots * a.group * 16);
  auto st = reinterpret_cast<cudaStream_t>(stream);
  // pages of 32 rows and more hold a tile whole (a kernel that takes both kinds needs
  // registers that the loads in flight then miss: 64 x 0..2000 keys 52 us for 48)
  const bool wide = a.pg.log_page >= kWideLog;
#define CDK_ATTN(FP8, NT) (int)(wide ? launch_attn<FP8, NT, true>(a, tiles, st) : launch_attn<FP8, NT, false>(a, tiles, st))
  if (cache->dtype == 1) return a.group <= 8 ? CDK_ATTN(true, 1) : CDK_ATTN(true, 2);
  return a.group <= 8 ? CDK_ATTN(false, 1) : CDK_ATTN(false, 2);
#undef CDK_ATTN
}

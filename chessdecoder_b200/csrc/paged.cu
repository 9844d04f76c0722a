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

// Value of a scale byte: 2^(e - 127).  Bytes 1..254 are exponent fields; byte 0
// (never written here) is the subnormal 2^-127 and 255 a NaN, as in e8m0.
__device__ __forceinline__ float scale_of(uint32_t e) {
  return e == 0 ? __uint_as_float(0x00400000u) : e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23);
}

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
// Append.  Eight lanes per (token, head) row of 64, eight values each.  The
// rotation is three separately rounded operations per value (no fused multiply-
// add), so that a quantised code does not depend on how a compiler contracts
// them.  Bound by HBM: one read of qkv, one write of each row.
// ---------------------------------------------------------------------------
template <bool F32, bool FP8>
__global__ void __launch_bounds__(256)
    paged_append_kernel(const void* __restrict__ qkv, long long ldq, const int32_t* __restrict__ pos,
                        const float* __restrict__ rope, long long rope_len, long long S_new, int H, Pages pg,
                        const int32_t* __restrict__ start, const int32_t* __restrict__ num_new,
                        __nv_bfloat16* __restrict__ q_out, long long ldo, long long rows) {
  const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
  const int sub = threadIdx.x & 7;
  const int heads = H + 2 * pg.kv_heads;
  const bool in = i < rows;
  const long long t = in ? i / heads : 0;
  const int h = in ? (int)(i - t * heads) : 0;
  const long long b = t / S_new;
  const long long s = t - b * S_new;
  bool live = in && (num_new == nullptr || s < num_new[b]);
  const bool is_q = h < H, is_v = h >= H + pg.kv_heads;
  if (is_q && q_out == nullptr) live = false;
  float x[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) x[c] = 0.f;
  if (live) {
    if (F32) {
      const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(qkv) + t * ldq + h * kHD + sub * 8);
      const float4 a = src[0], c = src[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = c.x; x[5] = c.y; x[6] = c.z; x[7] = c.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(qkv) + t * ldq + h * kHD + sub * 8);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 f = bf2f(w[c]);
        x[2 * c] = f.x;
        x[2 * c + 1] = f.y;
      }
    }
    if (rope != nullptr && !is_v) {
      const long long p = pos[t];
      if (p < 0 || p >= rope_len) {
        if (sub == 0) report_error(kErrIndex);
        live = false;
      } else {
        const float4* cs = reinterpret_cast<const float4*>(rope + (p * 32 + sub * 4) * 2);
        const float4 a = cs[0], c = cs[1];
        const float co[4] = {a.x, a.z, c.x, c.z}, si[4] = {a.y, a.w, c.y, c.w};
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          const float u = x[2 * c4], w = x[2 * c4 + 1];
          x[2 * c4] = __fsub_rn(__fmul_rn(u, co[c4]), __fmul_rn(w, si[c4]));
          x[2 * c4 + 1] = __fadd_rn(__fmul_rn(w, co[c4]), __fmul_rn(u, si[c4]));
        }
      }
    }
  }
  float amax = 0.f;
  if (FP8) {
#pragma unroll
    for (int c = 0; c < 8; ++c) amax = fmaxf(amax, fabsf(x[c]));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  if (!live) return;
  if (is_q) {
    *reinterpret_cast<uint4*>(q_out + t * ldo + h * kHD + sub * 8) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
    return;
  }
  const long long slot = (long long)start[b] + s;
  const int page = page_of(pg, b, slot);
  if (page < 0) return;
  const int kvh = is_v ? h - H - pg.kv_heads : h - H;
  const long long r = ((long long)kvh << pg.log_page) + (slot & ((1ll << pg.log_page) - 1));
  char* dst = (is_v ? pg.v : pg.k) + page * pg.ld_page + r * (kHD * (FP8 ? 1 : 2));
  if (FP8) {
    // least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), as an exponent field
    const uint32_t bits = __float_as_uint(amax);
    const int byte = max((int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
    uint32_t w[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
      w[c] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * c] * inv, x[4 * c + 1] * inv), __NV_SATFINITE,
                                                __NV_E4M3) |
             ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * c + 2] * inv, x[4 * c + 3] * inv), __NV_SATFINITE,
                                                 __NV_E4M3)
              << 16);
    *reinterpret_cast<uint2*>(dst + sub * 8) = make_uint2(w[0], w[1]);
    if (sub == 0) (is_v ? pg.vs : pg.ks)[page * pg.ld_scale + r] = (uint8_t)byte;
  } else {
    *reinterpret_cast<uint4*>(dst + sub * 16) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  }
}

// ---------------------------------------------------------------------------
// Read back.  Grid (row chunks, kv head, sequence); eight lanes per row, key and
// value of it.
// ---------------------------------------------------------------------------
template <bool FP8>
__device__ __forceinline__ uint4 load_row8(const char* base, long long row, int sub, const uint8_t* scale,
                                           long long srow) {
  if (!FP8) return *reinterpret_cast<const uint4*>(base + row + sub * 16);
  const uint2 c = *reinterpret_cast<const uint2*>(base + row + sub * 8);
  const float s = scale_of(scale[srow]);
  float2 f[4] = {e4m3x2_f(c.x), e4m3x2_f(c.x >> 16), e4m3x2_f(c.y), e4m3x2_f(c.y >> 16)};
  uint4 o;
  o.x = pack_bf16(f[0].x * s, f[0].y * s);
  o.y = pack_bf16(f[1].x * s, f[1].y * s);
  o.z = pack_bf16(f[2].x * s, f[2].y * s);
  o.w = pack_bf16(f[3].x * s, f[3].y * s);
  return o;
}

template <bool FP8>
__global__ void __launch_bounds__(256)
    paged_gather_kernel(Pages pg, const int32_t* __restrict__ lens, __nv_bfloat16* __restrict__ k_out,
                        __nv_bfloat16* __restrict__ v_out, long long sb, long long sh, long long ss, long long S) {
  const long long b = blockIdx.z;
  const int h = blockIdx.y;
  const long long j = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
  const int sub = threadIdx.x & 7;
  long long len = lens[b];
  if (len > S) {
    if (j == 0 && sub == 0 && h == 0) report_error(kErrIndex);
    len = S;
  }
  if (j >= len) return;
  const int page = page_of(pg, b, j);
  if (page < 0) return;
  const long long r = ((long long)h << pg.log_page) + (j & ((1ll << pg.log_page) - 1));
  const long long row = page * pg.ld_page + r * (kHD * (FP8 ? 1 : 2)), srow = page * pg.ld_scale + r;
  const long long o = b * sb + h * sh + j * ss + sub * 8;
  *reinterpret_cast<uint4*>(k_out + o) = load_row8<FP8>(pg.k, row, sub, pg.ks, srow);
  *reinterpret_cast<uint4*>(v_out + o) = load_row8<FP8>(pg.v, row, sub, pg.vs, srow);
}

// ---------------------------------------------------------------------------
// One new token per sequence.  One block per (query head, sequence): each warp
// takes every fourth key, lane l dims 2l and 2l + 1; a running maximum and sum
// per warp, merged through shared memory.
// ---------------------------------------------------------------------------
template <bool FP8>
__global__ void __launch_bounds__(128)
    paged_attn_kernel(const __nv_bfloat16* __restrict__ q, long long ldq, Pages pg, int group,
                      const int32_t* __restrict__ lens, __nv_bfloat16* __restrict__ out, long long ldo, float scale) {
  const long long b = blockIdx.y;
  const int h = blockIdx.x, kvh = h / group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long len = max(lens[b], 0);
  if (len > (pg.width << pg.log_page)) {
    if (threadIdx.x == 0) report_error(kErrIndex);
    len = pg.width << pg.log_page;
  }
  const float2 qf = bf2f(*reinterpret_cast<const uint32_t*>(q + b * ldq + h * kHD + 2 * lane));
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (long long j = warp; j < len; j += 4) {
    const int page = page_of(pg, b, j);
    if (page < 0) continue;
    const long long r = ((long long)kvh << pg.log_page) + (j & ((1ll << pg.log_page) - 1));
    const long long row = page * pg.ld_page + r * (kHD * (FP8 ? 1 : 2)), srow = page * pg.ld_scale + r;
    float2 kf, vf;
    if (FP8) {
      kf = e4m3x2_f(*reinterpret_cast<const uint16_t*>(pg.k + row + 2 * lane));
      vf = e4m3x2_f(*reinterpret_cast<const uint16_t*>(pg.v + row + 2 * lane));
      const float a = scale_of(pg.ks[srow]), c = scale_of(pg.vs[srow]);
      kf.x *= a; kf.y *= a;
      vf.x *= c; vf.y *= c;
    } else {
      kf = bf2f(*reinterpret_cast<const uint32_t*>(pg.k + row + 4 * lane));
      vf = bf2f(*reinterpret_cast<const uint32_t*>(pg.v + row + 4 * lane));
    }
    const float sc = warp_sum(qf.x * kf.x + qf.y * kf.y) * scale;
    const float mn = fmaxf(m, sc);
    const float al = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(sc - mn);
    l = l * al + p;
    o0 = o0 * al + p * vf.x;
    o1 = o1 * al + p * vf.y;
    m = mn;
  }
  __shared__ float sm[4][66];
  sm[warp][2 * lane] = o0;
  sm[warp][2 * lane + 1] = o1;
  if (lane == 0) {
    sm[warp][64] = m;
    sm[warp][65] = l;
  }
  __syncthreads();
  if (warp) return;
  const float M = fmaxf(fmaxf(sm[0][64], sm[1][64]), fmaxf(sm[2][64], sm[3][64]));
  float L = 0.f, x = 0.f, y = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float f = sm[w][64] == -INFINITY ? 0.f : __expf(sm[w][64] - M);
    L += sm[w][65] * f;
    x += sm[w][2 * lane] * f;
    y += sm[w][2 * lane + 1] * f;
  }
  const float inv = len > 0 && M != -INFINITY ? 1.f / L : 0.f;
  *reinterpret_cast<uint32_t*>(out + b * ldo + h * kHD + 2 * lane) = pack_bf16(x * inv, y * inv);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int take_pages(const CdkPagedCache* c, Pages* p) {
  if (!c || !c->k || !c->v || (!c->table && c->width != 0)) return -1;
  if (c->dtype != 0 && c->dtype != 1) return -2;
  if (c->dtype == 1 && (!c->k_scale || !c->v_scale)) return -3;
  if (c->kv_heads <= 0 || c->page_size <= 0 || (c->page_size & (c->page_size - 1)) || c->page_size > 65536) return -4;
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
  if (B > (1ll << 40) / S_new || B * S_new > (1ll << 40) / heads) return -14;
  const long long rows = B * S_new * heads;
  const long long blocks = (rows * 8 + 255) / 256;
  if (blocks > 0x7fffffff) return -14;
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  auto* qo = reinterpret_cast<__nv_bfloat16*>(q_out);
#define CDK_APPEND(F32, FP8)                                                                                     \
  paged_append_kernel<F32, FP8><<<(unsigned)blocks, 256, 0, st>>>(qkv, ldq, pos, rope, rope_len, S_new, (int)H, pg, \
                                                                  start, num_new, qo, ldo, rows)
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
  const long long chunks = (S + 31) / 32;
  if (B > 65535 || pg.kv_heads > 65535 || chunks > 0x7fffffff) return -12;
  const dim3 grid((unsigned)chunks, (unsigned)pg.kv_heads, (unsigned)B);
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  auto* ko = reinterpret_cast<__nv_bfloat16*>(k_out);
  auto* vo = reinterpret_cast<__nv_bfloat16*>(v_out);
  if (cache->dtype == 1) paged_gather_kernel<true><<<grid, 256, 0, st>>>(pg, lens, ko, vo, sb, sh, ss, S);
  else paged_gather_kernel<false><<<grid, 256, 0, st>>>(pg, lens, ko, vo, sb, sh, ss, S);
  return launched();
}

extern "C" int64_t cdk_paged_attn_workspace(int64_t B, int64_t H, int64_t kv_heads) {
  if (B < 0 || B > kMaxSeqs || H <= 0 || kv_heads <= 0 || H % kv_heads || H / kv_heads > kMaxGroup) return -1;
  return 16;
}

extern "C" int cdk_paged_attn(const void* q, int64_t ldq, const CdkPagedCache* cache, int64_t B, int64_t H,
                              const int32_t* lens, void* out, int64_t ldo, float scale, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (B == 0) return 0;
  Pages pg;
  if (const int rc = take_pages(cache, &pg)) return rc;
  if (!q || !lens || !out || B < 0 || H <= 0) return -10;
  const int64_t need = cdk_paged_attn_workspace(B, H, pg.kv_heads);
  if (need < 0) return -11;
  if (!workspace || workspace_bytes < need || !al16(workspace)) return -12;
  if (ldq < H * kHD || ldq % 8 || ldo < H * kHD || ldo % 8 || !al16(q) || !al16(out)) return -13;
  if (!(scale == scale)) return -14;
  const dim3 grid((unsigned)H, (unsigned)B);
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  auto* qq = reinterpret_cast<const __nv_bfloat16*>(q);
  auto* oo = reinterpret_cast<__nv_bfloat16*>(out);
  const int group = (int)(H / pg.kv_heads);
  if (cache->dtype == 1) paged_attn_kernel<true><<<grid, 128, 0, st>>>(qq, ldq, pg, group, lens, oo, ldo, scale);
  else paged_attn_kernel<false><<<grid, 128, 0, st>>>(qq, ldq, pg, group, lens, oo, ldo, scale);
  return launched();
}

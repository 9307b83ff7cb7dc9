// The paged key / value cache in microscaled floating point: rows quantised as they are written, and read back.
//
// A group of 32 channels x is held as codes c and one byte e: x ~ c 2^(e - 127). With k the smallest integer, within -127 ..
// 127, for which max|x| <= MAX 2^k (MAX 6 for e2m1, 448 for e4m3), e = k + 127 and c = RNE(x 2^-k): nothing saturates (the
// power of two below, which saturates what exceeds MAX, leaves a quarter of the largest value's binade off by up to 25% in
// e2m1). k comes from the bits of max|x|: its exponent, one more where the mantissa exceeds MAX's (1.5 and 1.75); scaling by a
// power of two is exact, so the codes are the nearest ones of the input itself. A group with an infinity or a NaN gets byte
// 255 and reads back as NaN.
//
// Both kernels only move bytes. A lane takes 8 channels of one head (16 or 32 bytes of a row, 4 or 8 of codes) and the four
// lanes of a group share its maximum through DPP; consecutive lanes take consecutive channels, so a wave reads whole rows. A
// workgroup takes consecutive rows, which fill consecutive bytes of a page.
#include <type_traits>

#include "common.h"
#include "serve.h"

namespace {

constexpr int NTH = 256;

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ unsigned quad_max(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, DPP_QUAD_XOR1, 0xF, 0xF, false));
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, DPP_QUAD_XOR2, 0xF, 0xF, false));
}

// 8 channels of a row in fp32.
template <int TYPE>
__device__ __forceinline__ void load8(const void* p, long at, float (&x)[8]) {
  if constexpr (TYPE == ROWS_F32) {
    const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at)[0];
    const float4 b = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (TYPE == ROWS_F16) {
    const f16x8 v = *reinterpret_cast<const f16x8*>(static_cast<const f16*>(p) + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
  } else {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(static_cast<const bf16*>(p) + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
  }
}
template <int TYPE>
__device__ __forceinline__ void store8(void* p, long at, const float (&x)[8]) {
  if constexpr (TYPE == ROWS_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else if constexpr (TYPE == ROWS_F16) {
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (f16)x[e];
    *reinterpret_cast<f16x8*>(static_cast<f16*>(p) + at) = v;
  } else {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_bf16(x[e]);
    *reinterpret_cast<bf16x8*>(static_cast<bf16*>(p) + at) = v;
  }
}

// The codes of 8 channels (4 or 8 bytes) and their group's scale byte, in all four lanes of the group.
template <int FMT>
__device__ __forceinline__ unsigned char quantise8(const float (&x)[8], uint2& codes) {
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  top = quad_max(top);
  // max|x| = 1.m 2^(ex - 127): k + 127 = ex - 2 for m <= 0.5 (e2m1, 6 = 1.5 2^2), ex - 8 for m <= 0.75 (e4m3, 448 = 1.75 2^8)
  const int ex = (int)(top >> 23), m = (int)(top & 0x7fffffu);
  const int e = max(0, FMT == CACHE_FP4 ? ex - 2 + (m > 0x400000) : ex - 8 + (m > 0x600000));
  const float down = __uint_as_float((unsigned)(254 - e) << 23);  // 2^-k
  if constexpr (FMT == CACHE_FP4) {
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0] * down, x[1] * down, 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2] * down, x[3] * down, 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4] * down, x[5] * down, 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6] * down, x[7] * down, 1.f, 3);
    codes.x = c;
  } else {
    int a = 0, b = 0;
    a = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * down, x[1] * down, a, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * down, x[3] * down, a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * down, x[5] * down, b, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * down, x[7] * down, b, true);
    codes = make_uint2((unsigned)a, (unsigned)b);
  }
  return ex == 255 ? 255 : (unsigned char)e;
}

// 2^(e - 127), NaN for 255
__device__ __forceinline__ float scale_of(unsigned e) {
  return __uint_as_float(e == 0 ? 0x400000u : e == 255 ? 0x7fc00000u : e << 23);
}

template <int FMT>
__device__ __forceinline__ void values8(uint2 codes, float scale, float (&x)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  f32x2 p[4];
  if constexpr (FMT == CACHE_FP4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes.x, 1.f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes.x, 1.f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes.x, 1.f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes.x, 1.f, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, false);
    p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, true);
    p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, false);
    p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, true);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[2 * e] = p[e].x * scale, x[2 * e + 1] = p[e].y * scale;
}

constexpr int ROWS_MAX = 16;  // rows of a workgroup

// Slots of the workgroup's rows into `slot`: -1 for a row at no place (no sequence, a negative position), -2 for a page that
// the cache does not have.
__device__ __forceinline__ void find_slots(const Cache& c, const Sequences& s, int r0, int nr, long* slot) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int r = wave; r < nr; r += NTH / 64) {
    const Place at = place_of(s, r0 + r);
    long x = -1;
    if (at.b >= 0 && at.pos >= 0) {
      x = slot_of(c, s, at.b, at.pos);
      if (x < 0) x = -2;
    }
    if ((threadIdx.x & 63) == 0) slot[r] = x;
  }
  __syncthreads();
}

// One workgroup: `nr` rows (the last one fewer), blockIdx.y 0 the keys, 1 the values.
template <int TYPE, int FMT>
__global__ void __launch_bounds__(NTH) cache_write_kernel(Cache c, Sequences s, Heads k, Heads v, int nr) {
  __shared__ long slot[ROWS_MAX];
  const int r0 = blockIdx.x * nr;
  nr = min(nr, s.rows - r0);
  find_slots(c, s, r0, nr, slot);
  const Heads in = blockIdx.y ? v : k;
  uint8_t *codes = blockIdx.y ? c.v : c.k, *scales = blockIdx.y ? c.vs : c.ks;
  const int ch = c.dim / 8, per = c.kv_heads * ch;  // chunks of a head, of a row
  constexpr int BYTES = FMT == CACHE_FP4 ? 4 : 8;
  for (int i = threadIdx.x; i < nr * per; i += NTH) {
    const int r = i / per, h = (i % per) / ch, d = i % ch;
    const long at = slot[r];
    float x[8];
    load8<TYPE>(in.p, (r0 + r) * in.ld + h * in.hs + 8 * d, x);
    uint2 q;
    const unsigned char e = quantise8<FMT>(x, q);
    if (at < 0) continue;
    // token row of this head: page * kv_heads * page size + h * page size + token
    const long page = at >> c.page_shift, row = ((page * c.kv_heads + h) << c.page_shift) + (at & ((1 << c.page_shift) - 1));
    uint8_t* o = codes + row * (ch * BYTES) + d * BYTES;
    if constexpr (FMT == CACHE_FP4)
      *reinterpret_cast<unsigned*>(o) = q.x;
    else
      *reinterpret_cast<uint2*>(o) = q;
    if (d % 4 == 0) scales[row * (ch / 4) + d / 4] = e;
  }
}

template <int TYPE, int FMT>
__global__ void __launch_bounds__(NTH) cache_read_kernel(Cache c, Sequences s, void* ko, void* vo, int nr) {
  __shared__ long slot[ROWS_MAX];
  const int r0 = blockIdx.x * nr;
  nr = min(nr, s.rows - r0);
  find_slots(c, s, r0, nr, slot);
  void* out = blockIdx.y ? vo : ko;
  const uint8_t *codes = blockIdx.y ? c.v : c.k, *scales = blockIdx.y ? c.vs : c.ks;
  const int ch = c.dim / 8, per = c.kv_heads * ch;
  constexpr int BYTES = FMT == CACHE_FP4 ? 4 : 8;
  for (int i = threadIdx.x; i < nr * per; i += NTH) {
    const int r = i / per, h = (i % per) / ch, d = i % ch;
    const long at = slot[r];
    float x[8];
    if (at >= 0) {
      const long page = at >> c.page_shift, row = ((page * c.kv_heads + h) << c.page_shift) + (at & ((1 << c.page_shift) - 1));
      const uint8_t* p = codes + row * (ch * BYTES) + d * BYTES;
      uint2 q = make_uint2(0, 0);
      if constexpr (FMT == CACHE_FP4)
        q.x = *reinterpret_cast<const unsigned*>(p);
      else
        q = *reinterpret_cast<const uint2*>(p);
      values8<FMT>(q, scale_of(scales[row * (ch / 4) + d / 4]), x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = at == -1 ? 0.f : __uint_as_float(0x7fc00000u);
    }
    store8<TYPE>(out, ((long)(r0 + r) * per + i % per) * 8, x);
  }
}

}  // namespace

bool bad_cache(const Cache& c, const Sequences& s) {
  return !c.k || !c.v || !c.ks || !c.vs || c.pages <= 0 || c.pages > 0x7fffffffL || c.page_shift < 4 || c.page_shift > 8 ||
         c.kv_heads <= 0 || c.kv_heads > 1024 || (c.dim != 64 && c.dim != 128) ||
         (c.format != CACHE_FP4 && c.format != CACHE_FP8) || (((uintptr_t)c.k | (uintptr_t)c.v) & 15) ||
         (((uintptr_t)c.ks | (uintptr_t)c.vs) & 3) || s.n <= 0 || s.rows <= 0 || !s.lengths || s.table_pages < 0 ||
         (s.table_pages > 0 && (!s.table || s.table_ld < s.table_pages)) || (!s.starts && s.rows != s.n);
}

namespace {

// Rows of a workgroup: 16 where that still gives every CU several workgroups, fewer for short calls.
int rows_per_group(const Cache& c, const Sequences& s) {
  int nr = ROWS_MAX;
  while (nr > 1 && (s.rows + nr - 1) / nr < 2 * num_cus()) nr /= 2;
  return nr;
}

// launch(type, format) with both as compile-time constants
template <class F>
void by_type(int type, int format, F launch) {
  auto of = [&](auto t) {
    if (format == CACHE_FP4)
      launch(t, std::integral_constant<int, CACHE_FP4>{});
    else
      launch(t, std::integral_constant<int, CACHE_FP8>{});
  };
  if (type == ROWS_BF16)
    of(std::integral_constant<int, ROWS_BF16>{});
  else if (type == ROWS_F16)
    of(std::integral_constant<int, ROWS_F16>{});
  else
    of(std::integral_constant<int, ROWS_F32>{});
}

}  // namespace

int cache_write_launch(const Cache& c, const Sequences& s, const Heads& k, const Heads& v, int type, hipStream_t stream) {
  if (bad_cache(c, s) || type < ROWS_BF16 || type > ROWS_F32) return NOISE_EINVAL;
  const int unit = type == ROWS_F32 ? 4 : 8;  // elements of a 16-byte load
  for (const Heads* h : {&k, &v})
    if (!h->p || ((uintptr_t)h->p & 15) || h->ld % unit || h->hs % unit || h->ld < 0 || h->hs < 0) return NOISE_EINVAL;
  const int nr = rows_per_group(c, s);
  const dim3 grid((unsigned)((s.rows + nr - 1) / nr), 2);
  by_type(type, c.format, [&](auto t, auto f) {
    hipLaunchKernelGGL((cache_write_kernel<decltype(t)::value, decltype(f)::value>), grid, dim3(NTH), 0, stream, c, s, k, v, nr);
  });
  NOISE_CHECK_LAUNCH();
  return NOISE_OK;
}

int cache_read_launch(const Cache& c, const Sequences& s, void* k, void* v, int type, hipStream_t stream) {
  if (bad_cache(c, s) || type < ROWS_BF16 || type > ROWS_F32 || !k || !v || (((uintptr_t)k | (uintptr_t)v) & 15))
    return NOISE_EINVAL;
  const int nr = rows_per_group(c, s);
  const dim3 grid((unsigned)((s.rows + nr - 1) / nr), 2);
  by_type(type, c.format, [&](auto t, auto f) {
    hipLaunchKernelGGL((cache_read_kernel<decltype(t)::value, decltype(f)::value>), grid, dim3(NTH), 0, stream, c, s, k, v, nr);
  });
  NOISE_CHECK_LAUNCH();
  return NOISE_OK;
}

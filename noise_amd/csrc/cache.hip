// The paged key / value cache in microscaled floating point: rows quantised as they are written, and read back.
//
// A group of 32 channels x is held as codes c and one byte e: x ~ c 2^(e - 127). With k the smallest integer, within -127 ..
// 127, for which max|x| <= MAX 2^k (MAX 6 for e2m1, 448 for e4m3), e = k + 127 and c = RNE(x 2^-k): nothing saturates (the
// power of two below, which saturates what exceeds MAX, leaves a quarter of the largest value's binade off by up to 25% in
// e2m1). k comes from the bits of max|x|: its exponent, one more where the mantissa exceeds MAX's (1.5 and 1.75); scaling by a
// power of two is exact, so the codes are the nearest ones of the input itself. A group with an infinity or a NaN gets byte
// 255 and reads back as NaN.
//
// Both kernels only move bytes. A workgroup takes up to 16 consecutive rows of up to 8 heads, of the keys or of the values, and
// turns them over in LDS: the rows are read or written in their own order (a lane 8 channels, 16 or 32 bytes; the four
// lanes of a group share its maximum through DPP), the codes in the cache's, head by head, where consecutive tokens of a page
// are consecutive bytes (a lane 16 bytes). Reading 64 bytes of a head here and there between the stores instead, without LDS, took
// 24 sequences of up to 8192 tokens, 8 heads of 128 in e2m1, 137 us where their stores alone take 85. Now 111 us, 5.1 TB/s, as a large
// copy; 32 prompts of up to 2048 rows, 8 heads of 64 in fp16 to e4m3, are written in 23 us and read in 23 (4.0 TB/s).
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

constexpr int ROWS_MAX = 16;  // rows of a workgroup, at most a wave's lanes
constexpr long NO_PLACE = -1, BAD_PLACE = -2;

// The code rows (of kv head 0) of the workgroup's rows into `base`, or NO_PLACE, or BAD_PLACE for a page that the cache does not
// have. A lane a row: the first row's sequence is found by the wave, and most rows are in the same one; the others search on.
// One wave, whose first thread is t0.
__device__ __forceinline__ void find_rows(const Cache& c, const Sequences& s, int r0, int nr, long* base, int t0) {
  const int r = threadIdx.x - t0, i = r0 + min(r, nr - 1);
  int b = i;
  long pos = -1;
  if (s.starts) {
    b = find_sequence(s.starts, s.n, r0);
    if (b < s.n && s.starts[b + 1] <= i) {
      int lo = b + 1, hi = s.n;  // the entries of starts[1 ..] that are <= i: at least lo, at most hi
      while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (s.starts[mid] <= i)
          lo = mid;
        else
          hi = mid - 1;
      }
      b = lo;
    }
    if (b < s.n) {
      const int s0 = s.starts[b], s1 = s.starts[b + 1];
      if (i >= s0 && i < s1) pos = (long)s.lengths[b] - s1 + i;
    }
  } else {
    pos = (long)s.lengths[b] - 1;
  }
  long x = NO_PLACE;
  if (pos >= 0) {
    x = slot_of(c, s, b, pos);
    const long page = x >> c.page_shift;
    x = x < 0 ? BAD_PLACE : ((page * c.kv_heads) << c.page_shift) + (x & ((1 << c.page_shift) - 1));
  }
  if (r < nr) base[r] = x;
}

constexpr int HEADS = 8;  // heads of a workgroup at most

// What a workgroup turns over in LDS: codes [head][row + one of padding][ROW bytes], so that the heads of a wave lie in different
// banks, and scale bytes [head][row][GROUPS].
template <int FMT, int DIM>
struct Turn {
  static constexpr int CH = DIM / 8, GROUPS = DIM / 32, ROW = FMT == CACHE_FP4 ? DIM / 2 : DIM, BYTES = ROW / CH;
  static __host__ __device__ int code_bytes(int heads, int nr) { return heads * (nr + 1) * ROW; }
  static __host__ __device__ int bytes(int heads, int nr) { return code_bytes(heads, nr) + heads * nr * GROUPS; }
};

// body(at, cache byte) for every 16 bytes of codes of the workgroup's rows, in the cache's order: from byte
// `at` of the LDS area; then scale() likewise for the scale bytes of every row and head.
template <int FMT, int DIM, class F, class G>
__device__ __forceinline__ void in_cache_order(const long* base, int page_shift, int h0, int heads, int nr, int log_nr, F body, G scale) {
  using T = Turn<FMT, DIM>;
  constexpr int PARTS = T::ROW / 16;
  const int all = (heads * PARTS) << log_nr;
  if (threadIdx.x >= NTH) return;
#pragma unroll 4
  for (int u = threadIdx.x; u < all; u += NTH) {
    const int part = u % PARTS, r = (u / PARTS) & ((1 << log_nr) - 1), h = (u / PARTS) >> log_nr;
    const long at = r < nr ? base[r] : NO_PLACE;
    if (at >= 0) body((h * ((1 << log_nr) + 1) + r) * T::ROW + 16 * part, (at + ((long)(h0 + h) << page_shift)) * T::ROW + 16 * part);
  }
  for (int u = threadIdx.x; u < heads << log_nr; u += NTH) {
    const int r = u & ((1 << log_nr) - 1), h = u >> log_nr;
    const long at = r < nr ? base[r] : NO_PLACE;
    if (at >= 0) scale(u * T::GROUPS, (at + ((long)(h0 + h) << page_shift)) * T::GROUPS);
  }
}

// One workgroup: 2^log_nr rows (the last one fewer) of a slab of heads; blockIdx.y even the keys, odd the values. A fifth wave looks
// the rows' places up (three loads, one after the other) while the others quantise.
template <int TYPE, int FMT, int DIM>
__global__ void __launch_bounds__(NTH + 64) cache_write_kernel(Cache c, Sequences s, Heads k, Heads v, int log_nr) {
  using T = Turn<FMT, DIM>;
  extern __shared__ __attribute__((aligned(16))) uint8_t turn[];
  __shared__ long base[ROWS_MAX];
  const int r0 = blockIdx.x << log_nr, nr = min(1 << log_nr, s.rows - r0);
  const int h0 = blockIdx.y / 2 * HEADS, heads = min(HEADS, c.kv_heads - h0);
  uint8_t* turned = turn + T::code_bytes(heads, 1 << log_nr);
  const Heads in = blockIdx.y & 1 ? v : k;
  uint8_t *codes = blockIdx.y & 1 ? c.v : c.k, *scales = blockIdx.y & 1 ? c.vs : c.ks;
  const int per = heads * T::CH, step = NTH / per, first = threadIdx.x / per, x0 = threadIdx.x % per, h = x0 / T::CH, d = x0 % T::CH;
  const long from = (long)(h0 + h) * in.hs + 8 * d;
  if (threadIdx.x >= NTH) {
    find_rows(c, s, r0, nr, base, NTH);
  } else if (first < step) {
#pragma unroll 4
    for (int r = first; r < nr; r += step) {
      float x[8];
      load8<TYPE>(in.p, (r0 + r) * in.ld + from, x);
      uint2 q;
      const unsigned char e = quantise8<FMT>(x, q);
      uint8_t* o = turn + (h * ((1 << log_nr) + 1) + r) * T::ROW + d * T::BYTES;
      if constexpr (FMT == CACHE_FP4)
        *reinterpret_cast<unsigned*>(o) = q.x;
      else
        *reinterpret_cast<uint2*>(o) = q;
      if (d % 4 == 0) turned[((h << log_nr) + r) * T::GROUPS + d / 4] = e;
    }
  }
  __syncthreads();
  in_cache_order<FMT, DIM>(
      base, c.page_shift, h0, heads, nr, log_nr,
      [&](int at, long to) { *reinterpret_cast<u32x4*>(codes + to) = *reinterpret_cast<const u32x4*>(turn + at); },
      [&](int at, long to) {
        if constexpr (DIM == 64)
          *reinterpret_cast<uint16_t*>(scales + to) = *reinterpret_cast<const uint16_t*>(turned + at);
        else
          *reinterpret_cast<unsigned*>(scales + to) = *reinterpret_cast<const unsigned*>(turned + at);
      });
}

template <int TYPE, int FMT, int DIM>
__global__ void __launch_bounds__(NTH) cache_read_kernel(Cache c, Sequences s, void* ko, void* vo, int log_nr) {
  using T = Turn<FMT, DIM>;
  extern __shared__ __attribute__((aligned(16))) uint8_t turn[];
  __shared__ long base[ROWS_MAX];
  const int r0 = blockIdx.x << log_nr, nr = min(1 << log_nr, s.rows - r0);
  const int h0 = blockIdx.y / 2 * HEADS, heads = min(HEADS, c.kv_heads - h0);
  uint8_t* turned = turn + T::code_bytes(heads, 1 << log_nr);
  if (threadIdx.x < 64) find_rows(c, s, r0, nr, base, 0);
  __syncthreads();
  void* out = blockIdx.y & 1 ? vo : ko;
  const uint8_t *codes = blockIdx.y & 1 ? c.v : c.k, *scales = blockIdx.y & 1 ? c.vs : c.ks;
  in_cache_order<FMT, DIM>(
      base, c.page_shift, h0, heads, nr, log_nr,
      [&](int at, long from) { *reinterpret_cast<u32x4*>(turn + at) = *reinterpret_cast<const u32x4*>(codes + from); },
      [&](int at, long from) {
        if constexpr (DIM == 64)
          *reinterpret_cast<uint16_t*>(turned + at) = *reinterpret_cast<const uint16_t*>(scales + from);
        else
          *reinterpret_cast<unsigned*>(turned + at) = *reinterpret_cast<const unsigned*>(scales + from);
      });
  __syncthreads();
  const int per = heads * T::CH, step = NTH / per, first = threadIdx.x / per, x0 = threadIdx.x % per, h = x0 / T::CH, d = x0 % T::CH;
  if (first >= step) return;
#pragma unroll 4
  for (int r = first; r < nr; r += step) {
    const long at = base[r];
    const uint8_t* p = turn + (h * ((1 << log_nr) + 1) + r) * T::ROW + d * T::BYTES;
    uint2 q = make_uint2(0, 0);
    if constexpr (FMT == CACHE_FP4)
      q.x = *reinterpret_cast<const unsigned*>(p);
    else
      q = *reinterpret_cast<const uint2*>(p);
    const unsigned e = turned[((h << log_nr) + r) * T::GROUPS + d / 4];
    if (at < 0) q = make_uint2(0, 0);  // (what LDS held before)
    float x[8];
    values8<FMT>(q, at == BAD_PLACE ? __uint_as_float(0x7fc00000u) : at < 0 ? 0.f : scale_of(e), x);
    store8<TYPE>(out, ((long)(r0 + r) * c.kv_heads * T::CH + h0 * T::CH + x0) * 8, x);
  }
}

}  // namespace

bool bad_cache(const Cache& c, const Sequences& s) {
  return !c.k || !c.v || !c.ks || !c.vs || c.pages <= 0 || c.pages > 0x7fffffffL || c.page_shift < 4 || c.page_shift > 8 ||
         c.kv_heads <= 0 || c.kv_heads > 1024 || (c.dim != 64 && c.dim != 128) ||
         (c.format != CACHE_FP4 && c.format != CACHE_FP8) || (((uintptr_t)c.k | (uintptr_t)c.v) & 15) ||
         (((uintptr_t)c.ks | (uintptr_t)c.vs) & 3) || s.n <= 0 || s.rows <= 0 || !s.lengths || s.table_pages < 0 ||
         (s.table_pages > 0 && (!s.table || s.table_ld < 0)) || (!s.starts && s.rows != s.n);
}

namespace {

// Rows of a workgroup, as a power of two: 16, fewer for short calls, but enough to keep its threads busy. (The read of the comment
// at the top: 16 rows 111 us, 32 115, 64 121: more workgroups that read and write at the same time.)
int log_rows(const Cache& c, const Sequences& s) {
  const int per = (c.kv_heads < HEADS ? c.kv_heads : HEADS) * (c.dim / 8);
  int l = 4;
  while (l > 0 && ((s.rows - 1) >> l) + 1 < 4 * num_cus() && (per << (l - 1)) >= NTH) --l;
  return l;
}
dim3 grid_of(const Cache& c, const Sequences& s, int l) {
  return dim3((unsigned)((s.rows - 1) >> l) + 1, 2u * (unsigned)((c.kv_heads + HEADS - 1) / HEADS));
}

// launch(type, format, dim) with all three as compile-time constants
template <class F>
void by_type(int type, const Cache& c, F launch) {
  auto of = [&](auto t) {
    auto with = [&](auto f) {
      if (c.dim == 64)
        launch(t, f, std::integral_constant<int, 64>{});
      else
        launch(t, f, std::integral_constant<int, 128>{});
    };
    if (c.format == CACHE_FP4)
      with(std::integral_constant<int, CACHE_FP4>{});
    else
      with(std::integral_constant<int, CACHE_FP8>{});
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
  const int l = log_rows(c, s), heads = c.kv_heads < HEADS ? c.kv_heads : HEADS;
  by_type(type, c, [&](auto t, auto f, auto d) {
    constexpr int TY = decltype(t)::value, F = decltype(f)::value, D = decltype(d)::value;
    const int lds = Turn<F, D>::bytes(heads, 1 << l);
    hipLaunchKernelGGL((cache_write_kernel<TY, F, D>), grid_of(c, s, l), dim3(NTH + 64), lds, stream, c, s, k, v, l);
  });
  NOISE_CHECK_LAUNCH();
  return NOISE_OK;
}

int cache_read_launch(const Cache& c, const Sequences& s, void* k, void* v, int type, hipStream_t stream) {
  if (bad_cache(c, s) || type < ROWS_BF16 || type > ROWS_F32 || !k || !v || (((uintptr_t)k | (uintptr_t)v) & 15))
    return NOISE_EINVAL;
  const int l = log_rows(c, s), heads = c.kv_heads < HEADS ? c.kv_heads : HEADS;
  by_type(type, c, [&](auto t, auto f, auto d) {
    constexpr int TY = decltype(t)::value, F = decltype(f)::value, D = decltype(d)::value;
    const int lds = Turn<F, D>::bytes(heads, 1 << l);
    hipLaunchKernelGGL((cache_read_kernel<TY, F, D>), grid_of(c, s, l), dim3(NTH), lds, stream, c, s, k, v, l);
  });
  NOISE_CHECK_LAUNCH();
  return NOISE_OK;
}

// Attention of whole prompts and of rows over the key / value cache: a query at position s sees key j when 0 <= j <= s and
// (s - j <= window or j < sinks). One wave per row and head: 64 keys at a time, a lane a key for the scores, a lane a channel
// for the values; the running maximum and sum of the softmax in fp32.
#include <type_traits>

#include "common.h"
#include "serve.h"

namespace {

typedef _Float16 f16;
constexpr int WAVES = 4, NTH = 64 * WAVES;

__device__ __forceinline__ float load1(const void* p, long at, int type) {
  return type == ROWS_F16 ? (float)static_cast<const f16*>(p)[at] : (float)static_cast<const bf16*>(p)[at];
}
__device__ __forceinline__ float wave_max(float x) {
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}
__device__ __forceinline__ float wave_add(float x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// key(j, d), value(j, d): channel d of key j
template <class K, class V>
__device__ void attend_row(const float* q, int dim, long pos, int window, int sinks, float scale, K key, V value, float (&y)[2]) {
  const int lane = threadIdx.x & 63;
  const long lo = max(0l, pos - window), first = min((long)sinks, lo), n = first + pos - lo + 1;
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (long t0 = 0; t0 < n; t0 += 64) {
    const long t = t0 + lane;
    float s = -INFINITY;
    if (t < n) {
      const long j = t < first ? t : lo + t - first;
      float d = 0.f;
      for (int c = 0; c < dim; ++c) d = fmaf(q[c], key(j, c), d);
      s = d * scale;
    }
    // a NaN score makes the maximum NaN, and so the row
    const float top = wave_max(s);
    const float mn = __any(s != s) ? __uint_as_float(0x7fc00000u) : fmaxf(m, top);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float alpha = __expf(m - base), p = __expf(s - base);
    m = mn;
    l = l * alpha + wave_add(p);
    o[0] *= alpha, o[1] *= alpha;
    const int cnt = (int)min(64l, n - t0);
    for (int k = 0; k < cnt; ++k) {
      const float pk = __shfl(p, k, 64);
      const long tk = t0 + k, j = tk < first ? tk : lo + tk - first;
      for (int c = 0; c < dim / 64; ++c) o[c] = fmaf(pk, value(j, lane + 64 * c), o[c]);
    }
  }
  for (int c = 0; c < 2; ++c) y[c] = l == 0.f ? 0.f : o[c] / l;
}

template <class T>
__device__ void put(T* y, int dim, const float (&v)[2]) {
  for (int c = 0; c < dim / 64; ++c) y[(threadIdx.x & 63) + 64 * c] = (T)v[c];
}
__device__ void put_row(void* y, long at, int type, int dim, const float (&v)[2]) {
  if (type == ROWS_F16)
    put(static_cast<f16*>(y) + at, dim, v);
  else
    put(static_cast<bf16*>(y) + at, dim, v);
}

__global__ void __launch_bounds__(NTH) sink_kernel(SinkArgs a) {
  __shared__ float sq[WAVES][128];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const long i = (long)blockIdx.x * WAVES + wave;
  if (i >= (long)a.rows * a.heads) return;
  const int row = (int)(i / a.heads), h = (int)(i % a.heads), kh = h / (a.heads / a.kv_heads);
  int s0 = 0;
  bool mine = true;
  if (!a.starts) {
    s0 = row / a.T * a.T;
  } else {
    const int b = __builtin_amdgcn_readfirstlane(find_sequence(a.starts, a.n, row));
    mine = b < a.n && a.starts[b] >= 0 && a.starts[b] <= row && row < a.starts[b + 1];
    if (mine) s0 = a.starts[b];
  }
  if (!mine && !a.fill) return;
  float y[2] = {0.f, 0.f};
  if (mine) {
    for (int d = lane; d < a.dim; d += 64) sq[wave][d] = load1(a.q.p, row * a.q.ld + h * a.q.hs + d, a.type);
    __builtin_amdgcn_wave_barrier();
    attend_row(sq[wave], a.dim, row - s0, a.window, a.sinks, a.scale,
               [&](long j, int d) { return load1(a.k.p, (s0 + j) * a.k.ld + kh * a.k.hs + d, a.type); },
               [&](long j, int d) { return load1(a.v.p, (s0 + j) * a.v.ld + kh * a.v.hs + d, a.type); }, y);
  }
  put_row(a.y, ((long)row * a.heads + h) * a.dim, a.type, a.dim, y);
}

}  // namespace

int sink_attention_launch(const SinkArgs& a, hipStream_t stream) {
  if (bad_heads(a.q) || bad_heads(a.k) || bad_heads(a.v) || !a.y || ((uintptr_t)a.y & 15) || (a.type != ROWS_BF16 && a.type != ROWS_F16) || (a.dim != 64 && a.dim != 128) ||
      a.heads <= 0 || a.heads > 1024 || a.kv_heads <= 0 || a.heads % a.kv_heads || a.window < 0 || a.sinks < 0 ||
      !(a.scale >= 0.f) || a.n <= 0 || a.rows <= 0 || (!a.starts && (a.T <= 0 || (long)a.n * a.T != a.rows)))
    return NOISE_EINVAL;
  const long waves = (long)a.rows * a.heads;
  if (waves > 0x7fffffffL) return NOISE_ENOTSUP;
  hipLaunchKernelGGL(sink_kernel, dim3((unsigned)((waves + WAVES - 1) / WAVES)), dim3(NTH), 0, stream, a);
  NOISE_CHECK_LAUNCH();
  return NOISE_OK;
}

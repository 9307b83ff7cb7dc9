// Causal attention of whole sequences with a left window and sinks: a query at position s sees key j <= s when s - j <= window or
// j < sinks. Sequences of any lengths are packed in one call, heads may be grouped over fewer kv heads.
//
// Bound: for dim 64 the softmax's vector work (an exponential, a fused multiply-add, half a maximum and half a conversion a score,
// beside 4 x 64 flop on the matrix cores), for dim 128 the matrix cores: 16384 tokens of 8 heads take 338 us (813 TFLOP/s of the
// seen scores) and 568 us (968 TFLOP/s; a matrix product of 8192^3 reaches 1248). Short windows pay for blocks seen in part and
// for beginnings: 16 sequences of 2048 tokens in windows of 1024 88 us (590 TFLOP/s).
//
// One workgroup takes 64 QB queries of one sequence and head, a wave 16 QB of them; key blocks of 64 go through a double-buffered
// LDS ring by direct global -> LDS loads, block j + 1 landing while block j is computed (a third slot, two blocks on their way,
// changed no time by more than 5% either way). With few tiles a second group of four waves takes every other block.
//   S^T = K Q^T (A = K rows, B = Q rows): a lane holds 16 scores of query lane % 16. K rows are interleaved at load time so that
//   the scores' layout is the B operand of O^T += V^T P^T: P never leaves registers. V stays row-major [key][channel] and
//   its A fragments come from transposing LDS reads.
//   Softmax in fp32 with a lazy running maximum; P is rounded once to the operands' type, and its row sums are taken of the rounded
//   values on the matrix cores (an all-ones operand), so that the rounding cancels in part.
// Blocks between the sinks and the window are skipped, and a wave skips the blocks none of its queries sees. Blocks seen in part are
// masked. A tile whose output comes out infinite or NaN is computed again row by row, with the values a row does not see taken
// out of the product, since 0 x NaN is not 0.
#include <type_traits>

#include "common.h"
#include "serve.h"

namespace {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int BKV = 64, NWAVE = 4, NTH = 64 * NWAVE;
constexpr int KB = BKV / 16, KC = BKV / 32;  // 16-key tiles of a block, 32-key steps of P V

template <bool F16>
struct Elem {
  using T = typename std::conditional<F16, f16, bf16>::type;
  typedef T x8 __attribute__((ext_vector_type(8)));
  typedef T x4 __attribute__((ext_vector_type(4)));
};
template <bool F16, class X>
__device__ __forceinline__ f32x4 mfma(const X& a, const X& b, const f32x4& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Key of LDS row R of a K block.
__device__ __forceinline__ int key_of_row(int R) {
  const int kb = R >> 4, r = R & 15;
  return 32 * (kb >> 1) + 8 * (r >> 2) + 4 * (kb & 1) + (r & 3);
}
// 16-byte chunk swizzle of LDS row R of a K block: the 16 rows of a fragment's read cover the banks once.
template <int DIM>
__device__ __forceinline__ int kswz(int R) {
  return DIM == 64 ? R & 7 : R & 15;
}

struct Args {
  SinkArgs a;
  float c2;          // scale in base-2 units
  int items, fills;  // workgroups of tiles, workgroups that zero rows
};

struct Tile {
  int s0, m, q0, h;  // first row and rows of the sequence, first query, head
  bool found;
};

// The tile of workgroup `id`. Workgroups reach the 8 XCDs in turn. Where heads divide by 8, XCD x takes the heads x heads / 8 .. of
// every sequence, so all XCDs have the same work and the tiles that share keys run on one XCD's L2 (12000 tokens, 16 heads over 4
// of 128: 591 us, every eighth tile 614); otherwise it takes every eighth tile. The tiles of 64 sequences come in the order of their
// last query, latest first: none sees fewer keys than one after it, and those that run together take about as long (workgroups
// start in order, and one that no CU of the next shader engine has room for holds up all behind it). 16 sequences of up to 2048
// tokens, 8 heads of 64, window 1024: 50 us, sequence by sequence 61.
template <int BQ>
__device__ Tile find_tile(const SinkArgs& a, int id) {
  const int lane = threadIdx.x & 63, x = id & 7;
  const bool even = a.heads % 8 == 0;
  const int per = even ? a.heads / 8 : a.heads;  // heads that an index runs over
  const int at = even ? id >> 3 : id, turn = at / per, h = at % per;
  Tile t{};
  // (all counts are below the grid's size)
  const Sequences rows{nullptr, 0, 0, nullptr, a.starts, a.n, a.rows};
  const int each = (a.T + BQ - 1) / BQ;
  auto first = [&](int b) { return a.starts ? first_tile(rows, b, 1, BQ) : b * each; };
  const int b0 = a.n <= 64 ? 0 : 64 * last_with((a.n - 1) / 64, [&](int c) { return first(64 * c) <= turn; });
  const int base = first(b0);
  const int b = b0 + lane;
  int s0 = 0, m = 0;
  if (b < a.n) {
    s0 = a.starts ? min(max(a.starts[b], 0), a.rows) : b * a.T;
    m = a.starts ? min(max(a.starts[b + 1], 0), a.rows) - s0 : a.T;
  }
  if (__any(m < 0) || turn < base) return t;  // (starts that decrease: nothing is found)
  const int tiles = (m + BQ - 1) / BQ;
  if (turn - base >= wave_sum(tiles)) return t;
  // the level, a tile's number in its sequence: the last from which on there are more tiles than come before this one
  int level = 0, over = (a.rows + BQ - 1) / BQ, before = 0;
  while (over - level > 1) {
    const int mid = (level + over) >> 1, from = wave_sum(max(tiles - mid, 0));
    if (from > turn - base)
      level = mid;
    else
      over = mid, before = from;
  }
  const unsigned long long has = __ballot(tiles > level);
  const int nth = __builtin_amdgcn_mbcnt_hi((unsigned)(has >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)has, 0));
  const int k = __builtin_ctzll(__ballot((tiles > level) & (nth == turn - base - before)));
  t.found = true;
  t.s0 = uniform(s0, k);
  t.m = uniform(m, k);
  t.q0 = level * BQ;
  t.h = even ? x * per + h : h;
  return t;
}

// KS groups of four waves, each with a KS-th of the tile's key blocks.
template <int DIM, bool F16, int QB, int KS>
__global__ void __launch_bounds__(NTH * KS, DIM == 128 ? 2 : KS == 2 ? 4 : 3) sink_kernel(Args g) {
  using E = Elem<F16>;
  using T = typename E::T;
  using x8 = typename E::x8;
  using x4 = typename E::x4;
  constexpr int BQ = 64 * QB, QS = DIM / 32, DT = DIM / 16;
  constexpr int ROWB = 2 * DIM, CH = DIM / 8;          // bytes and 16-byte chunks of a row
  constexpr int DH = BKV * ROWB / 1024 / NWAVE;        // load instructions of 1 KiB per wave, block and operand
  constexpr int RPI = 1024 / ROWB;                     // rows of one
  __shared__ __attribute__((aligned(1024))) char sk[KS][2][BKV * ROWB];
  __shared__ __attribute__((aligned(1024))) char sv[KS][2][BKV * ROWB];
  const SinkArgs& a = g.a;
  if ((int)blockIdx.x >= g.items) {
    fill_rows(a.starts, a.n, a.rows, a.y, a.heads * DIM, NTH * KS, blockIdx.x - g.items, g.fills);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, r16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NWAVE, part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 8);
  const Tile w = find_tile<BQ>(a, blockIdx.x);
  if (!w.found) return;
  const int kh = w.h / (a.heads / a.kv_heads), last = w.m - 1;
  const T* qp = static_cast<const T*>(a.q.p) + (long)w.s0 * a.q.ld + w.h * a.q.hs;
  const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(a.k.p) + (long)w.s0 * a.k.ld + kh * a.k.hs);
  const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(a.v.p) + (long)w.s0 * a.v.ld + kh * a.v.hs);

  // this wave's queries qw .. qe; rows past the sequence repeat its last one and are not stored
  const int qw = w.q0 + 16 * QB * wave, qe = min(qw + 16 * QB - 1, last);
  x8 qf[QB][QS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int i = 0; i < QS; ++i)
      qf[qb][i] = *reinterpret_cast<const x8*>(qp + (long)min(qw + 16 * qb + r16, last) * a.q.ld + 32 * i + 8 * grp);

  // the workgroup's blocks: the sinks', then from the window's first key to the last query
  const int qlast = min(w.q0 + BQ - 1, last), first = w.q0 > a.window ? w.q0 - a.window : 0;
  const int lo = first / BKV, sink = min((min(a.sinks, first) + BKV - 1) / BKV, lo), blocks = sink + qlast / BKV - lo + 1;
  auto block_key = [&](int i) { return (i < sink ? i : lo + i - sink) * BKV; };

  // Loads of block i into ring slot buf. Instruction q of this wave fills LDS rows RPI (DH wave + q) ..; lane L -> row L / CH of
  // them, chunk L % CH: of K the key kr0 + 16 q (8 q for dim 128), of V the key vr0 + RPI q, each at its swizzled chunk. Rows past
  // the sequence repeat its last one (no query sees them).
  const int lrow = lane / CH, lchunk = lane % CH;
  int kr0 = key_of_row(RPI * DH * wave + lrow), vr0 = RPI * DH * wave + lrow;
  unsigned kc0 = 16 * (lchunk ^ kswz<DIM>(RPI * DH * wave + lrow)), vc0 = 16 * (lchunk ^ vswz<DIM>(vr0));
  const unsigned kld = 2 * (unsigned)a.k.ld, vld = 2 * (unsigned)a.v.ld;
  auto issue = [&](int i, int buf) {
    const int j0 = block_key(i), lim = last - j0;
    // (opaque here and in block(): what is derived from these would be kept in registers over the loop)
    asm volatile("" : "+v"(kr0), "+v"(vr0), "+v"(kc0), "+v"(vc0));
    const char *k0 = kp + (long)j0 * kld, *v0 = vp + (long)j0 * vld;
    const char *kd = sk[part][buf] + DH * wave * 1024, *vd = sv[part][buf] + DH * wave * 1024;
#pragma unroll
    for (int q = 0; q < DH; ++q)
      dma_x4_s(k0, __umul24(min(kr0 + (DIM == 64 ? 16 : 8) * q, lim), kld) + (DIM == 64 ? kc0 : kc0 ^ (64 * q)), kd + 1024 * q);
#pragma unroll
    for (int q = 0; q < DH; ++q)
      dma_x4_s(v0, __umul24(min(vr0 + RPI * q, lim), vld) + (vc0 ^ (DIM == 64 ? 64 * q : 128 * (q >> 1))), vd + 1024 * q);
  };

  float mref[QB];
  f32x4 o[QB][DT], osum[QB];
  const x8 ones = {(T)1.f, (T)1.f, (T)1.f, (T)1.f, (T)1.f, (T)1.f, (T)1.f, (T)1.f};
  // fragment i of K tile kb: row 16 kb + r16, chunk 4 i + grp; of V: key 8 grp + t (+ 32 c + 4 x), chunk pair d
  int kro = r16 * ROWB + 16 * (grp ^ kswz<DIM>(r16));
  const int vrr = 8 * grp + (r16 >> 2);
  int vro = vrr * ROWB + 16 * (((lane & 3) >> 1) ^ vswz<DIM>(vrr)) + 8 * (lane & 1);

  // Block i from ring slot BUF. CAREFUL: with every row's unseen values taken out of the product.
  auto block = [&](int i, auto bufc, auto carefulc) {
    constexpr int buf = decltype(bufc)::value;
    constexpr bool CAREFUL = decltype(carefulc)::value;
    const int j0 = block_key(i);
    const char *kt = sk[part][buf], *vt = sv[part][buf];
    asm volatile("" : "+v"(kro), "+v"(vro));
    // blocks that this wave's queries see not at all, or in part
    if (j0 > qe || (qw - (j0 + BKV - 1) > a.window && j0 >= a.sinks)) return;
    const bool some = j0 + BKV - 1 > qw || (qe - j0 > a.window && j0 + BKV > a.sinks);
    f32x4 s[QB][KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      x8 kf[QS];
#pragma unroll
      for (int q = 0; q < QS; ++q) kf[q] = *reinterpret_cast<const x8*>(kt + (kro ^ (64 * q)) + 16 * kb * ROWB);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        s[qb][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < QS; ++q) s[qb][kb] = mfma<F16>(kf[q], qf[qb][q], s[qb][kb]);
      }
    }
    if (some) {
      // key j0 + 8 grp + t, t a constant, of query j0 + 8 grp + top: seen when 0 <= top - t <= window or t <= top, t < sinks'
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int top = qw + 16 * qb + r16 - j0 - 8 * grp;
        if (j0 >= a.sinks) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = 32 * (kb >> 1) + 4 * (kb & 1) + e;
              s[qb][kb][e] = (unsigned)(top - t) <= (unsigned)a.window ? s[qb][kb][e] : -INFINITY;
            }
        } else {
          const int few = min(top, a.sinks - 1 - j0 - 8 * grp);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = 32 * (kb >> 1) + 4 * (kb & 1) + e;
              s[qb][kb][e] = ((unsigned)(top - t) <= (unsigned)a.window) | (t <= few) ? s[qb][kb][e] : -INFINITY;
            }
        }
      }
    }
    x8 pf[QB][KC];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float mx = max_lanes4(max_scores(s[qb]));
      const bool move = mx * g.c2 > mref[qb] * g.c2 + LAZY;
      if (__any(move)) {
        const float mnew = move ? mx : mref[qb];
        const float alpha = move ? __builtin_amdgcn_exp2f((mref[qb] - mnew) * g.c2) : 1.f;
        mref[qb] = mnew;
        osum[qb] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[qb][d] *= alpha;
      }
      const float mc = mref[qb] == -INFINITY ? 0.f : mref[qb] * g.c2;
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int x = 0; x < 8; ++x)
          pf[qb][c][x] = (T)__builtin_amdgcn_exp2f(fmaf(s[qb][2 * c + (x >> 2)][x & 3], g.c2, -mc));
    }
    auto vfrag = [&](int c, int d) {
      const char* p = vt + (vro ^ (32 * d)) + 32 * c * ROWB;
      const x4 l = __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)p));
      const x4 h = __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p + 4 * ROWB)));
      return x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
    };
    if constexpr (!CAREFUL) {
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const x8 vf = vfrag(c, d);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) o[qb][d] = mfma<F16>(vf, pf[qb][c], o[qb][d]);
        }
    } else {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll 1
        for (int row = 0; row < 16; ++row) {
          const int top = qw + 16 * qb + row - j0 - 8 * grp, few = min(top, a.sinks - 1 - j0 - 8 * grp);
#pragma unroll 1
          for (int c = 0; c < KC; ++c) {
            u32x4 keep;  // a mask of the fragment's 8 keys 32 c + 8 grp ..
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int t = 32 * c + 2 * x;
              const bool one = ((unsigned)(top - t) <= (unsigned)a.window) | (t <= few);
              const bool two = ((unsigned)(top - t - 1) <= (unsigned)a.window) | (t + 1 <= few);
              keep[x] = (one ? 0xffffu : 0u) | (two ? 0xffff0000u : 0u);
            }
            const x8 pc = c == 0 ? pf[qb][0] : pf[qb][1];
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              f32x4 add = {0.f, 0.f, 0.f, 0.f};
              add = mfma<F16>(__builtin_bit_cast(x8, __builtin_bit_cast(u32x4, vfrag(c, d)) & keep), pc, add);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[qb][d][e] = r16 == row ? o[qb][d][e] + add[e] : o[qb][d][e];
            }
          }
        }
    }
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) osum[qb] = mfma<F16>(ones, pf[qb][c], osum[qb]);
  };
  // Each group of waves takes every KS-th block: its next one lands in its other slot while one is computed; then it has landed for
  // this wave, and the barrier makes every wave's part of it visible and retires the slot. (The loads are the only vector memory
  // operations in flight.)
  auto step = [&](int i, auto bufc, auto carefulc) {
    if (i + part + KS < blocks) issue(i + part + KS, decltype(bufc)::value ^ 1);
    if (KS == 1 || i + part < blocks) block(i + part, bufc, carefulc);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  auto pass = [&](auto carefulc) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      mref[qb] = -INFINITY;
      osum[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DT; ++d) o[qb][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (part < blocks) issue(part, 0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for (int i = 0; i < blocks; i += 2 * KS) {
      step(i, std::integral_constant<int, 0>{}, carefulc);
      if (i + KS < blocks) step(i + KS, std::integral_constant<int, 1>{}, carefulc);
    }
  };
  pass(std::false_type{});
  // An output that is not finite under a finite sum: infinities or NaN among the values, which in blocks seen in part reach rows that
  // do not see them (0 x NaN is not 0). All again, row by row.
  bool odd = false;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= !(fabsf(o[qb][d][e]) < INFINITY);
  if (__syncthreads_or(odd)) pass(std::true_type{});

  if constexpr (KS == 2) {
    // the second group's sums join the first's through LDS (its K slots: 16 DIM floats a wave)
    static_assert(QB == 1);
    f32x4* to = reinterpret_cast<f32x4*>(sk[1][0]) + wave * DT * 64 + lane;
    float2* ml = reinterpret_cast<float2*>(sv[1][0]) + wave * 64 + lane;
    if (part) {
#pragma unroll
      for (int d = 0; d < DT; ++d) to[64 * d] = o[0][d];
      *ml = make_float2(mref[0], osum[0][0]);
    }
    __syncthreads();
    if (part) return;
    // (a row may see none of one group's blocks, which then has no maximum and sums of zero; its own key is in the other's)
    const float m1 = ml->x, l1 = ml->y, m = fmaxf(mref[0], m1);
    const float a0 = mref[0] == m ? 1.f : __builtin_amdgcn_exp2f((mref[0] - m) * g.c2);
    const float a1 = m1 == m ? 1.f : __builtin_amdgcn_exp2f((m1 - m) * g.c2);
    osum[0][0] = osum[0][0] * a0 + l1 * a1;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[0][d] = o[0][d] * a0 + to[64 * d] * a1;
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int q = qw + 16 * qb + r16;
    if (q > last) continue;
    const float inv = 1.f / osum[qb][0];
    T* y = static_cast<T*>(a.y) + ((long)(w.s0 + q) * a.heads + w.h) * DIM + 4 * grp;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<x4*>(y + 16 * d) =
          x4{(T)(o[qb][d][0] * inv), (T)(o[qb][d][1] * inv), (T)(o[qb][d][2] * inv), (T)(o[qb][d][3] * inv)};
  }
}

}  // namespace

int sink_attention_launch(const SinkArgs& a, hipStream_t stream) {
  if (bad_heads(a.q) || bad_heads(a.k) || bad_heads(a.v) || !a.y || ((uintptr_t)a.y & 15) ||
      (a.type != ROWS_BF16 && a.type != ROWS_F16) || (a.dim != 64 && a.dim != 128) || a.heads <= 0 || a.heads > 1024 ||
      a.kv_heads <= 0 || a.heads % a.kv_heads || a.window < 0 || a.sinks < 0 || !(a.scale >= 0.f) || a.scale > 3.4e38f ||
      a.n <= 0 || a.rows <= 0 || (!a.starts && (a.T <= 0 || (long)a.n * a.T != a.rows)))
    return NOISE_EINVAL;
  // (byte strides of 24 bits: offsets inside a 64-key block are 24-bit products)
  if (a.k.ld >= (1 << 23) || a.v.ld >= (1 << 23)) return NOISE_ENOTSUP;
  // tiles' numbers: the full ones and one more for every sequence; the GPU finds which are tiles
  auto groups = [&](int bq) {
    const long tiles = a.starts ? a.rows / bq + a.n : (long)a.n * ((a.T + bq - 1) / bq);
    return a.heads % 8 == 0 ? tiles * a.heads : (tiles * a.heads + 7) / 8 * 8;
  };
  // Tiles of 64 queries where those of 128 leave the GPU empty for much of the time, and two groups of waves where those do too (8
  // heads, one sequence unless said otherwise; 128 queries / 64 / 64 in two groups. dim 64: 1000 tokens 20 / 14.3 / 12.0 us, 2048 34 /
  // 24.4 / 20.0, 6000 95 / 74 / 67, 8192 132 / 107 / 109, 4 of 2048 in windows of 1024 30.5 / 27.8 / 32.9, 2 of 6000 43.5 / 44.3 / 52;
  // dim 128: 2048 46 / 36 / 28, 4096 88 / 73 / 61, 6000 135 / 110 / 129, 8192 187 / 192, 4 of 2048 in windows 45.5 / 54).
  const long tiles = groups(128), cus = num_cus();
  const bool narrow = tiles <= (a.dim == 64 ? 3 : 2) * cus, split = 4 * tiles <= (a.dim == 64 ? 6 : 5) * cus;
  const long items = groups(narrow ? 64 : 128);
  Args g{a, 0.f, (int)items, a.fill && a.starts ? 32 : 0};
  if (items + g.fills > 0x7fffffffL) return NOISE_ENOTSUP;
  // (a scale of 0 is the smallest normal number: every seen key weighs the same, and a masked score stays -infinity)
  const float c2 = a.scale * 1.4426950408889634f;
  g.c2 = c2 > 1.17549435e-38f ? c2 : 1.17549435e-38f;
  auto launch = [&](auto dim, auto f16_, auto qb, auto ks) {
    hipLaunchKernelGGL((sink_kernel<decltype(dim)::value, decltype(f16_)::value, decltype(qb)::value, decltype(ks)::value>),
                       dim3((unsigned)(items + g.fills)), dim3(NTH * decltype(ks)::value), 0, stream, g);
  };
  const std::integral_constant<int, 1> one{};
  const std::integral_constant<int, 2> two{};
  auto with = [&](auto dim, auto f16_) {
    split ? launch(dim, f16_, one, two) : narrow ? launch(dim, f16_, one, one) : launch(dim, f16_, two, one);
  };
  const std::integral_constant<int, 64> d64{};
  const std::integral_constant<int, 128> d128{};
  if (a.type == ROWS_F16)
    a.dim == 64 ? with(d64, std::true_type{}) : with(d128, std::true_type{});
  else
    a.dim == 64 ? with(d64, std::false_type{}) : with(d128, std::false_type{});
  NOISE_CHECK_LAUNCH();
  return NOISE_OK;
}

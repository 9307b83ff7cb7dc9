// Internal interface of the serving kernels (not part of the C ABI): the microscaled key / value cache and the attention of
// prompts and of cached sequences.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

// Codes of a cache: e2m1 (two to a byte, the even channel in the low half) or e4m3. Values of the C ABI's format.
enum : int { CACHE_FP4 = 0, CACHE_FP8 = 1 };
// Types of rows handed in or out (values of the C ABI's type).
enum : int { ROWS_BF16 = 0, ROWS_F16 = 1, ROWS_F32 = 2 };

// keys / values [pages, kv_heads, page, dim / 2 or dim] codes; scales [pages, kv_heads, page, dim / 32] bytes: code * 2^(byte -
// 127), 255 = NaN.
struct Cache {
  uint8_t *k, *ks, *v, *vs;
  long pages;
  int page_shift, kv_heads, dim, format;
};

// `rows` packed rows of n sequences: sequence b owns rows starts[b] .. starts[b + 1] (starts null: row b alone), its m rows at
// the positions lengths[b] - m .. lengths[b] - 1; position p lies in page table[b * table_ld + p / page].
struct Sequences {
  const int* table;
  long table_ld;
  int table_pages;
  const int *lengths, *starts;
  int n, rows;
};

// 16- or 32-bit rows: head h of row r at p + r * ld + h * hs (elements).
struct Heads {
  const void* p;
  long ld, hs;
};

// Whether the description of a cache and its sequences is refused.
inline bool bad_heads(const Heads& h) {
  return !h.p || ((uintptr_t)h.p & 15) || h.ld < 0 || h.hs < 0 || h.ld % 8 || h.hs % 8;
}
bool bad_cache(const Cache& c, const Sequences& s);
int cache_write_launch(const Cache& c, const Sequences& s, const Heads& k, const Heads& v, int type, hipStream_t stream);
int cache_read_launch(const Cache& c, const Sequences& s, void* k, void* v, int type, hipStream_t stream);

struct AttendArgs {
  Heads q;
  int type, heads, window, sinks, fill;  // fill: rows of no sequence are set to zero (left as they were otherwise)
  float scale;
  void* y;  // [rows, heads, dim] of q's type
};
int cache_attend_launch(const Cache& c, const Sequences& s, const AttendArgs& a, void* ws, size_t ws_bytes, hipStream_t stream);
int cache_attend_workspace(const Cache& c, const Sequences& s, const AttendArgs& a, size_t* bytes);

// Attention of whole sequences: rows packed by starts (null: n sequences of T rows each).
struct SinkArgs {
  Heads q, k, v;
  const int* starts;
  int n, rows, T, heads, kv_heads, dim;
  int type, window, sinks, fill;
  float scale;
  void* y;
};
int sink_attention_launch(const SinkArgs& a, hipStream_t stream);

// ---------------------------------------------------------------- device helpers

// The largest b in [0, n] with in(b), where in(b) holds for no b after one for which it does not (in(0) is not asked); found by a
// wave 64 entries at a time (one round up to 64, two up to 4096). Called by whole waves.
template <class F>
__device__ __forceinline__ int last_with(int n, F in) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;  // the answer lies in [lo, hi]
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + (lane + 1) * step;
    const unsigned long long m = __ballot(at <= hi && in(at));
    const int k = m == ~0ull ? 64 : __builtin_ctzll(~m);
    const int nlo = lo + k * step;
    hi = max(nlo, min(hi, nlo + step - 1));
    lo = nlo;
  }
  const int at = lo + lane + 1;
  const unsigned long long m = __ballot(at <= hi && in(at));
  return lo + __builtin_popcountll(m);
}

// The sequence that owns row i: the number of entries of starts[1 .. n] that are <= i. Rows of no sequence give n.
__device__ __forceinline__ int find_sequence(const int* starts, int n, int i) {
  return last_with(n, [&](int b) { return starts[b] <= i; });
}

// Tiles of `per` units (a row is `mul` of them) that begin with every sequence are numbered with gaps, so that a sequence's first
// number follows from its start alone: rows mul / per + b, at least the tiles of all sequences in front (and of all, in front of
// sequence n: the numbers' limit).
__device__ __forceinline__ int first_tile(const Sequences& s, int b, int mul, int per) {
  return (int)((long)min(max(s.starts[b], 0), s.rows) * mul / per) + b;
}

constexpr int POSITIONS = 0x7fffff00;  // a position's limit: sums with a block's keys stay within an int

// The slot (page * page size + token) of a position, or -1 where the table names no page of the cache for it.
__device__ __forceinline__ long slot_of(const Cache& c, const Sequences& s, int b, long pos) {
  const long pg = pos >> c.page_shift;
  if (pos < 0 || pos >= POSITIONS || pg >= s.table_pages) return -1;
  const int id = s.table[b * s.table_ld + pg];
  if (id < 0 || id >= c.pages) return -1;
  return ((long)id << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}

// x of lane k in a scalar register (a lane shuffle's result counts as a lane's own, and so would all that follows from it)
__device__ __forceinline__ int uniform(int x, int k = 0) { return __builtin_amdgcn_readlane(x, k); }
__device__ __forceinline__ long uniform(long x, int k = 0) {
  return (long)((unsigned long long)(unsigned)uniform((int)(x >> 32), k) << 32 | (unsigned)uniform((int)x, k));
}

// The sum over a wave's lanes.
__device__ __forceinline__ int wave_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, DPP_QUAD_XOR1, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, DPP_QUAD_XOR2, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, DPP_ROW_HALF_MIRROR, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, DPP_ROW_MIRROR, 0xF, 0xF, false);
  return uniform(v) + uniform(v, 16) + uniform(v, 32) + uniform(v, 48);
}

// Zeroes the rows of no sequence, in front of the first one and behind the last: workgroup `part` of `parts` of nth threads.
__device__ __forceinline__ void fill_rows(const int* starts, int n, int rows, void* y, int width, int nth, int part, int parts) {
  const int lo = min(max(starts[0], 0), rows), hi = min(max(starts[n], lo), rows);
  const long units = width / 8, head = lo * units, all = head + (rows - hi) * units;
  for (long i = (long)part * nth + threadIdx.x; i < all; i += (long)parts * nth)
    static_cast<uint4*>(y)[i < head ? i : hi * units + i - head] = make_uint4(0, 0, 0, 0);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4_t;
constexpr float LAZY = 8.f;  // a running maximum moves only beyond 2^8 of headroom

// 16-byte chunk of V row R (16 dims' halves of 8): XOR-swizzled so that the rows of a transposing read (8 g + 4 h + t, four t of
// two lane groups g in a cycle of 32 lanes) cover the banks once.
template <int DIM>
__device__ __forceinline__ int vswz(int R) {
  return DIM == 64 ? 2 * (((R >> 1) & 1) | ((((R >> 3) ^ R) & 1) << 1)) : 2 * ((R & 3) | (((R >> 3) & 1) << 2));
}

// The largest of a lane's scores, 4 N of them: gfx950's three-operand maximum that passes a NaN on. (fmaxf first quiets each operand
// with an instruction of its own, as what left the matrix cores could be a signalling NaN for all the compiler knows; and inline
// assembly may not read it, since the compiler places the wait states that it needs in front of instructions it knows.)
template <int N>
__device__ __forceinline__ float max_scores(const f32x4 (&s)[N]) {
  float m = s[0][0];
#pragma unroll
  for (int x = 1; x < 4 * N; ++x) m = __builtin_elementwise_maximum(m, s[x / 4][x % 4]);
  return m;
}
// The same over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_lanes4(float x) {
  const f32pair a = rowpair16(x);
  const f32pair b = halves32(__builtin_elementwise_maximum(a.lo, a.hi));
  return __builtin_elementwise_maximum(b.lo, b.hi);
}

// Attention of a few new rows per sequence over the microscaled key / value cache (decoding, and drafted or prompt rows over what
// is cached): y = softmax(scale q K^T) V, a row at position s seeing key j when 0 <= j <= s and (s - j <= window or j < sinks).
//
// Bound: the visible tokens' bytes, read once per kv head (dim 64: 68 bytes a token in e2m1). The rows of one sequence and kv
// head, at most 16 (new tokens x query heads of the group), are the columns of one MFMA tile, so a group of heads costs what
// one head costs, and idle columns are free while memory is the bound. 48 sequences of up to 32768 tokens, 8 heads of 64 in e2m1, take
// 92 us (4.95 TB/s of what they see), 200000 tokens in e4m3 44 us (4.8 TB/s), a join 5 to 7 us more; 16 sequences of up to 16384,
// 32 heads over 4 of 128 in e2m1, 23 us (3.4 TB/s: start-up). A step of one short sequence takes 7 us, a few round trips to memory.
//
// A wave takes blocks of BK keys (64 of dim 64, 32 of dim 128) with its own running maximum and sum:
//   K codes go from global memory to registers (a lane holds a quarter of a key's channels, all of one scale group) and become
//   bf16 exactly, scale included, by the hardware's microscaling conversions; S^T = K Q^T on MFMA (A = keys, B = rows).
//   V codes become bf16 the same way and pass through the wave's LDS tile [key][channel], whose transposing reads give the A
//   operand of O^T += V^T P^T. The key of each K row is chosen so that the scores' layout is the B operand of that product.
//   The next block's codes are on their way meanwhile.
// fp16 queries and their probabilities enter as two bf16 terms (hi + lo: 16 significant bits, fp16 has 11); bf16 queries are
// exact and their probabilities are rounded once to bf16, the type of the output.
//
// Work is cut on the GPU from the sequences' lengths, which the host does not know. The rounds (a block for each wave) of all
// tiles, kv head by kv head, form one line, and each of the workgroups that fill the GPU once takes an equal stretch of it:
// every workgroup has the same to do whatever the lengths. A stretch may hold the end of one tile, whole tiles and
// the beginning of another; the waves join in LDS, and where a tile is spread over several workgroups their sums meet in a second
// kernel, in order (the same bits every time). Tables that name few keys, and very many sequences, go without it: a workgroup a tile.
#include <type_traits>

#include "common.h"
#include "serve.h"

namespace {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int RT = 16;         // rows of a tile

template <int DIM, int FMT>
struct Geo {
  static constexpr int BK = 4096 / DIM;                    // keys of a block
  static constexpr int GROUPS = DIM / 32;
  static constexpr int ROW = FMT == CACHE_FP4 ? DIM / 2 : DIM;  // code bytes of a token and head
  static constexpr int KT = BK / 16, KC = BK / 32, DT = DIM / 16, QS = DIM / 32;
  static constexpr int KW = ROW / 16;                      // 32-bit words of a lane's quarter of a key
  static constexpr int VW = FMT == CACHE_FP4 ? 4 : 8;      // 32-bit words of 32 channels
  static constexpr int VN = 2;                             // (key, group) pieces of V per lane and block
  static constexpr int TILE = BK * DIM * 2;                // bytes of a wave's V tile: 8 KiB
};

// 8 codes to bf16 under a scale, exactly (words 1 for e2m1, 2 for e4m3).
template <int FMT>
__device__ __forceinline__ u32x4 bf16_of(const unsigned* w, float scale) {
  u32x4 r;
  if constexpr (FMT == CACHE_FP4) {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 3));
  } else {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, true));
  }
  return r;
}

// One sequence's share of a call, as the kernels cut it.
struct Cut {
  int m, len, blocks, tiles;  // rows, tokens, key blocks of its longest tile, tiles of RT rows
  bool bad;                   // starts that decrease (the counts below would be of more rows than there are)
};
struct Plan {
  int group;        // query heads of a kv head
  int block_shift;  // log2 of a block's keys
  int cap;          // positions that a table names
  int groups;       // workgroups that share the line, or 0: a workgroup a tile (and a number without one)
  int waves;        // of a workgroup: the blocks of a round
};

__device__ __forceinline__ int first_key(int pos, int window) { return pos > window ? pos - window : 0; }

// The blocks of keys that rows at positions p0 .. p1 see, p1 >= 0: `sink` blocks from block 0, then from block `lo` on.
struct Range {
  int sink, lo, blocks;
};
__device__ __forceinline__ Range range_of(int p0, int p1, int window, int sinks, int shift) {
  const int first = first_key(max(p0, 0), window);
  const int lo = first >> shift;
  const int s = min(sinks, first);
  const int sink = min((s >> shift) + ((s & ((1 << shift) - 1)) != 0), lo);
  return Range{sink, lo, sink + (p1 >> shift) - lo + 1};
}

__device__ __forceinline__ Cut cut_of(const Sequences& s, const Plan& p, int window, int sinks, int b, int& s0) {
  Cut c{0, 0, 0, 0, false};
  s0 = 0;
  if (b >= s.n) return c;
  int s1;
  if (s.starts) {
    s0 = min(max(s.starts[b], 0), s.rows);
    s1 = min(max(s.starts[b + 1], 0), s.rows);
    c.bad = s1 < s0;
    if (c.bad) return c;
  } else {
    s0 = b;
    s1 = b + 1;
  }
  c.m = s1 - s0;
  c.len = max(s.lengths[b], 0);
  c.tiles = (c.m * p.group + RT - 1) / RT;
  // (positions past the table hold nothing: the rows there are NaN, and the others end in front of it)
  const int last = min(c.len, p.cap) - 1;
  if (c.m > 0 && last >= 0) {
    // a tile's rows are at most `span` tokens; its range is at most that of the last ones, and a block more by alignment
    const int span = min(c.m, (RT + p.group - 1) / p.group + 1);
    c.blocks = range_of(last + 1 - span, last, window, sinks, p.block_shift).blocks + (c.tiles > 1);
  }
  return c;
}

// The line: `units` rounds per kv head (a tile that sees no key counts as one), `share` of them to a workgroup.
struct Line {
  int units, share;
};
// A tile; on the line of its kv head `at` is its first round, `rounds` their number.
struct Work {
  int b, s0, m, len, tile, rounds, at;
  bool found;
};

// The cuts of up to 64 sequences in LDS, for the tiles after the first (every wave writes the same values).
struct Kept {
  int s0[64], m[64], len[64], blocks[64], tiles[64];
};

__device__ __forceinline__ int rounds_of(const Plan& p, const Cut& c) { return max((c.blocks + p.waves - 1) / p.waves, 1); }

// (the host keeps all rounds of a call below 2^31)
__device__ Line line_of(const Sequences& s, const Plan& p, int kv_heads, int window, int sinks, Kept& kept) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  bool bad = false;
  for (int b0 = 0; b0 < s.n; b0 += 64) {
    int s0;
    const Cut c = cut_of(s, p, window, sinks, b0 + lane, s0);
    total += c.tiles * rounds_of(p, c);
    bad |= c.bad;
    if (s.n <= 64) {
      kept.s0[lane] = s0;
      kept.m[lane] = c.m;
      kept.len[lane] = c.len;
      kept.blocks[lane] = c.blocks;
      kept.tiles[lane] = c.tiles;
    }
  }
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64);
  total = __any(bad) ? 0 : uniform(total);
  return Line{total, (total * kv_heads + p.groups - 1) / p.groups};
}

// The tile that holds round `unit` of a kv head's line (row < 0), or the one of row `row` and head `head` of its group. Whole waves.
__device__ Work find_work(const Sequences& s, const Plan& p, int window, int sinks, int unit, int row, int head, const Kept& kept) {
  const int lane = threadIdx.x & 63;
  Work w{};
  int base = 0;
  for (int b0 = 0; b0 < s.n; b0 += 64) {
    int s0;
    Cut c;
    if (s.n <= 64) {
      s0 = kept.s0[lane];
      c = Cut{kept.m[lane], kept.len[lane], kept.blocks[lane], kept.tiles[lane], false};
    } else {
      c = cut_of(s, p, window, sinks, b0 + lane, s0);
      if (__any(c.bad)) return w;
    }
    const int each = rounds_of(p, c);
    const int mine = c.tiles * each;
    int upto = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(upto, o, 64);
      if (lane >= o) upto += t;
    }
    const bool hit = row >= 0 ? row >= s0 && row < s0 + c.m : unit < base + upto;
    const unsigned long long hits = __ballot(hit);
    if (hits) {
      const int k = __builtin_ctzll(hits);
      w.found = true;
      w.b = b0 + k;
      w.s0 = uniform(s0, k);
      w.m = uniform(c.m, k);
      w.len = uniform(c.len, k);
      w.rounds = uniform(each, k);
      const int first = base + uniform(upto - mine, k);
      w.tile = row >= 0 ? ((row - w.s0) * p.group + head) / RT : (unit - first) / w.rounds;
      w.at = first + w.tile * w.rounds;
      return w;
    }
    base += uniform(upto, 63);
  }
  return w;
}

// Tile `i` of a kv head without a line: of up to 64 sequences without gaps (the workgroups with nothing to do come last: among the
// others, they would leave CUs idle beside CUs with two tiles: 5 rows of each of 32 sequences 24.8 us, so 15.1), of more by
// first_tile's numbers. Whole waves.
__device__ Work tile_of(const Sequences& s, const Plan& p, int i) {
  const int lane = threadIdx.x & 63, each = (p.group + RT - 1) / RT;
  Work w{};
  if (!s.starts) {
    w.b = i / each;
    w.tile = i % each;
  } else if (s.n <= 64) {
    const int lo = lane < s.n ? min(max(s.starts[lane], 0), s.rows) : 0, hi = lane < s.n ? min(max(s.starts[lane + 1], 0), s.rows) : 0;
    const int tiles = (max(hi - lo, 0) * p.group + RT - 1) / RT;
    int upto = tiles;
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(upto, o, 64);
      if (lane >= o) upto += t;
    }
    const unsigned long long hits = __ballot(i < upto);
    if (!hits || __any(hi < lo)) return w;
    w.b = __builtin_ctzll(hits);
    w.tile = i - uniform(upto - tiles, w.b);
  } else {
    w.b = last_with(s.n - 1, [&](int b) { return first_tile(s, b, p.group, RT) <= i; });
    w.tile = i - first_tile(s, w.b, p.group, RT);
  }
  if (w.b >= s.n) return w;
  w.s0 = s.starts ? min(max(s.starts[w.b], 0), s.rows) : w.b;
  w.m = s.starts ? min(max(s.starts[w.b + 1], 0), s.rows) - w.s0 : 1;
  w.len = max(s.lengths[w.b], 0);
  w.found = w.tile >= 0 && w.m > 0 && w.tile < (w.m * p.group + RT - 1) / RT;
  return w;
}

struct Args {
  Cache c;
  Sequences s;
  AttendArgs a;
  Plan p;
  float c2;         // scale in base-2 units
  int items, fills;  // workgroups of tiles or stretches, workgroups that zero rows
  float* part;      // [groups, 2, RT, dim] sums of a stretch's first and of its last tile, where others hold more of them,
  float2* ml;       // [groups, 2, RT] under these maxima, with these sums of probabilities
};

// Workgroups on a CU. e4m3: two, whose blocks on their way are as many bytes as e2m1's three (16 sequences of 16384 tokens, fp16
// queries, dim 64: 54 us, with three 59; dim 128 54 and 60); e2m1: three (48 sequences of up to 32768 tokens 93 us; two 101, four
// 95), or two where a third's registers would spill: a reload waits for all loads on their way.
constexpr int resident(int dim, int format, bool f16, bool wide, bool many) {
  return format == CACHE_FP8 || (many && (!wide || (f16 && dim == 128))) ? 2 : 3;
}

// WIDE: pages hold whole blocks. F16: fp16 queries (two bf16 terms). MANY: rows of a tile may lie at different positions (with one row
// a sequence, whatever one row sees all see, and what none sees is zero before it is multiplied). NW waves.
template <int DIM, int FMT, bool F16, bool WIDE, bool MANY, int NW>
__global__ void __launch_bounds__(64 * NW, NW == 8 ? 2 : resident(DIM, FMT, F16, WIDE, MANY)) attend_kernel(Args g) {
  using G = Geo<DIM, FMT>;
  constexpr int BK = G::BK, KT = G::KT, KC = G::KC, DT = G::DT, QS = G::QS, KW = G::KW, VW = G::VW, VN = G::VN;
  constexpr int SHIFT = DIM == 64 ? 6 : 5;
  __shared__ __attribute__((aligned(1024))) char sv[NW * G::TILE];
  __shared__ float2 sml[NW][RT];
  __shared__ Kept kept;
  const Cache& c = g.c;
  const Sequences& s = g.s;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if ((int)blockIdx.x >= g.items) {
    fill_rows(s.starts, s.n, s.rows, g.a.y, g.a.heads * DIM, 64 * NW, blockIdx.x - g.items, g.fills);
    return;
  }
  char* vt = sv + wave * G::TILE;
  const int page_mask = (1 << c.page_shift) - 1;
  Line line{};
  int unit = 0, end = 0;
  if (g.p.groups) {
    line = line_of(s, g.p, c.kv_heads, g.a.window, g.a.sinks, kept);
    unit = blockIdx.x * line.share;
    end = min(unit + line.share, line.units * c.kv_heads);
    if (unit >= end) return;
  }
#pragma unroll 1
  for (bool more = true; more;) {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // (opaque: what a lane derives from it would be kept in registers over the loop)
  const int lane = tid & 63, r16 = lane & 15, grp = lane >> 4;
  const int kh = g.p.groups ? unit / line.units : blockIdx.x % c.kv_heads;
  const Work w = g.p.groups ? find_work(s, g.p, g.a.window, g.a.sinks, unit - kh * line.units, -1, 0, kept)
                            : tile_of(s, g.p, blockIdx.x / c.kv_heads);
  if (!w.found) return;
  const int G_ = g.p.group, f0 = w.tile * RT, fn = min(RT, w.m * G_ - f0), back = w.len - w.m;
  const int p0 = back + f0 / G_, p1 = back + (f0 + fn - 1) / G_;  // positions of the tile's first and last row
  const int pmin = max(p0, -1), pmax = max(min(p1, g.p.cap - 1), -1);
  // this lane's row
  const int f = f0 + r16, tok = f / G_;
  const bool live = r16 < fn;
  const int pos = live ? max(back + tok, -1) : -1;

  // Q fragments (B operand): row lane % 16, channels (lane / 16) DIM / 4 + 8 i ..
  bf16x8 qh[QS], ql[F16 ? QS : 1];
#pragma unroll
  for (int i = 0; i < QS; ++i) {
    u32x4 raw = {0, 0, 0, 0};
    if (live) {
      const long at = (long)(w.s0 + tok) * g.a.q.ld + (long)(kh * G_ + f % G_) * g.a.q.hs + grp * (DIM / 4) + 8 * i;
      raw = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(g.a.q.p) + at);
    }
    if constexpr (F16) {
      const f16x8 x = __builtin_bit_cast(f16x8, raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bf16 hi = to_bf16((float)x[e]);
        qh[i][e] = hi;
        ql[i][e] = to_bf16((float)x[e] - (float)hi);
      }
    } else {
      qh[i] = __builtin_bit_cast(bf16x8, raw);
    }
  }

  float mref = -INFINITY, lsum = 0.f;
  f32x4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  const Range rg = pmax >= 0 && p0 < g.p.cap ? range_of(pmin, pmax, g.a.window, g.a.sinks, SHIFT) : Range{0, 0, 0};
  // this workgroup's blocks i0 .. i1 of the tile; `alone` when no other has any
  int i0 = 0, i1 = rg.blocks, slot = 0;
  bool alone = true;
  if (g.p.groups) {
    const int from = kh * line.units + w.at, stop = min(end, from + w.rounds);
    alone = unit == from && stop == from + w.rounds;
    slot = 2 * blockIdx.x + (unit != (int)blockIdx.x * line.share);
    i0 = (unit - from) * NW;
    i1 = min((stop - from) * NW, rg.blocks);
    unit = stop;
  }
  more = g.p.groups && unit < end;
  const int* table = s.table + (long)w.b * s.table_ld;

  // row lane % 16 of K tile kb is key 32 (kb / 2) + 4 (kb % 2) + krow0 of the block; piece n of V is 32 channels, vgr, of key
  // n * 64 / GROUPS + vrow0
  const int krow0 = 8 * (r16 >> 2) + (r16 & 3), vrow0 = lane / G::GROUPS, vgr = lane % G::GROUPS;
  struct Raw {
    unsigned k[KT][KW], v[VN][VW];
    unsigned ks[KT], vs[VN];
  };
  auto block_key = [&](int i) { return (i < rg.sink ? i : rg.lo + i - rg.sink) << SHIFT; };
  // page of key j (clamped to the last visible one), -1 for a bad one
  auto page_of = [&](int j) {
    const int id = table[min(j, pmax) >> c.page_shift];
    return (unsigned)id < (unsigned)c.pages ? id : -1;
  };
  // (page ids of one block: the wave's one page, or a lane's own)
  struct Ids {
    int k[WIDE ? 1 : KC], v[WIDE ? 1 : VN];
  };
  auto ids_of = [&](int i) {
    Ids d;
    const int j0 = block_key(i);
    if constexpr (WIDE) {
      d.k[0] = __builtin_amdgcn_readfirstlane(page_of(j0));
    } else {
#pragma unroll
      for (int h = 0; h < KC; ++h) d.k[h] = page_of(j0 + 32 * h + krow0);
#pragma unroll
      for (int n = 0; n < VN; ++n) d.v[n] = page_of(j0 + n * (64 / G::GROUPS) + vrow0);
    }
    return d;
  };
  // byte offsets of this lane's codes and scales from a block's first row of one page (WIDE): tile kb and piece n add constants
  // (kept opaque in the loop: hoisted sums of them with the cache's addresses would each hold a pair of registers)
  unsigned koff = krow0 * G::ROW + grp * (4 * KW), ksoff = krow0 * G::GROUPS + grp * G::GROUPS / 4;
  unsigned voff = vrow0 * G::ROW + vgr * (4 * VW), vsoff = vrow0 * G::GROUPS + vgr;
  auto load = [&](int i, const Ids& d, Raw& r) {
    const int j0 = block_key(i);
    if constexpr (WIDE) {
      asm volatile("" : "+v"(koff), "+v"(ksoff), "+v"(voff), "+v"(vsoff));
      const long row = (((long)max(d.k[0], 0) * c.kv_heads + kh) << c.page_shift) + (j0 & page_mask);
      const uint8_t *kp = c.k + row * G::ROW, *vp = c.v + row * G::ROW, *ksp = c.ks + row * G::GROUPS, *vsp = c.vs + row * G::GROUPS;
#pragma unroll
      for (int kb = 0; kb < KT; ++kb) {
        const int step = 32 * (kb >> 1) + 4 * (kb & 1);
#pragma unroll
        for (int x = 0; x < KW; ++x) r.k[kb][x] = reinterpret_cast<const unsigned*>(kp + step * G::ROW + koff)[x];
        r.ks[kb] = (ksp + step * G::GROUPS)[ksoff];
      }
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        constexpr int STEP = 64 / G::GROUPS;
#pragma unroll
        for (int x = 0; x < VW; ++x) r.v[n][x] = reinterpret_cast<const unsigned*>(vp + n * STEP * G::ROW + voff)[x];
        r.vs[n] = (vsp + n * STEP * G::GROUPS)[vsoff];
      }
      if (d.k[0] < 0) {
#pragma unroll
        for (int kb = 0; kb < KT; ++kb) r.ks[kb] = 255u;
#pragma unroll
        for (int n = 0; n < VN; ++n) r.vs[n] = 255u;
      }
    } else {
      auto row_of = [&](int id, int j) {
        return (((long)max(id, 0) * c.kv_heads + kh) << c.page_shift) + (min(j, pmax) & page_mask);
      };
#pragma unroll
      for (int kb = 0; kb < KT; ++kb) {
        const int id = d.k[kb >> 1];
        const long row = row_of(id, j0 + 32 * (kb >> 1) + 4 * (kb & 1) + krow0);
        const unsigned* src = reinterpret_cast<const unsigned*>(c.k + row * G::ROW) + grp * KW;
#pragma unroll
        for (int x = 0; x < KW; ++x) r.k[kb][x] = src[x];
        const unsigned e = c.ks[row * G::GROUPS + grp * G::GROUPS / 4];
        r.ks[kb] = id < 0 ? 255u : e;
      }
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        const int id = d.v[n];
        const long row = row_of(id, j0 + n * (64 / G::GROUPS) + vrow0);
        const unsigned* src = reinterpret_cast<const unsigned*>(c.v + row * G::ROW) + vgr * VW;
#pragma unroll
        for (int x = 0; x < VW; ++x) r.v[n][x] = src[x];
        const unsigned e = c.vs[row * G::GROUPS + vgr];
        r.vs[n] = id < 0 ? 255u : e;
      }
    }
  };
  // this lane's places in the V tile: pieces are written at chunks 4 vgr .. + 3 of key vrow0 (+ 64 / GROUPS a piece), read at chunk
  // pairs d of key 8 grp + t (+ 32 h + 4 x); the swizzle depends on none of what is added
  const int vwr = vrow0 * (2 * DIM) + 16 * ((4 * vgr) ^ vswz<DIM>(vrow0));
  const int vrt = (lane & 15) >> 2, vra = lane & 3, vrr = 8 * grp + vrt;
  const int vrd = vrr * (2 * DIM) + 16 * ((vra >> 1) ^ vswz<DIM>(vrr)) + 8 * (vra & 1);
  // Of block i: the scores, from its codes (V's go to the tile); then, while the next block's codes arrive, softmax and P V.
  f32x4 sc[KT];
  bool odd;  // a non-finite value in a block that some rows see only in part
  auto scores = [&](int i, Raw& r) {
    const int j0 = block_key(i);
    // blocks that every row sees whole need no mask
    const bool whole = j0 + BK - 1 <= pmin && (j0 + BK <= g.a.sinks || pmax - j0 <= g.a.window);
    odd = false;
#pragma unroll
    for (int n = 0; n < VN; ++n) {
      const int key = n * (64 / G::GROUPS) + vrow0;
      if (!whole) {
        // a value that no row sees is zero, whatever the slot holds
        const int j = j0 + key;
        if ((j > pmax) | ((j < pmin - g.a.window) & (j >= g.a.sinks))) {
#pragma unroll
          for (int x = 0; x < VW; ++x) r.v[n][x] = 0;
          r.vs[n] = 127;
        }
      }
      const float vs = __uint_as_float(r.vs[n] << 23);
      char* dst = vt + n * (64 / G::GROUPS) * (2 * DIM);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const u32x4 val = bf16_of<FMT>(&r.v[n][x * (VW / 4)], vs);
        *reinterpret_cast<u32x4*>(dst + ((vwr ^ (32 * (x >> 1))) + 16 * (x & 1))) = val;
        if (MANY && !whole)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            odd |= ((val[e] & 0x7f80u) == 0x7f80u) | ((val[e] & 0x7f800000u) == 0x7f800000u);
      }
    }
    // S^T = K Q^T
#pragma unroll
    for (int kb = 0; kb < KT; ++kb) {
      const float ks = __uint_as_float(r.ks[kb] << 23);
      sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < QS; ++q) {
        const bf16x8 kf = __builtin_bit_cast(bf16x8, bf16_of<FMT>(&r.k[kb][q * (KW / QS)], ks));
        sc[kb] = mfma16x16x32(kf, qh[q], sc[kb]);
        if constexpr (F16) sc[kb] = mfma16x16x32(kf, ql[q], sc[kb]);
      }
    }
    if (!whole) {
#pragma unroll
      for (int kb = 0; kb < KT; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 32 * (kb >> 1) + 8 * grp + 4 * (kb & 1) + e;
          const bool see = (j <= pos) & ((pos - j <= g.a.window) | (j < g.a.sinks));
          sc[kb][e] = see ? sc[kb][e] : -INFINITY;
        }
    }
  };
  auto values = [&](int i) {
    const int j0 = block_key(i);
    // the running maximum (lazy) of row lane % 16
    const float mx = max_lanes4(max_scores(sc));
    const bool move = mx * g.c2 > mref * g.c2 + LAZY;
    if (__any(move)) {
      const float mnew = move ? mx : mref;
      const float alpha = move ? __builtin_amdgcn_exp2f((mref - mnew) * g.c2) : 1.f;
      mref = mnew;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
    const float mc = mref == -INFINITY ? 0.f : mref * g.c2;
    bf16x8 ph[KC], pl[F16 ? KC : 1];
#pragma unroll
    for (int h = 0; h < KC; ++h)
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float p = __builtin_amdgcn_exp2f(fmaf(sc[2 * h + (x >> 2)][x & 3], g.c2, -mc));
        lsum += p;
        const bf16 hi = to_bf16(p);
        ph[h][x] = hi;
        if constexpr (F16) pl[h][x] = to_bf16(p - (float)hi);
      }
    // O^T += V^T P^T
    auto vfrag = [&](int h, int d) {
      s16x4 part[2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        part[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4_t*)(vt + (vrd ^ (32 * d)) + (32 * h + 4 * x) * (2 * DIM)));
      const bf16x4 lo = __builtin_bit_cast(bf16x4, part[0]), hi = __builtin_bit_cast(bf16x4, part[1]);
      return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    if (!MANY || !__any(odd)) {
#pragma unroll
      for (int h = 0; h < KC; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const bf16x8 vf = vfrag(h, d);
          o[d] = mfma16x16x32(vf, ph[h], o[d]);
          if constexpr (F16) o[d] = mfma16x16x32(vf, pl[h], o[d]);
        }
    } else {
      // infinities or NaN among the values: row by row, with what the row does not see taken out (0 x NaN would not be 0)
#pragma unroll 1
      for (int row = 0; row < fn; ++row) {
        const int rp = __builtin_amdgcn_readlane(pos, row);
        int k0 = j0 + 8 * grp;
        asm volatile("" : "+v"(k0));
        u32x4 keep[KC];  // a mask of the 8 keys of a fragment
#pragma unroll
        for (int h = 0; h < KC; ++h)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            unsigned m[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int j = k0 + 32 * h + 2 * x + y;
              m[y] = (j <= rp) & ((rp - j <= g.a.window) | (j < g.a.sinks)) ? 0xffffu : 0u;
            }
            keep[h][x] = m[0] | m[1] << 16;
          }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4 add = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < KC; ++h) {
            const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, vfrag(h, d)) & keep[h]);
            add = mfma16x16x32(vf, ph[h], add);
            if constexpr (F16) add = mfma16x16x32(vf, pl[h], add);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] = r16 == row ? o[d][e] + add[e] : o[d][e];
        }
      }
    }
  };

  // block i + NW's codes are loaded while block i's values are multiplied, its page ids one block earlier still
  int i = i0 + wave;
  if (i < i1) {
    Raw raw;
    load(i, ids_of(i), raw);
    Ids ids = ids_of(min(i + NW, i1 - 1));
    for (; i < i1; i += NW) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the tile's last reads stay in front of its next writes)
      scores(i, raw);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (i + NW < i1) {
        load(i + NW, ids, raw);
        ids = ids_of(min(i + 2 * NW, i1 - 1));
      }
      values(i);
    }
  }

  // ---- the waves' sums meet: [wave][row][dim] in the V tiles
  lsum = sum_rows4(lsum);
  if (grp == 0) sml[wave][r16] = make_float2(mref, lsum);
  {
    float* dst = reinterpret_cast<float*>(vt) + r16 * DIM + 4 * grp;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<float4*>(dst + 16 * d) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
  }
  __syncthreads();
  for (int e = 4 * tid; e < fn * DIM; e += 4 * 64 * NW) {
    const int row = e / DIM, d = e % DIM;
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, sml[x][row].x);
    float L = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float2 ml = sml[x][row];
      const float wt = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - M) * g.c2);
      const float4 v = *reinterpret_cast<const float4*>(sv + x * G::TILE + 4 * e);
      L = fmaf(wt, ml.y, L);
      sum[0] = fmaf(wt, v.x, sum[0]), sum[1] = fmaf(wt, v.y, sum[1]);
      sum[2] = fmaf(wt, v.z, sum[2]), sum[3] = fmaf(wt, v.w, sum[3]);
    }
    if (!alone) {
      *reinterpret_cast<f32x4*>(g.part + ((long)slot * RT + row) * DIM + d) = sum;
      if (d == 0) g.ml[(long)slot * RT + row] = make_float2(M, L);
      continue;
    }
    const int ff = f0 + row;
    const float inv = back + ff / G_ >= g.p.cap ? __uint_as_float(0x7fc00000u) : L == 0.f ? 0.f : 1.f / L;
    const long at = ((long)(w.s0 + ff / G_) * g.a.heads + kh * G_ + ff % G_) * DIM + d;
    uint16_t* dst = static_cast<uint16_t*>(g.a.y) + at;
    union {
      f16 h[4];
      bf16 b[4];
      uint2 u;
    } out;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if constexpr (F16)
        out.h[x] = (f16)(sum[x] * inv);
      else
        out.b[x] = to_bf16(sum[x] * inv);
    *reinterpret_cast<uint2*>(dst) = out.u;
  }
  if (more) __syncthreads();  // (the tiles are read before the next stretch writes them)
  }
}

// y of the rows whose tile several workgroups share: one workgroup a row and head, its waves taking the others' sums in turn.
template <int DIM, bool F16, int NW>
__global__ void __launch_bounds__(64 * NW) join_kernel(Args g) {
  constexpr int PER = DIM / 64;
  __shared__ float so[NW][DIM], sl[NW];
  __shared__ Kept kept;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x / g.a.heads, h = blockIdx.x % g.a.heads, kh = h / g.p.group;
  const Line line = line_of(g.s, g.p, g.c.kv_heads, g.a.window, g.a.sinks, kept);
  const Work w = find_work(g.s, g.p, g.a.window, g.a.sinks, 0, row, h % g.p.group, kept);
  if (!w.found || !line.units) return;
  const int from = kh * line.units + w.at, first = from / line.share, last = (from + w.rounds - 1) / line.share;
  if (first == last) return;
  const int n = last - first + 1, r = ((row - w.s0) * g.p.group + h % g.p.group) % RT;
  // the tile is the last of its first workgroup's stretch (its only one, if it begins there), and the first of the others'
  auto at = [&](int x) { return (2l * (first + x) + (x == 0 && from != first * line.share)) * RT + r; };
  float M = -INFINITY;
  for (int x = lane; x < n; x += 64) M = fmaxf(M, g.ml[at(x)].x);
  for (int q = 32; q; q >>= 1) M = fmaxf(M, __shfl_xor(M, q, 64));
  float L = 0.f, o[PER] = {};
#pragma unroll 8
  for (int x = wave; x < n; x += NW) {
    const float2 ml = g.ml[at(x)];
    const float wt = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - M) * g.c2);
    L = fmaf(wt, ml.y, L);
#pragma unroll
    for (int d = 0; d < PER; ++d) o[d] = fmaf(wt, g.part[at(x) * DIM + lane + 64 * d], o[d]);
  }
#pragma unroll
  for (int d = 0; d < PER; ++d) so[wave][lane + 64 * d] = o[d];
  if (lane == 0) sl[wave] = L;
  __syncthreads();
  if (threadIdx.x < DIM) {
    const int d = threadIdx.x;
    float l = 0.f, v = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) l += sl[x], v += so[x][d];
    const bool past = w.len - w.m + (row - w.s0) >= g.p.cap;
    const float y = past ? __uint_as_float(0x7fc00000u) : l == 0.f ? 0.f : v / l;
    const long dst = (long)blockIdx.x * DIM + d;
    if constexpr (F16)
      static_cast<f16*>(g.a.y)[dst] = (f16)y;
    else
      static_cast<bf16*>(g.a.y)[dst] = to_bf16(y);
  }
}

bool bad_attend(const Cache& c, const Sequences& s, const AttendArgs& a) {
  return bad_cache(c, s) || (a.type != ROWS_BF16 && a.type != ROWS_F16) || a.heads <= 0 || a.heads > 1024 ||
         a.heads % c.kv_heads || a.window < 0 || a.sinks < 0;
}

// Whether pages hold whole blocks.
bool wide_pages(const Cache& c) { return (1 << c.page_shift) >= 4096 / c.dim; }

// How a call is cut, by upper bounds of what the GPU finds from the lengths.
struct Shape {
  Plan p;
  long items;  // workgroups
};
Shape shape_of(const Cache& c, const Sequences& s, const AttendArgs& a) {
  Shape r{};
  r.p.group = a.heads / c.kv_heads;
  r.p.block_shift = c.dim == 64 ? 6 : 5;
  const long cap = (long)s.table_pages << c.page_shift;
  r.p.cap = (int)(cap < POSITIONS ? cap : POSITIONS);
  // tiles: at most one begun by every sequence beside the full ones; no tile sees more blocks than the table names, or its rows'
  // windows and the sinks (and some more by alignment)
  const long full = (long)s.rows * r.p.group / RT;
  const long tiles = (s.starts ? full + (s.n < s.rows ? s.n : s.rows) : (long)s.rows * ((r.p.group + RT - 1) / RT)) * c.kv_heads;
  const long all = r.p.cap >> r.p.block_shift, some = (((long)a.window + RT + 1) >> r.p.block_shift) + 1 + (a.sinks >> r.p.block_shift) + 1;
  const long blocks = (some < all ? some : all) + 2;
  const long fill = (long)resident(c.dim, c.format, a.type == ROWS_F16, wide_pages(c), s.starts) * num_cus();
  // A workgroup a tile, and no second kernel, where a tile sees so few keys that this costs no more than sharing them out (a
  // round takes about 1.4 us): 11 blocks of 8 heads on eight waves 8.2 us, shared 7.3 + 4.4; 64 sequences of 33 blocks 20.8,
  // shared 23.8 + 4.8; 5 rows of each of 32 sequences in windows of 2048 keys 15.1, shared 15.8 + 5.8; but one sequence of 63
  // blocks 17.5, shared 7.3 + 5.7.
  // Also where there are many tiles, or more rounds than fit; with more than 64 sequences, which every workgroup would search for its
  // stretch, a few times what fills the GPU: 512 of 8000 tokens, 8 heads, 370 us, shared 464 (3% of them of 8000, the others of 400: 80,
  // shared 134), 1000 of 6000, one head, 84, shared 217; but 160 of up to 20000, 8 heads, 212, shared 193.
  r.items = s.starts ? (full + s.n) * c.kv_heads : tiles;
  r.p.waves = 4;
  if (blocks <= 40 && tiles <= 2 * num_cus()) {
    r.p.waves = 8;
    return r;
  }
  const bool many = s.n <= 64 ? tiles >= 32 * fill : tiles >= (s.n < 512 ? 2 * fill : fill / 2);
  if (blocks <= 18 || (blocks <= 66 && tiles >= fill / 2) || many || tiles * (all + 2) > 0x3fffffffL) return r;
  const long most = tiles * ((blocks + r.p.waves - 1) / r.p.waves);
  r.items = r.p.groups = (int)(most < fill ? most : fill);
  return r;
}

size_t part_bytes(const Cache& c, const Shape& r) { return (size_t)r.p.groups * 2 * RT * c.dim * 4; }

}  // namespace

int cache_attend_workspace(const Cache& c, const Sequences& s, const AttendArgs& a, size_t* bytes) {
  // (for any window and sinks: a short window may need none)
  AttendArgs all = a;
  all.window = 0x7fffffff;
  if (bad_attend(c, s, all)) return NOISE_EINVAL;
  const Shape r = shape_of(c, s, all);
  *bytes = part_bytes(c, r) + (size_t)r.p.groups * 2 * RT * 8;
  return NOISE_OK;
}

int cache_attend_launch(const Cache& c, const Sequences& s, const AttendArgs& a, void* ws, size_t ws_bytes,
                        hipStream_t stream) {
  if (bad_attend(c, s, a) || bad_heads(a.q) || !a.y || ((uintptr_t)a.y & 15) || !(a.scale >= 0.f) || a.scale > 3.4e38f)
    return NOISE_EINVAL;
  const Shape r = shape_of(c, s, a);
  const size_t need = part_bytes(c, r) + (size_t)r.p.groups * 2 * RT * 8;
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) return NOISE_ENOSPC;
  Args g{c, s, a, r.p, 0.f, 0, 0, nullptr, nullptr};
  // (a scale of 0 is the smallest normal number: every seen key weighs the same, and a masked score stays -infinity)
  const float c2 = a.scale * 1.4426950408889634f;
  g.c2 = c2 > 1.17549435e-38f ? c2 : 1.17549435e-38f;
  g.fills = a.fill && s.starts ? 32 : 0;
  if ((long)s.rows * a.heads > 0x7fffff00L || r.items + g.fills > 0x7fffffffL) return NOISE_ENOTSUP;
  g.items = (int)r.items;
  g.part = static_cast<float*>(ws);
  g.ml = ws ? reinterpret_cast<float2*>(static_cast<char*>(ws) + part_bytes(c, r)) : nullptr;
  const bool wide = wide_pages(c);
  auto launch = [&](auto dim, auto fmt, auto f16_, auto wide_, auto many) {
    constexpr int D = decltype(dim)::value, F = decltype(fmt)::value;
    constexpr bool H = decltype(f16_)::value, W = decltype(wide_)::value, M = decltype(many)::value;
    const dim3 grid((unsigned)(g.items + g.fills));
    if (r.p.waves == 8)
      hipLaunchKernelGGL((attend_kernel<D, F, H, W, M, 8>), grid, dim3(512), 0, stream, g);
    else
      hipLaunchKernelGGL((attend_kernel<D, F, H, W, M, 4>), grid, dim3(256), 0, stream, g);
  };
  auto with = [&](auto dim, auto fmt) {
    const std::true_type yes{};
    const std::false_type no{};
    auto of = [&](auto f16_, auto wide_) { s.starts ? launch(dim, fmt, f16_, wide_, yes) : launch(dim, fmt, f16_, wide_, no); };
    if (a.type == ROWS_F16)
      wide ? of(yes, yes) : of(yes, no);
    else
      wide ? of(no, yes) : of(no, no);
  };
  const std::integral_constant<int, CACHE_FP4> fp4{};
  const std::integral_constant<int, CACHE_FP8> fp8{};
  if (c.dim == 64)
    c.format == CACHE_FP4 ? with(std::integral_constant<int, 64>{}, fp4) : with(std::integral_constant<int, 64>{}, fp8);
  else
    c.format == CACHE_FP4 ? with(std::integral_constant<int, 128>{}, fp4) : with(std::integral_constant<int, 128>{}, fp8);
  NOISE_CHECK_LAUNCH();
  if (r.p.groups) {
    const dim3 grid((unsigned)(s.rows * a.heads));
    // sixteen waves where few rows have many parts (8 rows of 64 parts 8.1 us with four, 6.5 with sixteen), four where rows fill the GPU
    auto join = [&](auto dim, auto f16_) {
      constexpr int D = decltype(dim)::value;
      constexpr bool H = decltype(f16_)::value;
      if (grid.x <= (unsigned)num_cus())
        hipLaunchKernelGGL((join_kernel<D, H, 16>), grid, dim3(1024), 0, stream, g);
      else
        hipLaunchKernelGGL((join_kernel<D, H, 4>), grid, dim3(256), 0, stream, g);
    };
    const std::integral_constant<int, 64> d64{};
    const std::integral_constant<int, 128> d128{};
    if (a.type == ROWS_F16)
      c.dim == 64 ? join(d64, std::true_type{}) : join(d128, std::true_type{});
    else
      c.dim == 64 ? join(d64, std::false_type{}) : join(d128, std::false_type{});
    NOISE_CHECK_LAUNCH();
  }
  return NOISE_OK;
}

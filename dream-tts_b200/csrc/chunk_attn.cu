// Attention of a ragged chunk of new tokens over a paged cache: row j of lane i's n new rows sits
// at position p = spans[i] - n + j and sees positions max(0, p + 1 - window) .. p of its lane
// (window 0: all of 0 .. p), grouped-query heads: o = sum_s w_s v_s / sum_s w_s,
// w_s = exp(scale q.k_s - m). A row that sees nothing (p < 0) is zero.
//
// Tiles. A lane's rows for one kv head are flattened token-major over the group's q heads (flat
// row f: token f / gqa, head f % gqa), so any group size shares one read of K and V. A work tile
// is 256 flat rows as two 128-row query tiles (MMA M); its keys go by in units of 128 positions
// (two MMAs a query tile and unit: S = Q.K^T, O += P.V). While one query tile's softmax runs, the
// tensor cores work on the other.
//
// Split. The units of all work tiles, one after another, are cut into equal runs, one per SM; a
// work tile that a cut falls into leaves its parts (O, row maximum, row sum) in the workspace and
// a second kernel joins them in order. So one long lane with one new token and a thousand short
// chunks both use every SM, and results do not depend on timing.
//
// Warps 0-3 and 4-7: one query row a thread through softmax and output, query tiles 0 and 1.
// Warp 8 loads K and V (TMA, 8 rows x 128 dims a box, so any page of a multiple of 8 rows, or any
// contiguous lane), warp 9 issues the MMAs, warp 10 walks the work. S and then P (f16, in place)
// stay in TMEM, O accumulates in TMEM.
//
// Softmax in powers of two against a reference r that is the row's maximum so far or up to 2^7
// below it: w = 2^(c s - r + 8), c = scale log2 e. O is rescaled only when the maximum passes r by
// more than that, which random scores hardly ever do after the first units. w is at most 2^15 and
// keeps f16's 11 bits down to 2^-22 of the row's largest; sums are f32.
#include <mutex>

#include "chunk_batch.cuh"

namespace tts {

namespace {

constexpr int kCaThreads = 384;
constexpr int kCaTile = 256;  // flat query rows of a work tile
constexpr int kCaKeys = 128;  // positions of a unit
constexpr int kCaSegs = 4;    // work descriptors in flight
constexpr float kCaSlack = 7.f, kCaBias = 8.f;

// 128 rows x 128 f16 for the MMAs: groups of 8 rows, in each two halves of 64 columns, rows of 128
// bytes with the 128-byte swizzle (what a TMA box of 8 rows x 2 halves x 64 columns writes).
constexpr int kCaTileBytes = 128 * 256;
TTS_DEV uint32_t ca_at(int r, int piece) {  // byte offset of 16-byte piece 0..15 of row r
  return uint32_t(r >> 3) * 2048u + uint32_t(piece >> 3) * 1024u + uint32_t(r & 7) * 128u +
         (uint32_t((piece & 7) ^ (r & 7)) << 4);
}

// One run of a work tile's units.
struct CaSeg {
  int row0, n, pos0;  // the lane's first row, its new rows, the first one's position
  int flat0, lane, head;
  int unit0, units;   // 0 units: no more work
  int begins, ends;   // whether the run has the work tile's first and last unit
};

template <int kStages, int kParts>  // kParts: f16 pieces a query element is held in
struct CaSmem {
  uint8_t ring[kStages][kCaTileBytes];
  uint8_t q[2][kParts][kCaTileBytes];
  uint64_t full[kStages], empty[kStages], q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t seg_full[kCaSegs], seg_empty[kCaSegs], tail, drain;
  CaSeg seg[kCaSegs];
  int start[4];  // the CTA's first lane, work tile, head and unit
  int count;     // its units
  int failed;
  uint32_t tmem;
};

// What a split work tile's part was, one per CTA for the run it takes over from the CTA before
// (slot 0) and one for the run it leaves unfinished to the next (slot 1).
struct CaPart {
  int valid, row0, n, flat0, head, more;
};
constexpr int kCaPartFloats = kCaTile * 130;  // O [32][256] float4, m [256], l [256]

struct CaArgs {
  ChunkAttnRequest r;
  float c;      // |scale| log2 e
  int negate;   // scale < 0: the queries change sign
  int odd;      // one page per lane of any size
  CaPart* parts;
  float* part_data;
};

TTS_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 32 columns of the warp's TMEM lanes, without the wait.
TTS_DEV void tmem_ld32(uint32_t a, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32"
      " {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
// Keeps uses of the 32 registers behind the wait that precedes it.
TTS_DEV void tmem_tie32(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
TTS_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
TTS_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
TTS_DEV void tmem_st16(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
// D += A . B with A (f16 pairs) in TMEM.
TTS_DEV void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}
// Boxes of the pool seen as [2 halves][rows][64 columns].
TTS_DEV void ca_load_group(void* dst, const void* map, uint64_t* bar, int row) {
  tma_load_3d(dst, map, bar, 0, row, 0);
}

// First unit and number of units of a lane's work tile k (at least one: rows that see nothing are
// written too).
TTS_DEV void ca_units(int n, int pos0, int gqa, int window, int k, int* first, int* count) {
  const int t0 = k * kCaTile / gqa, t1 = min(n, (k * kCaTile + kCaTile - 1) / gqa + 1);
  const int lo = window > 0 ? max(0, pos0 + t0 + 1 - window) : 0;
  const int last = max(0, pos0 + t1 - 1) / kCaKeys;
  *first = lo / kCaKeys;
  *count = last - *first + 1;
}
TTS_DEV int ca_tiles(int n, int gqa) { return (n * gqa + kCaTile - 1) / kCaTile; }

struct CaLane {
  int row0, n, pos0;
};
// A lane's rows; a span the block table cannot hold leaves the lane without any.
TTS_DEV CaLane ca_lane(const ChunkAttnRequest& r, int i) {
  CaLane l;
  l.row0 = r.row_start[i];
  l.n = r.row_start[i + 1] - l.row0;
  const int span = r.spans[i];
  if (span < 0 || span > r.max_blocks * r.block_size) l.n = 0;
  l.pos0 = span - l.n;
  return l;
}

template <typename TQ>
TTS_DEV float ca_q(const CaArgs& a, int row, int head, int d) {
  const float x =
      float(static_cast<const TQ*>(a.r.q)[((size_t)row * a.r.n_kv * a.r.gqa + head) * 128 + d]);
  return a.negate ? -x : x;
}

// The pool row of a lane's position, -1 where the page is outside the pool.
TTS_DEV long ca_pool_row(const CaArgs& a, int lane, int head, int pos) {
  const int page = a.r.block_table[(size_t)lane * a.r.max_blocks + pos / a.r.block_size];
  if (page < 0 || page >= a.r.num_blocks) return -1;
  return ((long)page * a.r.n_kv + head) * a.r.block_size + pos % a.r.block_size;
}

// Positions a row does not see have weight 0, but an infinity or NaN among their values makes 0
// times it NaN. Where a row's output is not finite, the warp looks at the values the row's units
// held beyond what it sees and, if one is not finite, sums the row again over what it sees (dims
// 4 lane .. + 3 of the result to each warp lane). Never reached by finite caches.
template <typename TQ>
__device__ __noinline__ bool ca_repair(const CaArgs& a, const CaSeg& s, int f, int hi, float ref,
                                       float4* o) {
  const int wl = threadIdx.x & 31;
  const int tok = f / a.r.gqa, head = s.head * a.r.gqa + f % a.r.gqa;
  const int pos = s.pos0 + tok;
  const int u0 = s.unit0 * kCaKeys, u1 = min(hi, (s.unit0 + s.units) * kCaKeys);
  const int lo = a.r.window > 0 ? max(0, pos + 1 - a.r.window) : 0;
  const auto finite4 = [&](int p) {
    const long at = ca_pool_row(a, s.lane, s.head, p);
    if (at < 0) return true;
    const uint2 u = *reinterpret_cast<const uint2*>(a.r.v_pool + at * 128 + wl * 4);
    const uint32_t e = 0x7c007c00u;  // an all-ones exponent in either half
    return (u.x & e & 0xffffu) != 0x7c00u && (u.x & e) >> 16 != 0x7c00u &&
           (u.y & e & 0xffffu) != 0x7c00u && (u.y & e) >> 16 != 0x7c00u;
  };
  bool clean = true;
  for (int p = u0; p < min(lo, u1); ++p) clean = clean && finite4(p);
  for (int p = max(u0, pos + 1); p < u1; ++p) clean = clean && finite4(p);
  if (__all_sync(0xffffffffu, clean)) return false;
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = ca_q<TQ>(a, s.row0 + tok, head, wl * 4 + i);
  *o = make_float4(0.f, 0.f, 0.f, 0.f);
  const float bias = ref == -INFINITY ? 0.f : kCaBias - ref;
  for (int p = max(u0, lo); p < min(u1, pos + 1); ++p) {
    const long at = ca_pool_row(a, s.lane, s.head, p);
    if (at < 0) continue;
    const __half2* k = reinterpret_cast<const __half2*>(a.r.k_pool + at * 128 + wl * 4);
    const __half2* v = reinterpret_cast<const __half2*>(a.r.v_pool + at * 128 + wl * 4);
    const float2 k0 = __half22float2(k[0]), k1 = __half22float2(k[1]);
    const float x = warp_sum(q[0] * k0.x + q[1] * k0.y + q[2] * k1.x + q[3] * k1.y);
    const float w = ex2(fmaf(x, a.c, bias));
    const float2 v0 = __half22float2(v[0]), v1 = __half22float2(v[1]);
    o->x += w * v0.x, o->y += w * v0.y, o->z += w * v1.x, o->w += w * v1.y;
  }
  return true;
}

// The CTA's share of the work: all CTAs compute the same totals from the lanes' lengths. Uses the
// (still empty) tile ring as scratch.
template <typename Smem>
TTS_DEV void ca_plan(Smem& S, const CaArgs& a) {
  const int t = threadIdx.x, warp = t >> 5, wl = t & 31;
  const ChunkAttnRequest& r = a.r;
  long long* tot = reinterpret_cast<long long*>(S.ring[0]);  // [lanes]: units before each lane
  for (int i = warp; i < r.lanes; i += kCaThreads / 32) {
    const CaLane l = ca_lane(r, i);
    long long u = 0;
    for (int k = wl; k < ca_tiles(l.n, r.gqa); k += 32) {
      int first, count;
      ca_units(l.n, l.pos0, r.gqa, r.window, k, &first, &count);
      u += count;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
    if (wl == 0) tot[i] = u * r.n_kv;
  }
  __syncthreads();
  if (warp == 0) {
    long long all = 0;
    for (int i0 = 0; i0 < r.lanes; i0 += 32) {
      const long long mine = i0 + wl < r.lanes ? tot[i0 + wl] : 0;
      long long inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (wl >= o) inc += x;
      }
      if (i0 + wl < r.lanes) tot[i0 + wl] = all + inc - mine;
      all += __shfl_sync(0xffffffffu, inc, 31);
    }
    __syncwarp();
    const long long per = (all + gridDim.x - 1) / gridDim.x;
    const long long lo = per * blockIdx.x, hi = lo + per < all ? lo + per : all;
    if (wl == 0) S.count = lo < hi ? int(hi - lo) : 0;
    if (lo < hi) {
      // the last lane that starts at or before `lo` (lanes without rows start where the next does)
      int lane = 0;
      for (int i0 = 0; i0 < r.lanes; i0 += 32) {
        const bool at = i0 + wl < r.lanes && tot[i0 + wl] <= lo;
        const unsigned m = __ballot_sync(0xffffffffu, at);
        if (m) lane = i0 + 31 - __clz(m);
      }
      long long rem = lo - tot[lane];
      const CaLane l = ca_lane(r, lane);
      for (int k0 = 0;; k0 += 32) {
        int first = 0, count = 0;
        if (k0 + wl < ca_tiles(l.n, r.gqa))
          ca_units(l.n, l.pos0, r.gqa, r.window, k0 + wl, &first, &count);
        const long long mine = (long long)count * r.n_kv;
        long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long x = __shfl_up_sync(0xffffffffu, inc, o);
          if (wl >= o) inc += x;
        }
        const unsigned m = __ballot_sync(0xffffffffu, rem < inc);
        if (m) {
          if (wl == __ffs(m) - 1) {
            const int in = int(rem - (inc - mine));
            S.start[0] = lane;
            S.start[1] = k0 + wl;
            S.start[2] = in / count;
            S.start[3] = in % count;
          }
          break;
        }
        rem -= __shfl_sync(0xffffffffu, inc, 31);
        if (k0 > ca_tiles(l.n, r.gqa)) {  // not reached: `lo` lies within the lane's units
          if (wl == 0) S.count = 0;
          break;
        }
      }
    }
  }
  __syncthreads();
}

template <typename TQ, int kStages, int kParts>
__global__ void __launch_bounds__(kCaThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ CaArgs a) {
  extern __shared__ uint8_t smem_raw[];
  typedef CaSmem<kStages, kParts> Smem;
  Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                     ~uintptr_t(1023));
  const int t = threadIdx.x, warp = t >> 5, wl = t & 31;
  const ChunkAttnRequest& r = a.r;
  pdl_launch_dependents();  // the join waits for this grid's end before it reads
  if (t < 2) a.parts[2 * blockIdx.x + t].valid = 0;
  if (!__syncthreads_and(chunk_starts_ok(r.row_start, r.lanes, r.rows, t, kCaThreads))) {
    if (t == 0 && blockIdx.x == 0) atomicOr(r.err, kFlagChunkStarts);
    return;
  }
  if (blockIdx.x == 0)
    for (int i = t; i < r.lanes; i += kCaThreads)
      if (r.spans[i] < 0 || r.spans[i] > r.max_blocks * r.block_size)
        atomicOr(r.err, kFlagSpanRange);
  ca_plan(S, a);
  if (S.count == 0) return;
  if (t == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&S.full[i], 1);
      mbar_init(&S.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.q_full[i], 4);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i], 4);
      mbar_init(&S.o_full[i], 1);
    }
    for (int i = 0; i < kCaSegs; ++i) {
      mbar_init(&S.seg_full[i], 1);
      mbar_init(&S.seg_empty[i], 10);
    }
    mbar_init(&S.tail, 1);
    mbar_init(&S.drain, 1);
    S.failed = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 9) {
    tmem_alloc(&S.tmem, 512);
    tmem_relinquish();
  }
  fence_proxy_async();  // the plan's scratch before the copies into the same memory
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  bool ok = true;
  int seg_slot = 0;
  uint32_t seg_phase = 0;
  // every role reads the work in order and frees its slot at once
  const auto next_seg = [&](CaSeg* s) {
    if (!mbar_wait_warp(&S.seg_full[seg_slot], seg_phase)) return false;
    *s = S.seg[seg_slot];
    __syncwarp();
    if (wl == 0) mbar_arrive(&S.seg_empty[seg_slot]);
    if (++seg_slot == kCaSegs) seg_slot = 0, seg_phase ^= 1;
    return true;
  };

  if (warp == 10) {
    // ---- the work walk: units in order of lane, work tile, head
    int lane = S.start[0], k = S.start[1], head = S.start[2], off = S.start[3], left = S.count;
    CaLane l = ca_lane(r, lane);
    for (;;) {
      CaSeg s{};
      if (left > 0) {
        int first, count;
        ca_units(l.n, l.pos0, r.gqa, r.window, k, &first, &count);
        const int take = min(left, count - off);
        s = CaSeg{l.row0, l.n, l.pos0, k * kCaTile, lane, head, first + off, take, off == 0,
                  off + take == count};
        left -= take;
        off = 0;
        if (++head == r.n_kv) {
          head = 0;
          if (++k == ca_tiles(l.n, r.gqa) && left > 0) {
            k = 0;
            do l = ca_lane(r, ++lane);
            while (l.n == 0 && lane + 1 < r.lanes);
          }
        }
        if (wl == 0 && !(s.begins && s.ends)) {
          CaPart& p = a.parts[2 * blockIdx.x + (s.begins ? 1 : 0)];
          p.row0 = s.row0, p.n = s.n, p.flat0 = s.flat0, p.head = s.head;
          p.more = !s.ends;
          p.valid = 1;
        }
      }
      ok = mbar_wait_warp(&S.seg_empty[seg_slot], seg_phase ^ 1);
      if (!ok) break;
      if (wl == 0) {
        S.seg[seg_slot] = s;
        mbar_arrive(&S.seg_full[seg_slot]);
      }
      __syncwarp();
      if (++seg_slot == kCaSegs) seg_slot = 0, seg_phase ^= 1;
      if (s.units == 0) break;
    }
  } else if (warp == 8) {
    // ---- K and V: warp lanes 0-15 a group of 8 K rows each, 16-31 of V rows
    const int g = wl & 15, is_v = wl >> 4;
    const CUtensorMap* map = is_v ? &tmV : &tmK;
    int slot = 0;
    uint32_t phase = 0, tail_phase = 0;
    CaSeg s;
    while (ok && (ok = next_seg(&s)) && s.units > 0) {
      const int last = min(s.n, (s.flat0 + kCaTile - 1) / r.gqa + 1);
      const int hi = s.pos0 + last;  // positions from here on are seen by no row of the tile
      const auto page_of = [&](int j) {
        const int p = (s.unit0 + j) * kCaKeys + g * 8;
        return j < s.units && p < hi
                   ? r.block_table[(size_t)s.lane * r.max_blocks + p / r.block_size]
                   : 0;
      };
      int page = page_of(0);
      for (int j = 0; j < s.units; ++j) {
        const int next = page_of(j + 1);
        const int p0 = (s.unit0 + j) * kCaKeys, p = p0 + g * 8;
        const bool seen = p < hi, bad = seen && (page < 0 || page >= r.num_blocks);
        if (bad) atomicOr(r.err, kFlagPageRange);
        const int row = (page * r.n_kv + s.head) * r.block_size + p % r.block_size;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          ok = ok && mbar_wait_warp(&S.empty[slot], phase ^ 1);
          if (!ok) break;
          uint8_t* tile = S.ring[slot];
          const bool mine = is_v == v;
          const int loads = __popc(__ballot_sync(0xffffffffu, mine && seen && !bad));
          // groups without a page read as zero; so do V rows that nothing sees, whose stale
          // bits times a weight of 0 could be NaN
          const bool tail = v && p0 + kCaKeys > hi;
          if (mine && (bad || (tail && !seen))) {
            for (int i = 0; i < 128; ++i)
              *reinterpret_cast<uint4*>(tile + g * 2048 + i * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
          }
          __syncwarp();
          uint64_t* bar = tail ? &S.tail : &S.full[slot];
          if (wl == 0) mbar_arrive_expect_tx(bar, uint32_t(loads) * 2048u);
          __syncwarp();
          if (mine && seen && !bad) ca_load_group(tile + g * 2048, map, bar, row);
          if (tail) {
            ok = mbar_wait_warp(&S.tail, tail_phase);
            tail_phase ^= 1;
            if (!ok) break;
            for (int i = wl; i < (8 - (hi & 7)) % 8 * 16 && hi > p0; i += 32)
              *reinterpret_cast<uint4*>(tile + ca_at(hi - p0 + (i >> 4), i & 15)) =
                  make_uint4(0, 0, 0, 0);
            fence_proxy_async();
            __syncwarp();
            if (wl == 0) mbar_arrive(&S.full[slot]);
          }
          if (++slot == kStages) slot = 0, phase ^= 1;
        }
        page = next;
        if (!ok) break;
      }
    }
    if (!ok)  // bounded: copies still on their way
      for (int i = 0; i < kStages; ++i) mbar_wait(&S.full[i], phase, 100000000ull);
  } else if (warp == 9) {
    // ---- the MMAs. Tile by tile and unit by unit: O_t += P_t.V(j), then S_t = Q_t.K(j + 1) over
    // the P just read (MMAs of one thread run in the order of their issue).
    const uint32_t idesc_s = idesc_f16_f32(128, kCaKeys);
    const uint32_t idesc_o = idesc_f16_f32(128, 128) | (1u << 16);  // B (V) MN-major
    int slot = 0;
    uint32_t phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
    const auto advance = [&] {
      if (++slot == kStages) slot = 0, phase ^= 1;
    };
    const auto scores = [&](int tl, int at) {
      const uint32_t kb = smem_u32(S.ring[at]);
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const uint32_t qb = smem_u32(S.q[tl][h]);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t o = (kk >> 2) * 1024 + (kk & 3) * 32;
          umma_f16(tmem + tl * 128, smem_desc(qb + o, 16, 2048, 2), smem_desc(kb + o, 16, 2048, 2),
                   idesc_s, (h | kk) != 0);
        }
      }
      umma_commit(&S.s_full[tl]);
    };
    CaSeg s;
    while (ok && (ok = next_seg(&s)) && s.units > 0) {
      const int tiles = s.flat0 + 128 < s.n * r.gqa ? 2 : 1;
      ok = mbar_wait_warp(&S.full[slot], phase);
      for (int tl = 0; tl < tiles && ok; ++tl) {
        ok = mbar_wait_warp(&S.q_full[tl], q_phase[tl]);
        q_phase[tl] ^= 1;
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) scores(tl, slot);
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) umma_commit(&S.empty[slot]);
      __syncwarp();
      advance();
      for (int j = 0; j < s.units && ok; ++j) {
        const int v_slot = slot;
        ok = mbar_wait_warp(&S.full[slot], phase);
        advance();
        const bool more = j + 1 < s.units;
        for (int tl = 0; tl < tiles && ok; ++tl) {
          ok = mbar_wait_warp(&S.p_full[tl], p_phase[tl]);
          p_phase[tl] ^= 1;
          if (tl == 0 && more && ok) ok = mbar_wait_warp(&S.full[slot], phase);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t vb = smem_u32(S.ring[v_slot]);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_f16_ts(tmem + 256 + tl * 128, tmem + tl * 128 + kk * 8,
                          smem_desc(vb + kk * 4096, 1024, 2048, 2), idesc_o, (j | kk) != 0);
            if (more)
              scores(tl, slot);
            else
              umma_commit(&S.o_full[tl]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elect_one()) {
          umma_commit(&S.empty[v_slot]);
          if (more) umma_commit(&S.empty[slot]);
        }
        __syncwarp();
        if (more) advance();
      }
    }
    if (!ok) {  // bounded: MMAs still running
      if (elect_one()) umma_commit(&S.drain);
      __syncwarp();
      mbar_wait(&S.drain, 0, 100000000ull);
    }
  } else if (warp < 8) {
    // ---- softmax and output, one query row a thread
    const int tl = warp >> 2, lane_row = t & 127;
    const uint32_t lanes_at = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes_at + uint32_t(tl * 128);
    const uint32_t o_at = tmem + lanes_at + 256u + uint32_t(tl * 128);
    uint32_t s_phase = 0, o_phase = 0;
    CaSeg s;
    while (ok && (ok = next_seg(&s)) && s.units > 0) {
      const int f = s.flat0 + tl * 128 + lane_row;
      if (s.flat0 + tl * 128 >= s.n * r.gqa) continue;  // this query tile has no rows
      const bool live = f < s.n * r.gqa;
      const int tok = f / r.gqa;
      const int head = s.head * r.gqa + f % r.gqa;
      const int pos = live ? s.pos0 + tok : -1;
      const int lo = r.window > 0 ? max(0, pos + 1 - r.window) : 0;
      const bool work = __any_sync(0xffffffffu, live);
      // the row as f16 pieces in the MMA's layout
      const uint4* src = reinterpret_cast<const uint4*>(
          static_cast<const TQ*>(r.q) +
          ((size_t)(s.row0 + tok) * r.n_kv * r.gqa + head) * 128);
      constexpr int kWords = int(sizeof(TQ)) / 2;  // 16-byte loads per 8 dims
#pragma unroll
      for (int e0 = 0; e0 < 16; e0 += 8) {
        uint4 x[8 * kWords];
#pragma unroll
        for (int i = 0; i < 8 * kWords; ++i)
          x[i] = live ? __ldg(src + e0 * kWords + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint4 piece[kParts];
          __half* h = reinterpret_cast<__half*>(piece);
          const TQ* v = reinterpret_cast<const TQ*>(x + e * kWords);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float rest = a.negate ? -float(v[i]) : float(v[i]);
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
              h[p * 8 + i] = __float2half_rn(rest);
              rest -= __half2float(h[p * 8 + i]);
            }
          }
#pragma unroll
          for (int p = 0; p < kParts; ++p)
            *reinterpret_cast<uint4*>(&S.q[tl][p][ca_at(lane_row, e0 + e)]) = piece[p];
        }
      }
      fence_proxy_async();
      tc_fence_before();
      __syncwarp();
      if (wl == 0) mbar_arrive(&S.q_full[tl]);
      // rows of a warp see contiguous ranges: a unit inside all of them needs no mask
      const int pos_min = __reduce_min_sync(0xffffffffu, live ? pos : INT_MAX);
      const int lo_max = __reduce_max_sync(0xffffffffu, live ? lo : 0);
      float ref = -INFINITY, sum = 0.f;
      for (int j = 0; j < s.units; ++j) {
        ok = mbar_wait_warp(&S.s_full[tl], s_phase);
        s_phase ^= 1;
        if (!ok) break;
        tc_fence_after();
        if (work) {
          uint32_t x[4][32];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld32(s_at + i * 32, x[i]);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_tie32(x[i]);
          const int p0 = (s.unit0 + j) * kCaKeys;
          if (p0 + kCaKeys - 1 > pos_min || p0 < lo_max) {
            const int first = lo - p0, last = pos - p0;  // columns the row sees
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (i * 32 + e < first || i * 32 + e > last) x[i][e] = 0xff800000u;  // -inf
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(x[i][e]));
          mx *= a.c;
          const bool up = mx > ref + kCaSlack;
          if (__any_sync(0xffffffffu, up)) {
            const float keep = up ? ex2(ref - mx) : 1.f;
            if (up) ref = mx;
            sum *= keep;
            if (j > 0) {  // the MMAs before S(j), O's among them, are complete
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float o[16];
                uint32_t y[16];
                tmem_ld16(o_at + i * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(o[e] * keep);
                tmem_st16(o_at + i * 16, y);
              }
            }
          }
          const float bias = ref == -INFINITY ? 0.f : kCaBias - ref;
          float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float w0 = ex2(fmaf(__uint_as_float(x[i][2 * e]), a.c, bias));
              const float w1 = ex2(fmaf(__uint_as_float(x[i][2 * e + 1]), a.c, bias));
              part[e & 1] += w0;
              part[2 + (e & 1)] += w1;
              const __half2 h = __floats2half2_rn(w0, w1);
              y[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            tmem_st16(s_at + i * 16, y);
          }
          sum += (part[0] + part[1]) + (part[2] + part[3]);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (wl == 0) mbar_arrive(&S.p_full[tl]);
      }
      if (!ok) break;
      ok = mbar_wait_warp(&S.o_full[tl], o_phase);
      o_phase ^= 1;
      if (!ok) break;
      tc_fence_after();
      if (!work) continue;
      // ---- out, or the part of a split work tile
      const bool whole = s.begins && s.ends;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      __half* dst = r.out + ((size_t)(s.row0 + tok) * r.n_kv * r.gqa + head) * 128;
      float* part = a.part_data + (size_t)(2 * blockIdx.x + (s.begins ? 1 : 0)) * kCaPartFloats;
      const int pr = tl * 128 + lane_row;
      float probe = 0.f;  // NaN once a value is not finite
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float o[16];
        tmem_ld16(o_at + i * 16, o);
#pragma unroll
        for (int e = 0; e < 16; ++e) probe = fmaf(o[e], 0.f, probe);
        if (!live) continue;
        if (whole) {
          uint4 y[2];
          __half2* h = reinterpret_cast<__half2*>(y);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = __floats2half2_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
          reinterpret_cast<uint4*>(dst)[2 * i] = y[0];
          reinterpret_cast<uint4*>(dst)[2 * i + 1] = y[1];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<float4*>(part)[(i * 4 + e) * kCaTile + pr] =
                make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
      if (!whole && live) {
        part[kCaTile * 128 + pr] = ref;
        part[kCaTile * 129 + pr] = sum;
      }
      unsigned again = __ballot_sync(0xffffffffu, live && probe != 0.f);
      const int hi = s.pos0 + min(s.n, (s.flat0 + kCaTile - 1) / r.gqa + 1);
      while (again) {
        const int src = __ffs(again) - 1;
        again &= again - 1;
        float4 o;
        const float sref = __shfl_sync(0xffffffffu, ref, src);
        const float sinv = __shfl_sync(0xffffffffu, inv, src);
        const int sf = __shfl_sync(0xffffffffu, f, src), spr = __shfl_sync(0xffffffffu, pr, src);
        if (!ca_repair<TQ>(a, s, sf, hi, sref, &o)) continue;
        if (whole) {
          __half2* h = reinterpret_cast<__half2*>(
              r.out + ((size_t)(s.row0 + sf / r.gqa) * r.n_kv * r.gqa + s.head * r.gqa +
                       sf % r.gqa) * 128 + wl * 4);
          h[0] = __floats2half2_rn(o.x * sinv, o.y * sinv);
          h[1] = __floats2half2_rn(o.z * sinv, o.w * sinv);
        } else {
          reinterpret_cast<float4*>(part)[wl * kCaTile + spr] = o;
        }
      }
    }
  }
  if (!ok && wl == 0) {
    atomicOr(r.err, kFlagAttnWait);
    S.failed = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of work tiles that a cut fell into: block (c, y) the tile that CTA c began and
// left unfinished (its slot 1, then slot 0 of the CTAs that took it over, in order), 32 of its
// rows; warp w dims 16 w .. + 15 of them, a row a warp lane.
constexpr int kCjThreads = 256;
__global__ void __launch_bounds__(kCjThreads) chunk_attn_join_kernel(const CaArgs a, int ctas) {
  pdl_wait();
  const int c = blockIdx.x, wl = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const CaPart p = a.parts[2 * c + 1];
  if (!p.valid) return;
  const int pr = blockIdx.y * 32 + wl, f = p.flat0 + pr;
  if (p.flat0 + (int)blockIdx.y * 32 >= p.n * a.r.gqa) return;
  int last = c + 1;
  while (last + 1 < ctas && a.parts[2 * last].more) ++last;
  const auto part = [&](int i) {
    return a.part_data + (size_t)(i == c ? 2 * c + 1 : 2 * i) * kCaPartFloats;
  };
  float m = -INFINITY;
  for (int i = c; i <= last; ++i) m = fmaxf(m, part(i)[kCaTile * 128 + pr]);
  float l = 0.f;
  float4 o[4] = {};
  for (int i = c; i <= last; ++i) {
    const float* x = part(i);
    const float mi = x[kCaTile * 128 + pr];
    const float w = mi == -INFINITY ? 0.f : ex2(mi - m);
    l = fmaf(x[kCaTile * 129 + pr], w, l);
    if (w == 0.f) continue;  // what it adds is below f32, or the row saw nothing there
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = reinterpret_cast<const float4*>(x)[(warp * 4 + e) * kCaTile + pr];
      o[e].x = fmaf(v.x, w, o[e].x), o[e].y = fmaf(v.y, w, o[e].y);
      o[e].z = fmaf(v.z, w, o[e].z), o[e].w = fmaf(v.w, w, o[e].w);
    }
  }
  if (f >= p.n * a.r.gqa) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint4 y[2];
  __half2* h = reinterpret_cast<__half2*>(y);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[2 * e] = __floats2half2_rn(o[e].x * inv, o[e].y * inv);
    h[2 * e + 1] = __floats2half2_rn(o[e].z * inv, o[e].w * inv);
  }
  uint4* dst = reinterpret_cast<uint4*>(
      a.r.out + ((size_t)(p.row0 + f / a.r.gqa) * a.r.n_kv * a.r.gqa + p.head * a.r.gqa +
                 f % a.r.gqa) * 128 + warp * 16);
  dst[0] = y[0];
  dst[1] = y[1];
}

}  // namespace

size_t chunk_attn_workspace(int device) {
  return size_t(num_sms(device)) * 2 * (sizeof(CaPart) + sizeof(float) * kCaPartFloats);
}

template <typename TQ, int kStages, int kParts>
static cudaError_t launch_as(const CUtensorMap& k, const CUtensorMap& v, const CaArgs& a, int ctas,
                             int device, cudaStream_t st) {
  const size_t smem = sizeof(CaSmem<kStages, kParts>) + 1024;
  {
    // the opt-in shared-memory limit is a per-device function attribute
    static std::mutex mu;
    static bool done[64] = {false};
    std::lock_guard<std::mutex> lock(mu);
    if (device >= 0 && device < 64 && !done[device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(chunk_attn_kernel<TQ, kStages, kParts>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
      if (e != cudaSuccess) return e;
      done[device] = true;
    }
  }
  chunk_attn_kernel<TQ, kStages, kParts><<<ctas, kCaThreads, smem, st>>>(k, v, a);
  return cudaGetLastError();
}

cudaError_t launch_chunk_attn(const ChunkAttnRequest& r, int device, cudaStream_t st) {
  const uint64_t rows = uint64_t(r.num_blocks) * r.n_kv * r.block_size;
  CUtensorMap tmK, tmV;
  if (!make_tmap_rows_f16(&tmK, r.k_pool, rows, 8) || !make_tmap_rows_f16(&tmV, r.v_pool, rows, 8)) {
    set_error("chunk_attention: cuTensorMapEncodeTiled failed (pools must be 16-byte aligned)");
    return cudaErrorInvalidValue;
  }
  const int ctas = num_sms(device);
  CaArgs a{};
  a.r = r;
  a.negate = r.scale < 0.f;
  // a scale of 0 still has to keep masked scores at -infinity
  a.c = fmaxf(fabsf(r.scale) * 1.4426950408889634f, 1e-30f);
  a.parts = static_cast<CaPart*>(r.workspace);
  a.part_data = reinterpret_cast<float*>(a.parts + 2 * ctas);
  cudaError_t e = r.q_f16 ? launch_as<__half, 5, 1>(tmK, tmV, a, ctas, device, st)
                          : launch_as<float, 3, 2>(tmK, tmV, a, ctas, device, st);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, kCaTile / 32, 1);
  cfg.blockDim = dim3(kCjThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, chunk_attn_join_kernel, a, ctas);
}

}  // namespace tts

// Attention of a ragged chunk of new tokens over a paged cache: row j of lane i's n new rows sits
// at position p = spans[i] - n + j and sees positions max(0, p + 1 - window) .. p of its lane
// (window 0: all of 0 .. p), grouped-query heads: o = sum_s w_s v_s / sum_s w_s,
// w_s = exp(scale q.k_s - m). A row that sees nothing (p < 0) is zero.
//
// Tiles. A lane's rows for one kv head are flattened token-major over the group's q heads (flat
// row f: token f / gqa, head f % gqa), so any group size shares one read of K and V. A work tile
// is 256 flat rows as two 128-row query tiles (MMA M); its keys go by in units of 128 positions
// (two MMAs a query tile and unit: S = Q.K^T, O += P.V). While one query tile's softmax runs, the
// tensor cores work on the other. Where there is one query tile only (a token or a few), its units
// alternate between the two score buffers and groups of softmax warps, each with an O of its own,
// and the first group reads both at the end (48 single rows over 4300 positions: 150 us; as two
// query tiles, one of them empty, 182).
//
// Split. The units of all work tiles, one after another, are cut into equal runs, one per SM; a
// work tile that a cut falls into leaves its parts (O, row maximum, row sum) in the workspace and
// a second kernel joins them in order. So one long lane with one new token and a thousand short
// chunks both use every SM, and results do not depend on timing.
//
// Warps 0-3 and 4-7: one query row a thread through softmax and output, query tiles 0 and 1. Warps
// 8 and 11 load K and V (TMA boxes of whole 256-byte rows within a page), warp 9 issues the MMAs,
// warp 10 walks the work. P (f16) takes the place of S in TMEM and is the A operand of O += P.V.
//
// Softmax in powers of two against a reference r: w = 2^(c s - r + 8), c = scale log2 e. r is the
// largest c s of the row's first unit and stays while the weights of 64 positions add up to no more
// than f16 holds; only then O and the sum are brought to a new one (random scores hardly ever ask
// for it after the first units), so no maximum is looked for in most units. Exponentials are the
// hardware's (2^-22), sums f32.
//
// Weights are f16, as the MMA takes them beside f16 values: 11 bits down to 2^-22 of r's, fewer
// below, none below 2^-33 (the f32 sum has those whole; over N positions they are at most N 2^-33
// of it). On N(0, 1) values results are 2.5e-4 to 2.9e-4 of their size off, where rounding the f16
// result alone gives 2.1e-4. The weights' lower halves would ask for a third product beside the
// two that a unit spends 2.4k of its 3.9k clocks on; the decode step's attention, which is bound
// by HBM at any length, does keep them.
//
// Measured (16 q heads, 8 kv heads; B200s differ by some percent): 4096 new rows over 12288
// positions 431 to 458 us, 1050 to 1120 TFLOP/s, 61 to 65 % of a large plain product's rate: a unit
// of two query tiles takes about 3.9k clocks, its MMAs 2.4k to 2.9k and its exponentials 2.0k (16 a
// clock) of them, the rest is their hand-overs. With f32 queries 550 to 578 us: the scores are two
// products. 48 single rows over 4300 positions 146 to 156 us, 5.4 to 5.8 TB/s, 84 to 90 % of a
// copy: bound by HBM. 448 single rows over 300: 181 to 218 us, and 74 chunks of 128 rows (592 work
// tiles) 39 to 45 us: runs of one to three units are too short to hide their start and end (about
// 10k clocks). There the fetch of instructions counts, so loops over a unit stay rolled, queries
// come by copies in short loops and divisions are multiplications: unrolled, those two took 325
// and 54.
#include <cfloat>
#include <mutex>

#include "chunk_batch.cuh"

namespace tts {

namespace {

constexpr int kCaThreads = 384;
constexpr int kCaTile = 256;  // flat query rows of a work tile
constexpr int kCaKeys = 128;  // positions of a unit
constexpr int kCaSegs = 4;    // work descriptors in flight
constexpr float kCaBias = 8.f, kCaMost = 65504.f;
// The MMAs get the weights of half a unit while the other half's are on their way (4096 rows over
// 12288 positions: in halves 436 us, 96 and 32 443, all 128 at once 518).
constexpr int kCaHalf = kCaKeys / 2;

// 128 rows x 128 f16 for the MMAs: groups of 8 rows, in each two halves of 64 columns, rows of 128
// bytes with the 128-byte swizzle (what a TMA box of 64 columns x 8 rows x 2 halves x groups
// writes).
constexpr int kCaTileBytes = 128 * 256;
TTS_DEV uint32_t ca_at(int r, int piece) {  // byte offset of 16-byte piece 0..15 of row r
  return uint32_t(r >> 3) * 2048u + uint32_t(piece >> 3) * 1024u + uint32_t(r & 7) * 128u +
         (uint32_t((piece & 7) ^ (r & 7)) << 4);
}

// 16 bytes from global to shared memory, zeros unless `any`, asynchronously.
TTS_DEV void ca_copy(void* to, const void* from, bool any) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from),
               "r"(any ? 16 : 0)
               : "memory");
}
TTS_DEV void ca_copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
TTS_DEV uint32_t ca_sign(uint32_t two_halves, int negate) {
  return negate ? two_halves ^ 0x80008000u : two_halves;
}
// The warp's 32 query rows (`rh`: each lane's row of q [rows * heads][128], -1: zeros) on their way
// to rows r0 .. r0 + 31 of the tile (copies in a short loop: unrolled loads to registers took
// longer to fetch their instructions than to arrive), and what is to be done once they are there.
// Half a warp takes a row of f16, a warp a row of f32, which is split into two f16 pieces so that
// the scores keep f32 queries' precision. Before that the row is multiplied by a power of two that
// brings its largest magnitude to [2^14, 2^15), just inside f16's range; its softmax factor is
// divided by it (ca_factor). So the pieces hold 22 bits of an element, or 2^-39 of the row's
// largest where that is more, whatever the row's magnitude (unscaled, elements past 65504 were
// infinite and a row near 1e-5 lost 1e-3 of its result; finding the rows' largest costs runs of f32
// queries: 4400 rows in chunks of up to 701 take 125 us for 117, 4096 rows 551 for 543).
TTS_DEV void ca_copy_q(uint8_t (*tile)[kCaTileBytes], const __half* q, int rh, int r0) {
  const int wl = threadIdx.x & 31, sub = wl >> 4, e = wl & 15;
#pragma unroll 2
  for (int k = 0; k < 16; ++k) {
    const int at = __shfl_sync(0xffffffffu, rh, 2 * k + sub);
    ca_copy(&tile[0][ca_at(r0 + 2 * k + sub, e)], q + (size_t)max(at, 0) * 128 + e * 8, at >= 0);
  }
}
TTS_DEV void ca_take_q(uint8_t (*tile)[kCaTileBytes], const __half*, int r0, int negate, uint8_t*) {
  const int wl = threadIdx.x & 31, sub = wl >> 4, e = wl & 15;
  ca_copy_wait();
  if (!negate) return;
#pragma unroll 1
  for (int k = 0; k < 16; ++k) {
    uint4* x = reinterpret_cast<uint4*>(&tile[0][ca_at(r0 + 2 * k + sub, e)]);
    *x = make_uint4(ca_sign(x->x, 1), ca_sign(x->y, 1), ca_sign(x->z, 1), ca_sign(x->w, 1));
  }
}
// A lane's four f32 wait in the 16 bytes of either tile where its and its neighbour's pieces go.
TTS_DEV void ca_copy_q(uint8_t (*tile)[kCaTileBytes], const float* q, int rh, int r0) {
  const int wl = threadIdx.x & 31;
#pragma unroll 2
  for (int k = 0; k < 32; ++k) {
    const int at = __shfl_sync(0xffffffffu, rh, k);
    ca_copy(&tile[wl & 1][ca_at(r0 + k, wl >> 1)], q + (size_t)max(at, 0) * 128 + wl * 4, at >= 0);
  }
}
// The exponent (biased) of a row whose largest magnitude has these bits, what the row is multiplied
// by and what its scores' factor is then; rows below 2^-112 are scaled like those at it (f32 has no
// finer element there than the pieces hold), infinities and NaN stay what they are.
TTS_DEV uint32_t ca_exponent(uint32_t largest) { return max(largest >> 23, 15u); }
TTS_DEV float ca_scale_up(uint32_t exponent) { return __uint_as_float((268u - exponent) << 23); }
// Factors are kept above 0 (times -infinity) and far below infinity: scores are multiples of 2^-48
// and below 2^39, so a factor of 2^80 parts any two of them as a larger one would.
constexpr float kCaFlat = 1e-30f, kCaSteep = 1.2089258196146292e24f;  // 2^80
TTS_DEV float ca_factor(float c, uint32_t exponent) {
  return fminf(fmaxf(c * __uint_as_float((exponent - 14u) << 23), kCaFlat), kCaSteep);
}
// Leaves the rows' exponents in `exponents` (null: rows of nothing).
TTS_DEV void ca_take_q(uint8_t (*tile)[kCaTileBytes], const float*, int r0, int negate,
                       uint8_t* exponents) {
  const int wl = threadIdx.x & 31;
  uint32_t mine = 0;
  ca_copy_wait();
#pragma unroll 1
  for (int k0 = 0; k0 < 32; k0 += 4) {
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      x[k] = *reinterpret_cast<const float4*>(&tile[wl & 1][ca_at(r0 + k0 + k, wl >> 1)]);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float most =
          fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
      const uint32_t e = ca_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      if (wl == k0 + k) mine = e;
      const float up = ca_scale_up(e);
      x[k] = make_float4(x[k].x * up, x[k].y * up, x[k].z * up, x[k].w * up);
      const __half2 h0 = __floats2half2_rn(x[k].x, x[k].y), h1 = __floats2half2_rn(x[k].z, x[k].w);
      const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
      const __half2 l0 = __floats2half2_rn(x[k].x - b0.x, x[k].y - b0.y),
                    l1 = __floats2half2_rn(x[k].z - b1.x, x[k].w - b1.y);
      const uint32_t to = ca_at(r0 + k0 + k, wl >> 1) + (wl & 1) * 8;
      *reinterpret_cast<uint2*>(&tile[0][to]) =
          make_uint2(ca_sign(*reinterpret_cast<const uint32_t*>(&h0), negate),
                     ca_sign(*reinterpret_cast<const uint32_t*>(&h1), negate));
      *reinterpret_cast<uint2*>(&tile[1][to]) =
          make_uint2(ca_sign(*reinterpret_cast<const uint32_t*>(&l0), negate),
                     ca_sign(*reinterpret_cast<const uint32_t*>(&l1), negate));
    }
  }
  if (exponents) exponents[wl] = uint8_t(mine);
}

// One run of a work tile's units.
struct CaSeg {
  int row0, n, pos0;  // the lane's first row, its new rows, the first one's position
  int flat0, lane, head;
  int unit0, units;   // 0 units: no more work
  int begins, ends;   // whether the run has the work tile's first and last unit
};

template <int kK, int kV, int kParts>  // tiles of K and V in flight; f16 pieces of a query element
struct CaSmem {
  uint8_t ring[kK + kV][kCaTileBytes];  // K's, then V's
  uint8_t q[2][kParts][kCaTileBytes];
  uint64_t full[kK + kV], empty[kK + kV];
  uint64_t q_full[2], s_full[2], h_full[2], h_done[2], p_full[2], o_full[2];
  uint64_t seg_full[kCaSegs], seg_empty[kCaSegs], seg_done[kCaSegs], tail, drain, x_full, x_empty;
  float x_ref[128], x_sum[128];  // the second group's, where one query tile has both groups
  CaSeg seg[kCaSegs];
  int start[4];  // the CTA's first lane, work tile, head and unit
  int count;     // its units
  int4 box_row[2][kCaKeys / 32];  // the loaders' boxes: their pool rows, -1 where none is read
  // f32 queries' exponents: of tiles that the softmax warps load, by tile (read by the warps that
  // wrote them or, of a lone tile, after they have met), of few rows by run (a run's place is
  // written again four runs later, when all warps have left it)
  uint8_t q_exp[kParts - 1 ? 2 : 1][128], few_exp[kCaSegs][32];
  uint32_t tmem;
  uint32_t patience;  // the waits' bound (ca_wait)
};

template <int N>
struct Int {
  static constexpr int value = N;
};

// A run of no more rows than a warp loads at once: its queries are loaded by the warp that walks
// the work, into the other buffer than the run before's if that was one too, while that is at work.
// Any other run's are loaded by the softmax warps, tile tl's into buffer tl, when the run before is
// done (a warp takes about a microsecond for 32 rows: 16 chunks of 512 rows over 512 took 149 us
// with all queries loaded by the one, 106 this way).
TTS_DEV bool ca_few(const CaSeg& s, int gqa) { return s.n * gqa - s.flat0 <= 32; }
TTS_DEV int ca_q_buffer(bool few, bool last_few, int last) {
  return few && last_few ? last ^ 1 : 0;
}

// A softmax thread's query row in a run.
struct CaRow {
  int pr, f, pos, lo;  // in the work tile, flat in the lane; its position, the first it sees
  int rh;              // its row of q and out [rows * heads][128], -1: none
  bool one, few, live, work;  // one query tile; ca_few; a row at all; any in the warp
};

// What a split work tile's part was, one per CTA for the run it takes over from the CTA before
// (slot 0) and one for the run it leaves unfinished to the next (slot 1).
struct CaPart {
  int valid, row0, n, flat0, head, more;
};
constexpr int kCaPartFloats = kCaTile * 130;  // O [32][256] float4, m [256], l [256]

// n / d for 0 <= n < 2^31: n m >> s, m = floor(2^s / d) + 1, s = 31 + ceil(log2 d) (Granlund and
// Montgomery 1994). A division of its own is some twenty instructions to fetch.
struct CaDiv {
  uint32_t m, s;
};
TTS_DEV int operator/(int n, CaDiv d) { return int((uint64_t(uint32_t(n)) * d.m) >> d.s); }

struct CaArgs {
  ChunkAttnRequest r;
  float c;      // |scale| log2 e; f32 queries' rows have their own (ca_factor)
  int negate;   // scale < 0: the queries change sign
  int box;      // rows of a page that one copy takes
  int odd;      // one page per lane, of no multiple of 8 rows
  CaDiv by_page, by_gqa;  // by block_size, by r.gqa
  int wide;     // out is 32-byte aligned: whole sectors at a time (4600 rows of 16 heads, in chunks
                // of up to 701: 138 us, in halves 144)
  CaPart* parts;
  float* part_data;
};

TTS_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Units of 2^32 clocks (about 2 s) of the SM.
TTS_DEV uint32_t ca_clock() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%clock_hi;" : "=r"(t));
  return t;
}
// mbar_wait_warp with its bound on the SM's own clock: the softmax and the MMAs hand over to each
// other several times a unit, and reading the global timer on each hand-over cost more than the
// hand-over. The bound is S.patience to S.patience + 1 units of ca_clock: 1 to 2, and more while
// rows are summed again (ca_repair, which ends by itself), as that may take any time at long
// contexts. (One word and one comparison: waits that looked for such rows' progress themselves took
// 448 single rows over 300 positions from 181 us to 198, 64-bit clocks a long prompt from 431 to
// 437.)
template <typename Smem>
TTS_DEV bool ca_wait(Smem& S, uint64_t* bar, uint32_t parity) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    const uint32_t t0 = ca_clock();
    do {
      ok = mbar_try_wait(bar, parity);
    } while (!ok && ca_clock() - t0 <= *static_cast<volatile uint32_t*>(&S.patience));
  }
  return __all_sync(0xffffffffu, ok);
}

// NaN if any of the three is.
TTS_DEV float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two f32 lanes in one instruction.
TTS_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 y;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return y;
}
TTS_DEV float2 add2(float2 a, float2 b) {
  float2 y;
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
// A row's weights are 2^(c s + bias). Past |ref| = 2^22 both are smaller by a power of two: c s is
// rounded by half a step of itself, beyond 2^27 by more than the weights' room of 2^8, and scores
// that the slope of 2^22 does not part differ by less than f32 sums of 128 products resolve.
struct CaAim {
  float c, bias;
};
TTS_DEV CaAim ca_aim(float c, float ref) {
  const uint32_t e = __float_as_uint(ref) >> 23 & 255u;
  const float less = __uint_as_float((127u - (e > 149u ? e - 149u : 0u)) << 23);
  return ref == -INFINITY ? CaAim{c, 0.f} : CaAim{c * less, kCaBias - ref * less};
}
// The f16 weights of N scores (-inf: not seen), two to a word, and their sum.
template <int N>
TTS_DEV float ca_weights(const uint32_t* v, uint32_t* y, float c, float bias) {
  const float2 c2 = make_float2(c, c), b2 = make_float2(bias, bias);
  // batches of 4 pairs, the exponentials of the next on their way while one is summed and packed
  float2 w[2][4], part[4];
  const auto start = [&](int b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 z = fma2(make_float2(__uint_as_float(v[8 * b + 2 * e]),
                                        __uint_as_float(v[8 * b + 2 * e + 1])), c2, b2);
      w[b & 1][e] = make_float2(ex2(z.x), ex2(z.y));
    }
  };
  start(0);
#pragma unroll
  for (int b = 0; b < N / 8; ++b) {
    if (b < N / 8 - 1) start(b + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = w[b & 1][e];
      part[e] = b == 0 ? x : add2(part[e], x);
      const __half2 h = __floats2half2_rn(x.x, x.y);
      y[4 * b + e] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  const float2 s = add2(add2(part[0], part[1]), add2(part[2], part[3]));
  return s.x + s.y;
}
// Which of columns 0..31 lie in first .. last.
TTS_DEV uint32_t ca_seen(int first, int last) {
  const uint32_t from = first <= 0 ? 0xffffffffu : first > 31 ? 0u : 0xffffffffu << first;
  const uint32_t to = last < 0 ? 0u : last >= 31 ? 0xffffffffu : (2u << last) - 1u;
  return from & to;
}
// max(ref, c times the largest of N scores), NaN if a score is.
template <int N>
TTS_DEV float ca_max(const uint32_t* v, float c, float ref) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < N / 2; ++e)
    m[e % 4] = max3(m[e % 4], __uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
  const float mx = max3(max3(m[0], m[1], m[2]), m[3], m[3]);
  return max3(ref, mx * c, mx * c);
}

// Two results as f16. A mean of f16 values is no larger than the largest of them, but weights are
// rounded and their sum is not: what that takes past f16's largest is brought back to it, and only
// an infinity of the values' own stays one. (Sums of the rounded weights would be exact here and took
// a long prompt from 434 us to 470.)
constexpr float kCaLargest = 65504.f;
TTS_DEV __half2 ca_halves(float x, float y) {
  const auto in = [](float v) {
    return fabsf(v) > kCaLargest && fabsf(v) < 1.01f * kCaLargest ? copysignf(kCaLargest, v) : v;
  };
  return __floats2half2_rn(in(x), in(y));
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
TTS_DEV void st_global_32(void* p, const uint32_t* r) {  // a whole 32-byte sector
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
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
// A shared-memory descriptor moved by `by` 16-byte units (its low 14 bits; they do not overflow).
TTS_DEV uint64_t ca_desc(uint64_t d, int by) {
  return (d & 0xffffffff00000000ull) | uint32_t(uint32_t(d) + by);
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
// The first position that the row at `pos` sees (0 for rows before position 0). The comparison
// keeps the difference in range: a window may be any size, a position as far below 0 as there are
// rows.
TTS_DEV int ca_first(int pos, int window) {
  return window > 0 && pos >= window ? pos + 1 - window : 0;
}
// First unit and number of units of a lane's work tile k (at least one: rows that see nothing are
// written too).
TTS_DEV void ca_units(int n, int pos0, CaDiv gqa, int window, int k, int* first, int* count) {
  const int t0 = k * kCaTile / gqa, t1 = min(n, (k * kCaTile + kCaTile - 1) / gqa + 1);
  const int lo = ca_first(pos0 + t0, window);
  const int last = max(0, pos0 + t1 - 1) / kCaKeys;
  *first = lo / kCaKeys;
  *count = last - *first + 1;
}
TTS_DEV int ca_tiles(int n, int gqa) { return (n * gqa + kCaTile - 1) / kCaTile; }

struct CaLane {
  int row0, n, pos0;
  bool bad;
};
// A lane's rows; a span the block table cannot hold leaves the lane without any.
TTS_DEV CaLane ca_lane(const ChunkAttnRequest& r, int start, int end, int span) {
  CaLane l;
  l.row0 = start;
  l.bad = span < 0 || span > r.max_blocks * r.block_size;
  l.n = l.bad ? 0 : end - start;
  l.pos0 = span - l.n;
  return l;
}
TTS_DEV CaLane ca_lane(const ChunkAttnRequest& r, int i) {
  return ca_lane(r, r.row_start[i], r.row_start[i + 1], r.spans[i]);
}

// The pool row of a lane's position, -1 where the page is outside the pool.
TTS_DEV int ca_pool_row(const CaArgs& a, int lane, int head, int pos) {
  const int block = pos / a.by_page;
  const int page = a.r.block_table[(size_t)lane * a.r.max_blocks + block];
  if (page < 0 || page >= a.r.num_blocks) return -1;
  return (page * a.r.n_kv + head) * a.r.block_size + (pos - block * a.r.block_size);
}

// Eight elements of a query as f32.
TTS_DEV void ca_load8(const float* p, float* x) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
TTS_DEV void ca_load8(const __half* p, float* x) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

// Positions a row does not see have weight 0, but an infinity or NaN among their values makes 0
// times it NaN. Where a row's output is not finite, the warp looks at the values the row's units
// held beyond what it sees and, if one is not finite, sums the row again over what it sees (dims
// 4 lane .. + 3 of the result to each warp lane). Never reached by finite caches. Half a warp takes
// a position, 16 positions' rows are on their way at once: a tile of such rows over a long cache
// should not keep the CTA for long (37 lanes of 128 rows of 8 heads over 8192 positions, the last
// of them NaN: 33 ms, one position at a time 185).
template <typename TQ>
__device__ __noinline__ bool ca_repair(const CaArgs& a, const CaSeg& s, int f, int hi, CaAim aim,
                                       float4* o) {
  const int wl = threadIdx.x & 31, half = wl >> 4, d0 = (wl & 15) * 8;
  const int tok = f / a.by_gqa, head = s.head * a.r.gqa + f - tok * a.r.gqa;
  const int pos = s.pos0 + tok;
  const int u0 = s.unit0 * kCaKeys, u1 = min(hi, (s.unit0 + s.units) * kCaKeys);
  const int lo = ca_first(pos, a.r.window);
  // the pool rows of 32 positions from p on, one a warp lane, -1 from `end` on
  const auto rows_at = [&](int p, int end) {
    return p + wl < end ? ca_pool_row(a, s.lane, s.head, p + wl) : -1;
  };
  const auto piece = [&](const __half* pool, int row) {
    return row < 0 ? make_uint4(0, 0, 0, 0)
                   : *reinterpret_cast<const uint4*>(pool + (size_t)row * 128 + d0);
  };
  bool clean = true;
  const auto look = [&](int from, int end) {
    for (int p = from; p < end; p += 32) {
      const int at = rows_at(p, end);
#pragma unroll 4
      for (int i = 0; i < 32; i += 2) {
        const uint4 v = piece(a.r.v_pool, __shfl_sync(0xffffffffu, at, i + half));
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)  // an all-ones exponent in either half
          clean = clean && (u[e] & 0x7c00u) != 0x7c00u && (u[e] >> 16 & 0x7c00u) != 0x7c00u;
      }
    }
  };
  look(u0, min(lo, u1));
  look(max(u0, pos + 1), u1);
  if (__all_sync(0xffffffffu, clean)) return false;
  float q[8];
  ca_load8(static_cast<const TQ*>(a.r.q) +
               ((size_t)(s.row0 + tok) * a.r.n_kv * a.r.gqa + head) * 128 + d0, q);
  float up = a.negate ? -1.f : 1.f;
  if (sizeof(TQ) == 4) {  // as the scores' queries were
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(q[e]));
    up *= ca_scale_up(ca_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(most))));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] *= up;
  float sum[8] = {};
  const int end = min(u1, pos + 1);
  for (int p = max(u0, lo); p < end; p += 32) {
    const int at = rows_at(p, end);
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += 16) {
      uint4 k[8], v[8];
      int row[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        row[i] = __shfl_sync(0xffffffffu, at, i0 + 2 * i + half);
        k[i] = piece(a.r.k_pool, row[i]);
        v[i] = piece(a.r.v_pool, row[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x[8], y = 0.f;
        ca_load8(reinterpret_cast<const __half*>(&k[i]), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) y = fmaf(q[e], x[e], y);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
        const float w = row[i] < 0 ? 0.f : ex2(fmaf(y, aim.c, aim.bias));
        ca_load8(reinterpret_cast<const __half*>(&v[i]), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = fmaf(w, x[e], sum[e]);
      }
    }
  }
  float out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float lower = sum[e] + __shfl_xor_sync(0xffffffffu, sum[e], 16);
    const float upper = sum[e + 4] + __shfl_xor_sync(0xffffffffu, sum[e + 4], 16);
    const float even = __shfl_sync(0xffffffffu, lower, wl >> 1);
    const float odd = __shfl_sync(0xffffffffu, upper, wl >> 1);
    out[e] = wl & 1 ? odd : even;
  }
  *o = make_float4(out[0], out[1], out[2], out[3]);
  return true;
}

// The CTA's share of the work: all CTAs compute the same totals from the lanes' lengths. Uses the
// (still empty) tile ring as scratch. False where the row starts are not in order.
template <typename Smem>
TTS_DEV bool ca_plan(Smem& S, const CaArgs& a) {
  const int t = threadIdx.x, warp = t >> 5, wl = t & 31;
  const ChunkAttnRequest& r = a.r;
  int* rows = reinterpret_cast<int*>(S.ring[0]);          // [lanes] new rows
  int* pos0 = rows + kChunkMaxLanes;                      // [lanes] the first one's position
  long long* tot = reinterpret_cast<long long*>(pos0 + kChunkMaxLanes);  // [lanes] units
  int* starts = reinterpret_cast<int*>(tot + kChunkMaxLanes);            // [lanes + 1]
  for (int i = t; i <= r.lanes; i += kCaThreads) {
    starts[i] = r.row_start[i];
    if (i < r.lanes) pos0[i] = r.spans[i];
  }
  __syncthreads();
  if (!__syncthreads_and(chunk_starts_ok(starts, r.lanes, r.rows, t, kCaThreads))) return false;
  const auto lane_units = [&](int n, int p, int from, int step) {
    long long u = 0;
    for (int k = from; k < ca_tiles(n, r.gqa); k += step) {
      int first, count;
      ca_units(n, p, a.by_gqa, r.window, k, &first, &count);
      u += count;
    }
    return u;
  };
  bool longer = false;
  for (int i = t; i < r.lanes; i += kCaThreads) {  // a thread a lane, if it has few work tiles
    const CaLane l = ca_lane(r, starts[i], starts[i + 1], pos0[i]);
    if (l.bad && blockIdx.x == 0) atomicOr(r.err, kFlagSpanRange);
    rows[i] = l.n;
    pos0[i] = l.pos0;
    const bool few = ca_tiles(l.n, r.gqa) <= 4;
    tot[i] = few ? lane_units(l.n, l.pos0, 0, 1) * r.n_kv : -1;
    longer = longer || !few;
  }
  if (__syncthreads_or(longer)) {
    for (int i = warp; i < r.lanes; i += kCaThreads / 32) {  // a warp a longer one
      if (tot[i] >= 0) continue;
      long long u = lane_units(rows[i], pos0[i], wl, 32);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      if (wl == 0) tot[i] = u * r.n_kv;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const auto before = [&](long long mine) {  // the sum over lower warp lanes
      long long inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (wl >= o) inc += x;
      }
      return inc - mine;
    };
    // a warp lane owns a run of lanes
    const int each = (r.lanes + 31) / 32, l0 = min(r.lanes, wl * each),
              l1 = min(r.lanes, l0 + each);
    long long mine = 0;
    for (int i = l0; i < l1; ++i) mine += tot[i];
    const long long pre = before(mine);
    const long long all = __shfl_sync(0xffffffffu, pre + mine, 31);
    const long long per = all <= INT_MAX ? (uint32_t(all) + gridDim.x - 1) / gridDim.x
                                         : (all + gridDim.x - 1) / gridDim.x;
    const long long lo = per * blockIdx.x, hi = lo + per < all ? lo + per : all;
    if (wl == 0) S.count = lo < hi ? int(hi - lo) : 0;
    if (lo < hi) {
      // the lane that unit `lo` belongs to, and its place there
      int lane = -1;
      long long rem = lo - pre;
      if (rem >= 0 && rem < mine) {
        lane = l0;
        while (rem >= tot[lane]) rem -= tot[lane++];
      }
      const int owner = __ffs(__ballot_sync(0xffffffffu, lane >= 0)) - 1;
      lane = __shfl_sync(0xffffffffu, lane, owner);
      rem = __shfl_sync(0xffffffffu, rem, owner);
      const int n = rows[lane], p = pos0[lane], tiles = ca_tiles(n, r.gqa);
      for (int k0 = 0; k0 < tiles; k0 += 32) {
        int first = 0, count = 0;
        if (k0 + wl < tiles) ca_units(n, p, a.by_gqa, r.window, k0 + wl, &first, &count);
        const long long here = (long long)count * r.n_kv, low = before(here);
        const unsigned m = __ballot_sync(0xffffffffu, rem >= low && rem < low + here);
        if (m) {
          if (wl == __ffs(m) - 1) {
            S.start[0] = lane;
            S.start[1] = k0 + wl;
            S.start[2] = int(rem - low) / count;
            S.start[3] = int(rem - low) % count;
          }
          break;
        }
        rem -= __shfl_sync(0xffffffffu, low + here, 31);
      }
    }
  }
  __syncthreads();
  return true;
}

template <typename TQ, int kK, int kV, int kParts>
__global__ void __launch_bounds__(kCaThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ CaArgs a) {
  extern __shared__ uint8_t smem_raw[];
  typedef CaSmem<kK, kV, kParts> Smem;
  Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                     ~uintptr_t(1023));
  const int t = threadIdx.x, warp = t >> 5, wl = t & 31;
  const ChunkAttnRequest& r = a.r;
  pdl_launch_dependents();  // the join waits for this grid's end before it reads
  if (t < 2) a.parts[2 * blockIdx.x + t].valid = 0;
  // what does not need the plan goes first, while its loads are on their way
  if (warp == 9) {
    tmem_alloc(&S.tmem, 512);
    tmem_relinquish();
  }
  if (warp == 11) {
    for (uint64_t* b = S.full + wl; b <= &S.x_empty; b += 32) {
      const auto one_of = [b](const uint64_t* s, int n) { return b >= s && b < s + n; };
      const bool warps = one_of(S.q_full, 2) || one_of(S.h_full, 2) || one_of(S.p_full, 2) ||
                         one_of(&S.x_full, 1) || one_of(&S.x_empty, 1);
      mbar_init(b, warps ? 4 : one_of(S.seg_empty, kCaSegs) ? 11 : 1);
    }
    fence_barrier_init();
    if (wl == 0) {
      S.patience = 1;
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  }
  const bool planned = ca_plan(S, a);
  if (!planned && t == 0 && blockIdx.x == 0) atomicOr(r.err, kFlagChunkStarts);
  fence_proxy_async();  // the plan's scratch before the copies into the same memory
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  if (!planned || S.count == 0) {
    if (warp == 9) tmem_dealloc(tmem, 512);
    return;
  }
  bool ok = true;
  int seg_slot = 0;
  uint32_t seg_phase = 0;
  // every role reads the work in order and frees its slot at once
  const auto next_seg = [&](CaSeg* s) {
    if (!ca_wait(S, &S.seg_full[seg_slot], seg_phase)) return false;
    *s = S.seg[seg_slot];
    __syncwarp();
    if (wl == 0) mbar_arrive(&S.seg_empty[seg_slot]);
    if (++seg_slot == kCaSegs) seg_slot = 0, seg_phase ^= 1;
    return true;
  };

  // the block's 384 x 168 registers, dealt out by need: 8 warps x 200 + 4 warps x 104
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 10) {
    // ---- the work walk: units in order of lane, work tile, head
    int lane = S.start[0], k = S.start[1], head = S.start[2], off = S.start[3], left = S.count;
    CaLane l = ca_lane(r, lane);
    int buf = 0;
    bool was_few = false;
    // The queries of run i, if they are this warp's (the first run's never are). Their buffer is
    // free once the scores of the run before are done, of the one before that if both are few. The
    // wait cannot miss its phase: the slot's next run is not out yet, and all before are done.
    const auto load_queries = [&](const CaSeg& s, int i) {
      const bool few = ca_few(s, r.gqa);
      const int free = i - (was_few ? 2 : 1);
      buf = ca_q_buffer(few, was_few, buf);
      was_few = few;
      if (!few || i == 0) return;
      if (free >= 0) ok = ca_wait(S, &S.seg_done[free % kCaSegs], (free / kCaSegs) & 1);
      if (!ok) return;
      const int f = s.flat0 + wl, tok = f / a.by_gqa;
      ca_copy_q(S.q[buf], static_cast<const TQ*>(r.q),
                f < s.n * r.gqa ? ((s.row0 + tok) * r.n_kv + s.head - tok) * r.gqa + f : -1,
                0);  // (the tile's other rows' scores are not read)
      ca_take_q(S.q[buf], static_cast<const TQ*>(r.q), 0, a.negate, S.few_exp[i % kCaSegs]);
      fence_proxy_async();
      __syncwarp();
      if (wl < 4) mbar_arrive(&S.q_full[buf]);
    };
    CaSeg before{};
    for (int i = 0;; ++i) {
      CaSeg s{};
      if (left > 0) {
        int first, count;
        ca_units(l.n, l.pos0, a.by_gqa, r.window, k, &first, &count);
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
      ok = ca_wait(S, &S.seg_empty[seg_slot], seg_phase ^ 1);
      if (!ok) break;
      if (wl == 0) {
        S.seg[seg_slot] = s;
        mbar_arrive(&S.seg_full[seg_slot]);
      }
      __syncwarp();
      if (++seg_slot == kCaSegs) seg_slot = 0, seg_phase ^= 1;
      // its queries, wanted in a few microseconds, into L2
      const int lines = int(sizeof(TQ)) * r.gqa;  // of 128 bytes, per token and kv head
      const int q0 = s.flat0 / a.by_gqa, q1 = min(s.n, (s.flat0 + kCaTile - 1) / a.by_gqa + 1);
      for (int e = wl; i > 0 && e < (q1 - q0) * lines; e += 32)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(
            static_cast<const char*>(r.q) +
            (((size_t)(s.row0 + q0 + e / lines) * r.n_kv + s.head) * lines + e % lines) * 128));
      if (i > 0) load_queries(before, i - 1);
      if (s.units == 0 || !ok) break;
      before = s;
    }
  } else if (warp != 9) {
    // ---- warp 8 K, warp 11 V, by boxes of `box` rows of one page: warp lane g looks up box g, one
    // elected lane issues them all in one go (a copy then takes it about 50 clocks; one per
    // reconvergence of the warp took 240)
    const int v = warp == 11, base = v ? kK : 0, ring = v ? kV : kK;
    const CUtensorMap* map = v ? &tmV : &tmK;
    const int boxes = kCaKeys / a.box;
    int slot = 0;
    uint32_t phase = 0, tail_phase = 0;
    CaSeg s;
    while (ok && (ok = next_seg(&s)) && s.units > 0) {
      const int last = min(s.n, (s.flat0 + kCaTile - 1) / a.by_gqa + 1);
      // the tile's rows see positions lo .. hi - 1; boxes before or behind them are not loaded
      // (their pages may be gone), and their values are zero
      const int lo = ca_first(s.pos0 + s.flat0 / a.by_gqa, r.window), hi = s.pos0 + last;
      const int* table = r.block_table + (size_t)s.lane * r.max_blocks;
      const int end = min(hi, (s.unit0 + s.units) * kCaKeys);
      // this warp lane's box of the next unit: its position, block and (once read) page
      int p = s.unit0 * kCaKeys + wl * a.box;
      const auto block = [&] { return a.odd ? 0 : p / a.by_page; };
      int blk = block(), page = wl < boxes && p < end ? table[blk] : -1;
      for (int j = 0; j < s.units; ++j) {
        const int p0 = (s.unit0 + j) * kCaKeys;
        const bool past = wl < boxes && p + a.box <= lo, seen = wl < boxes && p < hi && !past;
        const bool bad = seen && (page < 0 || page >= r.num_blocks);
        const int row =
            seen && !bad ? (page * r.n_kv + s.head) * r.block_size + (p - blk * r.block_size) : -1;
        const unsigned load = __ballot_sync(0xffffffffu, row >= 0);
        const unsigned flag = __ballot_sync(0xffffffffu, bad);
        const unsigned zero = __ballot_sync(0xffffffffu, bad || (past && v));
        p += kCaKeys;
        blk = block();
        page = wl < boxes && p < end ? table[blk] : -1;  // on its way while this tile is loaded
        const bool tail = v && p0 + kCaKeys > hi;
        uint64_t* full = &S.full[base + slot];
        ok = ca_wait(S, &S.empty[base + slot], phase ^ 1);
        if (!ok) break;
        uint8_t* tile = S.ring[base + slot];
        if (wl < kCaKeys / 8) reinterpret_cast<int*>(S.box_row[v])[wl] = row;
        const auto zero_rows = [&](int r0, int n) {
          for (int e = wl; e < n * 16; e += 32)
            *reinterpret_cast<uint4*>(tile + ca_at(r0 + (e >> 4), e & 15)) =
                make_uint4(0, 0, 0, 0);
        };
        if (flag && wl == 0) atomicOr(r.err, kFlagPageRange);
        if (zero) {  // pages outside the pool read as zero
          for (unsigned m = zero; m; m &= m - 1) zero_rows((__ffs(m) - 1) * a.box, a.box);
          fence_proxy_async();
        }
        __syncwarp();
        if (elect_one()) {
          uint64_t* bar = tail ? &S.tail : full;
          mbar_arrive_expect_tx(bar, uint32_t(__popc(load) * a.box) * 256u);
          for (int b = 0; b < boxes; b += 4) {
            const int4 at = S.box_row[v][b >> 2];
            const auto copy = [&](int i, int from) {
              uint8_t* dst = tile + (b + i) * a.box * 256;
              if (from < 0) return;
              if (a.odd)
                tma_load_3d(dst, map, bar, 0, from, 0);
              else
                tma_load_4d(dst, map, bar, 0, 0, 0, from >> 3);
            };
            copy(0, at.x);
            copy(1, at.y);
            copy(2, at.z);
            copy(3, at.w);
          }
        }
        __syncwarp();
        if (tail) {
          // rows that nothing sees: their stale bits times a weight of 0 could be NaN
          ok = ca_wait(S, &S.tail, tail_phase);
          tail_phase ^= 1;
          if (!ok) break;
          const int keep = max(hi - p0, 0);
          zero_rows(keep, kCaKeys - keep);
          fence_proxy_async();
          __syncwarp();
          if (wl == 0) mbar_arrive(full);
        }
        if (++slot == ring) slot = 0, phase ^= 1;
      }
    }
    if (!ok)  // bounded: copies still on their way
      for (int i = 0; i < ring; ++i) mbar_wait(&S.full[base + i], phase, 100000000ull);
  } else if (warp == 9) {
    // ---- the MMAs. Tile by tile and unit by unit: O_t += P_t.V(j), then S_t = Q_t.K(j + 1) over
    // the P just read (MMAs of one thread run in the order of their issue).
    const uint32_t idesc_s = idesc_f16_f32(128, kCaKeys);
    const uint32_t idesc_o = idesc_f16_f32(128, 128) | (1u << 16);  // B (V) MN-major
    int k_slot = 0, v_slot = 0, buf = 0, run = 0;
    bool was_few = false;
    uint32_t k_phase = 0, v_phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
    const auto next_k = [&] {
      if (++k_slot == kK) k_slot = 0, k_phase ^= 1;
    };
    // descriptors of the first tiles; others differ in the address alone (in 16 bytes)
    constexpr int kTile16 = kCaTileBytes / 16;
    const uint64_t q_desc = smem_desc(smem_u32(S.q), 16, 2048, 2);
    const uint64_t k_desc = smem_desc(smem_u32(S.ring), 16, 2048, 2);
    const uint64_t v_desc = smem_desc(smem_u32(S.ring[kK]), 1024, 2048, 2);
    // S_tl = Q.K^T, Q from buffer `from`
    const auto scores = [&](int tl, int from, int at, uint64_t* done) {
      const uint64_t q = ca_desc(q_desc, from * kParts * kTile16);
      const uint64_t k = ca_desc(k_desc, at * kTile16);
#pragma unroll
      for (int h = 0; h < kParts; ++h)
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          constexpr int kHalf16 = 1024 / 16;
          const int o = (kk >> 2) * kHalf16 + (kk & 3) * 2;
          umma_f16(tmem + tl * 128, ca_desc(q, h * kTile16 + o), ca_desc(k, o), idesc_s,
                   (h | kk) != 0);
        }
      umma_commit(&S.s_full[tl]);
      if (done) umma_commit(done);
    };
    CaSeg s;
    while (ok && (ok = next_seg(&s)) && s.units > 0) {
      // one query tile: units go to the two score buffers in turn, ahead of them the next but one
      const bool one = s.flat0 + 128 >= s.n * r.gqa;
      const int ahead = one ? 2 : 1;
      const bool few = ca_few(s, r.gqa);
      buf = ca_q_buffer(few, was_few, buf);
      was_few = few;
      uint64_t* const done = &S.seg_done[run++ % kCaSegs];  // after the run's last scores
      for (int b = 0; b < 2 && ok; ++b) {
        if (one && b >= s.units) break;
        if (b == 0 || one) ok = ca_wait(S, &S.full[k_slot], k_phase);
        if (ok && (b == 0 || !one)) {
          const int from = one ? buf : b;
          ok = ca_wait(S, &S.q_full[from], q_phase[from]);
          q_phase[from] ^= 1;
        }
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const bool last = s.units == (one ? b + 1 : 1) && (one || b == 1);
          scores(b, one ? buf : b, k_slot, last ? done : nullptr);
          if (one || b == 1) umma_commit(&S.empty[k_slot]);
        }
        __syncwarp();
        if (one || b == 1) next_k();
      }
      for (int j = 0; j < s.units && ok; ++j) {
        const bool more = j + ahead < s.units;
        ok = ca_wait(S, &S.full[kK + v_slot], v_phase);
        const uint64_t vd = ca_desc(v_desc, v_slot * kTile16);
        for (int b = one ? j & 1 : 0; b < (one ? (j & 1) + 1 : 2) && ok; ++b) {
          const auto values = [&](int kk) {
            umma_f16_ts(tmem + 256 + b * 128, tmem + b * 128 + kk * 8,
                        ca_desc(vd, kk * (4096 / 16)), idesc_o, j >= ahead || kk > 0);
          };
          ok = ca_wait(S, &S.h_full[b], p_phase[b]);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kCaHalf / 16; ++kk) values(kk);
            umma_commit(&S.h_done[b]);
          }
          __syncwarp();
          ok = ca_wait(S, &S.p_full[b], p_phase[b]);
          p_phase[b] ^= 1;
          if (ok && more && (b == 0 || one)) ok = ca_wait(S, &S.full[k_slot], k_phase);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = kCaHalf / 16; kk < 8; ++kk) values(kk);
            if (one || b == 1) umma_commit(&S.empty[kK + v_slot]);  // sooner than the scores
            if (more)
              scores(b, one ? buf : b, k_slot,
                     j + ahead == s.units - 1 && (one || b == 1) ? done : nullptr);
            else
              umma_commit(&S.o_full[b]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (more) {
          if (elect_one()) umma_commit(&S.empty[k_slot]);
          __syncwarp();
          next_k();
        }
        if (++v_slot == kV) v_slot = 0, v_phase ^= 1;
      }
    }
    if (!ok) {  // bounded: MMAs still running
      if (elect_one()) umma_commit(&S.drain);
      __syncwarp();
      mbar_wait(&S.drain, 0, 100000000ull);
    }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- softmax and output, one query row a thread
    const int tl = warp >> 2, lane_row = t & 127;
    const uint32_t lanes_at = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes_at + uint32_t(tl * 128);
    const uint32_t o_at = tmem + lanes_at + 256u + uint32_t(tl * 128);
    uint32_t s_phase = 0, o_phase = 0, x_phase = 0;
    const auto rows_of = [&](const CaSeg& s) {
      CaRow w;
      // one query tile only: its units alternate between the two groups of warps
      w.one = s.flat0 + 128 >= s.n * r.gqa;
      w.few = ca_few(s, r.gqa);
      w.pr = (w.one ? 0 : tl * 128) + lane_row;
      w.f = s.flat0 + w.pr;
      w.live = w.f < s.n * r.gqa;
      w.work = __any_sync(0xffffffffu, w.live);
      const int tok = w.f / a.by_gqa;
      w.pos = w.live ? s.pos0 + tok : -1;
      w.lo = ca_first(w.pos, r.window);
      w.rh = w.live ? ((s.row0 + tok) * r.n_kv + s.head - tok) * r.gqa + w.f : -1;
      return w;
    };
    CaSeg s{};
    CaRow w = rows_of(s);
    for (;;) {
      // rows of a warp see contiguous ranges: a unit inside all of them needs no mask
      const int pos_min = __reduce_min_sync(0xffffffffu, w.live ? w.pos : INT_MAX);
      const int lo_max = __reduce_max_sync(0xffffffffu, w.live ? w.lo : 0);
      float ref = w.live ? -INFINITY : 0.f, sum = 0.f;
      CaAim aim;
      bool fresh = true;  // some row has no reference yet
      float c = a.c;      // of scores as they come from the MMAs
      const int step0 = w.one ? tl : 0, steps = w.one ? 2 : 1;
      for (int j = step0; j < s.units; j += steps) {
        ok = ca_wait(S, &S.s_full[tl], s_phase);
        s_phase ^= 1;
        if (!ok) break;
        tc_fence_after();
        if (w.work) {
          const int p0 = (s.unit0 + j) * kCaKeys;
          const bool edge = p0 + kCaKeys - 1 > pos_min || p0 < lo_max;
          const int first = w.lo - p0, last = w.pos - p0;  // columns the row sees
          if (kParts > 1 && j == step0)
            c = ca_factor(a.c, w.few ? S.few_exp[(seg_slot + kCaSegs - 1) % kCaSegs][wl]
                                     : S.q_exp[(w.one ? 0 : tl) & (kParts - 1)][lane_row]);
          if (j == step0) aim = ca_aim(c, ref);
          // the unit's positions in two halves: their scores in x, their weights over them in TMEM
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            uint32_t x[kCaHalf];
            const int c0 = h * kCaHalf;
            tmem_ld32(s_at + c0, x);
            tmem_ld32(s_at + c0 + 32, x + 32);
            tmem_wait_ld();
            tmem_tie32(x);
            tmem_tie32(x + 32);
            if (edge) {
#pragma unroll
              for (int w32 = 0; w32 < 2; ++w32) {
                const uint32_t seen = ca_seen(first - c0 - w32 * 32, last - c0 - w32 * 32);
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (!(seen >> e & 1u)) x[w32 * 32 + e] = 0xff800000u;  // -inf
              }
            }
            float got = 0.f;
            bool raise = ref == -INFINITY, any = fresh;
#pragma unroll 1
            for (int pass = 0; pass < 2; ++pass) {
              if (any) {
                // O holds weights against the old reference: bring it, and the sum, to the new one
                float up = ref;
                if (raise) {
                  up = ca_max<kCaHalf>(x, c, ref);
                  if (up == INFINITY) up = NAN;  // as the row's formula has it
                }
                const float keep = up == -INFINITY ? 1.f : ex2(ref - up);
                ref = up;
                aim = ca_aim(c, ref);
                sum *= keep;
                fresh = __any_sync(0xffffffffu, ref == -INFINITY);
                if (h > 0) {  // the first half's MMAs; before that, S(j) came after all others
                  ok = ca_wait(S, &S.h_done[tl], s_phase ^ 1);
                  if (!ok) break;
                  tc_fence_after();
                }
                if (j > step0 || h > 0) {
#pragma unroll 1
                  for (int i = 0; i < 8; ++i) {
                    float o[16];
                    uint32_t z[16];
                    tmem_ld16(o_at + i * 16, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) z[e] = __float_as_uint(o[e] * keep);
                    tmem_st16(o_at + i * 16, z);
                  }
                }
              }
              uint32_t y[kCaHalf / 2];
              got = ca_weights<kCaHalf>(x, y, aim.c, aim.bias);
              tmem_st16(s_at + c0 / 2, y);
              tmem_st16(s_at + c0 / 2 + 16, y + 16);
              raise = !(got <= kCaMost) && ref == ref;
              any = __any_sync(0xffffffffu, raise);
              if (!any) break;
            }
            if (!ok) break;
            sum += got;
            tmem_wait_st();
            if (h == 0) {  // the MMAs can start on the first half of P
              tc_fence_before();
              __syncwarp();
              if (wl == 0) mbar_arrive(&S.h_full[tl]);
            }
          }
          if (!ok) break;
        } else if (wl == 0) {
          mbar_arrive(&S.h_full[tl]);
        }
        tc_fence_before();
        __syncwarp();
        if (wl == 0) mbar_arrive(&S.p_full[tl]);
      }
      if (!ok) break;
      CaSeg sn{};
      ok = next_seg(&sn);
      if (!ok) break;
      // The next run's queries, unless the walk loads them: this tile's scores are all done, of a
      // lone tile the other group's may not be.
      const CaRow wn = rows_of(sn);
      const bool load = sn.units > 0 && !(wn.one && tl == 1) && !(wn.few && s.units > 0);
      if (load && !w.one)
        ca_copy_q(S.q[tl], static_cast<const TQ*>(r.q), wn.rh, (warp & 3) * 32);
      if (step0 < s.units) {
        ok = ca_wait(S, &S.o_full[tl], o_phase);
        o_phase ^= 1;
        if (!ok) break;
        tc_fence_after();
      }
      float mine = 1.f, other = 0.f;  // what the two groups' O and sums over one query tile count
      if (w.one && s.units > 0) {
        // the second group leaves its O, in the same TMEM lanes, to the first (and does not run
        // ahead of it, to load a next run's queries over this one's)
        if (tl == 1) {
          S.x_ref[lane_row] = ref;
          S.x_sum[lane_row] = sum;
          tc_fence_before();
          __syncwarp();
          if (wl == 0) mbar_arrive(&S.x_full);
          ok = ca_wait(S, &S.x_empty, x_phase);
        } else {
          ok = ca_wait(S, &S.x_full, x_phase);
          tc_fence_after();
          if (s.units > 1) {
            const float ref1 = S.x_ref[lane_row], top = max3(ref, ref1, ref1);
            mine = ref == -INFINITY ? 0.f : ex2(ref - top);
            other = ref1 == -INFINITY ? 0.f : ex2(ref1 - top);
            sum = sum * mine + S.x_sum[lane_row] * other;
            ref = top;
          }
        }
        x_phase ^= 1;
        if (!ok) break;
      }
      if (load) {
        if (w.one) ca_copy_q(S.q[tl], static_cast<const TQ*>(r.q), wn.rh, (warp & 3) * 32);
        // (few rows here: the first run's)
        uint8_t* const exponents = kParts == 1 ? nullptr
                                   : !wn.few   ? &S.q_exp[tl & (kParts - 1)][(warp & 3) * 32]
                                   : warp == 0 ? S.few_exp[0]
                                               : nullptr;
        ca_take_q(S.q[tl], static_cast<const TQ*>(r.q), (warp & 3) * 32, a.negate, exponents);
        fence_proxy_async();
        tc_fence_before();
        __syncwarp();
        if (wl == 0) mbar_arrive(&S.q_full[tl]);
      }
      if (w.work && (!w.one || tl == 0)) {
        // ---- out, or the part of a split work tile
        const bool whole = s.begins && s.ends;
        const float total = ref == -INFINITY ? 0.f : sum;  // 0: the row saw nothing
        const float inv = total == 0.f ? 0.f : 1.f / total;
        float* part = a.part_data + (size_t)(2 * blockIdx.x + (s.begins ? 1 : 0)) * kCaPartFloats;
        float largest = 0.f;  // magnitude of O, NaN if one is
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          uint32_t v[32];
          tmem_ld32(o_at + i * 32, v);
          if (w.one && s.units > 1) {
            uint32_t o1[32];
            tmem_ld32(o_at + 128 + i * 32, o1);
            tmem_wait_ld();
            tmem_tie32(v);
            tmem_tie32(o1);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              v[e] = __float_as_uint(
                  fmaf(__uint_as_float(o1[e]), other, __uint_as_float(v[e]) * mine));
          } else {
            tmem_wait_ld();
            tmem_tie32(v);
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            largest = max3(largest, fabsf(__uint_as_float(v[e])), fabsf(__uint_as_float(v[e + 1])));
          if (!w.live) continue;
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              uint32_t y[8];
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                const __half2 h = __floats2half2_rn(__uint_as_float(v[e + 2 * d]) * inv,
                                                    __uint_as_float(v[e + 2 * d + 1]) * inv);
                y[d] = *reinterpret_cast<const uint32_t*>(&h);
              }
              __half* to = r.out + (size_t)w.rh * 128 + i * 32 + e;
              if (a.wide) {
                st_global_32(to, y);
              } else {
                reinterpret_cast<uint4*>(to)[0] = make_uint4(y[0], y[1], y[2], y[3]);
                reinterpret_cast<uint4*>(to)[1] = make_uint4(y[4], y[5], y[6], y[7]);
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              reinterpret_cast<uint4*>(part)[(i * 8 + e) * kCaTile + w.pr] =
                  make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
        }
        if (!whole && w.live) {
          part[kCaTile * 128 + w.pr] = ref;
          part[kCaTile * 129 + w.pr] = total;
        }
        const bool finite = largest < INFINITY;
        if (whole && w.live && finite && largest * inv > kCaLargest) {  // see ca_halves
          __half* to = r.out + (size_t)w.rh * 128;
          for (int d = 0; d < 128; ++d)
            if (__hisinf(to[d])) to[d] = __float2half(copysignf(kCaLargest, float(to[d])));
        }
        unsigned again = __ballot_sync(0xffffffffu, w.live && !finite);
        const int hi = s.pos0 + min(s.n, (s.flat0 + kCaTile - 1) / a.by_gqa + 1);
        // a bound of waits ahead of the time that the rows take, one for each that passes
        const long long began = clock64();
        long long granted = 0;
        while (again) {
          if ((clock64() - began) >> 32 >= granted) {
            ++granted;
            if (wl == 0) atomicAdd(&S.patience, 1u);
          }
          const int src = __ffs(again) - 1;
          again &= again - 1;
          float4 y;
          const CaAim own = ca_aim(c, ref);
          const CaAim saim{__shfl_sync(0xffffffffu, own.c, src),
                           __shfl_sync(0xffffffffu, own.bias, src)};
          const float sinv = __shfl_sync(0xffffffffu, inv, src);
          const int sf = __shfl_sync(0xffffffffu, w.f, src);
          const int spr = __shfl_sync(0xffffffffu, w.pr, src);
          const int at = __shfl_sync(0xffffffffu, w.rh, src);
          if (!ca_repair<TQ>(a, s, sf, hi, saim, &y)) continue;
          __syncwarp();  // after the row's own stores
          if (whole) {
            __half2* h = reinterpret_cast<__half2*>(r.out + (size_t)at * 128 + wl * 4);
            h[0] = ca_halves(y.x * sinv, y.y * sinv);
            h[1] = ca_halves(y.z * sinv, y.w * sinv);
          } else {
            reinterpret_cast<float4*>(part)[wl * kCaTile + spr] = y;
          }
        }
      }
      if (w.one && tl == 0 && s.units > 0) {  // both groups' O have been read
        tc_fence_before();
        __syncwarp();
        if (wl == 0) mbar_arrive(&S.x_empty);
      }
      if (sn.units == 0) break;
      s = sn;
      w = wn;
    }
  }
  if (!ok) {
    ca_copy_wait();
    if (wl == 0) atomicOr(r.err, kFlagAttnWait);
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
  const int tok = f / a.by_gqa;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint4 y[2];
  __half2* h = reinterpret_cast<__half2*>(y);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[2 * e] = ca_halves(o[e].x * inv, o[e].y * inv);
    h[2 * e + 1] = ca_halves(o[e].z * inv, o[e].w * inv);
  }
  uint4* dst = reinterpret_cast<uint4*>(
      a.r.out + ((size_t)((p.row0 + tok) * a.r.n_kv + p.head - tok) * a.r.gqa + f) * 128 +
      warp * 16);
  dst[0] = y[0];
  dst[1] = y[1];
}

}  // namespace

size_t chunk_attn_workspace(int device) {
  return size_t(num_sms(device)) * 2 * (sizeof(CaPart) + sizeof(float) * kCaPartFloats);
}

template <typename TQ, int kK, int kV, int kParts>
static cudaError_t launch_as(const CUtensorMap& k, const CUtensorMap& v, const CaArgs& a, int ctas,
                             int device, cudaStream_t st) {
  constexpr size_t smem = sizeof(CaSmem<kK, kV, kParts>) + 1024;
  static_assert(smem <= 232448, "227 KB a block");
  {
    // the opt-in shared-memory limit is a per-device function attribute
    static std::mutex mu;
    static bool done[64] = {false};
    std::lock_guard<std::mutex> lock(mu);
    if (device >= 0 && device < 64 && !done[device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(chunk_attn_kernel<TQ, kK, kV, kParts>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
      if (e != cudaSuccess) return e;
      done[device] = true;
    }
  }
  chunk_attn_kernel<TQ, kK, kV, kParts><<<ctas, kCaThreads, smem, st>>>(k, v, a);
  return cudaGetLastError();
}

cudaError_t launch_chunk_attn(const ChunkAttnRequest& r, int device, cudaStream_t st) {
  const uint64_t rows = uint64_t(r.num_blocks) * r.n_kv * r.block_size;
  CUtensorMap tmK, tmV;
  // a copy never leaves its page: the largest power of two that divides the page, 8 rows where
  // only the whole lane is contiguous (pages of 64, 4096 rows over 12288 positions: boxes of 64
  // rows 443 us, of 16 446)
  const bool odd = r.block_size % 8 != 0;
  int box = 8;
  while (!odd && box < kCaKeys && r.block_size % (2 * box) == 0) box *= 2;
  if (!make_tmap_rows_f16(&tmK, r.k_pool, rows, box, odd) ||
      !make_tmap_rows_f16(&tmV, r.v_pool, rows, box, odd)) {
    set_error("chunk_attention: cuTensorMapEncodeTiled failed (pools must be 16-byte aligned)");
    return cudaErrorInvalidValue;
  }
  const int ctas = num_sms(device);
  CaArgs a{};
  a.r = r;
  a.box = box;
  a.odd = odd;
  a.wide = (reinterpret_cast<uintptr_t>(r.out) & 31) == 0;
  const auto div = [](int d) {
    int l = 0;
    while ((1ll << l) < d) ++l;
    return CaDiv{uint32_t((1ull << (31 + l)) / uint32_t(d) + 1), uint32_t(31 + l)};
  };
  a.by_page = div(r.block_size);
  a.by_gqa = div(r.gqa);
  a.negate = r.scale < 0.f;
  // f32 queries: kept in range row by row (ca_factor); f16: here
  const double c = fabs(double(r.scale)) * 1.4426950408889634;
  a.c = r.q_f16 ? float(fmin(fmax(c, double(kCaFlat)), double(kCaSteep)))
                : float(fmin(c, double(FLT_MAX)));
  a.parts = static_cast<CaPart*>(r.workspace);
  a.part_data = reinterpret_cast<float*>(a.parts + 2 * ctas);
  cudaError_t e = r.q_f16 ? launch_as<__half, 3, 2, 1>(tmK, tmV, a, ctas, device, st)
                          : launch_as<float, 2, 1, 2>(tmK, tmV, a, ctas, device, st);
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

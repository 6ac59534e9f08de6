// The tensor-core products of the vocabulary head, on CTA pairs (tcgen05 cta_group::2): one 256 x BN tile per pair of
// SMs, operands by TMA into a ring of shared-memory stages, accumulators double-buffered in TMEM, so that the
// epilogue of a tile runs under the products of the next.  Persistent: one pair of CTAs per pair of SMs walks the tiles.
//
//   STAT, GRAD   logits tile = x w^T; a thread of the epilogue owns one row (a TMEM lane) and 128 of its logits, so
//                the softmax statistics need no exchange between threads, and the row's few targets in those
//                columns are met by walking its ascending list
//   (the loss of a few rows without gradient has a kernel of its own, below)
//   WHOLE        the same of a vocabulary of up to two tiles, whose logits stay in TMEM until the row's softmax is known:
//                a second pass over them makes the row's loss and its gradient.  One launch in place of three and 2 of
//                the 8 N V D operations less: loss and gradients of 2048 rows of 256 against 256 take 28.2 us,
//                37.1 the other way; of 131072 rows of 768 against 512, 527 and 617.  A loss alone is
//                quicker without g (2048 rows of 768 against 512: 18 us, 26), so this is for losses with a backward
//   BWD          dw = g^T x (rows = vocabulary, K = counted rows) and dx = g w (rows = counted rows, K = vocabulary)
//                as one list of tiles: neither product fills whole waves of 74 pairs by itself, the two share g in
//                L2, and a small batch saves a launch.  K is split where there are few tiles; the parts go to fp32
//                slabs that are added in order, not through atomics.
//
// The number of counted rows is known on the device only; every role derives the same tile list from it.  All waits are
// bounded.  No load uses cluster multicast.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "common.cuh"
#include "vocab_gemm.cuh"

namespace pcb {
namespace head {

constexpr int kBM = 128;   // rows per CTA (256 per pair)
constexpr int kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;

template <int MODE, int BN>
struct Cfg {
  static constexpr int A_BYTES = kBM * kBK * 2;
  static constexpr int B_BYTES = (BN / 2) * kBK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int TMEM_COLS = 2 * BN;
  // per epilogue warp: two [32 x 64] bf16 boxes for TMA stores, of which the fp32 path uses one as scratch
  static constexpr int EPI_WARP_BYTES = MODE == HEAD_STAT ? 0 : 8192;
  // WHOLE: (max, sum) of both halves of a row, losses of one, partial sums of the losses
  static constexpr int ROW_BYTES = MODE == HEAD_WHOLE ? kBM * 20 + 8 * kEpiWarps + 8 : 0;
  static constexpr int STAGES_FIT = (232448 - 2048 - kEpiWarps * EPI_WARP_BYTES - ROW_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT > 8 ? 8 : STAGES_FIT;
  static constexpr int EPI_OFF = STAGES * STAGE_BYTES + 1024;
  static constexpr int ROW_OFF = EPI_OFF + kEpiWarps * EPI_WARP_BYTES;
  static constexpr int SMEM_BYTES = ROW_OFF + ROW_BYTES + 1024;
  static_assert(SMEM_BYTES <= 232448, "dynamic shared memory above the 227 KB per-block limit");
  static_assert(8 * (2 * STAGES + 4) + 8 <= 1024, "barriers do not fit behind the ring");
};

struct Shape {   // what the number of counted rows makes of a launch
  int rows;      // counted rows
  int num_n;     // column blocks
  int num_m;     // row blocks (BWD: of dx)
  int kb_dw, kb_dx;   // k-blocks of the whole contraction (STAT, GRAD: kb_dx)
  int dw_tiles;
  int tiles;     // STAT, GRAD: all; BWD: of dx
  int dx_more;   // BWD: the pairs below this one have one dx tile more than the others
  int dx_least;  // dx tiles of the others
  int catch_up;  // dw tiles that the others do in the time of one dx tile
  int dw_splits, dx_splits;   // 0: not wanted
  bool two;      // two-term g
};

struct Tile {
  bool dw;
  int mb, nb, split;
  int kb0, kb1;
};

template <int MODE, int BN>
PCB_DEVICE Shape shape_of(const HeadGemm& a, int pairs) {
  Shape s;
  const int count = *a.count;
  int plan_dw = 0, plan_dx = 0;
  if (MODE == HEAD_BWD) {   // asked for together
    plan_dw = a.plan[0];
    plan_dx = a.plan[1];
  }
  s.rows = min(count, a.N);
  const int r = max(s.rows, 1);   // one tile at least: gradients of a batch without counted rows are zeros
  s.num_m = (r + 2 * kBM - 1) / (2 * kBM);
  s.two = MODE != HEAD_STAT && s.rows <= kTwoTermRows;
  s.dw_tiles = s.kb_dw = s.dx_more = s.dx_least = s.catch_up = s.dw_splits = s.dx_splits = 0;
  if (MODE == HEAD_BWD) {
    if (a.want_dw) s.dw_splits = plan_dw;
    if (a.want_dx) s.dx_splits = plan_dx;
    s.num_n = (a.D + BN - 1) / BN;
    s.kb_dw = (r + kBK - 1) / kBK;
    s.kb_dx = (a.cols + kBK - 1) / kBK;
    s.dw_tiles = (a.cols + 2 * kBM - 1) / (2 * kBM) * s.num_n * s.dw_splits;
    s.tiles = s.num_m * s.num_n * s.dx_splits;
    s.dx_more = s.tiles % pairs;
    s.dx_least = s.tiles / pairs;
    if (s.dx_more > 0 && s.dw_splits > 0) {
      const int k = s.two ? 2 : 1;
      const int c_dx = k * s.kb_dx / s.dx_splits + kTileOverhead, c_dw = k * s.kb_dw / s.dw_splits + kTileOverhead;
      s.catch_up = (c_dx + c_dw / 2) / c_dw;
    }
  } else {
    s.num_n = (a.cols + BN - 1) / BN;
    s.kb_dx = (a.D + kBK - 1) / kBK;
    s.tiles = s.num_m * s.num_n;
  }
  return s;
}

// The u-th tile of a pair; false behind its last.  BWD: dx's few long tiles go round first.  The pairs that got one
// less do dw's first tiles among themselves for that time, then dw's other tiles go round all pairs: the order in
// which pairs become free when all tiles take their expected time, so neighbouring tiles of dw run side by side and
// share their operands in L2, and the pairs end within about one of its tiles of one another.
template <int MODE>
PCB_DEVICE bool tile_at(const HeadGemm& a, const Shape& s, int pair, int pairs, int u, Tile& r) {
  if (MODE == HEAD_WHOLE) {   // a pair takes all columns of its rows
    r.mb = pair + (s.num_n == 2 ? u >> 1 : u) * pairs;
    r.nb = s.num_n == 2 ? u & 1 : 0;
    r.dw = false;
    r.split = 0;
    r.kb0 = 0;
    r.kb1 = s.kb_dx;
    return r.mb < s.num_m;
  }
  if (MODE != HEAD_BWD) {
    const int t = pair + u * pairs;
    if (t >= s.tiles) return false;
    r.dw = false;
    r.split = 0;
    if (a.row_blocks_last) {
      r.nb = t % s.num_n;
      r.mb = t / s.num_n;
    } else {
      r.mb = t % s.num_m;
      r.nb = t / s.num_m;
    }
    r.kb0 = 0;
    r.kb1 = s.kb_dx;
    return true;
  }
  const bool more = pair < s.dx_more;
  const int mine = s.dx_least + (more ? 1 : 0);
  int t;
  r.dw = u >= mine;
  if (!r.dw) {
    t = pair + u * pairs;
  } else {
    const int j = u - mine, fewer = pairs - s.dx_more, early = s.catch_up * fewer;
    if (!more && j < s.catch_up) t = pair - s.dx_more + j * fewer;
    else t = early + pair + (j - (more ? 0 : s.catch_up)) * pairs;
    if (t >= s.dw_tiles) return false;
  }
  const int splits = r.dw ? s.dw_splits : s.dx_splits, kb = r.dw ? s.kb_dw : s.kb_dx;
  r.nb = t % s.num_n;
  t /= s.num_n;
  r.split = t % splits;
  r.mb = t / splits;
  r.kb0 = (int)((long long)kb * r.split / splits);
  r.kb1 = (int)((long long)kb * (r.split + 1) / splits);
  if (s.two) {   // the two terms of g take turns, k-block by k-block
    r.kb0 *= 2;
    r.kb1 *= 2;
  }
  return true;
}

// ---------------------------------------------------------------- epilogues of the logits
PCB_DEVICE void load32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld_32x32b_x32(taddr, r);
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
}

// v[o] for a run-time o: a tree of selects, since registers have no run-time index
PCB_DEVICE float pick32(const float (&v)[32], int o) {
  float a[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) a[j] = (o & 16) ? v[16 + j] : v[j];
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1) {
#pragma unroll
    for (int j = 0; j < w; ++j) a[j] = (o & w) ? a[w + j] : a[j];
  }
  return a[0];
}

// One packed row's part of the target list: the entries whose ids fall in this thread's 128 columns.  Its loads depend on
// one another (row -> first entry -> ids): each of the three steps only asks, and the next one, 32 columns of
// arithmetic later, uses the answer.  The next kAhead entries are kept in registers, so that one is asked for long
// before it is met.
struct RowTargets {
  static constexpr int kAhead = 4;
  static constexpr int kNone = 0x7fffffff;
  bool live;        // a counted row
  float2 norm;      // GRAD: p = 2^(c l - x) y
  int n, m;         // the row's place in the batch and among the packed rows
  int lo;           // vocabulary id of the first of the 128 columns
  int entry, end;   // next entry of the row's list, and the first behind these columns
  int id[kAhead];   // its id and those behind it; kNone behind `end`
  float q[kAhead];  // their weights (GRAD)

  template <int MODE>
  PCB_DEVICE void ask_row(const HeadGemm& h, int packed, int col0, int rows) {
    m = packed;
    lo = h.v0 + col0;
    live = packed < rows;
    const int at = max(min(packed, rows - 1), 0);
    norm = MODE == HEAD_GRAD ? h.norm[at] : make_float2(0.f, 0.f);
    n = h.start != nullptr ? h.row[at] : h.ids[at];   // class targets stand by packed row
  }
  PCB_DEVICE void ask_entries(const HeadGemm& h) {
    if (h.start == nullptr) return;
    if (!live) n = 0;   // with no row counted at all there is no first one either
    const unsigned short* s = h.start + (long long)(lo >> 7) * h.N + n;
    entry = s[0];
    end = s[h.N];
  }
  template <int MODE>
  PCB_DEVICE void ask_ids(const HeadGemm& h) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      id[i] = kNone;
      q[i] = 1.f;
    }
    if (h.start == nullptr) {
      if (live && n >= lo && n < lo + 128) id[0] = n;
      entry = n = end = 0;
    } else {
      if (!live) end = entry;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fill<MODE>(h, i);
    }
  }
  template <int MODE>
  PCB_DEVICE void fill(const HeadGemm& h, int i) {   // slot i: entry + i
    id[i] = kNone;
    if (entry + i < end) {
      const long long at = (long long)n * h.K + entry + i;
      id[i] = h.ids[at];
      if (MODE != HEAD_STAT) q[i] = h.q[at];
    }
  }
  PCB_DEVICE float* z(const HeadGemm& h) const { return h.z + (long long)m * h.K + entry; }
  template <int MODE>
  PCB_DEVICE void advance(const HeadGemm& h) {
    ++entry;
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) {
      id[i] = id[i + 1];
      q[i] = q[i + 1];
    }
    fill<MODE>(h, kAhead - 1);
  }
};

PCB_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// (a0, a1) * b + (c, c)
PCB_DEVICE void scale2(float& d0, float& d1, float a0, float a1, float b, float c) { ffma2v(d0, d1, a0, a1, b, c, c); }
PCB_DEVICE void add2(float& d0, float& d1, float a0, float a1) {
  asm("{\n\t.reg .b64 ra, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rd, {%0, %1};\n\t"
      "add.rn.f32x2 rd, rd, ra;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "+f"(d0), "+f"(d1)
      : "f"(a0), "f"(a1));
}

PCB_DEVICE void mul2(float& d0, float& d1, float a0, float a1, float b) {
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %4};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b));
}

// tcgen05.wait::ld that names the registers it completes, so that no use of them moves above it while the next
// load is in flight
PCB_DEVICE void wait32(uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
        "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
        "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
        "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}

// the other accumulator's part of 32 logits
PCB_DEVICE void add_half(uint32_t taddr, uint32_t (&v)[32]) {
  uint32_t o[32];
  tmem_ld_32x32b_x32(taddr + 256, o);
  wait32(o);
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(o[j]));
}

// 32 logits, `nvalid` of them in the vocabulary, joined to a running (max, sum 2^(c l - max))
PCB_DEVICE void join32(float c, float (&v)[32], int nvalid, float& mx, float& sum) {
  if (nvalid < 32) {   // warp-uniform
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = j < nvalid ? v[j] : -INFINITY;
  }
  float cm[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) cm[j] = max3(v[8 * j], v[8 * j + 1], v[8 * j + 2]);
#pragma unroll
  for (int j = 0; j < 4; ++j) cm[j] = max3(cm[j], v[8 * j + 3], v[8 * j + 4]);
#pragma unroll
  for (int j = 0; j < 4; ++j) cm[j] = max3(cm[j], v[8 * j + 5], v[8 * j + 6]);
#pragma unroll
  for (int j = 0; j < 4; ++j) cm[j] = fmaxf(cm[j], v[8 * j + 7]);
  const float nm = fmaxf(mx, max3(fmaxf(cm[0], cm[1]), cm[2], cm[3]) * c);
  const float ref = nm == -INFINITY ? 0.f : nm;
  float s[8] = {};
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float e0, e1;
    scale2(e0, e1, v[j], v[j + 1], c, -ref);
    add2(s[j & 7], s[(j & 7) + 1], ex2_approx(e0), ex2_approx(e1));
  }
#pragma unroll
  for (int j = 0; j < 4; j += 2) add2(s[j], s[j + 1], s[j + 4], s[j + 5]);
  add2(s[0], s[1], s[2], s[3]);
  sum = fmaf(sum, ex2_approx(mx - ref), s[0] + s[1]);
  mx = nm;
}

// (max, sum 2^(c l - max)) of this thread's 128 logits, in one pass with a running maximum, and the logits at the
// row's targets.  The maximum stays in units of c l, and the sum is taken against that rounded value, so the
// log-sum-exp made of the pair carries no error of the product c * max.  The next 32 columns come from TMEM while
// these are worked on; `between(i)` runs after 32 columns.
template <bool HALVES, typename F>
PCB_DEVICE void stat128(const HeadGemm& a, RowTargets& r, uint32_t taddr, int col0, F between) {
  float mx = -INFINITY, sum = 0.f;
  uint32_t buf[2][32];
  tmem_ld_32x32b_x32(taddr, buf[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    wait32(buf[i & 1]);
    if constexpr (HALVES) add_half(taddr + 32 * i, buf[i & 1]);
    if (i < 3) tmem_ld_32x32b_x32(taddr + 32 * (i + 1), buf[(i + 1) & 1]);
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(buf[i & 1][j]);
    while (r.id[0] < r.lo + 32 * (i + 1)) {
      *r.z(a) = pick32(v, r.id[0] - r.lo - 32 * i);
      r.advance<HEAD_STAT>(a);
    }
    __syncwarp();
    join32(a.c, v, a.cols - (col0 + 32 * i), mx, sum);
    between(i);
  }
  if (r.live) a.part[(long long)(r.lo >> 7) * a.N + r.m] = make_float2(mx, sum);
}

// 128 columns of softmax - target distribution as bf16, 64 at a time handed to `store` (high terms, and with TWO the low
// ones).  The factor 1 / count is applied in fp32 behind the products that read them: rounding a shared factor into
// every entry would bias all of them alike.
template <bool TWO, bool HALVES, typename F, typename S>
PCB_DEVICE void grad128(const HeadGemm& a, RowTargets& r, uint32_t taddr, int col0, F between, S store) {
  const bool all = __all_sync(0xffffffffu, r.live);
  uint32_t buf[2][32];
  uint32_t hi[32], low[TWO ? 32 : 1];
  tmem_ld_32x32b_x32(taddr, buf[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    wait32(buf[i & 1]);
    if constexpr (HALVES) add_half(taddr + 32 * i, buf[i & 1]);
    if (i < 3) tmem_ld_32x32b_x32(taddr + 32 * (i + 1), buf[(i + 1) & 1]);
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      float e0, e1;
      scale2(e0, e1, __uint_as_float(buf[i & 1][j]), __uint_as_float(buf[i & 1][j + 1]), a.c, -r.norm.x);
      mul2(v[j], v[j + 1], ex2_approx(e0), ex2_approx(e1), r.norm.y);
    }
    if (!all) {   // what stands in a row that is not counted may be anything
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = r.live ? v[j] : 0.f;
    }
    const int nvalid = a.cols - (col0 + 32 * i);   // warp-uniform
    if (nvalid < 32) {   // the rest of the last panel: K of dx's product
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = j < nvalid ? v[j] : 0.f;
    }
    while (r.id[0] < r.lo + 32 * (i + 1)) {
      const int o = r.id[0] - r.lo - 32 * i;
      const float q = r.q[0];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] -= j == o ? q : 0.f;
      r.advance<HEAD_GRAD>(a);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t p = pack_bf16x2(v[2 * j], v[2 * j + 1]);
      hi[16 * (i & 1) + j] = p;
      if constexpr (TWO) low[16 * (i & 1) + j] = pack_bf16x2(v[2 * j] - bf16_lo(p), v[2 * j + 1] - bf16_hi(p));
    }
    if (i & 1) {
      store(i >> 1, hi, false);
      if constexpr (TWO) store(i >> 1, low, true);
    }
    between(i);
  }
}

// ---------------------------------------------------------------- stores
// TMA store that adds the fp32 box to what is there; one launch adds to a place once
PCB_DEVICE void tma_add_2d(const CUtensorMap* map, const void* smem_src, int c0, int c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
               : "memory");
}

// a lane's 64 bf16 as its row of the 128-byte-swizzled [32 x 64] box, written by one TMA store; the two boxes of a warp
// alternate
PCB_DEVICE void store_box64(const CUtensorMap* map, uint8_t* stg, int& box_at, const uint32_t (&pk)[32], int col, int row,
                            int lane) {
  uint8_t* box = stg + box_at * 4096;
  box_at ^= 1;
  if (lane == 0) bulk_group_wait_read<1>();   // the store that last read this box is done with it
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
        make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, box, col, row);
    bulk_group_commit();
  }
}

// Behind a wait that ran out, copies into this block's shared memory and matrix instructions that read it or write TMEM may
// still be on their way, and the barriers that they would have completed may lie in the other CTA.  A thread that sees
// the abort stays 2 ms, a thousand times as long as any of them takes, before it meets the block's last barrier, so none
// of them finds the memory in other hands.
constexpr long long kSettleCycles = 4000000;
PCB_DEVICE void settle() {
  const long long t0 = clock64();
  while (clock64() - t0 < kSettleCycles) __nanosleep(1000);
}

PCB_DEVICE void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// whether `p` holds for all of them
PCB_DEVICE bool bar_and(int id, int threads, bool p) {
  int r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %1, 0;\n\tbar.red.and.pred b, %2, %3, a;\n\tselp.s32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"((int)p), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

// The accumulator of this warp is free again, at the leader's barrier.  Relaxed: what the leader waits for is that the loads
// from TMEM are complete, which tcgen05.wait::ld and the fence before this see to; a release at cluster scope would also wait
// for this thread's own loads and stores in global memory, 1500 cycles in the other CTA at every tile (epilogues of
// 128 columns of statistics 3300 cycles in the leader, 4800 in the other).
PCB_DEVICE void arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---------------------------------------------------------------- WHOLE's epilogue
// Two threads share a row: each owns 128 columns of every tile.  The first pass makes their softmax statistics, which
// the two exchange; the second the row's entries of g and, where it meets a target, the loss.  Both go through 32 columns
// at a time in a loop that is not unrolled: most launches run this code once on an SM, and fetching it counts (2048
// rows, 256 x 256: 13.1 us for the launch, 14.3 with the four steps written out; 512 rows, 260 x 256, 16 targets
// each: 19.2, 22.6).
PCB_DEVICE void whole_rows(const HeadGemm& a, const Shape& sh, uint8_t* smem, uint8_t* stg, const CUtensorMap* tmC,
                           uint32_t tmem_base, uint64_t* tfull, const uint32_t (&tempty_leader)[2], int pair, int pairs,
                           uint32_t rank, volatile int* abort_flag) {
  constexpr int kEpi = 32 * kEpiWarps;
  float2* stats = reinterpret_cast<float2*>(smem);                          // [2][kBM]
  float* losses = reinterpret_cast<float*>(smem + kBM * 16);                // [kBM]
  double* sums = reinterpret_cast<double*>(smem + kBM * 20);
  volatile int* last = reinterpret_cast<volatile int*>(sums + kEpiWarps);
  const int tid = threadIdx.x - 64, lane = tid & 31, q = (threadIdx.x >> 5) & 3, half = tid >> 7;
  const int mine = q * 32 + lane;
  Tile tile;
  RowTargets ahead;
  bool all_ok = true;
  auto row_of = [&](const Tile& t) { return t.mb * 2 * kBM + (int)rank * kBM + q * 32; };
  if (tile_at<HEAD_WHOLE>(a, sh, pair, pairs, 0, tile)) {
    ahead.ask_row<HEAD_WHOLE>(a, row_of(tile) + lane, half * 128, sh.rows);
    ahead.ask_entries(a);
    ahead.ask_ids<HEAD_WHOLE>(a);
  }
  for (int u = 0; tile_at<HEAD_WHOLE>(a, sh, pair, pairs, u, tile); u += sh.num_n) {
    const int row0 = row_of(tile);
    const bool live = row0 + lane < sh.rows;
    const int place = live ? a.row[row0 + lane] : 0;
    float mx = -INFINITY, sum = 0.f;
    bool ok = true;
#pragma unroll 1
    for (int nb = 0; nb < sh.num_n; ++nb) {
      const int acc = (u + nb) & 1, col0 = nb * 256 + half * 128;
      // behind a wait that ran out the barriers below are still met, and both threads of a row leave together; the lanes of
      // a warp are together again before its loads from TMEM
      ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], ((u + nb) >> 1) & 1, a.err, kErrTimeoutTmemFull, abort_flag)) && ok;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256 + half * 128;
#pragma unroll 1
      for (int i = 0; i < 4 && col0 + 32 * i < a.cols; ++i) {
        float v[32];
        load32(taddr + 32 * i, v);
        join32(a.c, v, a.cols - (col0 + 32 * i), mx, sum);
      }
    }
    stats[half * kBM + mine] = make_float2(mx, sum);
    ok = bar_and(1 + q, 64, ok);
    const float2 s0 = stats[mine], s1 = stats[kBM + mine];
    const float m = fmaxf(s0.x, s1.x), ref = m == -INFINITY ? 0.f : m;
    const float tot = s0.y * exp2f(s0.x - ref) + s1.y * exp2f(s1.x - ref);
    const float lt = log2f(tot), over = 1.f / tot;
    float l = 0.f;
#pragma unroll 1
    for (int nb = 0; nb < sh.num_n; ++nb) {
      const int acc = (u + nb) & 1, col0 = nb * 256 + half * 128;
      RowTargets r = ahead;
      Tile after;
      const bool more = tile_at<HEAD_WHOLE>(a, sh, pair, pairs, u + nb + 1, after);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256 + half * 128;
      uint4 low[4];   // of the panel's first half
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        if (more) {   // the next tile's targets, under this one's arithmetic
          if (i == 0) ahead.ask_row<HEAD_WHOLE>(a, row_of(after) + lane, after.nb * 256 + half * 128, sh.rows);
          if (i == 1) ahead.ask_entries(a);
          if (i == 2) ahead.ask_ids<HEAD_WHOLE>(a);
        }
        const int col = col0 + 32 * i, panel = col / 64;
        if (64 * panel >= a.cols) continue;   // warp-uniform
        float z[32], v[32];
        load32(taddr + 32 * i, z);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float e0, e1;
          scale2(e0, e1, z[j], z[j + 1], a.c, -ref);
          mul2(v[j], v[j + 1], ex2_approx(e0), ex2_approx(e1), over);
        }
        const int nvalid = live ? a.cols - col : 0;   // what stands in a row that is not counted may be anything
        if (!__all_sync(0xffffffffu, nvalid >= 32)) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = j < nvalid ? v[j] : 0.f;
        }
        // a panel's box of high terms and one of low terms, as TMA stores them; until the latter is filled, each lane's row of
        // it holds its 32 entries while the targets are taken off
        if ((i & 1) == 0) {
          if (lane == 0) bulk_group_wait_read<0>();   // the last panel's stores are done with the boxes
          __syncwarp();
        }
        uint8_t* box = stg + lane * 128;
        float4* cells = reinterpret_cast<float4*>(box + 4096);
        const int end = r.lo + 32 * (i + 1);
        if (r.id[0] < end) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            cells[j ^ (lane & 7)] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          do {
            const int o = r.id[0] - r.lo - 32 * i;
            const float w = r.q[0];
            // sum_k q_k (log2 q_k - log2 p_k); the difference of the logit and ref first, in one rounding; 0 log 0 = 0
            if (w != 0.f) l += w * (log2f(w) + (fmaf(-a.c, pick32(z, o), ref) + lt));
            reinterpret_cast<float*>(cells + ((o >> 2) ^ (lane & 7)))[o & 3] -= w;
            r.advance<HEAD_WHOLE>(a);
          } while (r.id[0] < end);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 f = cells[j ^ (lane & 7)];
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) p[k] = pack_bf16x2(v[8 * j + 2 * k], v[8 * j + 2 * k + 1]);
          const int at = (4 * (i & 1) + j) ^ (lane & 7);
          reinterpret_cast<uint4*>(box)[at] = make_uint4(p[0], p[1], p[2], p[3]);
          if (sh.two) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              p[k] = pack_bf16x2(v[8 * j + 2 * k] - bf16_lo(p[k]), v[8 * j + 2 * k + 1] - bf16_hi(p[k]));
            if (i & 1) {
              reinterpret_cast<uint4*>(cells)[j ^ (lane & 7)] = low[j];
              reinterpret_cast<uint4*>(cells)[at] = make_uint4(p[0], p[1], p[2], p[3]);
            } else {
              low[j] = make_uint4(p[0], p[1], p[2], p[3]);
            }
          }
        }
        if (i & 1) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(tmC, stg, 0, panel * a.g_rows + row0);
            if (sh.two) tma_store_2d(tmC, stg + 4096, 0, panel * a.g_rows + row0 + a.g_low);
            bulk_group_commit();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(tempty_leader[acc]);
    }
    if (half) losses[mine] = l;
    bar_sync(1 + q, 64);
    if (!half && live) a.loss[place] = (l + losses[mine]) * a.factor;
    all_ok = ok;
    if (!ok) break;
  }
  if (lane == 0) bulk_group_wait_all();   // every TMA store has landed
  if (a.total == nullptr) return;
  if (!all_ok) record_error(a.err, kErrTimeoutTmemFull);   // known to the last block, whichever role gave up first
  bar_sync(5, kEpi);
  if (tid == 0) *last = arrive_last(a.done, (int)gridDim.x);
  bar_sync(5, kEpi);
  if (!*last) return;
  add_losses<kEpi>(a.loss, a.N, sh.rows, a.mean, a.err, a.total, a.inverse, sums, tid, [] { bar_sync(5, kEpi); });
}

PCB_DEVICE bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

PCB_DEVICE void store4(float* c, float (&o)[4], int nv, bool add) {
  if (nv == 4 && aligned(c, 16)) {
    float4* p = reinterpret_cast<float4*>(c);
    if (add) {
      const float4 f = *p;
      o[0] += f.x; o[1] += f.y; o[2] += f.z; o[3] += f.w;
    }
    *p = make_float4(o[0], o[1], o[2], o[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < nv) c[j] = add ? c[j] + o[j] : o[j];
  }
}
PCB_DEVICE void store4(__nv_bfloat16* c, float (&o)[4], int nv, bool add) {
  if (nv == 4 && aligned(c, 8)) {
    uint2* p = reinterpret_cast<uint2*>(c);
    if (add) {
      const uint2 u = *p;
      o[0] += bf16_lo(u.x); o[1] += bf16_hi(u.x); o[2] += bf16_lo(u.y); o[3] += bf16_hi(u.y);
    }
    *p = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < nv) c[j] = __float2bfloat16_rn(add ? __bfloat162float(c[j]) + o[j] : o[j]);
  }
}

// The tensor cores cut a sum off at every step, which takes D / 16 units of its last digit from a logit.  A batch of one
// row block is bound by reading w and needs no second accumulator to work ahead: with HALVES the two take half of the
// sum each, and the losses come out at half of the error (32 rows of 2048 against 32000: 4e-7 in 38 us, 9e-7 in 36
// with the tiles overlapped; below 1024 columns the error is under half of that and the overlap stays).  Both logits'
// modes go by the same rule: what a row that is sure of its target has in p - q is the sum of its other entries.
static bool in_halves(int N, int D) { return N <= kTwoTermRows && D >= 1024; }

// ---------------------------------------------------------------- kernel
// STAT, GRAD, WHOLE: tmA = packed x, tmX = x, tmB = w, tmC = g.   BWD: tmA = g, tmB = w, tmC = dw, tmD = packed x, tmX = x,
// tmS = fp32 slabs.
template <int MODE, int BN, bool HALVES>
__global__ void __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmD,
                const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmS, const HeadGemm a) {
  using C = Cfg<MODE, BN>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&tfull[s], 1);
      mbar_init(&tempty[s], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    if (MODE != HEAD_STAT) prefetch_tmap(&tmC);
    if (MODE == HEAD_BWD) {
      prefetch_tmap(&tmD);
      prefetch_tmap(&tmS);
    }
    prefetch_tmap(&tmX);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();   // barriers of both CTAs initialised, TMEM allocated in both
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_begin();
  const Shape sh = shape_of<MODE, BN>(a, num_pairs);
  Tile tile;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer (both CTAs) ----------------
      const bool whole = a.dense && sh.rows == a.N;
      const CUtensorMap* x = whole ? &tmX : MODE == HEAD_BWD ? &tmD : &tmA;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = 0; ok && tile_at<MODE>(a, sh, pair_id, num_pairs, u, tile); ++u) {
        const int m0 = tile.mb * 2 * kBM + rank * kBM;
        const int n0 = tile.nb * BN + rank * (BN / 2);
        for (int kb = tile.kb0; kb < tile.kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, a.err, kErrTimeoutEmpty, abort_flag)) { ok = false; break; }
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * C::STAGE_BYTES);
          uint8_t* sa = smem + stage * C::STAGE_BYTES;
          uint8_t* sb = sa + C::A_BYTES;
          if (MODE == HEAD_BWD) {
            const int k0 = (sh.two ? kb >> 1 : kb) * kBK;
            const int low = sh.two && (kb & 1) ? a.g_low : 0;
#pragma unroll
            for (int p = 0; p < kBM / 64; ++p) {
              const int panel = tile.dw ? m0 / 64 + p : k0 / 64, at = tile.dw ? k0 : m0 + 64 * p;
              tma_load_2d_pair(sa + p * 8192, &tmA, &full[stage], 0, panel * a.g_rows + at + low);
            }
#pragma unroll
            for (int p = 0; p < BN / 128; ++p)
              tma_load_2d_pair(sb + p * 8192, tile.dw ? x : &tmB, &full[stage], n0 + 64 * p, k0);
          } else {
            tma_load_2d_pair(sa, x, &full[stage], kb * kBK, m0);
            tma_load_2d_pair(sb, &tmB, &full[stage], kb * kBK, n0);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    if ((MODE == HEAD_GRAD || MODE == HEAD_WHOLE) && lane == 0 && !leader && pair_id == 0 && a.v0 == 0) plan_splits(a, sh.rows, a.bwd_pairs, a.plan);
    if (lane == 0 && leader) {
      // ---------------- MMA issuer (leader only) ----------------
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int u = 0; ok && tile_at<MODE>(a, sh, pair_id, num_pairs, u, tile); ++u) {
        // Shared-memory descriptors advance by additions to their low words (address / 16): the issue of one k-block has
        // to take less than the 512 cycles that its matrix instructions do.
        const bool a_mn = MODE == HEAD_BWD && tile.dw;
        constexpr bool b_mn = MODE == HEAD_BWD;
        const uint32_t idesc = make_idesc_bf16(2 * kBM, BN, a_mn, b_mn);
        const uint64_t a0 = a_mn ? make_smem_desc(smem_u32(smem), 8192, 1024, 2) : make_smem_desc(smem_u32(smem), 16, 1024, 2);
        const uint64_t b0 = make_smem_desc(smem_u32(smem) + C::A_BYTES, b_mn ? 8192 : 16, 1024, 2);
        const uint32_t a_step = a_mn ? 2048 / 16 : 32 / 16;
        constexpr uint32_t b_step = b_mn ? 2048 / 16 : 32 / 16;
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1u, a.err, kErrTimeoutTmemEmpty, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = tile.kb0; kb < tile.kb1; ++kb) {
          if (!mbar_wait(&full[stage], phase, a.err, kErrTimeoutFull, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = a0 + static_cast<uint32_t>(stage) * (C::STAGE_BYTES / 16);
          const uint64_t bd = b0 + static_cast<uint32_t>(stage) * (C::STAGE_BYTES / 16);
          uint32_t d = d_tmem;
          bool fresh = kb == tile.kb0;
          if (HALVES && kb >= sh.kb_dx / 2) {
            d += BN;
            fresh = kb == sh.kb_dx / 2;
          }
          umma_bf16_pair(d, ad, bd, idesc, fresh ? 0u : 1u);
#pragma unroll
          for (int k = 1; k < kBK / 16; ++k) umma_bf16_pair(d, ad + k * a_step, bd + k * b_step, idesc, 1u);
          umma_commit_pair(&empty[stage], 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair(&tfull[acc], 0x3);
        if (!HALVES) acc ^= 1;   // two halves: always the same pair of accumulators
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  } else if (MODE == HEAD_WHOLE) {
    const uint32_t tempty_leader[2] = {mapa_shared(smem_u32(&tempty[0]), 0), mapa_shared(smem_u32(&tempty[1]), 0)};
    whole_rows(a, sh, smem + C::ROW_OFF, smem + C::EPI_OFF + (warp - 2) * C::EPI_WARP_BYTES, &tmC, tmem_base, tfull,
               tempty_leader, pair_id, num_pairs, rank, abort_flag);
  } else {
    // ---------------- epilogue warps (both CTAs, 128 rows each) ----------------
    const int q = warp & 3;
    const int half = (warp - 2) >> 2;
    const uint32_t tempty_leader0 = mapa_shared(smem_u32(&tempty[0]), 0);
    const uint32_t tempty_leader1 = mapa_shared(smem_u32(&tempty[1]), 0);
    uint8_t* stg = smem + C::EPI_OFF + (warp - 2) * C::EPI_WARP_BYTES;
    int acc = 0;
    uint32_t acc_phase = 0;
    int box_at = 0;
    float scale = 1.f;
    if (MODE == HEAD_BWD && sh.dw_splits == 1) {
      scale = a.alpha;
      if (a.scale != nullptr) scale *= *a.scale;
      if (a.scale2 != nullptr) scale *= *a.scale2;
    }
    RowTargets ahead;
    if (MODE != HEAD_BWD && tile_at<MODE>(a, sh, pair_id, num_pairs, 0, tile)) {
      ahead.template ask_row<MODE>(a, tile.mb * 2 * kBM + rank * kBM + q * 32 + lane, tile.nb * BN + half * 128, sh.rows);
      ahead.ask_entries(a);
      ahead.template ask_ids<MODE>(a);
    }
    for (int u = 0; tile_at<MODE>(a, sh, pair_id, num_pairs, u, tile); ++u) {
      const int row0 = tile.mb * 2 * kBM + rank * kBM + q * 32;
      const int n0 = tile.nb * BN;
      // the next tile's rows and targets are fetched under this one's arithmetic
      RowTargets r = ahead;
      int row0_next = 0, n0_next = 0, rows_next = 0;
      Tile after;
      if (MODE != HEAD_BWD && tile_at<MODE>(a, sh, pair_id, num_pairs, u + 1, after)) {
        row0_next = after.mb * 2 * kBM + rank * kBM + q * 32;
        n0_next = after.nb * BN;
        rows_next = sh.rows;
      }
      auto between = [&](int i) {
        if (i == 0) ahead.template ask_row<MODE>(a, row0_next + lane, n0_next + half * 128, rows_next);
        if (i == 1) ahead.ask_entries(a);
        if (i == 2) ahead.template ask_ids<MODE>(a);
      };
      // the warp leaves together: what follows is warp-wide
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, a.err, kErrTimeoutTmemFull, abort_flag))) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN);
      if (MODE == HEAD_STAT) {
        stat128<HALVES>(a, r, tbase + half * 128, n0 + half * 128, between);
      } else if (MODE == HEAD_GRAD) {
        auto store = [&](int b, const uint32_t (&pk)[32], bool low) {
          const int col = n0 + half * 128 + 64 * b;
          if (col < a.cols)   // warp-uniform
            store_box64(&tmC, stg, box_at, pk, 0, col / 64 * a.g_rows + row0 + (low ? a.g_low : 0), lane);
        };
        if (HALVES || sh.two) grad128<true, HALVES>(a, r, tbase + half * 128, n0 + half * 128, between, store);
        else grad128<false, false>(a, r, tbase + half * 128, n0 + half * 128, between, store);
      } else if (tile.dw && a.dw_tma && sh.dw_splits == 1) {
#pragma unroll 1
        for (int c2 = half; c2 < BN / 64; c2 += 2) {
          const int col = n0 + c2 * 64;
          if (row0 >= a.cols || col >= a.D) break;   // nothing of the box inside dw (warp-uniform)
          uint32_t r0[32], r1[32], pk[32];
          tmem_ld_32x32b_x32(tbase + c2 * 64, r0);
          tmem_ld_32x32b_x32(tbase + c2 * 64 + 32, r1);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            pk[j] = pack_bf16x2(scale * __uint_as_float(r0[2 * j]), scale * __uint_as_float(r0[2 * j + 1]));
            pk[16 + j] = pack_bf16x2(scale * __uint_as_float(r1[2 * j]), scale * __uint_as_float(r1[2 * j + 1]));
          }
          store_box64(&tmC, stg, box_at, pk, col, row0, lane);
        }
      } else if (!tile.dw || sh.dw_splits > 1) {
        // fp32 slabs: [32 x 32] boxes of 128-byte rows, stored (or, behind the first piece of the vocabulary, added) by
        // TMA; the rows up to the next multiple of 256 belong to the slab
        const int at = tile.dw ? a.slab_rows + tile.split * ((a.cols + 255) / 256 * 256) : tile.split * (sh.num_m * 256);
        const bool none = tile.kb0 == tile.kb1;   // a split without k-blocks: nothing was accumulated
#pragma unroll 1
        for (int c = half; c < BN / 32; c += 2) {
          const int col = n0 + c * 32;
          if (col >= a.D) break;   // warp-uniform
          float v[32];
          load32(tbase + c * 32, v);
          uint8_t* box = stg + box_at * 4096;
          box_at ^= 1;
          if (lane == 0) bulk_group_wait_read<1>();   // the store that last read this box is done with it
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (!tile.dw && a.dx_add) tma_add_2d(&tmS, box, col, at + row0);
            else tma_store_2d(&tmS, box, col, at + row0);
            bulk_group_commit();
          }
        }
      } else {
        // gradients of the weights that no TMA store takes (fp32, added to, rows not 16-byte aligned): each 32 x 32 chunk
        // goes through this warp's scratch (16-byte cells, XOR-swizzled by row), then 8 lanes write one row segment
        float4* scr = reinterpret_cast<float4*>(stg);
        if (lane == 0) bulk_group_wait_read<0>();   // TMA stores of earlier tiles read the same memory
        __syncwarp();
#pragma unroll 1
        for (int c = half; c < BN / 32; c += 2) {
          float v[32];
          load32(tbase + c * 32, v);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            scr[lane * 8 + (j ^ (lane & 7))] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          __syncwarp();
          const int c4 = lane & 7, col = n0 + c * 32 + c4 * 4;
          const int nv = min(4, a.D - col);
#pragma unroll
          for (int it = 0; it < 8; ++it) {
            const int rr = it * 4 + (lane >> 3), m = row0 + rr;
            const float4 x = scr[rr * 8 + (c4 ^ (rr & 7))];
            float e[4] = {scale * x.x, scale * x.y, scale * x.z, scale * x.w};
            if (m < a.cols && nv > 0) {
              if (a.dw_f32) store4(reinterpret_cast<float*>(a.dw) + m * a.lddw + col, e, nv, a.dw_add);
              else store4(reinterpret_cast<__nv_bfloat16*>(a.dw) + m * a.lddw + col, e, nv, a.dw_add);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive(&tempty[acc]);
        else arrive_leader(acc ? tempty_leader1 : tempty_leader0);
      }
      if (!HALVES) acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (MODE != HEAD_STAT && lane == 0) bulk_group_wait_all();   // every TMA store has landed
  }
  if (*abort_flag) settle();
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();   // both CTAs done with TMEM and with each other's barriers
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
}

// ---------------------------------------------------------------- the loss of a few rows
// STAT for up to kScoreRows rows of which only the loss is wanted.  Reading w bounds it, so the product is turned round: 128
// rows of w are the matrix instruction's M and the batch its N, no operand is padded to 256 rows, and a block of 100
// KB of stages leaves room for another one on the SM, whose loads go on while this one is in its epilogue.  Nothing
// before the launch in this stream writes w that has not ended (the kernel that packs the rows waited for it), so the
// first stages of w are asked for before the wait for the packed rows.  The sum over D is taken in up to eight parts,
// each in an accumulator of its own: the tensor cores cut off what D / 16 / 8 steps lose, not D / 16.
// 32 rows of 2048 against 32000: 31.7 us for the call and losses 1e-7 off, 38 and 4e-7 by tiles of 256 rows; 64 rows 33
// against 42 to 49, 128 rows 40 against 50; this kernel alone 25.8 us at 32 rows, of which 131 MB take 20.  The gradient
// has to make the same logits again, bit for bit, so a loss that it follows is not taken here.
constexpr int kScoreThreads = 128;

template <int NB>   // rows of a block
struct Score {
  static constexpr int W = 128 * kBK * 2, X = NB * kBK * 2, STAGE = W + X;
  static constexpr int STAGES = 110 * 1024 / STAGE;   // 5, 4, 3
  static constexpr int PARTS = 256 / NB;
  static constexpr int SMEM = STAGES * STAGE + 256 + 1024;
  static constexpr int LD = 132;   // floats between the rows of the logits in shared memory
  static_assert(NB * LD * 4 <= STAGES * STAGE, "logits do not fit in the ring");
  static_assert(2 * (SMEM + 1024) <= 233472, "two blocks on an SM");
};

template <int NB>
__global__ void __launch_bounds__(kScoreThreads, 2)
    score_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                 const __grid_constant__ CUtensorMap tmX, const HeadGemm a) {
  using C = Score<NB>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = blockIdx.x * 128;
  const int kbs = (a.D + kBK - 1) / kBK, parts = min(kbs, C::PARTS), pre = min(kbs, C::STAGES);
  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    for (int i = 0; i < pre; ++i) {
      mbar_arrive_expect_tx(&full[i], C::STAGE);
      tma_load_2d(smem + i * C::STAGE, &tmW, &full[i], i * kBK, lo);
    }
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();
  // behind the product a few threads have a row: what they need of it
  constexpr int kPer = kScoreThreads / NB;
  const int m = tid / kPer, first = tid % kPer;
  const int rows = min(*a.count, a.N);
  const bool live = m < rows;
  const int n = !live ? 0 : a.start != nullptr ? a.row[m] : a.ids[m];   // batch row, or the class
  int entry = 0, end = 0;
  if (live && a.start != nullptr) {
    const unsigned short* s = a.start + (long long)blockIdx.x * a.N + n;
    entry = s[0];
    end = s[a.N];
  }
  if (warp == 0 && lane == 0) {
    const CUtensorMap* x = a.dense && rows == a.N ? &tmX : &tmA;
    for (int i = 0; i < pre; ++i) tma_load_2d(smem + i * C::STAGE + C::W, x, &full[i], i * kBK, 0);
    for (int i = pre; i < kbs; ++i) {
      const int s = i % C::STAGES;
      if (!mbar_wait(&empty[s], ((i / C::STAGES) & 1) ^ 1u, a.err, kErrTimeoutEmpty, abort_flag)) break;
      mbar_arrive_expect_tx(&full[s], C::STAGE);
      tma_load_2d(smem + s * C::STAGE, &tmW, &full[s], i * kBK, lo);
      tma_load_2d(smem + s * C::STAGE + C::W, x, &full[s], i * kBK, 0);
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = make_idesc_bf16(128, NB, 0, 0);
    int part = -1, next = 0;   // k-block at which the next part begins
    for (int i = 0; i < kbs; ++i) {
      const int s = i % C::STAGES;
      const bool fresh = i == next;
      if (fresh) {
        ++part;
        next = kbs * (part + 1) / parts;
      }
      if (!mbar_wait(&full[s], (i / C::STAGES) & 1, a.err, kErrTimeoutFull, abort_flag)) break;
      tc_fence_after();
      const uint32_t sw = smem_u32(smem + s * C::STAGE);
#pragma unroll
      for (int k = 0; k < kBK / 16; ++k)
        umma_bf16(tmem + part * NB, make_smem_desc(sw + k * 32, 16, 1024, 2),
                  make_smem_desc(sw + C::W + k * 32, 16, 1024, 2), idesc, fresh && k == 0 ? 0u : 1u);
      umma_commit(&empty[s]);
    }
    umma_commit(done);
  }
  __syncwarp();
  // the product ends with `done` even where a wait for an operand ran out in front of it
  const bool ok = mbar_wait(done, 0, a.err, kErrTimeoutTmemFull, abort_flag) && !*abort_flag;
  tc_fence_after();
  if (!__syncthreads_and(ok)) {   // the status says so, and the row losses are NaN
    settle();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, 256);
    return;
  }
  // every warp is past the wait: no copy or product uses the ring
  float* logits = reinterpret_cast<float*>(smem);   // [NB][LD]
#pragma unroll 1
  for (int b = 0; b < NB; b += 32) {
    const uint32_t at = tmem + (static_cast<uint32_t>(warp * 32) << 16) + b;
    float v[32];
    load32(at, v);
#pragma unroll 1
    for (int p = 1; p < parts; ++p) {
      float o[32];
      load32(at + p * NB, o);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += o[j];
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) logits[(b + j) * C::LD + tid] = v[j];
  }
  __syncthreads();
  const float* mine = logits + m * C::LD;
  const int nvalid = min(128, a.cols - lo);
  float mx = -INFINITY;
#pragma unroll 8
  for (int j = first; j < nvalid; j += kPer) mx = fmaxf(mx, mine[j]);
#pragma unroll
  for (int o = 1; o < kPer; o *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  mx *= a.c;
  const float ref = mx == -INFINITY ? 0.f : mx;
  float t = 0.f;
#pragma unroll 8
  for (int j = first; j < nvalid; j += kPer) t += ex2_approx(fmaf(mine[j], a.c, -ref));
#pragma unroll
  for (int o = 1; o < kPer; o *= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (live) {
    if (first == 0) a.part[(long long)blockIdx.x * a.N + m] = make_float2(mx, t);
    if (a.start == nullptr) {
      if (first == 0 && n >= lo && n < lo + 128) a.z[m] = mine[n - lo];
    } else {
      for (int e = entry + first; e < end; e += kPer) a.z[(long long)m * a.K + e] = mine[a.ids[(long long)n * a.K + e] - lo];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 256);
}

// ---------------------------------------------------------------- host
static PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [outer, inner] rows of stride ld, bf16 in boxes of [rows, 64] or fp32 in boxes of [rows, 32], with the 128-byte swizzle
static bool map2(CUtensorMap* m, const void* ptr, long long inner, long long outer, long long ld, int rows,
                 bool f32 = false) {
  auto fn = encoder();
  if (fn == nullptr || !((reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && ld % (f32 ? 4 : 8) == 0)) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * (f32 ? 4 : 2)};
  const cuuint32_t box[2] = {f32 ? 32u : 64u, (cuuint32_t)rows};   // 128 bytes wide
  const cuuint32_t es[2] = {1, 1};
  return fn(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE, int BN, bool HALVES = false>
static int launch(const CUtensorMap (&t)[6], const HeadGemm& a, int tiles, int num_sms, cudaStream_t s) {
  using C = Cfg<MODE, BN>;
  static SmemLimit limit;
  if (!limit.raise(head_kernel<MODE, BN, HALVES>, C::SMEM_BYTES)) return -3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(tiles, num_sms / 2), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_env_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, head_kernel<MODE, BN, HALVES>, t[0], t[1], t[2], t[3], t[4], t[5], a) == cudaSuccess ? 0 : -3;
}

}  // namespace head
}  // namespace pcb

using namespace pcb;
using namespace pcb::head;

template <int NB>
static int launch_score(HeadGemm a, const void* x, long long ldx, const void* x_all, long long ldx_all, const void* w,
                        long long ldw, cudaStream_t s) {
  CUtensorMap tw, ta, tx;
  if (!map2(&tw, w, a.D, a.cols, ldw, 128) || !map2(&ta, x, a.D, a.N, ldx, NB)) return -5;
  a.dense = x_all != nullptr;
  if (!a.dense) tx = ta;
  else if (!map2(&tx, x_all, a.D, a.N, ldx_all, NB)) return -5;
  static SmemLimit limit;
  if (!limit.raise(score_kernel<NB>, Score<NB>::SMEM)) return -3;
  return pdl_launch(score_kernel<NB>, dim3((a.cols + 127) / 128), dim3(kScoreThreads), Score<NB>::SMEM, s, tw, ta, tx, a) == cudaSuccess ? 0 : -3;
}

int pcb_head_score(HeadGemm a, const void* x, long long ldx, const void* x_all, long long ldx_all, const void* w, long long ldw,
                   cudaStream_t s) {
  if (a.N < 1 || a.N > kScoreRows || a.D < 1 || a.cols < 1) return -1;
  return a.N <= 32   ? launch_score<32>(a, x, ldx, x_all, ldx_all, w, ldw, s)
         : a.N <= 64 ? launch_score<64>(a, x, ldx, x_all, ldx_all, w, ldw, s)
                     : launch_score<128>(a, x, ldx, x_all, ldx_all, w, ldw, s);
}

bool pcb_head_whole(int N, int V, int D) { return V <= kWholeColumns && !in_halves(N, D); }

int pcb_head_gemm(int mode, HeadGemm a, const void* x, long long ldx, const void* x_all, long long ldx_all,
                  const void* w, long long ldw, void* g, int num_sms, cudaStream_t s) {
  if (a.N < 1 || a.D < 1 || a.cols < 1 || num_sms < 2) return -1;
  a.bwd_pairs = num_sms / 2;   // tiles of the gradients are split until there are enough; a pair without one ends at once
  CUtensorMap t[6];
  memset(t, 0, sizeof(t));
  const int num_m = (a.N + 255) / 256;
  const bool bwd = mode == HEAD_BWD;
  const long long panels = (a.cols + 63) / 64;
  if (panels * a.g_rows > 0x7fffffffLL) return -1;   // rows of g's panels are addressed by an int
  const int xrows = bwd ? 64 : kBM;
  CUtensorMap& tx = t[bwd ? 3 : 0];
  if (!map2(&tx, x, a.D, a.N, ldx, xrows)) return -5;
  a.dense = x_all != nullptr;
  if (!a.dense) t[4] = tx;
  else if (!map2(&t[4], x_all, a.D, a.N, ldx_all, xrows)) return -5;
  if (!bwd) {
    if (!map2(&t[1], w, a.D, a.cols, ldw, 128)) return -5;
    if (mode != HEAD_STAT && !map2(&t[2], g, 64, panels * a.g_rows, 64, 32)) return -5;
    if (mode == HEAD_WHOLE) {
      if (!pcb_head_whole(a.N, a.cols, a.D)) return -1;
      return launch<HEAD_WHOLE, 256>(t, a, num_m, num_sms, s);
    }
    // the blocks that run side by side share the operand with the larger footprint
    a.row_blocks_last = a.N > a.cols;
    const int tiles = num_m * ((a.cols + 255) / 256);
    if (in_halves(a.N, a.D))
      return mode == HEAD_STAT ? launch<HEAD_STAT, 256, true>(t, a, tiles, num_sms, s)
                               : launch<HEAD_GRAD, 256, true>(t, a, tiles, num_sms, s);
    return mode == HEAD_STAT ? launch<HEAD_STAT, 256>(t, a, tiles, num_sms, s) : launch<HEAD_GRAD, 256>(t, a, tiles, num_sms, s);
  }
  if (!map2(&t[0], g, 64, panels * a.g_rows, 64, 64) || !map2(&t[1], w, a.D, a.cols, ldw, 64)) return -5;
  const long long slab_rows = a.slab_rows + (a.dw_max > 1 ? (long long)a.dw_max * ((a.cols + 255) / 256 * 256) : 0);
  if (a.slab == nullptr) t[5] = t[0];
  else if (!map2(&t[5], a.slab, a.D, slab_rows, a.ld_slab, 32, true)) return -5;
  a.dw_tma = a.want_dw && !a.dw_f32 && !a.dw_add && map2(&t[2], a.dw, a.D, a.cols, a.lddw, 32);
  if (!a.dw_tma) t[2] = t[0];
  const int bn = head_bn(a.D);
  return bn == 256 ? launch<HEAD_BWD, 256>(t, a, a.bwd_pairs, num_sms, s) : launch<HEAD_BWD, 128>(t, a, a.bwd_pairs, num_sms, s);
}

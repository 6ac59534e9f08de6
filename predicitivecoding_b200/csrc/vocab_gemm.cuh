// Products of the vocabulary head (csrc/vocab_gemm.cu): what one launch reads and writes.
#pragma once
#include <atomic>
#include <cmath>

#include <cuda_runtime.h>

namespace pcb {

// Up to this many counted rows, p - q is carried as two bf16 terms.  A gradient of few rows has few large entries,
// so one rounding of them to 8 bits shows in its norm (up to 2^-8); over more rows the roundings average to about the
// one that the bf16 result takes anyway.  It is the rows of one tile: the second term costs one more pass of
// matrix instructions over a tile that reading the weights bounds: 256 rows of 768 against 32000 take 71.2 us for the
// backward, 257 with one term 69.8, and fp32 dx and dw are 7e-6 and 0.7e-6 off in norm, 5.6e-5 and 5.8e-5.  Their
// rounding to bf16, where it is asked for, is 1.7e-3.
constexpr int kTwoTermRows = 256;

// Up to this many rows, a loss without gradient is made by a product with the vocabulary as its rows.
constexpr int kScoreRows = 128;

// Raises a kernel's limit of dynamic shared memory, once on each device.
struct SmemLimit {
  std::atomic<unsigned long long> done{0};
  template <typename F>
  bool raise(F* kernel, int bytes) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return false;
    if ((done.load(std::memory_order_relaxed) >> dev) & 1) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return true;
  }
};

enum HeadMode : int {
  HEAD_STAT = 0,   // logits -> (max, sum) of every 128 of a row, and the logits at its targets
  HEAD_GRAD = 1,   // logits -> g = softmax - target distribution, bf16
  HEAD_BWD = 2,    // dw = g^T x and dx = g w in one launch
  HEAD_WHOLE = 3,  // a vocabulary of up to kWholeColumns: logits -> row losses, their sum and g
};

// Columns of logits that the accumulators of a tile row hold together: up to there the softmax of a row is known before
// its logits are gone, and they need not be made again for the gradient.
constexpr int kWholeColumns = 512;

struct HeadGemm {
  int N, D;               // rows of the batch, width
  int cols;               // columns of the vocabulary in this launch
  int v0;                 // the first of them (a multiple of 256)
  const int* count;       // device: counted rows, packed in front
  int* err;               // device: status of a wait that ran out (0: none)
  int dense;              // x itself may be read in place of the packed rows when all are counted
  float c;                // log2(e) / temperature: exponents are taken to base 2
  int row_blocks_last;    // order of tiles: 1 = the column blocks of one row block run side by side
  // target distribution: K entries a row, ids ascending, by batch row; without `start`, one id of weight 1, by packed row
  const int* row;         // [N] batch row of each packed row
  const int* ids;         // [N, K]
  const float* q;
  int K;
  const unsigned short* start;   // [2 ceil(V / 256) + 1, N]: first entry with id >= 128 g, by batch row
  // STAT
  float2* part;           // [2 ceil(V / 256), N] (max, sum), by packed row
  float* z;               // [N, K] logits at the ids, by packed row
  // WHOLE
  float* loss;            // [N] by batch row: factor * the divergence in bits
  float factor;
  float *total, *inverse; // as row_loss_kernel leaves them (nullptr: not wanted)
  int mean;
  int* done;              // CTAs that are done, 0 before the launch
  // GRAD, BWD
  const float2* norm;     // [N] (r, 1 / sum of 2^(c l - r)), by packed row
  // g: panels of 64 columns, each [g_rows, 64], so that every box that is stored or loaded (32 or 64 rows of a panel) is
  // one run of memory, whichever of its two dimensions the product contracts
  int g_rows;
  int g_low;              // row of a panel where the second terms begin: behind the one tile of rows that has them
  // BWD.  The K splits of the two products depend on the number of counted rows: GRAD of the first
  // piece of the vocabulary works them out and leaves them in plan[0] (dw) and plan[1] (dx).
  int* plan;
  int want_dw, want_dx;
  int bwd_pairs;          // pairs of CTAs of the BWD launch (set by pcb_head_gemm)
  int dw_max;             // most splits of dw
  int slab_rows;          // rows of dx's slabs: its splits times the counted rows, rounded up to 256, fit in
  void* dw;               // [cols, D], row stride lddw (unsplit)
  long long lddw;
  int dw_f32, dw_add, dw_tma;
  float alpha;            // dw *= alpha * scale * scale2 (not the slabs)
  const float* scale;
  const float* scale2;
  // fp32 slabs, rows of ld_slab (nullptr: neither needs one): dx's, packed rows rounded up to 256 for each split; from row
  // slab_rows on dw's, when it may be split, cols rounded up to 256 for each split
  float* slab;
  long long ld_slab;
  int dx_add;             // add to dx's slabs instead of writing them
};

// Columns of a tile of the gradients' products.  A k-block of a 256 x 256 tile brings 32 KB into each SM for 512 cycles of
// matrix instructions, just what L2 delivers (64 bytes a cycle); one of 256 x 128 brings 24 KB for 256 cycles and is
// bound by that.  So 256 even where a quarter of the columns is empty (3001 x 384 x 16001, 40% counted: 37 us, 42 in
// three tiles of 128).
constexpr int kMaxDxSplits = 16;
__host__ __device__ inline int head_bn(int D) { return D <= 128 ? 128 : 256; }

// k-blocks that a tile costs besides its own
constexpr int kTileOverhead = 4;

// K splits of dw and dx.  With the schedule below all pairs of SMs are busy for the mean of the work and half a tile of
// dw, unless either product has too few tiles; slabs cost their bytes, written and read once, of which the time of
// one k-block of a 256-column tile moves 2.4 MB.  As if both were wanted, so that a gradient is the same with and
// without the other.
__device__ inline void plan_splits(const HeadGemm& a, int rows, int pairs, int* plan) {
  const int bn = head_bn(a.D), num_n = (a.D + bn - 1) / bn;
  const int r = max(rows, 1), two = rows <= kTwoTermRows ? 2 : 1;
  const float kb_dw = two * ((r + 63) / 64), kb_dx = two * ((a.cols + 63) / 64);
  const int dw = (a.cols + 255) / 256 * num_n, dx = (r + 255) / 256 * num_n;
  const float slab = 8.f * a.D / 2.4e6f * (256 / bn);   // per row
  const int dx_max = min(kMaxDxSplits, a.slab_rows / ((r + 255) / 256 * 256));
  float best = INFINITY;
  for (int s1 = 1; s1 <= a.dw_max && (s1 == 1 || kb_dw >= 4 * s1); s1 *= 2) {
    const float c1 = kb_dw / s1 + kTileOverhead;
    const float alone = (dw * s1 + pairs - 1) / pairs * c1;
    for (int s2 = 1; s2 <= dx_max && (s2 == 1 || kb_dx >= 4 * s2); ++s2) {
      const float c2 = kb_dx / s2 + kTileOverhead;
      const float even = (dw * s1 * c1 + dx * s2 * c2) / pairs + 0.5f * c1;
      const float c = fmaxf(fmaxf(even, alone), (dx * s2 + pairs - 1) / pairs * c2) + slab * ((s1 > 1 ? s1 * a.cols : 0) + s2 * r);
      if (c < best) {
        best = c;
        plan[0] = s1;
        plan[1] = s2;
      }
    }
  }
}

// Whether this block is the last of `blocks` to come here, called by one thread between two barriers of the block: its
// release covers what all of the block's threads wrote before the first, its acquire what they read after the second.
__device__ inline bool arrive_last(int* done, int blocks) {
  int before;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(done) : "memory");
  return before == blocks - 1;
}

// The last step of a loss: the rows' losses added up by THREADS threads in a fixed order and in 64 bits.  *total = their sum
// or mean, *inverse = 1 / counted rows (both 0 when there are none); *total = NaN behind a wait that ran out.  `sync`
// joins the threads.
template <int THREADS, typename F>
__device__ inline void add_losses(const float* loss, int N, int rows, int mean, const int* status, float* total, float* inverse,
                                  double* sums, int tid, F sync) {
  const int spoilt = tid == 0 ? __ldcg(status) : 0;
  double t = 0.0;
#pragma unroll 8
  for (int i = tid; i < N; i += THREADS) t += __ldcg(loss + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((tid & 31) == 0) sums[tid >> 5] = t;
  sync();
  if (tid < 32) {
    t = tid < THREADS / 32 ? sums[tid] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (tid == 0) {
      *total = spoilt != 0 ? NAN : (float)(mean ? (rows > 0 ? t / rows : 0.0) : t);
      *inverse = rows > 0 ? 1.f / (float)rows : 0.f;
    }
  }
}

}  // namespace pcb

// x: packed rows [N, ldx]; x_all: the batch itself (nullptr: cannot be read in place); w: [cols, D] rows v0..; g: panels of 64
// columns.  Returns 0, -1 (operands), -3 (launch), -5 (tensor map).
int pcb_head_gemm(int mode, pcb::HeadGemm a, const void* x, long long ldx, const void* x_all, long long ldx_all,
                  const void* w, long long ldw, void* g, int num_sms, cudaStream_t s);
// whether HEAD_WHOLE takes these sizes
bool pcb_head_whole(int N, int V, int D);
// STAT of up to kScoreRows rows; operands as in pcb_head_gemm
int pcb_head_score(pcb::HeadGemm a, const void* x, long long ldx, const void* x_all, long long ldx_all, const void* w,
                   long long ldw, cudaStream_t s);

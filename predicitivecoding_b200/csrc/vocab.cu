// The two ends of a decoder over its vocabulary: embedding lookup and its gradient, and the vocabulary head's losses
// (softmax cross entropy; distillation from a teacher's top logits) with their gradients.
//
// Head.  With x [N, D], w [V, D], logits l = x w^T and a target distribution per row (one id of weight 1, or the
// softmax q of K teacher logits at temperature T):
//     loss_n = T^2 sum_k q_k (log q_k - log p_k),  p = softmax(l / T)   (T = 1, one target: lse(l) - l_t)
//     d loss_n / d l = T (p - q),   dx = c (p - q) w,   dw = c (p - q)^T x,   c = T gout / counted rows
// The logits [N, V] are never kept.  The forward's product (csrc/vocab_gemm.cu) reduces each row's 128 columns to (max,
// sum) and picks the logits at the targets; the backward makes the logits again, a piece of the vocabulary at a
// time, and turns them into bf16 p - q, which two more products read: dw of the piece is finished there, dx is
// accumulated over the pieces in fp32.  8 N V D operations instead of 6, for workspaces that do not grow with N * V.
// (A vocabulary of up to 512 columns is taken whole where a gradient follows: its loss and p - q come of one product.)
// Rows without a target (masked prompts, padding) are taken out first: the counted rows are packed in order,
// the products run over their number, known on the device only, and what stands in the other rows (NaN too) is
// never read.  When all rows are counted the products read x itself.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "vocab_api.h"
#include "vocab_gemm.cuh"

namespace pcb {
namespace vocab {

constexpr int kThreads = 256;
constexpr int kMaxK = kVocabMaxEntries;

PCB_DEVICE long long load_id(const void* p, int is64, long long i) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

// Exclusive prefix sum of one int per thread over the block's first nw warps (all threads call it); total in *sum.
PCB_DEVICE int block_scan(int v, int* warp_sums, int* sum, int nw) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();   // the sums of the previous call have been read
  if (lane == 31 && w < nw) warp_sums[w] = inc;
  __syncthreads();
  int before = 0, total = 0;
  for (int i = 0; i < nw; ++i) {
    if (i < w) before += warp_sums[i];
    total += warp_sums[i];
  }
  *sum = total;
  return before + inc - v;
}

template <typename T> PCB_DEVICE float to_f32(T v);
template <> PCB_DEVICE float to_f32<float>(float v) { return v; }
template <> PCB_DEVICE float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> PCB_DEVICE T from_f32(float v);
template <> PCB_DEVICE float from_f32<float>(float v) { return v; }
template <> PCB_DEVICE __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC>
PCB_DEVICE void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
    static_assert(VEC % 4 == 0, "16-byte vectors");
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 f = reinterpret_cast<const float4*>(p)[i];
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
  } else if constexpr (VEC == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
    v[4] = bf16_lo(u.z); v[5] = bf16_hi(u.z); v[6] = bf16_lo(u.w); v[7] = bf16_hi(u.w);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
  }
}
// the same vector as loaded, for loads kept in flight in registers
template <typename T, int VEC>
struct Raw {
  using type = std::conditional_t<VEC == 1, T, std::conditional_t<VEC * sizeof(T) == 16, uint4, uint2>>;
};
template <typename T, int VEC>
PCB_DEVICE void unpack(const typename Raw<T, VEC>::type& r, float (&v)[VEC]) {
  load_vec<T, VEC>(reinterpret_cast<const T*>(&r), v);
}
template <typename T, int VEC>
PCB_DEVICE void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else if constexpr (VEC == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
}

// ---------------------------------------------------------------- packing
struct PackArgs {
  const void* tgt;       // class targets, or
  int tgt64;
  long long ignore;
  const int* len;        // entries of each row's target list
  int V, N, D;
  const __nv_bfloat16* x;
  long long ldx;
  int vec;               // x in 16-byte vectors
  int in_place;          // x may be read in place when every row is counted
  const int* counts;     // counted rows of every kCountRows (nullptr: each block counts for itself)
  __nv_bfloat16* xc;
  long long ldxc;
  int *row, *pos, *tgt32, *count;
  float* loss;
};
constexpr int kCountRows = kThreads;
// Longer batches are counted by a launch of their own.  Losses of N x 64 against 700, half of the rows counted, each
// block counting for itself and a launch: 13.5 and 18.0 us at 2048 rows, 18.0 and 18.9 at 4096, 23.1 and 20.5 at 8192,
// 30.8 and 27.7 at 16384, 54.7 and 39.9 at 32768.
constexpr int kSelfCountRows = 8192;

PCB_DEVICE bool counted(const PackArgs& a, int n) {
  if (a.len != nullptr) return a.len[n] > 0;
  const long long t = load_id(a.tgt, a.tgt64, n);
  return t >= 0 && t < a.V && t != a.ignore;
}

__global__ void __launch_bounds__(kCountRows) count_rows_kernel(PackArgs a, int* __restrict__ counts) {
  pdl_begin();
  const int n = blockIdx.x * kCountRows + threadIdx.x;
  const int c = __syncthreads_count(n < a.N && counted(a, n));
  if (threadIdx.x == 0) counts[blockIdx.x] = c;
}

// Packs the counted rows in order; block b owns rows [b R, (b + 1) R).  In a short batch each block counts the rows
// before and behind its own by itself (8 bytes a row from L2 against 2 D a row copied), which saves a launch.
__global__ void __launch_bounds__(kThreads) pack_rows_kernel(PackArgs a, int R) {
  __shared__ int sums[kThreads / 32];
  __shared__ int src[kThreads];
  pdl_begin();
  auto zero_or_copy = [&](int n, long long j) {   // one warp: packed row j from row n, or zeros (n < 0)
    const int lane = threadIdx.x & 31;
    __nv_bfloat16* d = a.xc + j * a.ldxc;
    const __nv_bfloat16* s = a.x + (long long)max(n, 0) * a.ldx;
    if (a.vec) {
      const int nv = (int)(a.ldxc / 8);
      for (int i0 = lane; i0 < nv; i0 += 128) {
        uint4 r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          r[u] = n >= 0 && i0 + 32 * u < nv ? reinterpret_cast<const uint4*>(s)[i0 + 32 * u] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i0 + 32 * u < nv) reinterpret_cast<uint4*>(d)[i0 + 32 * u] = r[u];
      }
    } else {
      for (int i = lane; i < (int)a.ldxc; i += 32) d[i] = n >= 0 && i < a.D ? s[i] : __float2bfloat16_rn(0.f);
    }
  };
  const int r0 = (int)min((long long)a.N, (long long)blockIdx.x * R), r1 = (int)min((long long)a.N, (long long)r0 + R);
  int before = 0, others = 0;   // counted rows in front of this block's, and in all other blocks
  if (a.counts != nullptr) {
    const int blocks = (a.N + kCountRows - 1) / kCountRows;   // R is kCountRows
    for (int i = threadIdx.x; i < blocks; i += kThreads) {
      const int c = a.counts[i];
      if (i < (int)blockIdx.x) before += c;
      if (i != (int)blockIdx.x) others += c;
    }
  } else {
    for (int n = threadIdx.x; n < a.N; n += kThreads) {
      if (n >= r0 && n < r1) continue;
      const int c = counted(a, n) ? 1 : 0;
      if (n < r0) before += c;
      others += c;
    }
  }
  int base, rest;
  block_scan(before, sums, &base, kThreads / 32);
  block_scan(others, sums, &rest, kThreads / 32);
  const int n = r0 + threadIdx.x;   // R is at most kThreads
  const bool c = n < r1 && counted(a, n);
  int total;
  const int k = block_scan(c ? 1 : 0, sums, &total, kThreads / 32);
  if (n < r1) {
    a.pos[n] = c ? base + k : -1;
    if (!c) a.loss[n] = 0.f;
  }
  if (c) {
    a.row[base + k] = n;
    if (a.tgt32 != nullptr) a.tgt32[base + k] = (int)load_id(a.tgt, a.tgt64, n);
    src[k] = n;
  }
  __syncthreads();
  if (!(a.in_place && rest + total == a.N))
    for (int i = threadIdx.x >> 5; i < total; i += kThreads / 32) zero_or_copy(src[i], base + i);
  base += total;
  if (blockIdx.x == gridDim.x - 1) {
    if (threadIdx.x == 0) {
      a.count[0] = base;
      a.count[1] = 0;   // blocks of row_loss_kernel that are done
      a.count[4] = 0;   // status
    }
    const int end = min(a.N, (max(base, 1) + 63) / 64 * 64);
    for (int j = base + (threadIdx.x >> 5); j < end; j += kThreads / 32) zero_or_copy(-1, j);
  }
}

__global__ void pad_rows_kernel(const __nv_bfloat16* __restrict__ src, long long ld, __nv_bfloat16* __restrict__ dst,
                                long long ldd, long long total, int D) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / ldd;
    const int c = (int)(i - r * ldd);
    dst[i] = c < D ? src[r * ld + c] : __float2bfloat16_rn(0.f);
  }
}

// ---------------------------------------------------------------- the teacher's lists
// One warp per row: the softmax of the entries present, and the entries in ascending id (rank = number of smaller
// ids, ties by place), so that a thread of the product's epilogue meets its row's targets in column order.  A lane
// holds R entries; their ranks are counted together, four other entries at a time.  The table of first entries lies by
// row, so a block collects it for its rows in shared memory and stores 16 bytes of a column at a time (2048 rows, K
// 64, V 32000: 12.0 us with a store per entry from 4 rows a block, 14.1 with 32 rows a block, 10.1 as it is).
constexpr int kSortRows = 8;
constexpr int kStartPass = 256;   // columns of the table at a time

template <int R>
__global__ void __launch_bounds__(32 * kSortRows)
    sort_targets_kernel(const void* __restrict__ ids, int ids64, long long ld_ids, const void* __restrict__ logits,
                        int bf16, long long ld_logits, int N, int V, int K, float c, int* __restrict__ out_ids,
                        float* __restrict__ out_q, float* __restrict__ out_lq, int* __restrict__ out_len,
                        unsigned short* __restrict__ start, int granules) {
  constexpr int kRows = kSortRows;
  __shared__ __align__(16) int s_id[kRows][32 * R];
  __shared__ int s_sorted[kRows][32 * R];
  __shared__ unsigned short s_start[kStartPass][kRows];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = blockIdx.x * kRows + w;
  const bool in = n < N;   // whole warps
  constexpr int kAbsent = 0x7fffffff;   // behind every id
  int id[R], rank[R];
  float y[R];
  float mx = -INFINITY;
  int mine = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int k = lane + 32 * r;
    id[r] = kAbsent;
    y[r] = -INFINITY;
    rank[r] = 0;
    if (in && k < K) {
      const long long t = load_id(ids, ids64, n * ld_ids + k);
      const long long at = n * ld_logits + k;
      const float l = bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(logits)[at])
                           : reinterpret_cast<const float*>(logits)[at];
      if (t >= 0 && t < V && l != -INFINITY) {
        id[r] = (int)t;
        y[r] = l * c;
        ++mine;
      }
    }
    s_id[w][k] = id[r];
    mx = fmaxf(mx, y[r]);
  }
  mx = warp_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (id[r] != kAbsent) sum += exp2f(y[r] - mx);
  sum = warp_sum(sum);
  const int present = __reduce_add_sync(0xffffffffu, mine);
  const float ls = log2f(sum);
  __syncwarp();
  for (int i = 0; i < K; i += 4) {
    const int4 o = *reinterpret_cast<const int4*>(&s_id[w][i]);
    const int ov[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) rank[r] += ov[e] < id[r] || (ov[e] == id[r] && i + e < lane + 32 * r) ? 1 : 0;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (id[r] == kAbsent) continue;
    s_sorted[w][rank[r]] = id[r];
    const long long at = (long long)n * K + rank[r];
    out_ids[at] = id[r];
    out_q[at] = exp2f(y[r] - mx) / sum;
    out_lq[at] = y[r] - mx - ls;
  }
  __syncwarp();
  if (in && lane == 0) out_len[n] = present;
  // entries with an id below 128 g, for every g: four searches at a time
  for (int pass = 0; pass <= granules; pass += kStartPass) {
    const int columns = min(kStartPass, granules + 1 - pass);
    for (int g0 = lane; g0 < columns; g0 += 128) {
      int lo[4] = {}, hi[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) hi[u] = present;
      for (int span = present; span > 0; span >>= 1) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (lo[u] < hi[u]) {
            const int mid = (lo[u] + hi[u]) >> 1;
            if (s_sorted[w][mid] < (pass + g0 + 32 * u) * 128LL) lo[u] = mid + 1;
            else hi[u] = mid;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (g0 + 32 * u < kStartPass) s_start[g0 + 32 * u][w] = (unsigned short)lo[u];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns * kRows; i += 32 * kRows) {
      const int g = pass + i / kRows, r = i % kRows;
      if (blockIdx.x * kRows + r < N) start[(long long)g * N + blockIdx.x * kRows + r] = s_start[i / kRows][r];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- logits of a few rows
// What the STAT and GRAD products do, for up to kFewRows rows on the FMA units: such a call reads the weights once and has
// nothing else to do, so it is bound by that; sums in fp32 rounded to nearest keep digits that the tensor cores'
// accumulation, cut off at each of its D / 16 steps, loses (one row, D 1600: a loss 7e-6 off), and which the loss of
// few rows does not average out.  Both modes make the same logits, bit for bit: a row that is sure of its target has
// the sum of its other probabilities in p - q.  A block takes 128 rows of w, a warp four of them at a time, its lanes
// 8 columns each in turn; x stands in shared memory.  Losses of 1, 2, 4 and 8 rows of 2048 against 32000: 36, 35, 41 and
// 57 us, on the tensor cores 43, 39, 41 and 39, where they are 0.2 to 0.7e-6 off instead of 0.05e-6.  (A loss without
// gradient over many columns is score_kernel's: 31.5, 33.0, 31.9 us, at most 0.15e-6 off.)
constexpr int kFewRows = 4;
constexpr int few_threads(int rows) { return rows <= 2 ? 1024 : 512; }   // as many as registers allow: a small w has few blocks
constexpr int kFewColumns = 24 * 1024;   // of x in shared memory

struct FewRowsArgs {
  const __nv_bfloat16* x;      // the batch, read in place when all rows are counted (nullptr: never)
  long long ldx;
  const __nv_bfloat16* xc;     // packed rows
  long long ldxc;
  const __nv_bfloat16* w;      // [cols, D]
  long long ldw;
  __nv_bfloat16* g;            // GRAD
  HeadGemm h;
};

// (c0, c1) += (a0, a1) * (b0, b1)
PCB_DEVICE void fma2(float (&c)[2], float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 ra, rb, rc;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%0, %1};\n\t"
      "fma.rn.f32x2 rc, ra, rb, rc;\n\tmov.b64 {%0, %1}, rc;\n\t}"
      : "+f"(c[0]), "+f"(c[1])
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

template <int NR, bool GRAD>
__global__ void __launch_bounds__(few_threads(NR)) few_rows_kernel(FewRowsArgs a) {
  constexpr int kThreads = few_threads(NR), kPerWarp = 128 / (kThreads / 32);
  extern __shared__ __align__(16) __nv_bfloat16 xs[];   // [NR][ld]
  __shared__ float logits[NR][128];
  pdl_begin();
  const HeadGemm& h = a.h;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int nvec = (h.D + 7) / 8, ld = nvec * 8, whole = h.D / 8;
  const int rows = min(h.count[0], h.N);
  const bool direct = a.x != nullptr && rows == h.N;
  const __nv_bfloat16* src = direct ? a.x : a.xc;
  const long long lds = direct ? a.ldx : a.ldxc;
  for (int i = threadIdx.x; i < NR * nvec; i += kThreads) {   // rows of either are 16-byte aligned, packed ones padded
    const int n = i / nvec, v = i - n * nvec;
    reinterpret_cast<uint4*>(xs)[i] = n < rows ? *reinterpret_cast<const uint4*>(src + n * lds + v * 8) : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  const int col0 = blockIdx.x * 128;
#pragma unroll 1
  for (int r0 = 0; r0 < kPerWarp; r0 += 4) {
    const int v0 = col0 + w * kPerWarp + r0;
    if (v0 < h.cols) {   // warp-uniform
      const __nv_bfloat16* p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = a.w + (long long)min(v0 + r, h.cols - 1) * a.ldw;
      float acc[4][NR][2] = {};   // even and odd columns: products and sums are taken in pairs
#pragma unroll 2
      for (int v = lane; v < whole; v += 32) {
        float f[4][8];
#pragma unroll
        for (int r = 0; r < 4; ++r) load_vec<__nv_bfloat16, 8>(p[r] + v * 8, f[r]);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          float xv[8];
          load_vec<__nv_bfloat16, 8>(xs + n * ld + v * 8, xv);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 8; e += 2) fma2(acc[r][n], f[r][e], f[r][e + 1], xv[e], xv[e + 1]);
        }
      }
      if (whole * 8 + lane < h.D) {   // the columns that fill no vector
        const int d = whole * 8 + lane;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < NR; ++n)
            acc[r][n][0] = fmaf(__bfloat162float(p[r][d]), __bfloat162float(xs[n * ld + d]), acc[r][n][0]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float s = warp_sum(acc[r][n][0] + acc[r][n][1]);
          if (lane == 0) logits[n][w * kPerWarp + r0 + r] = s;
        }
    }
  }
  __syncthreads();
  const int lo = h.v0 + col0;   // vocabulary id of the first column
  const bool mine = w < NR && w < rows;   // a warp per row
  int e0 = 0, e1 = 0;           // this row's entries in these columns
  const int* ids = nullptr;
  const float* q = nullptr;
  if (mine) {
    if (h.start != nullptr) {
      const int n = h.row[w];
      const unsigned short* s = h.start + (long long)(lo >> 7) * h.N + n;
      e0 = s[0];
      e1 = s[h.N];
      ids = h.ids + (long long)n * h.K;
      if (GRAD) q = h.q + (long long)n * h.K;
    } else {
      ids = h.ids + w;
      e1 = ids[0] >= lo && ids[0] < lo + 128 ? 1 : 0;
    }
  }
  if constexpr (!GRAD) {
    if (!mine) return;
    float v[4], mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = col0 + lane + 32 * i < h.cols ? logits[w][lane + 32 * i] : -INFINITY;
      mx = fmaxf(mx, v[i]);
    }
    mx = warp_max(mx) * h.c;
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += exp2f(fmaf(v[i], h.c, -ref));
    sum = warp_sum(sum);
    if (lane == 0) h.part[(long long)(lo >> 7) * h.N + w] = make_float2(mx, sum);
    for (int e = e0 + lane; e < e1; e += 32) h.z[(long long)w * h.K + e] = logits[w][ids[e] - lo];
  } else {
    if (mine) {
      const float2 norm = h.norm[w];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        logits[w][c] = col0 + c < h.cols ? exp2f(fmaf(logits[w][c], h.c, -norm.x)) * norm.y : 0.f;
      }
      __syncwarp();
      if (lane == 0)
        for (int e = e0; e < e1; ++e) logits[w][ids[e] - lo] -= q != nullptr ? q[e] : 1.f;   // in order: ids may repeat
    }
    __syncthreads();
    // the two panels' rows up to the first k-block of dw's product, in both terms: 8 columns a thread and turn
    for (int i = threadIdx.x; i < 2 * 64 * 8; i += kThreads) {
      const int c = (i & 7) * 8, n = (i >> 3) & 63, panel = i >> 9;
      if (col0 + panel * 64 >= h.cols) break;
      uint32_t hi[4] = {}, low[4] = {};
      if (n < rows) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x0 = logits[n % NR][panel * 64 + c + 2 * j], x1 = logits[n % NR][panel * 64 + c + 2 * j + 1];
          hi[j] = pack_bf16x2(x0, x1);
          low[j] = pack_bf16x2(x0 - bf16_lo(hi[j]), x1 - bf16_hi(hi[j]));
        }
      }
      __nv_bfloat16* g = a.g + ((long long)(col0 / 64 + panel) * h.g_rows + n) * 64 + c;
      *reinterpret_cast<uint4*>(g) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(g + (long long)h.g_low * 64) = make_uint4(low[0], low[1], low[2], low[3]);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0 && h.v0 == 0) plan_splits(h, rows, h.bwd_pairs, h.plan);
  }
}

// ---------------------------------------------------------------- row losses
// 32 rows a block, a warp a row: the row's (max, sum) pairs become one, its target list its loss.  The pairs
// lie by row, so they are read with a row per lane and change hands through shared memory; the targets, which wait
// for nothing, are read in the meantime.  The last block to finish adds the losses up, in a fixed order and in 64
// bits: *total = their sum or mean, *inverse = 1 / counted rows (both 0 when there are none).
constexpr int kLossParts = 32;

__global__ void __launch_bounds__(32 * kLossParts)
    row_loss_kernel(const float2* __restrict__ part, int granules, const int* __restrict__ row,
                    const float* __restrict__ z, const float* __restrict__ q, const float* __restrict__ lq,
                    const int* __restrict__ len, int N, int K, float c, float factor, float2* __restrict__ norm,
                    float* loss, int* count, int mean, float* __restrict__ total, float* __restrict__ inverse) {
  __shared__ float sm[kLossParts][33], ss[kLossParts][33];
  __shared__ double sums[kLossParts];
  __shared__ int last;
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + w;   // this warp's packed row
  const int place = j < N ? row[j] : 0;   // asked for together with the count: a row behind it holds anything
  const int rows = min(count[0], N);
  const bool spoilt = count[4] != 0;   // a wait ran out: the pairs and the logits at the targets may be anything
  const bool live = j < rows;
  const int n = live ? place : 0;
  // the first two targets of a lane: weight, its logarithm, logit
  constexpr int kAhead = 2;
  const int e = !live ? 0 : len != nullptr ? len[n] : 1;
  const long long at_q = (long long)n * K, at_z = (long long)j * K;
  float qk[kAhead], lk[kAhead], zk[kAhead];
  auto target = [&](int k, float& weight, float& lw, float& logit) {
    weight = q != nullptr ? q[at_q + k] : 1.f;
    lw = lq != nullptr ? lq[at_q + k] : 0.f;
    logit = z[at_z + k];
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    qk[i] = lk[i] = zk[i] = 0.f;
    if (lane + 32 * i < e) target(lane + 32 * i, qk[i], lk[i], zk[i]);
  }
  {
    const int jl = blockIdx.x * 32 + lane;
    float m = -INFINITY, s = 0.f;
    if (jl < rows) {
#pragma unroll 8
      for (int g = w; g < granules; g += kLossParts) {
        const float2 p = part[(long long)g * N + jl];
        const float nm = fmaxf(m, p.x);
        const float ref = nm == -INFINITY ? 0.f : nm;
        s = s * exp2f(m - ref) + p.y * exp2f(p.x - ref);
        m = nm;
      }
    }
    sm[w][lane] = m;
    ss[w][lane] = s;
  }
  __syncthreads();
  const float m = sm[lane][w];   // lane = part
  const float mm = warp_max(m);
  const float ref = mm == -INFINITY ? 0.f : mm;
  const float tot = warp_sum(ss[lane][w] * exp2f(m - ref));
  const float lt = log2f(tot);
  // sum_k q_k (log2 q_k - log2 p_k), log2 p_k = (c z_k - ref) - log2(tot).  The difference of the two large numbers is
  // taken first and in one rounding: what ref itself was rounded by is in tot, so a row that is sure of its target
  // keeps the digits of its small loss.
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (lane + 32 * i < e && qk[i] != 0.f) l += qk[i] * (lk[i] + (fmaf(-c, zk[i], ref) + lt));   // 0 log 0 = 0
  for (int k = lane + 32 * kAhead; k < e; k += 32) {
    float weight, lw, logit;
    target(k, weight, lw, logit);
    if (weight != 0.f) l += weight * (lw + (fmaf(-c, logit, ref) + lt));
  }
  l = warp_sum(l);
  if (live && lane == 0) {
    loss[n] = spoilt ? NAN : l * factor;
    norm[j] = make_float2(ref, 1.f / tot);
  }
  if (total == nullptr) return;
  __syncthreads();
  if (threadIdx.x == 0) last = arrive_last(&count[1], (int)gridDim.x);
  __syncthreads();
  if (!last) return;
  add_losses<32 * kLossParts>(loss, N, rows, mean, count + 4, total, inverse, sums, threadIdx.x, [] { __syncthreads(); });
}

// Gradients from their fp32 slabs: the sum in slab order, times the gradient's factor.  The first N rows are dx's, found
// by their packed place, zero where the row is not counted; the others dw's, when it was split.  A warp per row
// and slice of columns.
constexpr int kFinishVecs = 4;

struct FinishArgs {
  const float* slab;
  int slab_rows;         // of dx, dw's behind them
  const int* count;
  const int* plan;       // K splits of dw and dx
  const int* status;     // of the waits of all launches before
  const int* pos;
  void *dx, *dw;
  long long ld_slab, lddx, lddw;
  int dx_f32, dw_f32, dw_add;
  int N, V, D;           // N = 0 where dx is not wanted, V = 0 where dw cannot be in slabs
  int dw_rows;           // 0 where dw is not wanted
  float alpha;
  const float* scale;
  const float* scale2;
};

// [rows, D] of NaN, by all threads of the grid; not a part of the code that every launch fetches
__device__ __noinline__ void spoil(void* p, int f32, long long ld, int rows, int D) {
  const long long step = (long long)gridDim.x * gridDim.y * kThreads;
  for (long long i = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * kThreads + threadIdx.x; i < (long long)rows * D; i += step) {
    const long long r = i / D, at = r * ld + (i - r * D);
    if (f32) reinterpret_cast<float*>(p)[at] = NAN;
    else reinterpret_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(NAN);
  }
}

template <int VEC>
__global__ void __launch_bounds__(kThreads) finish_kernel(FinishArgs a) {
  pdl_begin();
  int n = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const bool in = n < a.N + a.V, w = n >= a.N;
  if (w) n -= a.N;
  const int status = *a.status, slabs = a.plan[w ? 0 : 1], j = w ? n : a.pos[n];   // asked for together
  if (__builtin_expect(status != 0, 0)) {   // some launch gave up a wait: what the products wrote, dw itself too, may be anything
    if (a.N > 0) spoil(a.dx, a.dx_f32, a.lddx, a.N, a.D);
    spoil(a.dw, a.dw_f32, a.lddw, a.dw_rows, a.D);
    return;
  }
  if (!in || (w && slabs == 1)) return;   // slabs == 1: written by the product itself
  float f = a.alpha;
  if (a.scale != nullptr) f *= *a.scale;
  if (a.scale2 != nullptr) f *= *a.scale2;
  const int d0 = (blockIdx.y * kFinishVecs * 32 + (threadIdx.x & 31)) * VEC;
  const float* src = a.slab + ((long long)max(j, 0) + (w ? a.slab_rows : 0)) * a.ld_slab + d0;
  const long long stride = ((w ? a.V : max(a.count[0], 1)) + 255) / 256 * 256 * a.ld_slab;
  float v[kFinishVecs][VEC] = {};
  if (j >= 0) {
    for (int k = 0; k < slabs; ++k, src += stride) {
      float r[kFinishVecs][VEC];
#pragma unroll
      for (int i = 0; i < kFinishVecs; ++i)
        if (d0 + i * 32 * VEC < a.D) load_vec<float, VEC>(src + i * 32 * VEC, r[i]);
#pragma unroll
      for (int i = 0; i < kFinishVecs; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (d0 + i * 32 * VEC < a.D) v[i][e] += r[i][e];
    }
  }
  const bool f32 = w ? a.dw_f32 : a.dx_f32;
  const long long at = n * (w ? a.lddw : a.lddx) + d0;
  float* of = (float*)(w ? a.dw : a.dx) + at;
  __nv_bfloat16* oh = (__nv_bfloat16*)(w ? a.dw : a.dx) + at;
#pragma unroll
  for (int i = 0; i < kFinishVecs; ++i) {
    if (d0 + i * 32 * VEC >= a.D) break;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i][e] = j >= 0 ? f * v[i][e] : 0.f;
    if (w && a.dw_add) {
      float p[VEC];
      if (f32) load_vec<float, VEC>(of + i * 32 * VEC, p);
      else load_vec<__nv_bfloat16, VEC>(oh + i * 32 * VEC, p);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] += p[e];
    }
    if (f32) store_vec<float, VEC>(of + i * 32 * VEC, v[i]);
    else store_vec<__nv_bfloat16, VEC>(oh + i * 32 * VEC, v[i]);
  }
}

// ---------------------------------------------------------------- embedding
// A warp copies kLookupVecs vectors a lane of one row; wide rows take several warps.  All loads of a lane are issued
// before its first store.
constexpr int kLookupVecs = 4;

template <typename TW, typename TX, int VEC>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(const void* __restrict__ tok, int tok64, const TW* __restrict__ w, long long ldw, TX* __restrict__ x,
                  int N, int V, int D, float scale) {
  pdl_begin();
  const int n = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (n >= N) return;
  const long long t = load_id(tok, tok64, n);
  const bool in = t >= 0 && t < V;
  const int d0 = (blockIdx.y * kLookupVecs * 32 + (threadIdx.x & 31)) * VEC;
  const TW* src = w + (in ? t : 0) * ldw;
  TX* dst = x + (long long)n * D;
  float v[kLookupVecs][VEC];
#pragma unroll
  for (int i = 0; i < kLookupVecs; ++i) {
    const int d = d0 + i * 32 * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
    if (in && d < D) load_vec<TW, VEC>(src + d, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kLookupVecs; ++i) {
    const int d = d0 + i * 32 * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i][e] *= scale;
    if (d < D) store_vec<TX, VEC>(dst + d, v[i]);
  }
}

// ---- stable sort of (token, place) by token: least significant digit first, 8 bits a pass.  Tokens outside
// [0, V) take the key V and end up behind all others.
constexpr int kSortTile = 2048;   // keys per block
constexpr int kSortWarps = kThreads / 32;
constexpr int kPerWarp = kSortTile / kSortWarps;

PCB_DEVICE uint32_t sort_key(const void* tok, int tok64, const uint32_t* keys, int n, int V) {
  if (keys != nullptr) return keys[n];
  const long long t = load_id(tok, tok64, n);
  return t >= 0 && t < V ? (uint32_t)t : (uint32_t)V;
}

__global__ void __launch_bounds__(kThreads)
    sort_hist_kernel(const void* tok, int tok64, const uint32_t* __restrict__ keys, int N, int V, int shift,
                     uint32_t* __restrict__ hist, int blocks) {
  __shared__ uint32_t h[256];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * kSortTile;
  for (int i = threadIdx.x; i < kSortTile && t0 + i < N; i += kThreads)
    atomicAdd(&h[(sort_key(tok, tok64, keys, t0 + i, V) >> shift) & 255], 1u);   // counts: any order gives the same
  __syncthreads();
  hist[(long long)threadIdx.x * blocks + blockIdx.x] = h[threadIdx.x];
}

__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* __restrict__ hist, int total, int* __restrict__ list) {
  __shared__ int sums[32];
  if (threadIdx.x == 0) list[0] = 0;
  int base = 0;
  for (int t0 = 0; t0 < total; t0 += 1024) {
    const int i = t0 + threadIdx.x;
    const int v = i < total ? (int)hist[i] : 0;
    int sum;
    const int before = block_scan(v, sums, &sum, 32);
    if (i < total) hist[i] = base + before;
    base += sum;
  }
}

// A warp owns kPerWarp consecutive keys.  Digit counts per warp give each warp its first place of every digit;
// lanes with the same digit take places in lane order.
__global__ void __launch_bounds__(kThreads)
    sort_scatter_kernel(const void* tok, int tok64, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ idx,
                        int N, int V, int shift, const uint32_t* __restrict__ hist, int blocks,
                        uint32_t* __restrict__ keys_out, uint32_t* __restrict__ idx_out) {
  __shared__ uint32_t place[kSortWarps][256];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i = lane; i < 256; i += 32) place[w][i] = 0;
  __syncwarp();
  const int t0 = blockIdx.x * kSortTile + w * kPerWarp;
  for (int i = 0; i < kPerWarp; i += 32) {
    const int n = t0 + i + lane;
    if (n < N) atomicAdd(&place[w][(sort_key(tok, tok64, keys, n, V) >> shift) & 255], 1u);
  }
  __syncthreads();
  {
    uint32_t p = hist[(long long)threadIdx.x * blocks + blockIdx.x];
#pragma unroll
    for (int i = 0; i < kSortWarps; ++i) {
      const uint32_t c = place[i][threadIdx.x];
      place[i][threadIdx.x] = p;
      p += c;
    }
  }
  __syncthreads();
  for (int i = 0; i < kPerWarp; i += 32) {
    const int n = t0 + i + lane;
    const bool in = n < N;
    const uint32_t key = in ? sort_key(tok, tok64, keys, n, V) : 0u;
    const uint32_t digit = in ? (key >> shift) & 255 : 256u;   // lanes past the end match one another only
    const uint32_t same = __match_any_sync(0xffffffffu, digit);
    const uint32_t rank = __popc(same & ((1u << lane) - 1));
    uint32_t at = 0;
    if (in) at = place[w][digit] + rank;
    __syncwarp();
    if (in && rank == 0) place[w][digit] += __popc(same);
    __syncwarp();
    if (in) {
      keys_out[at] = key;
      idx_out[at] = idx != nullptr ? idx[n] : (uint32_t)n;
    }
  }
}

// ---- the same sort in one launch for up to 64 K keys: a cluster of 8 blocks holds them in registers and exchanges
// them through distributed shared memory, so a pass costs two cluster barriers instead of three launches.  The
// other clusters of the grid meanwhile write the zeros of the gradient, which bound this part when the matrix is large.
constexpr int kCluster = 8;
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;

template <int ITEMS>
constexpr int cluster_sort_smem() {
  return kClusterWarps * 256 * 4 + kCluster * 256 * 4 + 4 * 256 * 4 + 256 * 4 + ITEMS * kClusterThreads * 8;
}

PCB_DEVICE void write_zeros(char* p, long long bytes, int part, int parts) {
  const long long head = min(bytes, (long long)(-reinterpret_cast<uintptr_t>(p) & 15));
  const long long vecs = (bytes - head) / 16, tail = head + vecs * 16;
  uint4* q = reinterpret_cast<uint4*>(p + head);
  for (long long i = part * (long long)blockDim.x + threadIdx.x; i < vecs; i += (long long)parts * blockDim.x)
    q[i] = make_uint4(0, 0, 0, 0);
  if (part == 0) {
    for (long long i = threadIdx.x; i < head; i += blockDim.x) p[i] = 0;
    for (long long i = tail + threadIdx.x; i < bytes; i += blockDim.x) p[i] = 0;
  }
}

template <int ITEMS>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kClusterThreads)
    cluster_sort_kernel(const void* __restrict__ tok, int tok64, int N, int V, int bits, uint32_t* __restrict__ keys_out,
                        uint32_t* __restrict__ idx_out, int* __restrict__ list, char* zeros, long long zero_bytes) {
  extern __shared__ __align__(16) uint32_t sm[];
  uint32_t* warp_count = sm;                                     // [warps][256]: keys of a digit, then its first place
  uint32_t* count = warp_count + kClusterWarps * 256;            // [blocks][256], the same in every block
  uint32_t* quarter = count + kCluster * 256;                    // [4][256]
  uint32_t* first = quarter + 4 * 256;                           // [256] first place of this block's digit
  unsigned long long* pairs = reinterpret_cast<unsigned long long*>(first + 256);   // [ITEMS * 1024] place << 32 | key
  __shared__ int sums[32];
  pdl_begin();
  if (blockIdx.x >= kCluster) {   // whole clusters
    write_zeros(zeros, zero_bytes, blockIdx.x - kCluster, gridDim.x - kCluster);
    return;
  }
  constexpr int PER = ITEMS * kClusterThreads;
  if (blockIdx.x == 0 && threadIdx.x == 0) list[0] = 0;
  cluster_sync_all();   // every block of the cluster runs before another one writes to its shared memory
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int rank = (int)cluster_ctarank();
  const int mine = max(0, min(PER, N - rank * PER));
  uint32_t key[ITEMS], idx[ITEMS], place[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int k = (w * ITEMS + i) * 32 + lane;
    key[i] = k < mine ? sort_key(tok, tok64, nullptr, rank * PER + k, V) : 0u;
    idx[i] = (uint32_t)(rank * PER + k);
  }
  for (int shift = 0; shift < bits; shift += 8) {
    const bool last = shift + 8 >= bits;
    for (int i = tid; i < kClusterWarps * 256 / 4; i += kClusterThreads)
      reinterpret_cast<uint4*>(warp_count)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t* wc = warp_count + w * 256;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {   // place among the warp's keys of the same digit, in order
      const bool in = (w * ITEMS + i) * 32 + lane < mine;
      const uint32_t digit = in ? (key[i] >> shift) & 255 : 256u;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      const uint32_t before = __popc(same & ((1u << lane) - 1));
      const uint32_t have = in ? wc[digit] : 0u;
      place[i] = have + before;
      __syncwarp();
      if (in && before == 0) wc[digit] = have + __popc(same);
      __syncwarp();
    }
    __syncthreads();
    {   // over the warps: 4 threads a digit, 8 warps each
      const int d = tid & 255, part = tid >> 8;
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c[j] = warp_count[(part * 8 + j) * 256 + d];
        sum += c[j];
      }
      quarter[part * 256 + d] = sum;
      __syncthreads();
      uint32_t base = 0, all = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t v = quarter[j * 256 + d];
        if (j < part) base += v;
        all += v;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        warp_count[(part * 8 + j) * 256 + d] = base;
        base += c[j];
      }
#pragma unroll
      for (int j = 0; j < kCluster / 4; ++j)   // this block's count of the digit, to every block
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                         mapa_shared(smem_u32(count + rank * 256 + d), part * (kCluster / 4) + j)),
                     "r"(all)
                     : "memory");
    }
    cluster_sync_all();
    {
      uint32_t before = 0, all = 0;
      if (tid < 256) {
#pragma unroll
        for (int j = 0; j < kCluster; ++j) {
          const uint32_t v = count[j * 256 + tid];
          if (j < rank) before += v;
          all += v;
        }
      }
      int total;
      const int start = block_scan((int)all, sums, &total, 8);
      if (tid < 256) first[tid] = start + before;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if ((w * ITEMS + i) * 32 + lane < mine) {
        const uint32_t digit = (key[i] >> shift) & 255;
        const uint32_t at = first[digit] + wc[digit] + place[i];
        if (last) {
          keys_out[at] = key[i];
          idx_out[at] = idx[i];
        } else {
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(pairs + at % PER), at / PER)),
                       "l"((unsigned long long)idx[i] << 32 | key[i])
                       : "memory");
        }
      }
    }
    if (last) break;
    cluster_sync_all();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int k = (w * ITEMS + i) * 32 + lane;
      const unsigned long long p = k < mine ? pairs[k] : 0ull;
      key[i] = (uint32_t)p;
      idx[i] = (uint32_t)(p >> 32);
    }
  }
}

// ---- sums over runs of equal tokens.  A warp owns kChunk consecutive sorted entries and 32 VEC of the columns.  A run of
// up to kChunk entries is summed whole by the warp where it begins, which reads past its own entries for it.  A longer
// one leaves a partial row in every chunk that it touches (slot 1 where it begins, slot 0 behind) and is put on a
// list, and join_kernel adds its parts in order: however many tokens are the same, no warp sums more than two chunks.
constexpr int kChunk = 8;

template <typename TX, typename TW, int VEC>
PCB_DEVICE void emit(TW* dw, uint32_t id, int D, int d0, float (&a)[VEC], float scale, int add) {
  TW* o = dw + (long long)id * D + d0;
#pragma unroll
  for (int e = 0; e < VEC; ++e) a[e] *= scale;
  if (add) {
    float p[VEC];
    load_vec<TW, VEC>(o, p);
#pragma unroll
    for (int e = 0; e < VEC; ++e) a[e] += p[e];
  }
  store_vec<TW, VEC>(o, a);
}

template <typename TX, typename TW, int VEC>
__global__ void __launch_bounds__(kThreads)
    run_sums_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ idx, const TX* __restrict__ dx,
                    long long lddx, TW* __restrict__ dw, float* __restrict__ partial, int* __restrict__ list, int N, int V,
                    int D, float scale, int add) {
  using R = typename Raw<TX, VEC>::type;
  constexpr uint32_t kAll = 0xffffffffu;
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const int slices = (D + 32 * VEC - 1) / (32 * VEC);
  const long long item = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const long long chunk = item / slices;
  const int slice = (int)(item - chunk * slices);
  if (chunk * kChunk >= N) return;   // whole warps
  // lane l holds the key of entry l - kChunk of the chunk, with a chunk of keys on either side, and its place
  const long long n = chunk * kChunk + lane - kChunk;
  const bool in = lane < 3 * kChunk && n >= 0 && n < N;
  const uint32_t key = in ? keys[n] : kAll - lane;   // outside: no two alike
  const uint32_t place = in && lane >= kChunk ? idx[n] : 0u;
  const uint32_t before = __shfl_up_sync(kAll, key, 1), behind8 = __shfl_down_sync(kAll, key, kChunk);
  // per entry: the same token as the entry before; as the entry kChunk behind (of a run's first: it is a long run); a
  // token with a row
  const uint32_t same = __ballot_sync(kAll, lane > 0 && key == before);
  const uint32_t longer = __ballot_sync(kAll, lane < 2 * kChunk && key == behind8);
  const uint32_t live = __ballot_sync(kAll, in && key < (uint32_t)V);
  // the chunk's first entry that is this warp's: behind a short run that began in the chunk before
  int first = kChunk;
  bool late = (same >> kChunk) & 1;   // the run at hand began in an earlier chunk
  if (late) {
    const int s = 31 - __clz(~same & ((2u << kChunk) - 1));   // its first entry in sight
    if (!((longer >> s) & 1)) {
      first = min(2 * kChunk, kChunk - 1 + __ffs(~(same >> kChunk)));
      late = false;
    }
  }
  // entries of the next chunk that belong to a short run which begins here
  int more = 0;
  {
    const int s = 31 - __clz(~same & ((1u << (2 * kChunk)) - 1));   // first entry of the chunk's last run
    if (s >= first && !((longer >> s) & 1)) more = __ffs(~(same >> (2 * kChunk))) - 1;
  }
  const int d0 = (slice * 32 + lane) * VEC;
  const bool mine = d0 < D;
  // All rows are asked for at once: behind the zeros of a large matrix, which are still on their way to memory, a
  // read takes microseconds.
  constexpr int kAhead = 4;
  R r[kChunk], ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const uint32_t at = __shfl_sync(kAll, place, kChunk + i);
    if (mine && kChunk + i >= first && ((live >> (kChunk + i)) & 1)) r[i] = *reinterpret_cast<const R*>(dx + at * lddx + d0);
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const uint32_t at = __shfl_sync(kAll, place, 2 * kChunk + i);
    if (mine && i < more && ((live >> (2 * kChunk + i)) & 1)) ahead[i] = *reinterpret_cast<const R*>(dx + at * lddx + d0);
  }
  float acc[VEC] = {};
  bool whole = false;   // the run at hand is summed here to its end
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const int l = kChunk + i;
    if (l < first) continue;
    if (!((live >> l) & 1)) return;   // only tokens without a row follow
    if (!late && (l == first || !((same >> l) & 1))) whole = !((longer >> l) & 1);
    float v[VEC];
    unpack<TX, VEC>(r[i], v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] += v[e];
    if (i < kChunk - 1 && ((same >> (l + 1)) & 1)) continue;
    const uint32_t id = __shfl_sync(kAll, key, l);
    if (late || !whole) {   // the run's part in this chunk
      if (mine) store_vec<float, VEC>(partial + (chunk * 2 + (late ? 0 : 1)) * D + d0, acc);
      if (!late && slice == 0 && lane == 0) list[1 + atomicAdd(list, 1)] = (int)chunk;   // in any order
    } else {
      if (i == kChunk - 1) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (j >= more) break;
          unpack<TX, VEC>(ahead[j], v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += v[e];
        }
        for (int j = kAhead; j < more; ++j) {
          const uint32_t at = __shfl_sync(kAll, place, 2 * kChunk + j);
          if (mine) load_vec<TX, VEC>(dx + at * lddx + d0, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += v[e];
        }
      }
      if (mine) emit<TX, TW, VEC>(dw, id, D, d0, acc, scale, add);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    late = false;
  }
}

// The long runs.  A block takes a run of the list and 32 VEC columns at a time; its warps share the run's parts, and the
// first warp adds the warps' sums in order.
template <typename TW, int VEC>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ partial, const int* __restrict__ list,
                TW* __restrict__ dw, int N, int V, int D, float scale, int add) {
  constexpr int kWarps = kThreads / 32, U = 8;
  __shared__ float s_sum[kWarps][32][VEC + 1];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int slices = (D + 32 * VEC - 1) / (32 * VEC);
  const long long items = (long long)list[0] * slices;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int d0 = ((int)(item % slices) * 32 + lane) * VEC;
    const long long c = list[1 + item / slices], next = (c + 1) * kChunk;
    const uint32_t id = keys[next];
    int parts = 1;   // chunks that the run touches
    for (int more = blockDim.x; more == (int)blockDim.x;) {
      const long long at = next + ((long long)parts - 1 + threadIdx.x) * kChunk;
      more = __syncthreads_count(at < N && keys[at] == id);
      parts += more;
    }
    const int per = (parts + kWarps - 1) / kWarps, p0 = min(parts, w * per), p1 = min(parts, p0 + per);
    float acc[VEC] = {};
    if (d0 < D) {
      for (int p = p0; p < p1; p += U) {
        float r[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (p + u < p1) load_vec<float, VEC>(partial + ((c + p + u) * 2 + (p + u == 0 ? 1 : 0)) * D + d0, r[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (p + u < p1) acc[e] += r[u][e];
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_sum[w][lane][e] = acc[e];
    __syncthreads();
    if (w == 0 && d0 < D) {
#pragma unroll
      for (int k = 1; k < kWarps; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += s_sum[k][lane][e];
      emit<float, TW, VEC>(dw, id, D, d0, acc, scale, add);
    }
    __syncthreads();
  }
}

// ---- a batch of few tokens, in one launch and without sorting.  Every block reads all tokens.  A block of sums has a token
// a warp and 32 VEC columns: a warp whose token stands at no earlier place finds the later ones by comparing and adds
// their rows in order; a token with more than kFewTogether of them is left to all warps of the block, which list its
// places, add an eighth of them each and join the sums in order.  The warps of a block take places far apart, since the
// first places of a batch are where its frequent tokens are met first.  The other blocks write the zeros of the
// rows without a token.  Sorting against this, tokens that fall off as 1 / rank: 32 tokens into 5003 x 101 8.0 -> 2.9 us,
// 512 10.3 -> 5.5, 1024 11.4 -> 6.8; 1024 that are all the same 10.7 -> 11.3.  A large matrix's zeros are in the
// way of the rows: into 32000 x 768 fp32 512 tokens take 20.9 -> 19.7 us, 21.3 -> 21.9 all the same, but 1024 22.1 ->
// 23.5 and 22.3 -> 31.6.  A warp takes up to 16 places alone: 1024 tokens in runs of 12 into 5003 x 101 take 6.0 us, 9.3 with
// up to 8; in runs of 24 8.4, 6.2 with up to 32, and all else (1 / rank: 7.1) the same.
constexpr int kFewTokens = 1024;
constexpr long long kFewZeros = 32 << 20;   // more zeros than this: half as many tokens
constexpr int kFewTogether = 16;
constexpr int kFewZeroRows = 1024;   // most rows of a block of zeros

template <typename TX, typename TW, int VEC>
__global__ void __launch_bounds__(kThreads, 4)
    few_tokens_kernel(const void* __restrict__ tok, int tok64, const TX* __restrict__ dx, long long lddx,
                      TW* __restrict__ dw, int N, int V, int D, float scale, int add, int slices, int sum_blocks) {
  using R = typename Raw<TX, VEC>::type;
  constexpr int kWarps = kThreads / 32, U = VEC == 1 && sizeof(TX) == 4 ? 16 : 8;
  constexpr uint32_t kAll = 0xffffffffu;
  __shared__ uint32_t keys[kFewTokens];
  __shared__ float s_sum[kWarps][32][VEC + 1];
  __shared__ unsigned short s_at[kWarps][kFewTogether], s_all[kFewTokens];
  __shared__ int s_count[kWarps];
  __shared__ int s_many[kWarps];
  __shared__ uint32_t used[kFewZeroRows / 32];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < N; i += kThreads) {
    const long long t = load_id(tok, tok64, i);
    keys[i] = t >= 0 && t < V ? (uint32_t)t : kAll;
  }
  if ((int)blockIdx.x >= sum_blocks) {
    const int z = blockIdx.x - sum_blocks, parts = gridDim.x - sum_blocks;
    const int v0 = (int)((long long)V * z / parts), rows = (int)((long long)V * (z + 1) / parts) - v0;
    if (threadIdx.x < kFewZeroRows / 32) used[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < N; i += kThreads) {
      const uint32_t at = keys[i] - (uint32_t)v0;
      if (at < (uint32_t)rows) atomicOr(&used[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    float none[VEC] = {};
    for (int r = w; r < rows; r += kWarps) {
      if ((used[r >> 5] >> (r & 31)) & 1) continue;
      for (int d = lane * VEC; d < D; d += 32 * VEC) store_vec<TW, VEC>(dw + (long long)(v0 + r) * D + d, none);
    }
    return;
  }
  __syncthreads();
  const int apart = sum_blocks / slices, n = (int)blockIdx.x / slices + w * apart;
  const int d0 = ((int)blockIdx.x % slices * 32 + lane) * VEC;
  const bool mine = d0 < D;
  uint32_t key = n < N ? keys[n] : kAll;
  bool earlier = key == kAll;
#pragma unroll 4
  for (int m = lane; m < n; m += 32) earlier = earlier || keys[m] == key;
  const bool first = !__any_sync(kAll, earlier);
  int count = 0;
  if (first) {
#pragma unroll 4
    for (int base = n & ~31; base < N; base += 32) {
      const int m = base + lane;
      const uint32_t same = __ballot_sync(kAll, m >= n && m < N && keys[m] == key);
      if ((same >> lane) & 1) {
        const int at = count + __popc(same & ((1u << lane) - 1));
        if (at < kFewTogether) s_at[w][at] = (unsigned short)m;
      }
      count += __popc(same);
    }
    __syncwarp();
  }
  const bool many = count > kFewTogether;
  if (lane == 0) s_many[w] = many;
  float acc[VEC] = {};
  auto add_rows = [&](const unsigned short* at, int n0, int n1) {
    for (int i = n0; i < n1; i += U) {
      R r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (mine && i + u < n1) r[u] = *reinterpret_cast<const R*>(dx + at[i + u] * lddx + d0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u >= n1) break;
        float v[VEC];
        unpack<TX, VEC>(r[u], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[e];
      }
    }
  };
  if (first && !many) {
    add_rows(s_at[w], 0, count);
    if (mine) emit<TX, TW, VEC>(dw, key, D, d0, acc, scale, add);
  }
  __syncthreads();
  for (int k = 0; k < kWarps; ++k) {
    if (!s_many[k]) continue;
    key = keys[n + (k - w) * apart];
    // the token's places in order: a warp lists those of an eighth of the batch, behind what the warps before it have
    const int steps = (N + 31) / 32, s0 = steps * w / kWarps, s1 = steps * (w + 1) / kWarps;
    uint32_t same[kFewTokens / 32 / kWarps];
    int here = 0;
#pragma unroll
    for (int i = 0; i < kFewTokens / 32 / kWarps; ++i) {
      const int m = (s0 + i) * 32 + lane;
      same[i] = __ballot_sync(kAll, s0 + i < s1 && m < N && keys[m] == key);
      here += __popc(same[i]);
    }
    if (lane == 0) s_count[w] = here;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) {
      if (j < w) at += s_count[j];
      total += s_count[j];
    }
#pragma unroll
    for (int i = 0; i < kFewTokens / 32 / kWarps; ++i) {
      if ((same[i] >> lane) & 1) s_all[at + __popc(same[i] & ((1u << lane) - 1))] = (unsigned short)((s0 + i) * 32 + lane);
      at += __popc(same[i]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    add_rows(s_all, total * w / kWarps, total * (w + 1) / kWarps);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_sum[w][lane][e] = acc[e];
    __syncthreads();
    if (w == 0 && mine) {
#pragma unroll
      for (int j = 1; j < kWarps; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += s_sum[j][lane][e];
      emit<TX, TW, VEC>(dw, key, D, d0, acc, scale, add);
    }
    __syncthreads();
  }
}

inline bool al(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline int launched() { return cudaGetLastError() == cudaSuccess ? 0 : -3; }

}  // namespace vocab

using namespace vocab;

VocabLayout vocab_layout(int N, int V, int D, int K, bool distill) {
  VocabLayout l{};
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  l.ldxc = (D + 7) / 8 * 8;
  l.granules = 2 * ((V + 255) / 256);
  l.xc = take((long long)N * l.ldxc * 2);
  l.count = take(32);
  l.row = take(4LL * N);
  l.pos = take(4LL * N);
  l.norm = take(8LL * N);
  l.z = take(4LL * N * K);
  l.ids = take(4LL * N * K);
  if (distill) {
    l.q = take(4LL * N * K);
    l.lq = take(4LL * N * K);
    l.len = take(4LL * N);
    l.start = take(2LL * N * (l.granules + 1));
  }
  l.bytes = at;
  return l;
}

// Rows of g: the counted ones up to the next tile; behind the one tile that a second term is made for, that term.
long long vocab_g_rows(int N) { return std::max((N + 255LL) / 256 * 256, 2LL * kTwoTermRows); }

static bool few_rows(int N, int D) { return N <= kFewRows && D <= kFewColumns; }

VocabPlan vocab_plan(int N, int V, int D, int want_piece, bool gradient, int num_sms) {
  VocabPlan r{};
  const long long all = (V + 255LL) / 256 * 256;
  // 256 MiB of g: the backward of 16384 x 768 x 32000 takes 1868 us (128 MiB: 1970, 64: 2648, 512: 1830, 1024, which is one
  // piece: 1756)
  long long p = want_piece > 0 ? (want_piece + 255LL) / 256 * 256 : (256LL << 20) / (2 * vocab_g_rows(N)) / 256 * 256;
  p = std::max(256LL, std::min(p, all));
  r.pieces = (int)((all + p - 1) / p);
  p = (all / 256 + r.pieces - 1) / r.pieces * 256;   // pieces of one size
  r.piece = (int)p;
  r.pieces = (int)((all + p - 1) / p);
  // dw is split where its tiles do not fill the GPU; dx has room for a few splits of every row, and for all splits of a
  // few rows
  const int bn = head_bn(D);
  const long long tiles = p / 256 * ((D + bn - 1) / bn);
  r.dw_max = r.pieces == 1 ? (int)std::max(1LL, std::min(8LL, num_sms / 2 / tiles)) : 1;
  r.slab_rows = (int)std::min((N + 255LL) / 256 * 256 + 16 * 256, 1LL << 30);
  r.all_rows = r.slab_rows + (r.dw_max > 1 ? r.dw_max * all : 0);
  // a block of 128 columns an SM at least, or the FMA units are quicker: one row of 1600 against 300 takes 12.4 us, 16.2
  // by score_kernel; one of 2048 against 32000 35.8 and 31.5
  r.score = !gradient && N <= kScoreRows && !(few_rows(N, D) && V <= 128LL * num_sms);
  // g then lives as long as the forward's state, so it is bounded as a piece is
  r.whole = gradient && r.pieces == 1 && !few_rows(N, D) && pcb_head_whole(N, V, D);
  return r;
}

}  // namespace pcb

using namespace pcb;
using namespace pcb::vocab;

int pcb_vocab_pad_rows(const void* src, long long ld, void* dst, long long ldd, int rows, int D, cudaStream_t s) {
  const long long total = rows * ldd;
  const int grid = (int)std::min<long long>((total + 255) / 256, 148 * 16);
  pad_rows_kernel<<<grid, 256, 0, s>>>((const __nv_bfloat16*)src, ld, (__nv_bfloat16*)dst, ldd, total, D);
  return launched();
}

static char* at(void* base, long long off) { return (char*)base + off; }

// whether the products may read x itself: rows that a tensor map can describe
static bool readable(const void* x, long long ldx, int D) {
  return D % 8 == 0 && ldx % 8 == 0 && ldx >= D && al(x, 16);
}

template <bool GRAD>
static int launch_few_rows(const HeadGemm& h, const void* xc, long long ldxc, const void* x, long long ldx, const void* w,
                           long long ldw, void* g, cudaStream_t s) {
  FewRowsArgs f{};
  f.x = (const __nv_bfloat16*)x;
  f.ldx = ldx;
  f.xc = (const __nv_bfloat16*)xc;
  f.ldxc = ldxc;
  f.w = (const __nv_bfloat16*)w;
  f.ldw = ldw;
  f.g = (__nv_bfloat16*)g;
  f.h = h;
  auto go = [&](auto nr) {
    constexpr int NR = decltype(nr)::value;
    static SmemLimit limit;
    if (!limit.raise(few_rows_kernel<NR, GRAD>, NR * kFewColumns * 2)) return cudaErrorInvalidValue;
    return pdl_launch(few_rows_kernel<NR, GRAD>, dim3((h.cols + 127) / 128), dim3(few_threads(NR)), (size_t)(NR * ldxc * 2), s, f);
  };
  const cudaError_t e = h.N == 1   ? go(std::integral_constant<int, 1>{})
                        : h.N == 2 ? go(std::integral_constant<int, 2>{})
                                   : go(std::integral_constant<int, 4>{});
  return e == cudaSuccess ? 0 : -3;
}

// what the backward's launches, and the forward's where it makes g, know of the gradients' products
static void plan_products(HeadGemm& g, const VocabPlan& plan, int N, int* splits, int num_sms) {
  g.g_low = kTwoTermRows;
  g.g_rows = (int)vocab_g_rows(N);
  g.plan = splits;
  g.dw_max = plan.dw_max;
  g.slab_rows = plan.slab_rows;
  g.bwd_pairs = num_sms / 2;
}

int pcb_vocab_fwd(const VocabHeadArgs& a, const VocabPlan& plan, void* saved, void* part, void* dlogits, int mean,
                  int num_sms, cudaStream_t s) {
  const bool distill = a.tgt == nullptr;
  if (a.N < 1 || a.V < 1 || a.D < 1 || a.K < 1 || a.K > kMaxK) return -1;
  const VocabLayout l = vocab_layout(a.N, a.V, a.D, a.K, distill);
  int *row = (int*)at(saved, l.row), *ids = (int*)at(saved, l.ids), *count = (int*)at(saved, l.count);
  float2* norm = (float2*)at(saved, l.norm);
  float* z = (float*)at(saved, l.z);
  float *q = distill ? (float*)at(saved, l.q) : nullptr, *lq = distill ? (float*)at(saved, l.lq) : nullptr;
  int* len = distill ? (int*)at(saved, l.len) : nullptr;
  unsigned short* start = distill ? (unsigned short*)at(saved, l.start) : nullptr;
  const float T = distill ? a.temperature : 1.f;
  const float c = 1.4426950408889634f / T, factor = 0.6931471805599453f * T * T;
  if (distill) {
    auto sort = [&](auto r) {
      constexpr int R = decltype(r)::value, rows = kSortRows;
      return pdl_launch(sort_targets_kernel<R>, dim3((a.N + rows - 1) / rows), dim3(32 * rows), 0, s, a.ids, a.ids64, a.ld_ids, a.logits, a.logits_bf16, a.ld_logits, a.N, a.V,
                        a.K, c, ids, q, lq, len, start, l.granules);
    };
    const cudaError_t e = a.K <= 32    ? sort(std::integral_constant<int, 1>{})
                          : a.K <= 64  ? sort(std::integral_constant<int, 2>{})
                          : a.K <= 128 ? sort(std::integral_constant<int, 4>{})
                                       : sort(std::integral_constant<int, 8>{});
    if (e != cudaSuccess) return -3;
  }
  PackArgs p{};
  p.tgt = a.tgt;
  p.tgt64 = a.tgt64;
  p.ignore = a.ignore;
  p.len = len;
  p.V = a.V;
  p.N = a.N;
  p.D = a.D;
  p.x = (const __nv_bfloat16*)a.x;
  p.ldx = a.ldx;
  p.vec = a.D % 8 == 0 && a.ldx % 8 == 0 && al(a.x, 16);
  p.in_place = readable(a.x, a.ldx, a.D);
  p.xc = (__nv_bfloat16*)at(saved, l.xc);
  p.ldxc = l.ldxc;
  p.row = row;
  p.pos = (int*)at(saved, l.pos);
  p.tgt32 = distill ? nullptr : ids;
  p.count = count;
  p.loss = a.loss;
  int blocks, R;
  if (a.N > kSelfCountRows) {
    blocks = (a.N + kCountRows - 1) / kCountRows;
    R = kCountRows;
    int* counts = (int*)part;   // the pairs are written later
    if (pdl_launch(count_rows_kernel, dim3(blocks), dim3(kCountRows), 0, s, p, counts) != cudaSuccess) return -3;
    p.counts = counts;
  } else {
    blocks = std::max(1, std::min(2 * num_sms, (a.N + 7) / 8));   // 64 or more: at most 128 rows each
    R = (a.N + blocks - 1) / blocks;
  }
  if (pdl_launch(pack_rows_kernel, dim3(blocks), dim3(kThreads), 0, s, p, R) != cudaSuccess) return -3;
  auto finish = [&](const VocabLayout& l, int pairs) {   // row losses from `pairs` (max, sum) pairs a row
    return pdl_launch(row_loss_kernel, dim3((a.N + 31) / 32), dim3(32 * kLossParts), 0, s, (const float2*)part, pairs,
                      (const int*)row, (const float*)z, (const float*)q, (const float*)lq, (const int*)len, a.N, a.K, c,
                      factor, norm, a.loss, count, mean, a.total, (float*)(count + 5)) == cudaSuccess ? 0 : -3;
  };
  HeadGemm g{};
  g.N = a.N;
  g.D = a.D;
  g.cols = a.V;
  g.count = count;
  g.err = count + 4;
  g.c = c;
  g.row = row;
  g.ids = ids;
  g.K = a.K;
  g.start = start;
  g.part = (float2*)part;
  g.z = z;
  if (plan.score) {
    const int rc = pcb_head_score(g, p.xc, l.ldxc, p.in_place ? a.x : nullptr, a.ldx, a.w, a.ldw, s);
    return rc ? rc : finish(l, (a.V + 127) / 128);
  }
  if (few_rows(a.N, a.D)) {
    const int rc = launch_few_rows<false>(g, p.xc, l.ldxc, p.in_place ? a.x : nullptr, a.ldx, a.w, a.ldw, nullptr, s);
    return rc ? rc : finish(l, (a.V + 127) / 128);
  }
  if (plan.whole) {
    plan_products(g, plan, a.N, count + 2, num_sms);
    g.q = q;
    g.loss = a.loss;
    g.factor = factor;
    g.total = a.total;
    g.inverse = (float*)(count + 5);
    g.mean = mean;
    g.done = count + 1;
    return pcb_head_gemm(HEAD_WHOLE, g, p.xc, l.ldxc, p.in_place ? a.x : nullptr, a.ldx, a.w, a.ldw, dlogits, num_sms, s);
  }
  const int rc = pcb_head_gemm(HEAD_STAT, g, p.xc, l.ldxc, p.in_place ? a.x : nullptr, a.ldx, a.w, a.ldw, nullptr, num_sms, s);
  if (rc) return rc;
  return finish(l, l.granules);
}

// the lists' sort, a long batch's count, the packing; the product, which makes the row losses too where it is whole
int pcb_vocab_fwd_launches(const VocabPlan& plan, int N, bool distill) {
  return (distill ? 1 : 0) + (N > kSelfCountRows ? 1 : 0) + 1 + (plan.whole ? 1 : 2);
}

// for each piece g, unless the forward made it, and the products; the gather
int pcb_vocab_bwd_launches(const VocabPlan& plan) { return (plan.whole ? 1 : 2) * plan.pieces + 1; }

int pcb_vocab_bwd(const VocabGradArgs& a, int num_sms, cudaStream_t s) {
  const VocabLayout l = vocab_layout(a.N, a.V, a.D, a.K, a.distill != 0);
  void* sv = a.saved;
  const void* x_all = readable(a.x, a.ldx, a.D) ? a.x : nullptr;
  const float T = a.distill ? a.temperature : 1.f;
  HeadGemm g{};
  g.N = a.N;
  g.D = a.D;
  g.count = (const int*)at(sv, l.count);
  g.err = (int*)at(sv, l.count) + 4;
  g.c = 1.4426950408889634f / T;
  g.row = (const int*)at(sv, l.row);
  g.ids = (const int*)at(sv, l.ids);
  g.K = a.K;
  if (a.distill) {
    g.q = (const float*)at(sv, l.q);
    g.start = (const unsigned short*)at(sv, l.start);
  }
  g.norm = (const float2*)at(sv, l.norm);
  plan_products(g, a.plan, a.N, a.plan.whole ? (int*)at(sv, l.count) + 2 : a.splits, num_sms);
  g.want_dw = a.dw != nullptr;
  g.want_dx = a.dx != nullptr;
  g.lddw = a.lddw;
  g.dw_f32 = a.dw_f32;
  g.dw_add = a.dw_add;
  g.alpha = a.gout * T;
  g.scale = a.mean ? (const float*)(g.count + 5) : nullptr;
  g.scale2 = a.gout_dev;
  g.slab = a.slab;
  g.ld_slab = a.ld_slab;
  for (int v0 = 0; v0 < a.V; v0 += a.plan.piece) {
    g.v0 = v0;
    g.cols = std::min(a.plan.piece, a.V - v0);
    g.dx_add = v0 > 0;
    g.dw = a.dw == nullptr ? nullptr : (char*)a.dw + (long long)v0 * a.lddw * (a.dw_f32 ? 4 : 2);
    const __nv_bfloat16* w = (const __nv_bfloat16*)a.w + (long long)v0 * a.ldw;
    for (int mode : {HEAD_GRAD, HEAD_BWD}) {
      if (mode == HEAD_GRAD && a.plan.whole) continue;   // the forward made g
      const int rc = mode == HEAD_GRAD && few_rows(a.N, a.D)
                         ? launch_few_rows<true>(g, at(sv, l.xc), l.ldxc, x_all, a.ldx, w, a.ldw, a.g, s)
                         : pcb_head_gemm(mode, g, at(sv, l.xc), l.ldxc, x_all, a.ldx, w, a.ldw, a.g, num_sms, s);
      if (rc) return rc;
    }
  }
  FinishArgs f{};
  f.slab = a.slab;
  f.slab_rows = a.plan.slab_rows;
  f.count = g.count;
  f.plan = g.plan;
  f.status = g.err;
  f.pos = (const int*)at(sv, l.pos);
  f.dx = a.dx;
  f.dw = a.dw;
  f.ld_slab = a.ld_slab;
  f.lddx = a.lddx;
  f.lddw = a.lddw;
  f.dx_f32 = a.dx_f32;
  f.dw_f32 = a.dw_f32;
  f.dw_add = a.dw_add;
  f.N = a.dx != nullptr ? a.N : 0;
  f.V = a.dw != nullptr && a.plan.dw_max > 1 ? a.V : 0;
  f.dw_rows = a.dw != nullptr ? a.V : 0;
  f.D = a.D;
  f.alpha = g.alpha;
  f.scale = g.scale;
  f.scale2 = g.scale2;
  const bool v4 = a.D % 4 == 0 && (f.N == 0 || (a.lddx % 4 == 0 && al(a.dx, a.dx_f32 ? 16 : 8))) &&
                  (f.V == 0 || (a.lddw % 4 == 0 && al(a.dw, a.dw_f32 ? 16 : 8)));
  const int vecs = v4 ? a.D / 4 : a.D;
  // with nothing to gather the launch is there for the status alone
  const dim3 grid(std::max((f.N + f.V + 7) / 8, 1), (vecs + 32 * kFinishVecs - 1) / (32 * kFinishVecs));
  if (grid.y > 65535) return -1;
  return pdl_launch(v4 ? finish_kernel<4> : finish_kernel<1>, grid, dim3(kThreads), 0, s, f) == cudaSuccess ? 0 : -3;
}

template <typename F>
static void by_type(int w_bf16, int x_bf16, F f) {
  if (w_bf16) {
    if (x_bf16) f((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr);
    else f((__nv_bfloat16*)nullptr, (float*)nullptr);
  } else {
    if (x_bf16) f((float*)nullptr, (__nv_bfloat16*)nullptr);
    else f((float*)nullptr, (float*)nullptr);
  }
}

int pcb_vocab_embed_fwd(const void* tok, int tok64, const void* w, int w_bf16, long long ldw, void* x, int x_bf16,
                        int N, int V, int D, float scale, cudaStream_t s) {
  int rc = 0;
  by_type(w_bf16, x_bf16, [&](auto* tw, auto* tx) {
    using TW = std::remove_pointer_t<decltype(tw)>;
    using TX = std::remove_pointer_t<decltype(tx)>;
    auto go = [&](auto v) {
      constexpr int VEC = decltype(v)::value;
      const int vecs = (D + VEC - 1) / VEC;
      const dim3 grid((N + 7) / 8, (vecs + 32 * kLookupVecs - 1) / (32 * kLookupVecs));
      if (grid.y > 65535) { rc = -1; return; }
      rc = pdl_launch(lookup_kernel<TW, TX, VEC>, grid, dim3(kThreads), 0, s, tok, tok64, (const TW*)w, ldw, (TX*)x, N, V,
                      D, scale) == cudaSuccess ? 0 : -3;
    };
    if (D % 4 == 0 && ldw % 4 == 0 && al(w, w_bf16 ? 8 : 16) && al(x, x_bf16 ? 8 : 16)) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 1>{});
  });
  return rc;
}

static long long up256(long long b) { return (b + 255) / 256 * 256; }

// keys of one cluster's sort; longer batches take the launch-per-step sort
constexpr int kClusterKeys = 8 * kCluster * kClusterThreads;

long long pcb_vocab_embed_bwd_bytes(int N, int V, int D) {
  const long long blocks = (N + kSortTile - 1) / kSortTile, chunks = (N + kChunk - 1) / kChunk;
  return (N <= kClusterKeys ? 2 : 4) * up256(4LL * N) + (N <= kClusterKeys ? 0 : up256(4LL * 256 * blocks)) +
         up256(8LL * chunks * D) + up256(4LL * (chunks + 1));
}

static long long zeros_of(int V, int D, int dw_bf16, int add) { return add ? 0 : (long long)V * D * (dw_bf16 ? 2 : 4); }
static bool few_tokens(int N, long long zero_bytes) { return N <= (zero_bytes <= kFewZeros ? kFewTokens : kFewTokens / 2); }

int pcb_vocab_embed_bwd_launches(int N, int V, int D, int dw_bf16, int add) {
  if (few_tokens(N, zeros_of(V, D, dw_bf16, add))) return 1;
  if (N <= kClusterKeys) return 3;
  int passes = 1;
  while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
  return 3 * passes + 2;
}

template <int ITEMS>
static int launch_cluster_sort(const void* tok, int tok64, int N, int V, int bits, uint32_t* keys, uint32_t* idx, int* list,
                               void* zeros, long long zero_bytes, int num_sms, cudaStream_t s) {
  constexpr int smem = cluster_sort_smem<ITEMS>();
  static SmemLimit limit;
  if (!limit.raise(cluster_sort_kernel<ITEMS>, smem)) return -3;
  // as many more clusters as there is for them to write, 64 KB a block, up to 7 blocks an SM: of 131 MB (4096 tokens, V
  // 32000, D 2048) 16 clusters made 55 us of the gradient, 34 made 44, 128 made 38 and 512 made 41
  const int most = 7 * num_sms / kCluster;
  const int clusters = zero_bytes > 0 ? 1 + (int)std::min<long long>(most, (zero_bytes >> 19) + 1) : 1;
  return pdl_launch(cluster_sort_kernel<ITEMS>, dim3(clusters * kCluster), dim3(kClusterThreads), smem, s, tok, tok64, N,
                    V, bits, keys, idx, list, (char*)zeros, zero_bytes) == cudaSuccess ? 0 : -3;
}

int pcb_vocab_embed_bwd(const void* tok, int tok64, const void* dx, int dx_bf16, long long lddx, void* dw, int dw_bf16,
                        int N, int V, int D, float scale, int add, void* ws, int num_sms, cudaStream_t s) {
  const int blocks = (N + kSortTile - 1) / kSortTile, chunks = (N + kChunk - 1) / kChunk;
  if (blocks > (1 << 22)) return -1;   // 256 counts a block are scanned as ints
  const long long zero_bytes = zeros_of(V, D, dw_bf16, add);
  char* p = (char*)ws;
  auto take = [&](long long bytes) {
    char* q = p;
    p += up256(bytes);
    return q;
  };
  int bits = 1;
  while (bits < 32 && (V >> bits) != 0) ++bits;   // keys run up to V
  const uint32_t *keys = nullptr, *idx = nullptr;
  int* list = (int*)take(4LL * (chunks + 1));   // number of long runs, then the chunks where they begin; emptied by the sort
  int rc = 0;
  const bool few = few_tokens(N, zero_bytes);   // nothing to sort
  if (few) {
  } else if (N <= kClusterKeys) {
    uint32_t *k = (uint32_t*)take(4LL * N), *i = (uint32_t*)take(4LL * N);
    auto sort = [&](auto items) {
      return launch_cluster_sort<decltype(items)::value>(tok, tok64, N, V, bits, k, i, list, dw, zero_bytes, num_sms, s);
    };
    if (N <= kClusterKeys / 8) rc = sort(std::integral_constant<int, 1>{});
    else if (N <= kClusterKeys / 4) rc = sort(std::integral_constant<int, 2>{});
    else if (N <= kClusterKeys / 2) rc = sort(std::integral_constant<int, 4>{});
    else rc = sort(std::integral_constant<int, 8>{});
    if (rc) return rc;
    keys = k;
    idx = i;
  } else {
    uint32_t* buf[4];
    for (auto& b : buf) b = (uint32_t*)take(4LL * N);
    uint32_t* hist = (uint32_t*)take(4LL * 256 * blocks);
    if (zero_bytes > 0 && cudaMemsetAsync(dw, 0, (size_t)zero_bytes, s) != cudaSuccess) return -3;
    int side = 0;
    for (int shift = 0; shift < bits; shift += 8) {
      sort_hist_kernel<<<blocks, kThreads, 0, s>>>(tok, tok64, keys, N, V, shift, hist, blocks);
      sort_scan_kernel<<<1, 1024, 0, s>>>(hist, 256 * blocks, list);
      sort_scatter_kernel<<<blocks, kThreads, 0, s>>>(tok, tok64, keys, idx, N, V, shift, hist, blocks, buf[2 * side],
                                                      buf[2 * side + 1]);
      if (launched()) return -3;
      keys = buf[2 * side];
      idx = buf[2 * side + 1];
      side ^= 1;
    }
  }
  float* partial = (float*)take(8LL * chunks * D);
  by_type(dw_bf16, dx_bf16, [&](auto* tw, auto* tx) {
    using TW = std::remove_pointer_t<decltype(tw)>;
    using TX = std::remove_pointer_t<decltype(tx)>;
    auto go = [&](auto v) {
      constexpr int VEC = decltype(v)::value;
      const int cols = (D + VEC - 1) / VEC;
      const int slices = (cols + 31) / 32;
      const long long warps = (long long)chunks * slices, blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
      if (blocks > 0x7fffffffLL) { rc = -1; return; }
      if (few) {
        const long long sums = (long long)((N + kThreads / 32 - 1) / (kThreads / 32)) * slices;
        long long zeros = 0;   // blocks of 16 KB or more, 2 an SM; of 128 KB where that is not enough
        if (!add) {
          zeros = std::max(std::min<long long>(zero_bytes >> 14, 2 * num_sms), zero_bytes >> 17);
          zeros = std::max(zeros, (long long)V / (kFewZeroRows - 1) + 1);
        }
        if (sums + zeros > 0x7fffffffLL) { rc = -1; return; }
        rc = pdl_launch(few_tokens_kernel<TX, TW, VEC>, dim3((unsigned)(sums + zeros)), dim3(kThreads), 0, s, tok, tok64,
                        (const TX*)dx, lddx, (TW*)dw, N, V, D, scale, add, slices, (int)sums) == cudaSuccess ? 0 : -3;
        return;
      }
      const int joins = (int)std::min<long long>(4 * num_sms, warps);
      if (pdl_launch(run_sums_kernel<TX, TW, VEC>, dim3((unsigned)blocks), dim3(kThreads), 0, s, keys, idx, (const TX*)dx, lddx, (TW*)dw,
                     partial, list, N, V, D, scale, add) != cudaSuccess ||
          pdl_launch(join_kernel<TW, VEC>, dim3(joins), dim3(kThreads), 0, s, keys, (const float*)partial, (const int*)list,
                     (TW*)dw, N, V, D, scale, add) != cudaSuccess)
        rc = -3;
    };
    const bool wide = dx_bf16 && D % 8 == 0 && lddx % 8 == 0 && al(dx, 16) && al(dw, 16);
    if (wide) go(std::integral_constant<int, 8>{});
    else if (D % 4 == 0 && lddx % 4 == 0 && al(dx, dx_bf16 ? 8 : 16) && al(dw, dw_bf16 ? 8 : 16))
      go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 1>{});
  });
  return rc;
}

// Epilogues of the vocabulary head (csrc/vocab.cu) on the CTA-pair GEMM: a thread owns one row of the tile (a TMEM
// lane) and 128 consecutive logits of it, so softmax statistics need no exchange between threads, and the few target
// ids of a row inside those 128 columns are found from its ascending target list.
#pragma once

#include "gemm_epilogue.cuh"

namespace pcb {

template <int EPI>
PCB_DEVICE constexpr bool epi_vocab() {
  return EPI == EPI_VH_STAT || EPI == EPI_VH_GRAD || EPI == EPI_VH_DX || EPI == EPI_VH_DW;
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

// One packed row's part of the target list: the entries whose ids fall in this thread's 128 columns.
struct VocabRow {
  int n;        // the row's place in the batch
  bool live;    // a counted row
  float lse;
  long long at; // entry index of the next target
  int left;     // entries left in these columns
  int next;     // its column relative to the first of the 128; past them when none is left
  int lo;       // vocabulary id of the first of the 128 columns

  template <int EPI>
  PCB_DEVICE void fetch(const VocabHead& h, int m, int col0, int rows) {
    n = 0;
    lse = 0.f;
    at = 0;
    left = 0;
    next = 1 << 30;
    lo = h.v0 + col0;
    live = m < rows;
    if (!live) return;
    n = h.row[m];
    if (EPI == EPI_VH_GRAD) lse = h.lse[n];
    at = (long long)n * h.K;
    if (h.start != nullptr) {
      const unsigned short* s = h.start + (long long)(lo >> 7) * h.ld_start + n;
      const int e = s[0];
      left = s[h.ld_start] - e;
      at += e;
    } else {
      const int t = h.ids[n] - lo;
      left = t >= 0 && t < 128 ? 1 : 0;
    }
    if (left > 0) next = h.ids[at] - lo;
  }
  PCB_DEVICE void advance(const VocabHead& h) {
    ++at;
    next = --left > 0 ? h.ids[at] - lo : 1 << 30;
  }
};

// (max, sum 2^(c l - max)) of this thread's 128 logits, in one pass with a running maximum, and the logits at the
// row's targets.  The maximum stays in units of c l, and the sum is taken against that rounded value, so the
// log-sum-exp made of the pair carries no error of the product c * max.
PCB_DEVICE void vocab_stat(const GemmArgs& a, VocabRow& r, uint32_t taddr, int m, int col0) {
  float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int nvalid = a.N - (col0 + 32 * i);   // warp-uniform
    if (nvalid <= 0) break;
    float v[32];
    tmem_load_f32x32(taddr + 32 * i, v);
    while (r.next < 32 * (i + 1)) {
      a.vh.z[r.at] = pick32(v, r.next - 32 * i);
      r.advance(a.vh);
    }
    __syncwarp();
    if (nvalid < 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = j < nvalid ? v[j] : -INFINITY;
    }
    float cm = v[0];
#pragma unroll
    for (int j = 1; j < 32; ++j) cm = fmaxf(cm, v[j]);
    const float nm = fmaxf(mx, cm * a.vh.c);
    const float ref = nm == -INFINITY ? 0.f : nm;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      s0 += ex2_approx(fmaf(v[j], a.vh.c, -ref));
      s1 += ex2_approx(fmaf(v[j + 1], a.vh.c, -ref));
    }
    sum = sum * ex2_approx(mx - ref) + (s0 + s1);
    mx = nm;
  }
  if (r.live) a.vh.part[(long long)((a.vh.v0 + col0) >> 7) * a.vh.ld_part + m] = make_float2(mx, sum);
}

// 64 columns of softmax - target distribution as packed bf16.  The difference is rounded once to the type of the
// matrix product's operand; its factor 1 / count is applied in fp32 behind that product, because rounding a shared
// factor into every entry would bias all of them alike.
PCB_DEVICE void vocab_grad64(const GemmArgs& a, VocabRow& r, uint32_t taddr, int col0, uint32_t (&pk)[32]) {
  const int base = col0 + a.vh.v0 - r.lo;   // 0 or 64
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[32];
    tmem_load_f32x32(taddr + 32 * h, v);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = r.live ? ex2_approx(fmaf(v[j], a.vh.c, -r.lse)) : 0.f;
    while (r.next < base + 32 * (h + 1)) {
      const int o = r.next - (base + 32 * h);
      const float q = a.vh.q != nullptr ? a.vh.q[r.at] : 1.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] -= j == o ? q : 0.f;
      r.advance(a.vh);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) pk[16 * h + j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
  }
}

PCB_DEVICE float vocab_scale(const GemmArgs& a) {
  float s = a.alpha;
  if (a.vh.scale != nullptr) s *= *a.vh.scale;
  if (a.vh.scale2 != nullptr) s *= *a.vh.scale2;
  return s;
}

// 4 consecutive columns of one row of dx's fp32 slab, or of the weights' gradient
template <int EPI>
PCB_DEVICE void vocab_store4(const GemmArgs& a, int split, int m, int n, const float (&e)[4]) {
  const int nv = min(4, a.N - n);
  if (nv <= 0) return;
  float o[4] = {e[0], e[1], e[2], e[3]};
  if (EPI == EPI_VH_DX || a.vh.out_f32) {
    float* c = reinterpret_cast<float*>(a.C) + split * a.vh.slab + (long long)m * a.ldc + n;
    if (a.vh.add) {
      float p[4];
      ld_f32x4(c, p, nv);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += p[j];
    }
    st_f32x4(c, o, nv);
  } else {
    __nv_bfloat16* c = reinterpret_cast<__nv_bfloat16*>(a.C) + (long long)m * a.ldc + n;
    if (a.vh.add) {
      float p[4];
      ld_bf16x4(c, p, nv);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += p[j];
    }
    st_bf16x4(c, o, nv);
  }
}

}  // namespace pcb

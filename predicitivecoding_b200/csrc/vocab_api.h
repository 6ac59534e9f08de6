// Host-safe API of the operators at the two ends of a decoder (csrc/vocab.cu).
#pragma once
#include <cuda_runtime.h>

namespace pcb {

constexpr int kVocabMaxEntries = 256;   // teacher entries per row

// Loss of the vocabulary head: softmax cross entropy, or distillation from a list of teacher logits per row.
struct VocabHeadArgs {
  const void* x;        // [N, D] bf16, row stride ldx
  long long ldx;
  const void* w;        // [V, D] bf16, row stride ldw (a multiple of 8, 16-byte aligned base)
  long long ldw;
  int N, V, D;
  // cross entropy
  const void* tgt;      // [N] int32 or int64 (nullptr: distillation)
  int tgt64;
  long long ignore;     // rows with this target are not counted; neither are targets outside [0, V)
  // distillation
  const void* ids;      // [N, K] int32 or int64; entries outside [0, V) are absent
  int ids64;
  long long ld_ids;
  const void* logits;   // [N, K] fp32 or bf16; -inf entries are absent
  int logits_bf16;
  long long ld_logits;
  int K;                // entries per row (1 for cross entropy)
  float temperature;
  float* loss;          // [N] row losses
  float* total;         // sum or mean of the row losses (nullptr: not wanted)
};

// Workspaces of the backward.  The vocabulary is taken `piece` columns at a time.
struct VocabPlan {
  int piece, pieces;
  int dw_max;            // most K splits of the dw product
  int slab_rows;         // rows of the fp32 slabs that dx takes
  long long all_rows;    // with those of dw
  bool score;            // a few rows' loss alone
  bool whole;            // a small vocabulary: the forward makes the gradient of the logits, g, along with the loss
};
// `gradient`: for a forward that a backward follows
VocabPlan vocab_plan(int N, int V, int D, int want_piece, bool gradient, int num_sms);

// Where the forward keeps what the backward reads: byte offsets into one buffer.  A kernel that gives up a wait records it
// in the status and leaves its outputs unfinished; the losses and the gradients are then NaN.
struct VocabLayout {
  long long xc;      // [N, ldxc] bf16: the counted rows of x, packed; zero rows up to the next multiple of 64
  long long ldxc;
  long long count;   // int [6]: counted rows, finished blocks of the loss kernel, K splits of dw and dx (where the forward
                     // makes g), status of a wait; float 1 / counted rows, where the losses are summed up
  long long row;     // int [N]: batch place of each packed row
  long long pos;     // int [N]: packed place of each row, -1 where it is not counted
  long long norm;    // float2 [N], by packed row: r and 1 / s, the sum of 2^(logit log2(e) / temperature - r)
  long long z;       // float [N, K]: logits at the target ids, by packed row
  long long ids;     // int [N, K] ascending ids (cross entropy: the targets by packed row)
  long long q;       // float [N, K] weights (distillation)
  long long lq;      // float [N, K] log2 of the weights (distillation)
  long long len;     // int [N] entries present (distillation)
  long long start;   // unsigned short [granules + 1, N] (distillation)
  int granules;      // 128-column halves of the 256-column tiles
  long long bytes;
};
VocabLayout vocab_layout(int N, int V, int D, int K, bool distill);

struct VocabGradArgs {
  const void* x;         // as the forward read it
  long long ldx;
  const void* w;
  long long ldw;
  int N, V, D, K;
  int distill;
  float temperature;
  void* saved;           // buffer of the forward
  float gout;            // gradient of the loss: gout * *gout_dev (nullptr: 1) / (counted rows, for the mean)
  const float* gout_dev;
  int mean;
  void* dx;              // [N, D] bf16 or fp32, row stride lddx (nullptr: not wanted)
  long long lddx;
  int dx_f32;
  void* dw;              // [V, D] bf16 or fp32, row stride lddw (nullptr: not wanted)
  long long lddw;
  int dw_f32;
  int dw_add;
  VocabPlan plan;
  void* g;               // bf16, vocab_g_rows(N) * piece: workspace, or as the forward left it
  int* splits;           // int [2], K splits of dw and dx: workspace (not used where the forward made g).  The backward writes
                         // nothing into `saved` but a status, so two of one state may run at the same time
  float* slab;           // workspace: fp32 [all_rows, ld_slab]
  long long ld_slab;
};
long long vocab_g_rows(int N);

}  // namespace pcb

int pcb_vocab_pad_rows(const void* src, long long ld, void* dst, long long ldd, int rows, int D, cudaStream_t s);
// `part`: [granules, N] float2 workspace; `g`: bf16 [vocab_g_rows(N) * piece] where plan.whole
int pcb_vocab_fwd(const pcb::VocabHeadArgs& a, const pcb::VocabPlan& plan, void* saved, void* part, void* g, int mean,
                  int num_sms, cudaStream_t s);
// kernels that these launch
int pcb_vocab_fwd_launches(const pcb::VocabPlan& plan, int N, bool distill);
int pcb_vocab_bwd_launches(const pcb::VocabPlan& plan);
int pcb_vocab_bwd(const pcb::VocabGradArgs& a, int num_sms, cudaStream_t s);

// x[n] = scale * w[tok[n]]; rows of tokens outside [0, V) are zero
int pcb_vocab_embed_fwd(const void* tok, int tok64, const void* w, int w_bf16, long long ldw, void* x, int x_bf16,
                        int N, int V, int D, float scale, cudaStream_t s);
// bytes of workspace of the embedding gradient
long long pcb_vocab_embed_bwd_bytes(int N, int V, int D);
// kernels that the gradient launches
int pcb_vocab_embed_bwd_launches(int N, int V, int D, int dw_bf16, int add);
// dw[v] (+)= scale * sum of dx[n] over tok[n] == v in ascending n
int pcb_vocab_embed_bwd(const void* tok, int tok64, const void* dx, int dx_bf16, long long lddx, void* dw, int dw_bf16,
                        int N, int V, int D, float scale, int add, void* ws, int num_sms, cudaStream_t s);

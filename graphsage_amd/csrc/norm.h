// Layer norm and dropout, host side: what norm.hip (the C entries) hands to the kernels of one type of table, and which
// kernel a width takes.
#pragma once
#include "gsage_common.h"

struct NormDrop {          // p = 0: no mask
  float p, inv_keep;
  uint64_t seed;
  const int64_t *seed_dev;
};

struct NormFwd {
  const void *x, *res, *w, *b;
  int64_t M, F;
  int wdtype;
  float eps;
  NormDrop d;
  void *y, *sum;
  float *mean, *rstd;
};

struct NormBwd {
  const void *g, *gsum, *x, *res, *w;
  const float *mean, *rstd;
  int64_t M, F;
  int wdtype;
  NormDrop d;
  void *gx, *gres, *gw, *gb;
  float *ws;
  bool joined() const { return res || d.p > 0.f || gsum || gres; }
};

// Which kernel a row takes: K vectors of 16 bytes (V elements each) in each of R lanes of a wave, or of `row` threads of a
// workgroup (B, W); NORM_ONE: rows shorter than a vector, an element a lane.  A row's sums and addresses cost its threads
// the same whatever they hold, so a row takes the fewest lanes that need no more than three vectors each, which also
// leaves few of them idle (fp16 240 000 x 264, joined: 16 lanes x 3 78 us forward and 135 backward, 32 x 2 92 and 167).
// Past a vector each of four lanes at least eight: a wave's accesses then take whole lines (4 M x 64 bf16 forward 0.167
// ms, at four lanes x 2 0.220).  Two or four waves a row rather than three or five: eight fit a compute unit (40 000 x 1544
// fp16 joined forward 79 us, 80); where that would be three or four waves of three vectors, nine to twelve of one (NORM_W1:
// of tables rotated past the caches 8191 x 5120 bf16 joined with its sum forward 65 us, backward 115; in fours 66 and 122;
// 9000 x 2600 fp32 34 and 62, joined 51 and 90; 36 and 62, 54 and 94).  Past 8192 columns (NORM_W) 16 elements a thread in up to sixteen waves, as many as a
// compute unit has room for: 8192 x 16000 bf16 forward 97 us, backward 176, joined 143 and 304; as eight waves with 32
// elements a thread 103, 190, 174 and 367 (fp32 179, 288, 291, 661; 194, 315, 363, 956).  Large fp32 tables of whole cache
// lines without residual or dropout stream best where neighbouring lanes hold neighbouring vectors (`stream`: 10 M x 64
// forward 0.81 ms at 16 lanes x 1, 0.85 at 8 x 2, backward 1.25 and 1.34; 4 M x 128 0.65 and 0.68, 1.01 and 1.08: 6.2 to
// 6.4 TB/s; widths between, whose lanes do not all hold one vector, 6.1 at 3 M x 96, 5.9 at 2 M x 160, 5.6 to 5.9 at 192;
// bf16 2 M x 256 0.325 and 0.319, 0.548 and 0.541).
enum NormKind { NORM_ONE, NORM_R4, NORM_R8, NORM_R8x2, NORM_R8x3, NORM_R16, NORM_R16x2, NORM_R16x3, NORM_R32, NORM_R32x2,
                NORM_R32x3, NORM_R64, NORM_R64x2, NORM_R64x3, NORM_B2, NORM_B3, NORM_B4, NORM_W1, NORM_W, NORM_LONG };
struct NormForm { NormKind kind; int row; };      // threads of a row
static inline NormForm norm_form(int64_t F, int V, bool stream) {
  stream = stream && V == 4;
  if (F < V) return {NORM_ONE, 8};
  const int64_t nv = (F + V - 1) / V;
  const auto waves = [&](int k) { return (int)((nv + 64 * k - 1) / (64 * k)) * 64; };
  if (nv <= 4) return {NORM_R4, 4};
  if (nv <= 8) return {NORM_R8, 8};
  if (stream && nv == 16) return {NORM_R16, 16};
  if (stream && nv == 32) return {NORM_R32, 32};
  if (stream && nv == 64) return {NORM_R64, 64};
  if (nv <= 16) return {NORM_R8x2, 8};
  if (nv <= 24) return {NORM_R8x3, 8};
  if (nv <= 32) return {NORM_R16x2, 16};
  if (nv <= 48) return {NORM_R16x3, 16};
  if (nv <= 64) return {NORM_R32x2, 32};
  if (nv <= 96) return {NORM_R32x3, 32};
  if (nv <= 128) return {NORM_R64x2, 64};
  if (nv <= 192) return {NORM_R64x3, 64};
  if (nv <= 256) return {NORM_B2, 128};
  if (nv <= 384) return {NORM_B3, 128};
  if (nv <= 512) return {NORM_B2, 256};
  if (nv <= 768) return {NORM_W1, waves(1)};
  if (nv <= 1024) return {NORM_B2, waves(2)};
  if (nv <= 2048 && V == 4) return {NORM_B4, waves(4)};
  if (nv <= 16384 / V) return {NORM_W, waves(16 / V)};
  return {NORM_LONG, 1024};
}

// Workgroups for M rows, `rows` at once each, at most `cap`, with the same number of turns each (but for the last)
static inline int norm_blocks(int64_t M, int rows, int cap) {
  const int64_t groups = (M + rows - 1) / rows, turns = (groups + cap - 1) / cap;
  return groups ? (int)((groups + turns - 1) / turns) : 0;
}
// Tables too large for any cache (256 MB behind the L2s) are read and written past them, if their rows share no cache
// lines: 1 M x 128 fp32 joined forward 0.263 -> 0.242 ms, backward 0.454 -> 0.414; 10 M x 64 backward 1.43 -> 1.25.
// Smaller ones lose that way, for the caches serve them (60 000 x 64 joined forward 9.1 -> 9.8 us), and so do rows that end
// inside a line (1 M x 196 fp16 forward 0.141 -> 0.156 ms, joined backward 0.388 -> 0.476).
static inline bool norm_large(int64_t n, size_t size) { return n * (int64_t)size >= ((int64_t)256 << 20); }
static inline bool norm_streams(int64_t M, int64_t F, size_t size) { return norm_large(M * F, size) && F * (int64_t)size % 128 == 0; }

// Slabs of column sums that a backward call writes at most: one for every two turns of a workgroup where streamed rows are
// short (and 256 more, to which those are added up first), otherwise as few as keep the GPU busy
constexpr int NORM_FOLD_TURNS = 2, NORM_FOLD_THREADS = 512;
static inline int norm_fold_rows(int64_t F) { return NORM_FOLD_TURNS * (NORM_FOLD_THREADS / norm_form(F, 4, true).row); }
static inline bool norm_folds(int64_t M, int64_t F, size_t size, bool join) {
  return !join && size == 4 && norm_streams(M, F, size) && F <= 128 && M <= (int64_t)1 << 27;      // (its launch's threads fit 32 bits)
}
static inline int norm_max_slabs(int64_t M, int64_t F) {
  const int64_t cap = F <= 512 ? 1024 : F <= 8192 ? 512 : 256;
  return (int)(M < cap ? M : cap);
}
static inline int64_t norm_ws_floats(int64_t M, int64_t F, size_t size, bool join) {
  const int64_t few = norm_max_slabs(M, F), rows = norm_folds(M, F, size, join) ? norm_fold_rows(F) : 0;
  const int64_t many = rows ? (M + rows - 1) / rows + 256 : 0;
  return 2 * F * (many > few ? many : few > 0 ? few : 1);
}

int norm_dropout_f32(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st);
int norm_dropout_bf16(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st);
int norm_dropout_f16(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st);
int norm_fwd_f32(const NormFwd &n, hipStream_t st);
int norm_fwd_bf16(const NormFwd &n, hipStream_t st);
int norm_fwd_f16(const NormFwd &n, hipStream_t st);
int norm_bwd_f32(const NormBwd &n, hipStream_t st);
int norm_bwd_bf16(const NormBwd &n, hipStream_t st);
int norm_bwd_f16(const NormBwd &n, hipStream_t st);

// Kernels and launches of layer norm and dropout for one type of table: included by norm_f32.hip, norm_bf16.hip and
// norm_f16.hip, which are compiled side by side.
//
//   z = residual + dropout(x);  y = (z - mean) rstd w + b
//   a = g w;  h = (z - mean) rstd;  dz = rstd (a - mean(a) - h mean(a h)) + grad_sum
//   grad_residual = dz;  grad_x = dropout'(dz);  grad_w = sum_rows g h;  grad_b = sum_rows g
//
// Neither the mask nor z is stored: both are formed again from (seed, index) and from x and residual.  A row is read
// once: it lies in the registers of the threads that share it while its sums are taken.
#pragma once
#include <atomic>

#include "gsage_common.h"
#include "gsage_dropout.h"
#include "norm.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// by value: __builtin_bit_cast straight from an element of a vector reads element 0, whatever the index
__device__ __forceinline__ float as_f(unsigned w) { return __builtin_bit_cast(float, w); }
__device__ __forceinline__ unsigned as_u(float f) { return __builtin_bit_cast(unsigned, f); }

// ------------------------------------------------------------------ 16 bytes of a table as fp32
// Rows start wherever they start: 16-byte accesses at element alignment, which global memory takes on this hardware
// (the compiler emits one global_{load,store}_dwordx4 for them).
template <typename T> struct Tab;
template <> struct Tab<float> {
  static constexpr int V = 4;
  typedef u32x4 __attribute__((aligned(4), may_alias)) mem;
  static __device__ __forceinline__ void open(u32x4 r, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = as_f(r[i]);
  }
  static __device__ __forceinline__ u32x4 close(const float (&f)[4]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = as_u(f[i]);
    return r;
  }
};
template <> struct Tab<__bf16> {
  static constexpr int V = 8;
  typedef u32x4 __attribute__((aligned(2), may_alias)) mem;
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void open(u32x4 r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = as_f(r[i] << 16);
      f[2 * i + 1] = as_f(r[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ u32x4 close(const float (&f)[8]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, pair{(__bf16)f[2 * i], (__bf16)f[2 * i + 1]});
    return r;
  }
};
template <> struct Tab<_Float16> {
  static constexpr int V = 8;
  typedef u32x4 __attribute__((aligned(2), may_alias)) mem;
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void open(u32x4 r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned word = r[i];
      const pair h = __builtin_bit_cast(pair, word);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ u32x4 close(const float (&f)[8]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, pair{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
    return r;
  }
};

// V = 16 / sizeof(T) elements in four words, or (V = 1: rows shorter than that) one element.
// NT: accesses that are not to be kept in the caches
template <typename T, int V> struct Raw {
  u32x4 w;
  __device__ __forceinline__ void keep(bool on) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = on ? w[i] : 0u;
  }
  template <bool NT = false> __device__ __forceinline__ void load(const T *p) {
    const auto *q = (const typename Tab<T>::mem *)p;
    if constexpr (NT) w = __builtin_nontemporal_load(q);
    else w = *q;
  }
  __device__ __forceinline__ void open(float (&f)[V]) const { Tab<T>::open(w, f); }
  template <bool NT = false> static __device__ __forceinline__ void store(T *p, const float (&f)[V]) {
    auto *q = (typename Tab<T>::mem *)p;
    if constexpr (NT) __builtin_nontemporal_store(Tab<T>::close(f), q);
    else *q = Tab<T>::close(f);
  }
};
template <typename T> struct Raw<T, 1> {
  T w;
  __device__ __forceinline__ void keep(bool on) { w = on ? w : (T)0.f; }
  template <bool NT = false> __device__ __forceinline__ void load(const T *p) { w = *p; }
  __device__ __forceinline__ void open(float (&f)[1]) const { f[0] = (float)w; }
  template <bool NT = false> static __device__ __forceinline__ void store(T *p, const float (&f)[1]) { *p = (T)f[0]; }
};

// ------------------------------------------------------------------ dropout
__device__ __forceinline__ uint64_t drop_key(const NormDrop &d) { return d.seed_dev ? (uint64_t)*d.seed_dev : d.seed; }

// kept[i] = keep(idx + i).  The V indices share their upper word but for one vector in 2^32 / V.
template <int V>
__device__ __forceinline__ void draw_vec(bool (&kept)[V], uint64_t idx, uint64_t key, uint32_t thr, float p) {
  const uint32_t lo = (uint32_t)idx, hi = (uint32_t)(idx >> 32);
  if (V > 1 && lo > 0xFFFFFFFFu - (V - 1)) {
#pragma unroll
    for (int i = 0; i < V; ++i) kept[i] = dropout_keep(key, idx + i, p);
    return;
  }
  const uint32_t k = dropout_word(key, hi), m0 = lo * DROPOUT_STEP;
#pragma unroll
  for (int i = 0; i < V; ++i) kept[i] = dropout_draw(k, m0 + (uint32_t)i * DROPOUT_STEP) >= thr;
}
template <int V> __device__ __forceinline__ void drop_vec(float (&f)[V], const bool (&kept)[V], float inv_keep) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = kept[i] ? f[i] * inv_keep : 0.f;
}

// A vector a thread and as many workgroups as that takes: they start in order, so at any time the GPU reads and writes one
// short stretch of each table, and the memory stays on its open pages.  The same loop over a grid the GPU holds at once,
// whose workgroups drift apart, reaches three quarters of it (10 M x 64 fp32: 0.80 ms, 6.4 TB/s; 1.11 ms with four vectors
// a turn, 1.00 with one).
template <typename T, bool NT>
__global__ void __launch_bounds__(256) dropout_k(const T *x, int64_t n, int64_t begin, NormDrop d, T *out) {
  constexpr int V = Tab<T>::V;
  const uint64_t key = drop_key(d);
  const uint32_t thr = dropout_threshold(d.p);
  const int64_t i = begin + (int64_t)blockIdx.x * 256 + threadIdx.x, nv = n / V;
  if (i < nv) {
    Raw<T, V> r;
    r.template load<NT>(x + i * V);
    float f[V];
    bool kept[V];
    draw_vec<V>(kept, (uint64_t)i * V, key, thr, d.p);
    r.open(f);
    drop_vec<V>(f, kept, d.inv_keep);
    Raw<T, V>::template store<NT>(out + i * V, f);
  } else if (i - nv < n - nv * V) {      // the last n mod V elements
    const int64_t e = nv * V + (i - nv);
    out[e] = (T)(dropout_keep(key, (uint64_t)e, d.p) ? (float)x[e] * d.inv_keep : 0.f);
  }
}

// ------------------------------------------------------------------ sums over the threads of a row
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// over aligned groups of N lanes (4 .. 64), in every lane; all lanes of the wave take part
template <int N> __device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<0xB1>(v);                 // quad_perm: lane ^ 1
  v += dpp<0x4E>(v);                 // quad_perm: lane ^ 2
  if (N >= 8) v += dpp<0x141>(v);    // row_half_mirror: the other four of eight
  if (N >= 16) v += dpp<0x140>(v);   // row_mirror: the other eight of a row
  if (N >= 32) {                     // rows 0 <-> 1, 2 <-> 3
    const auto r = __builtin_amdgcn_permlane16_swap(as_u(v), as_u(v), false, false);
    v = as_f(r[0]) + as_f(r[1]);
  }
  if (N >= 64) {                     // the two halves of the wave
    const auto r = __builtin_amdgcn_permlane32_swap(as_u(v), as_u(v), false, false);
    v = as_f(r[0]) + as_f(r[1]);
  }
  return v;
}

// V weights from a column on, fp32 or of the tables' type: loaded in one place, made fp32 in another, so that the loads
// of a row's operands go out between (NULL: `other` V times)
template <typename T, int V> struct Weights {
  u32x4 r[V > 4 ? 2 : 1];
  __device__ __forceinline__ void load(const void *w, int wdtype, int c) {
    if (!w) return;
    if constexpr (V == 1) {
      if (wdtype == GSAGE_F32) r[0][0] = as_u(((const float *)w)[c]);
      else r[0][0] = as_u((float)((const T *)w)[c]);
    } else if (wdtype == GSAGE_F32) {
      const float *p = (const float *)w + c;
      r[0] = *(const Tab<float>::mem *)p;
      if constexpr (V > 4) r[1] = *(const Tab<float>::mem *)(p + 4);
    } else r[0] = *(const typename Tab<T>::mem *)((const T *)w + c);
  }
  __device__ __forceinline__ void open(const void *w, int wdtype, float other, float (&f)[V]) const {
    if (!w) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = other;
    } else if constexpr (V == 1) f[0] = as_f(r[0][0]);
    else if (wdtype == GSAGE_F32) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = as_f(r[i / 4][i % 4]);
    } else Tab<T>::open(r[0], f);
  }
};
__device__ __forceinline__ void store_w(void *w, int wdtype, int64_t c, float v) {
  if (wdtype == GSAGE_F32) ((float *)w)[c] = v;
  else if (wdtype == GSAGE_BF16) ((__bf16 *)w)[c] = (__bf16)v;
  else ((_Float16 *)w)[c] = (_Float16)v;
}

template <typename T> struct Ln {
  const T *x, *res;
  const void *w, *b;
  int64_t M;
  int F, wdtype, row;      // row: threads of a row, where that is not the kernel's own constant
  NormDrop d;
};

// A row takes TPR lanes of a wave, or a.row threads: up to 8 (TPR = 0) or 16 (TPR = -1) whole waves.  A workgroup takes as
// many rows at once as fit.  Thread t of the row holds K vectors of V columns, a row's threads apart.  A vector that would
// go past the row's end is moved back to end with it; its first `lo` elements (all of them, where the thread has nothing
// left to do) then belong to vectors before it: both threads form and store the same values, the sums count them once.
constexpr int MAXW = 8;
constexpr int ln_waves(int TPR) { return TPR < 0 ? 16 : MAXW; }
template <int V, int TPR, int K> struct Cols {
  int t, threads, col[K], lo[K];
  bool on[K], full;
  __device__ __forceinline__ Cols(int F, int row) {
    threads = TPR > 0 ? TPR : row;
    t = threadIdx.x % threads;
    full = F == threads * K * V;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int v = (t + k * threads) * V;
      on[k] = v < F;
      col[k] = v < F - V ? v : F - V;
      lo[k] = v - col[k];
    }
  }
  __device__ __forceinline__ bool live(int k, int i) const { return i >= lo[k]; }
  // live elements of wave i of a row's
  __device__ __forceinline__ int wave_count(int i, int F) const {
    int n = 0;
    if (i < threads >> 6)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int left = F - (i * 64 + k * threads) * V;
        n += left < 0 ? 0 : left < 64 * V ? left : 64 * V;
      }
    return n;
  }
};

// The operands of z of one row.  Loaded without a branch a vector: where a thread has no column it loads its neighbour's
// (and row `row` must be one of the table's), and drops it at use.
template <typename T, int V, int TPR, int K, bool JOIN, bool NT> struct Operands {
  Raw<T, V> x[K], r[JOIN ? K : 1];
  __device__ __forceinline__ void load(const Ln<T> &a, const Cols<V, TPR, K> &c, int64_t row) {
#pragma unroll
    for (int k = 0; k < K; ++k) x[k].template load<NT>(a.x + row * a.F + c.col[k]);
    if (JOIN && a.res)
#pragma unroll
      for (int k = 0; k < K; ++k) r[k].template load<NT>(a.res + row * a.F + c.col[k]);
  }
  // (zero where the thread has no column)
  __device__ __forceinline__ void z(const Ln<T> &a, const Cols<V, TPR, K> &c, int64_t row, uint64_t key, uint32_t thr,
                                    float (&z)[K][V], bool (&kept)[K][V]) {
    if (!c.full)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        x[k].keep(c.on[k]);
        if (JOIN) r[k].keep(c.on[k]);
      }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k].open(z[k]);
      if (JOIN && a.d.p > 0.f) {
        draw_vec<V>(kept[k], (uint64_t)(row * a.F + c.col[k]), key, thr, a.d.p);
        drop_vec<V>(z[k], kept[k], a.d.inv_keep);
      }
    }
    if (JOIN && a.res)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float q[V];
        r[k].open(q);
#pragma unroll
        for (int i = 0; i < V; ++i) z[k][i] += q[i];
      }
  }
};

// Rows of a workgroup: those it takes at once from begin + blockIdx apart on, then `step` further for each of `turns`
struct Walk { int64_t begin, apart, step; int turns; };

// ------------------------------------------------------------------ forward
// LOOP: several turns, the row after in flight; otherwise one turn and as many workgroups as that takes, which start in
// order (see dropout_k: 1 M x 128 fp32 0.163 ms, 0.178 as a loop over the grid the GPU holds, joined 0.242 and 0.272: the
// memory's rate for such a stream, 6.3 TB/s).
template <typename T, int V, int TPR, int K, bool JOIN, bool NT, bool LOOP>
__global__ void __launch_bounds__(TPR > 0 || K == 3 ? 256 : 64 * ln_waves(TPR)) ln_fwd_k(Ln<T> a, Walk g, float eps, T *y, T *sum, float *mean, float *rstd) {
  constexpr int WAVES = ln_waves(TPR);
  __shared__ float part[TPR > 0 ? 1 : 2][TPR > 0 ? 1 : WAVES][2];
  const Cols<V, TPR, K> c(a.F, a.row);
  const int first = TPR > 0 ? threadIdx.x / (TPR > 0 ? TPR : 1) : 0;      // this thread's among the rows at once
  int64_t row = g.begin + (int64_t)blockIdx.x * g.apart + first;
  Operands<T, V, TPR, K, JOIN, NT> next;
  const auto fetch = [&](int64_t r) { next.load(a, c, r < a.M ? r : a.M - 1); };
  fetch(row);
  Weights<T, V> wr[K], br[K];
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) wr[k].load(a.w, a.wdtype, c.col[k]);
#pragma unroll
  for (int k = 0; k < K; ++k) br[k].load(a.b, a.wdtype, c.col[k]);
  const auto weights = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      wr[k].open(a.w, a.wdtype, 1.f, w[k]);
      br[k].open(a.b, a.wdtype, 0.f, b[k]);
    }
  };
  const uint64_t key = JOIN ? drop_key(a.d) : 0;
  const uint32_t thr = JOIN ? dropout_threshold(a.d.p) : 0;
  const float inv_f = 1.0f / (float)a.F;
  // (rows of several waves) this wave's elements, and those of the wave whose sums this lane puts together
  const int mine = TPR > 0 ? 0 : c.wave_count(c.t >> 6, a.F), other = TPR > 0 ? 0 : c.wave_count(threadIdx.x % WAVES, a.F);
  const float inv_mine = mine ? 1.0f / (float)mine : 0.f, inv_other = other ? 1.0f / (float)other : 0.f;
  if (LOOP) weights();
  const int turns = LOOP ? g.turns : 1;
  for (int turn = 0; turn < turns; ++turn, row += g.step) {
    float z[K][V];
    bool kept[K][V];
    next.z(a, c, row, key, thr, z, kept);
    if (LOOP && turn + 1 < turns) fetch(row + g.step);
    float s = 0.f, q = 0.f, m, var;
    const auto squares = [&](float about) {
      if (c.full) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) { const float e = z[k][i] - about; q = fmaf(e, e, q); }
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) { const float e = c.live(k, i) ? z[k][i] - about : 0.f; q = fmaf(e, e, q); }
      }
    };
    // (z is zero where a thread has no column; a moved vector's first elements are not counted again)
    if (a.F % V == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s += z[k][i];
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s += c.live(k, i) ? z[k][i] : 0.f;
    }
    if constexpr (TPR > 0) {
      m = lanes_sum<TPR>(s) * inv_f;
      squares(m);
      var = lanes_sum<TPR>(q) * inv_f;
    } else {
      // each wave about its own mean, the waves' (sum, sum of squares about it) then put together: one barrier a row
      // (the slots alternate), and no difference of large sums
      const float sw = lanes_sum<64>(s);
      squares(sw * inv_mine);
      q = lanes_sum<64>(q);
      float(*slot)[2] = part[turn & 1];
      if (gs_lane() == 0) { slot[c.t >> 6][0] = sw; slot[c.t >> 6][1] = q; }
      __syncthreads();
      // (waves that are not there have no elements; their slots hold whatever LDS held)
      const float so = other ? slot[threadIdx.x % WAVES][0] : 0.f, qo = other ? slot[threadIdx.x % WAVES][1] : 0.f;
      m = lanes_sum<WAVES>(so) * inv_f;
      const float e = other ? so * inv_other - m : 0.f;      // (m^2 times no elements: a mean past 2^64 would make it NaN)
      var = lanes_sum<WAVES>(fmaf(e * e, (float)other, qo)) * inv_f;
    }
    const float rs = rsqrtf(var + eps);
    if (!LOOP) weights();
    if (row < a.M) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!c.on[k]) continue;
        if (JOIN && sum) Raw<T, V>::template store<NT>(sum + row * a.F + c.col[k], z[k]);
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = fmaf((z[k][i] - m) * rs, w[k][i], b[k][i]);
        Raw<T, V>::template store<NT>(y + row * a.F + c.col[k], o);
      }
      if (mean && c.t == 0) { mean[row] = m; rstd[row] = rs; }
    }
  }
}

template <typename T> struct Grads {
  const T *g, *gsum;
  const float *mean, *rstd;
  T *gx, *gres;
  float *ws;               // slabs; NULL: no column sums wanted
  void *gw, *gb;           // written by the kernel itself where one workgroup is the whole grid
};

// ------------------------------------------------------------------ backward
// A thread's column sums: in registers for `flush` rows, then added in double to its own words of LDS, which so hold
// thousands of rows without losing bits (fp32 words: 33 M rows x 64 of one gradient off by 24 roundings, doubles by none).
// Doubles cost a flush 0.8 us where a thread has 16 elements, so they come from `doubles` rows a thread on (fewer stay in
// registers to the end), rows that share waves with others flush a wave at a time (`late`; 1 M x 196 fp16 208 us, all at
// once 215, in fp32 words 207) and rows of several waves half as often (40 000 x 1544 fp16 72 us, every 16 rows 75, in
// fp32 words 72).  Joined rows that share a wave have neither: tests of the turn's number beside the loop's own cost more there
// (4 M x 3 fp32 82 us, 116 to 120 with them; the doubles themselves 1 to 2 %).
// Where there are no registers for the first level (ln_bwd_ahead) every row goes to LDS, in fp32: two words for each of 24
// elements, or of 16 in sixteen waves, do not fit there.  A thread's sum of n rows of either sign is then off by some
// sqrt(n) / 2.4 roundings: 6 at the 200 rows of 3 M x 192 bf16.
constexpr int ln_bwd_flush(int TPR) { return TPR > 0 ? 16 : 32; }
constexpr int ln_bwd_doubles(int TPR, bool JOIN) { return TPR > 0 && JOIN ? 16 : 2 * ln_bwd_flush(TPR); }

// Workgroups of eight waves (fewer slabs than four would leave), or of the row's up to sixteen.  The row after is loaded a
// row ahead where there are registers for it: not at 24 elements a thread (fp16 257 columns 39 us, joined 71; with four
// waves that have them 42 and 83), nor at 16 of fp32 joined, nor at 16 in sixteen waves, which have 128 each and, joined,
// keep some in scratch (fp32 156 bytes a lane, forward 68; 16-bit 16); those read grad_sum, too, only when the weights are
// used up (fp32 8192 x 16000 joined 661 us; with the other operands 758).  The doubles of nine to twelve waves of 16-bit rows
// leave room for one workgroup a compute unit, which is the better half: 8191 x 5120 bf16 59 us, as two 66.
constexpr bool ln_bwd_ahead(int V, int TPR, int K, bool JOIN) {
  return (TPR >= 0 || K == 1) && K * V < 24 && !(JOIN && K * V == 16 && V == 4);
}
constexpr int ln_bwd_threads(int TPR) { return 64 * ln_waves(TPR); }

// Nothing of this wave is under way (vmcnt = 0).  The loops over the grid that the GPU holds wait so before their stores and
// after them on streamed tables: reads and writes then come in turns, which the memory takes better than both at once
// (1 M x 256 fp32 backward 0.52 ms against 0.54, joined 0.90 against 0.98; 1 M x 128 joined 0.414 against 0.434).
__device__ __forceinline__ void settle() { __builtin_amdgcn_s_waitcnt(0x0F70); }

template <typename T, int V, int TPR, int K, bool JOIN, bool NT>
__global__ void __launch_bounds__(ln_bwd_threads(TPR)) ln_bwd_k(Ln<T> a, Walk g, Grads<T> d) {
  constexpr bool AHEAD = ln_bwd_ahead(V, TPR, K, JOIN);
  constexpr int FLUSH = ln_bwd_flush(TPR), DOUBLES = ln_bwd_doubles(TPR, JOIN);
  constexpr bool LATE = TPR < 0 && !AHEAD;      // grad_sum is read when the weights are used up
  constexpr int A = AHEAD ? K : 1;
  // [2 K V][threads] column sums: grad_w, then grad_b; a thread's words are its own.  Doubles where registers come first
  extern __shared__ __attribute__((aligned(8))) char lds[];
  constexpr int WAVES = ln_waves(TPR);
  __shared__ float part[TPR > 0 ? 1 : 2][TPR > 0 ? 1 : WAVES][2];
  constexpr int threads = ln_bwd_threads(TPR);      // (a workgroup a row may have fewer)
  const Cols<V, TPR, K> c(a.F, a.row);
  const int rows = TPR > 0 ? threads / (TPR > 0 ? TPR : 1) : blockDim.x / c.threads, first = TPR < 0 ? 0 : threadIdx.x / c.threads;
  int64_t base = g.begin + (int64_t)blockIdx.x * g.apart, row = base + first;
  Operands<T, V, TPR, K, JOIN, NT> next;
  Raw<T, V> gnext[K], snext[JOIN ? K : 1];
  float mnext, rnext;
  const auto fetch = [&](int64_t at) {
    const int64_t r = at < a.M ? at : a.M - 1;
    next.load(a, c, r);
#pragma unroll
    for (int k = 0; k < K; ++k) gnext[k].template load<NT>(d.g + r * a.F + c.col[k]);
    if (JOIN && d.gsum && !LATE)
#pragma unroll
      for (int k = 0; k < K; ++k) snext[k].template load<NT>(d.gsum + r * a.F + c.col[k]);
    mnext = d.mean[r];
    rnext = d.rstd[r];
  };
  fetch(row);
  Weights<T, V> wr[K];
  float w[K][V], dw[A][V], db[A][V];
  float *const mine = (float *)lds + threadIdx.x;      // (without registers for them)
#pragma unroll
  for (int k = 0; k < K; ++k) wr[k].load(a.w, a.wdtype, c.col[k]);
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (AHEAD) dw[k % A][i] = db[k % A][i] = 0.f;
      else mine[(k * V + i) * threads] = mine[((K + k) * V + i) * threads] = 0.f;
    }
    wr[k].open(a.w, a.wdtype, 1.f, w[k]);
  }
  const uint64_t key = JOIN ? drop_key(a.d) : 0;
  const uint32_t thr = JOIN ? dropout_threshold(a.d.p) : 0;
  const float inv_f = 1.0f / (float)a.F;
  const bool doubles = g.turns >= DOUBLES;      // (every wave has flushed by then)
  const int late = TPR > 0 && !JOIN ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const auto flush = [&](auto *sums, bool first) {      // (the first one writes, for there is nothing to add to)
    if constexpr (AHEAD) {
      sums += threadIdx.x;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          auto &uw = sums[(k * V + i) * threads], &ub = sums[((K + k) * V + i) * threads];
          uw = first ? dw[k][i] : uw + dw[k][i];
          ub = first ? db[k][i] : ub + db[k][i];
          dw[k][i] = db[k][i] = 0.f;
        }
    }
  };
  for (int turn = 0; turn < g.turns; ++turn, base += g.step, row += g.step) {
    float h[K][V], gv[K][V];
    Raw<T, V> sv[JOIN ? K : 1];
    bool kept[K][V];
    if (!AHEAD && turn > 0) fetch(row);
    next.z(a, c, row, key, thr, h, kept);
    if (!c.full || base + rows > a.M)                             // no column, or no row: nothing for the sums
#pragma unroll
      for (int k = 0; k < K; ++k) gnext[k].keep(c.on[k] && row < a.M);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      gnext[k].open(gv[k]);
      if (JOIN && !LATE) sv[k] = snext[k];
    }
    const float m = mnext, rs = rnext;
    if (AHEAD && turn + 1 < g.turns) fetch(row + g.step);
    if (AHEAD && (DOUBLES == FLUSH || doubles)) {
      const int since = turn + 1 - late;
      if (since > 0 && since % FLUSH == 0) flush((double *)lds, since == FLUSH);
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float mk = c.on[k] ? m : 0.f;      // h = 0 without a column: m rs may pass the range, and g = 0 times that is NaN
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[k][i] = (h[k][i] - mk) * rs;
        if constexpr (AHEAD) {
          dw[k][i] = fmaf(gv[k][i], h[k][i], dw[k][i]);
          db[k][i] += gv[k][i];
        } else {
          mine[(k * V + i) * threads] += gv[k][i] * h[k][i];
          mine[((K + k) * V + i) * threads] += gv[k][i];
        }
        gv[k][i] *= w[k][i];
      }
    }
    if (JOIN && LATE && d.gsum)
#pragma unroll
      for (int k = 0; k < K; ++k) sv[k].template load<NT>(d.gsum + (row < a.M ? row : a.M - 1) * a.F + c.col[k]);
    if (a.F % V == 0) {                     // (g is zero where a thread has no column)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) { s1 += gv[k][i]; s2 = fmaf(gv[k][i], h[k][i], s2); }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) { const float e = c.live(k, i) ? gv[k][i] : 0.f; s1 += e; s2 = fmaf(e, h[k][i], s2); }
    }
    if constexpr (TPR > 0) {
      s1 = lanes_sum<TPR>(s1);
      s2 = lanes_sum<TPR>(s2);
    } else {
      s1 = lanes_sum<64>(s1);
      s2 = lanes_sum<64>(s2);
      float(*slot)[2] = part[turn & 1] + first * (c.threads >> 6);
      if (gs_lane() == 0) { slot[c.t >> 6][0] = s1; slot[c.t >> 6][1] = s2; }
      __syncthreads();
      const bool there = threadIdx.x % WAVES < c.threads >> 6;
      s1 = lanes_sum<WAVES>(there ? slot[threadIdx.x % WAVES][0] : 0.f);
      s2 = lanes_sum<WAVES>(there ? slot[threadIdx.x % WAVES][1] : 0.f);
    }
    s1 *= inv_f;
    s2 *= inv_f;
    if constexpr (NT) settle();
    if (row < a.M) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!c.on[k]) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = rs * fmaf(-h[k][i], s2, gv[k][i] - s1);
        if (JOIN && d.gsum) {
          float q[V];
          sv[k].open(q);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] += q[i];
        }
        if (JOIN && d.gres) Raw<T, V>::template store<NT>(d.gres + row * a.F + c.col[k], o);
        if (d.gx) {
          if (JOIN && a.d.p > 0.f) drop_vec<V>(o, kept[k], a.d.inv_keep);
          Raw<T, V>::template store<NT>(d.gx + row * a.F + c.col[k], o);
        }
      }
    }
    if constexpr (NT) settle();
  }
  if (!d.ws) return;
  // this workgroup's column sums -> its slab, or (one workgroup) the result: element e of thread t's columns, over the
  // threads of the workgroup's rows that hold the same columns (up to 128: in double)
  const auto finish = [&](const auto *sums) {
    __syncthreads();
    float *slab = d.ws + (int64_t)blockIdx.x * 2 * a.F;
    for (int j = threadIdx.x; j < K * V * c.threads; j += blockDim.x) {
      const int t = j % c.threads, e = j / c.threads, v = (t + e / V * c.threads) * V, at = v < a.F - V ? v : a.F - V;
      if (v >= a.F || e % V < v - at) continue;
      double u = 0., q = 0.;
      for (int r = 0; r < rows; ++r) {
        u += sums[e * threads + r * c.threads + t];
        q += sums[(K * V + e) * threads + r * c.threads + t];
      }
      const int col = at + e % V;
      if (gridDim.x > 1) { slab[col] = (float)u; slab[a.F + col] = (float)q; continue; }
      if (d.gw) store_w(d.gw, a.wdtype, col, (float)u);
      if (d.gb) store_w(d.gb, a.wdtype, col, (float)q);
    }
  };
  if (AHEAD && doubles) {
    flush((double *)lds, false);
    finish((const double *)lds);
  } else {      // (the registers' sums as they are)
    flush((float *)lds, true);
    finish((const float *)lds);
  }
}

// Thousands of slabs -> gridDim.y of them: 64 columns of the 2 F a workgroup, `per` slabs
__global__ void __launch_bounds__(1024) ln_fold_k(const float *ws, int slabs, int per, int F, float *out) {
  __shared__ double part[16][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + gs_lane();
  const int s0 = blockIdx.y * per, s1 = s0 + per < slabs ? s0 + per : slabs, w = threadIdx.x >> 6;
  double v = 0.;
  if (c < 2 * (int64_t)F)
#pragma unroll 8
    for (int s = s0 + w; s < s1; s += 16) v += (double)ws[(int64_t)s * 2 * F + c];
  part[w][gs_lane()] = v;
  __syncthreads();
  if (w == 0 && c < 2 * (int64_t)F) {
#pragma unroll
    for (int i = 1; i < 16; ++i) v += part[i][gs_lane()];
    out[(int64_t)blockIdx.y * 2 * F + c] = (float)v;
  }
}

// The slabs' sum, in slab order per thread and in double: 16 columns of the 2 F a workgroup, 64 slabs at a time
__global__ void __launch_bounds__(1024) ln_slabs_k(const float *ws, int slabs, int F, int wdtype, void *gw, void *gb) {
  __shared__ double part[64][16];
  const int64_t c = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const int s0 = threadIdx.x >> 4;
  double v = 0.;
  if (c < 2 * (int64_t)F)
#pragma unroll 8
    for (int s = s0; s < slabs; s += 64) v += (double)ws[(int64_t)s * 2 * F + c];
  part[s0][threadIdx.x & 15] = v;
  __syncthreads();
  if (threadIdx.x < 16 && c < 2 * (int64_t)F) {
    v = 0.;
    for (int s = 0; s < 64; ++s) v += part[s][threadIdx.x];
    if (c < F) { if (gw) store_w(gw, wdtype, c, (float)v); }
    else if (gb) store_w(gb, wdtype, c - F, (float)v);
  }
}

// ------------------------------------------------------------------ rows longer than a workgroup's registers (16 384)
__device__ __forceinline__ float block_sum(float v) {      // over 1024 threads, in every thread
  __shared__ float part[16];
  v = lanes_sum<64>(v);
  __syncthreads();
  if (gs_lane() == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += part[i];
  return v;
}

// Thread t's vectors of a row are t, t + 1024, ... ; the last of the row is moved back as in Cols
template <typename T> struct LongVec {
  static constexpr int V = Tab<T>::V;
  int c, lo;
  __device__ __forceinline__ LongVec(int v, int F) : c(v < F - V ? v : F - V) { lo = v - c; }
  __device__ __forceinline__ void z(const Ln<T> &a, int64_t base, uint64_t key, uint32_t thr, float (&z)[V], bool (&kept)[V]) const {
    Raw<T, V> x, r;
    x.load(a.x + base + c);
    if (a.res) r.load(a.res + base + c);
    x.open(z);
    if (a.d.p > 0.f) {
      draw_vec<V>(kept, (uint64_t)(base + c), key, thr, a.d.p);
      drop_vec<V>(z, kept, a.d.inv_keep);
    }
    if (!a.res) return;
    float q[V];
    r.open(q);
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] += q[i];
  }
  __device__ __forceinline__ void weight(const void *w, int wdtype, float other, float (&f)[V]) const {
    Weights<T, V> r;
    r.load(w, wdtype, c);
    r.open(w, wdtype, other, f);
  }
};

// A row is read twice (from the caches where it has stayed there): for its mean and squares about it, which a thread takes
// along from vector to vector (each vector about its own mean, then the two put together), and for y.  Bound by the second
// read and by a thread's few loads in flight: 4096 x 32768 fp32 0.28 ms, joined 0.38, backward 0.66 and 0.99 (bf16 0.17,
// 0.27, 0.36, 0.57).
template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_long_k(Ln<T> a, float eps, T *y, T *sum, float *mean, float *rstd) {
  constexpr int V = Tab<T>::V;
  const uint64_t key = drop_key(a.d);
  const uint32_t thr = dropout_threshold(a.d.p);
  const float inv_f = 1.0f / (float)a.F;
  for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
    const int64_t base = r * a.F;
    float n = 0.f, m = 0.f, q = 0.f, z[V];
    bool kept[V];
    for (int v = threadIdx.x * V; v < a.F; v += 1024 * V) {
      const LongVec<T> at(v, a.F);
      at.z(a, base, key, thr, z, kept);
      float s = 0.f, qv = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) s += i >= at.lo ? z[i] : 0.f;
      const float nv = (float)(V - at.lo), mv = s / nv;
#pragma unroll
      for (int i = 0; i < V; ++i) { const float e = i >= at.lo ? z[i] - mv : 0.f; qv = fmaf(e, e, qv); }
      const float all = n + nv, e = n > 0.f ? mv - m : 0.f;      // (the first vector's mean is no distance from another)
      m = n > 0.f ? fmaf(e, nv / all, m) : mv;
      q += fmaf(e * e, n * nv / all, qv);
      n = all;
    }
    const float mr = block_sum(m * n) * inv_f, e = m - mr;
    const float rs = 1.0f / sqrtf(block_sum(fmaf(e * e, n, q)) * inv_f + eps);
    for (int v = threadIdx.x * V; v < a.F; v += 1024 * V) {
      const LongVec<T> at(v, a.F);
      float w[V], b[V];
      at.z(a, base, key, thr, z, kept);
      at.weight(a.w, a.wdtype, 1.f, w);
      at.weight(a.b, a.wdtype, 0.f, b);
      if (sum) Raw<T, V>::store(sum + base + at.c, z);
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = fmaf((z[i] - mr) * rs, w[i], b[i]);
      Raw<T, V>::store(y + base + at.c, z);
    }
    if (mean && threadIdx.x == 0) { mean[r] = mr; rstd[r] = rs; }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_dz_long_k(Ln<T> a, const T *g, const T *gsum, const float *mean,
                                                     const float *rstd, T *gx, T *gres) {
  constexpr int V = Tab<T>::V;
  const uint64_t key = drop_key(a.d);
  const uint32_t thr = dropout_threshold(a.d.p);
  const float inv_f = 1.0f / (float)a.F;
  for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
    const int64_t base = r * a.F;
    const float m = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f, h[V], e[V], w[V];
    bool kept[V];
    const auto row = [&](const LongVec<T> &at) {      // h and g w of these columns
      Raw<T, V> gr;
      gr.load(g + base + at.c);
      at.z(a, base, key, thr, h, kept);
      at.weight(a.w, a.wdtype, 1.f, w);
      gr.open(e);
#pragma unroll
      for (int i = 0; i < V; ++i) { h[i] = (h[i] - m) * rs; e[i] *= w[i]; }
    };
    for (int v = threadIdx.x * V; v < a.F; v += 1024 * V) {
      const LongVec<T> at(v, a.F);
      row(at);
#pragma unroll
      for (int i = 0; i < V; ++i) { const float one = i >= at.lo ? e[i] : 0.f; s1 += one; s2 = fmaf(one, h[i], s2); }
    }
    s1 = block_sum(s1) * inv_f;
    s2 = block_sum(s2) * inv_f;
    for (int v = threadIdx.x * V; v < a.F; v += 1024 * V) {
      const LongVec<T> at(v, a.F);
      row(at);
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = rs * fmaf(-h[i], s2, e[i] - s1);
      if (gsum) {
        Raw<T, V> sr;
        float q[V];
        sr.load(gsum + base + at.c);
        sr.open(q);
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] += q[i];
      }
      if (gres) Raw<T, V>::store(gres + base + at.c, e);
      if (!gx) continue;
      if (a.d.p > 0.f) drop_vec<V>(e, kept, a.d.inv_keep);
      Raw<T, V>::store(gx + base + at.c, e);
    }
  }
}

// A vector of columns a thread, rows blockIdx.y, blockIdx.y + gridDim.y, ... -> slab blockIdx.y.  Summed in double: an fp32
// sum with its error carried along costs the same registers, and an infinite gradient leaves NaN in the carry.
template <typename T>
__global__ void __launch_bounds__(256) ln_dw_long_k(Ln<T> a, const T *g, const float *mean, const float *rstd, float *ws) {
  constexpr int V = Tab<T>::V;
  const int v = (blockIdx.x * 256 + threadIdx.x) * V;
  if (v >= a.F) return;
  const LongVec<T> at(v, a.F);
  const uint64_t key = drop_key(a.d);
  const uint32_t thr = dropout_threshold(a.d.p);
  double dw[V] = {}, db[V] = {};
  float h[V], e[V];
  bool kept[V];
  for (int64_t r = blockIdx.y; r < a.M; r += gridDim.y) {
    Raw<T, V> gr;
    gr.load(g + r * a.F + at.c);
    at.z(a, r * a.F, key, thr, h, kept);
    gr.open(e);
    const float m = mean[r], rs = rstd[r];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[i] += (double)(e[i] * ((h[i] - m) * rs));
      db[i] += (double)e[i];
    }
  }
  float *slab = ws + (int64_t)blockIdx.y * 2 * a.F;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i < at.lo) continue;
    slab[at.c + i] = (float)dw[i];
    slab[a.F + at.c + i] = (float)db[i];
  }
}

// ------------------------------------------------------------------ launches
constexpr int64_t MAX_GRID = 1 << 20;      // workgroups of a launch (a launch's threads are counted in 32 bits)

// Workgroups of this kernel that the GPU holds at once: the rows are dealt out to these, none waits for a place
template <auto KERNEL> int ln_resident(int threads, int lds) {
  static std::atomic<int> known[16 + 1];
  if (lds >= 65536) {      // (the kernels have a little LDS of their own besides; the attribute is a device's own)
    static std::atomic<bool> done[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
      (void)hipFuncSetAttribute((const void *)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
  }
  std::atomic<int> &n = known[threads / 64];
  int blocks = n.load(std::memory_order_relaxed);
  if (blocks == 0) {
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, KERNEL, threads, lds) != hipSuccess || blocks < 1) blocks = 1;
    n.store(blocks, std::memory_order_relaxed);
  }
  return 256 * blocks;
}

template <typename T, int V, int TPR, int K, bool JOIN, bool NT, bool LOOP>
void ln_fwd_launch(const Ln<T> &a, int turns, float eps, T *y, T *sum, float *mean, float *rstd, hipStream_t st) {
  constexpr auto kernel = ln_fwd_k<T, V, TPR, K, JOIN, NT, LOOP>;
  const int threads = TPR > 0 ? 256 : a.row, rows = threads / a.row;
  if (turns > 0) {      // neighbouring rows, workgroups in order
    const int64_t apart = (int64_t)rows * turns;
    for (int64_t begin = 0; begin < a.M; begin += MAX_GRID * apart) {
      const int64_t left = (a.M - begin + apart - 1) / apart;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(left < MAX_GRID ? left : MAX_GRID)), dim3(threads), 0, st, a,
                         Walk{begin, apart, rows, turns}, eps, y, sum, mean, rstd);
    }
  } else {              // the grid that the GPU holds
    const int blocks = norm_blocks(a.M, rows, ln_resident<kernel>(threads, 0));
    const int64_t step = (int64_t)blocks * rows;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, st, a, Walk{0, rows, step, (int)((a.M + step - 1) / step)}, eps, y,
                       sum, mean, rstd);
  }
}

// One turn a workgroup, where it has 3200 bytes of rows to spread its weights over (fp32 2 M x 28: 81 us, 83 as a loop of
// two turns; 2 M x 20: 70 us, as a loop 60; 4 M x 4 59 and 41); 16-bit rows without dropout or a residual need two (less
// arithmetic a byte: 4 M x 64 bf16 0.167 against 0.181 ms), and so do rows of two or four waves.  Rows of several waves
// with three vectors a thread or more, and of more than eight waves, run as loops over the grid that the GPU holds (8191 x
// 5120 bf16 in three waves 33 us, 42 in order).
template <typename T, int V, int TPR, int K, bool JOIN, bool NT>
void ln_fwd_go(const Ln<T> &a, float eps, T *y, T *sum, float *mean, float *rstd, hipStream_t st) {
  const int64_t bytes = 256 / (TPR > 0 ? TPR : 256) * (int64_t)a.F * sizeof(T);
  constexpr bool thin = sizeof(T) == 2 && !JOIN;
  if constexpr (TPR <= 0) ln_fwd_launch<T, V, TPR, K, JOIN, NT, true>(a, K == 2 && TPR == 0 ? 2 : 0, eps, y, sum, mean, rstd, st);
  else if constexpr (thin || K == 1) {
    if (thin || bytes < 3200)
      ln_fwd_launch<T, V, TPR, K, JOIN, NT, true>(a, bytes < 4096 ? (int)((8191 + bytes) / bytes) : 2, eps, y, sum, mean, rstd, st);
    else if constexpr (!thin) ln_fwd_launch<T, V, TPR, K, JOIN, NT, false>(a, 1, eps, y, sum, mean, rstd, st);
  } else ln_fwd_launch<T, V, TPR, K, JOIN, NT, false>(a, 1, eps, y, sum, mean, rstd, st);
}

// -> the slabs of column sums that are left in ws
template <typename T, int V, int TPR, int K, bool JOIN, bool NT>
int ln_bwd_go(const Ln<T> &a, const Grads<T> &d, hipStream_t st) {
  constexpr auto kernel = ln_bwd_k<T, V, TPR, K, JOIN, NT>;
  constexpr bool AHEAD = ln_bwd_ahead(V, TPR, K, JOIN);
  constexpr int few = 2 * K * V * ln_bwd_threads(TPR) * (int)sizeof(float), lds = AHEAD ? 2 * few : few;
  const int rows = ln_bwd_threads(TPR) / a.row, threads = rows * a.row, resident = ln_resident<kernel>(threads, lds);
  // Streamed fp32 tables of short rows in order, as the forward takes them, two turns a workgroup and a slab for each:
  // 10 M x 64 1.37 -> 1.25 ms, 4 M x 128 1.06 -> 1.01 (joined, and in 16 bits, nothing is gained: more arithmetic a byte).
  // A slab is written once and read once: 2 % of the traffic at its 64 rows of 64 columns, 4 % at 32 rows of 128.
  constexpr int turns = NORM_FOLD_TURNS;
  if (NT && !JOIN && d.ws && norm_folds(a.M, a.F, sizeof(T), JOIN)) {
    const int blocks = (int)((a.M + rows * turns - 1) / (rows * turns)), folded = norm_blocks(blocks, 1, 256);
    static_assert(!AHEAD || turns < ln_bwd_doubles(TPR, JOIN), "the column sums are fp32 words");
    static_assert(TPR <= 0 || ln_bwd_threads(TPR) == NORM_FOLD_THREADS, "the workspace counts their rows a workgroup");
    // (room for two workgroups a compute unit: 1 M x 96 192 us, 218 with doubles')
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), few, st, a, Walk{0, (int64_t)rows * turns, rows, turns}, d);
    const int per = (blocks + folded - 1) / folded;
    float *out = d.ws + (int64_t)blocks * 2 * a.F;
    hipLaunchKernelGGL(ln_fold_k, dim3((unsigned)((2 * a.F + 63) / 64), folded), dim3(1024), 0, st, d.ws, blocks, per, a.F, out);
    hipLaunchKernelGGL(ln_slabs_k, dim3((unsigned)((2 * a.F + 15) / 16)), dim3(1024), 0, st, out, folded, a.F, a.wdtype, d.gw, d.gb);
    return 0;
  }
  // Of the large tables sixteen waves a compute unit keep the memory busy where a lane holds one vector, or two of a plain
  // fp32 row; 24 of them were slower (1 M x 256 fp32 0.56 against 0.52 ms).  Joined rows of two vectors, plain ones of two in
  // 16 bits and all of three run eight: registers (129 and more; of plain fp32 rows the doubles in LDS) allow no more.
  // Sixteen of the joined fp32 ones, from a build that needed 115 registers, were slower: 1 M x 128 478 us against 433,
  // 1 M x 256 965 against 905.
  const int most = norm_max_slabs(a.M, a.F), held = NT && resident > 512 ? 512 : resident;
  const int slabs = norm_blocks(a.M, rows, held < most ? held : most);
  const int64_t step = (int64_t)slabs * rows;
  hipLaunchKernelGGL(kernel, dim3(slabs), dim3(threads), lds, st, a, Walk{0, rows, step, (int)((a.M + step - 1) / step)}, d);
  return slabs > 1 ? slabs : 0;
}

// every form: CASE(kind, V, TPR, K); LINE: those of large plain fp32 tables only
#define LN_FORMS(CASE, LINE)                                                                                  \
  CASE(NORM_ONE, 1, 8, 1) CASE(NORM_R4, V, 4, 1) CASE(NORM_R8, V, 8, 1) CASE(NORM_R8x2, V, 8, 2)              \
  CASE(NORM_R8x3, V, 8, 3) LINE(NORM_R16, V, 16, 1) CASE(NORM_R16x2, V, 16, 2) CASE(NORM_R16x3, V, 16, 3)     \
  LINE(NORM_R32, V, 32, 1) CASE(NORM_R32x2, V, 32, 2) CASE(NORM_R32x3, V, 32, 3) LINE(NORM_R64, V, 64, 1)     \
  CASE(NORM_R64x2, V, 64, 2) CASE(NORM_R64x3, V, 64, 3) CASE(NORM_B2, V, 0, 2) CASE(NORM_B3, V, 0, 3)                          \
  CASE(NORM_W1, V, -1, 1) CASE(NORM_W, V, -1, 16 / V)

template <typename T>
int ln_fwd(const NormFwd &n, hipStream_t st) {
  constexpr int V = Tab<T>::V;
  const bool join = n.res || n.d.p > 0.f || n.sum, nt = norm_streams(n.M, n.F, sizeof(T));
  const NormForm f = norm_form(n.F, V, nt && !join);
  const Ln<T> a{(const T *)n.x, (const T *)n.res, n.w, n.b, n.M, (int)n.F, n.wdtype, f.row, n.d};
  T *y = (T *)n.y, *sum = (T *)n.sum;
#define ARGS a, n.eps, y, sum, n.mean, n.rstd, st
#define CASE(KIND, V, TPR, K)                                                                        \
  case KIND:                                                                                         \
    if (join) { if (nt) ln_fwd_go<T, V, TPR, K, true, true>(ARGS); else ln_fwd_go<T, V, TPR, K, true, false>(ARGS); } \
    else { if (nt) ln_fwd_go<T, V, TPR, K, false, true>(ARGS); else ln_fwd_go<T, V, TPR, K, false, false>(ARGS); }    \
    break;
#define LINE(KIND, V, TPR, K) \
  case KIND: if constexpr (V == 4) ln_fwd_go<T, V, TPR, K, false, true>(ARGS); break;
  switch (f.kind) {
    LN_FORMS(CASE, LINE)
    case NORM_B4:      // (16-bit rows as long take NORM_W)
      if constexpr (V == 4) {
        if (join) { if (nt) ln_fwd_go<T, V, 0, 4, true, true>(ARGS); else ln_fwd_go<T, V, 0, 4, true, false>(ARGS); }
        else { if (nt) ln_fwd_go<T, V, 0, 4, false, true>(ARGS); else ln_fwd_go<T, V, 0, 4, false, false>(ARGS); }
      }
      break;
    case NORM_LONG:
      hipLaunchKernelGGL(ln_fwd_long_k<T>, dim3(gs_grid(n.M, 1, 512)), dim3(1024), 0, st, a, n.eps, y, sum, n.mean, n.rstd);
  }
#undef CASE
#undef LINE
#undef ARGS
  GSAGE_CHECK_LAUNCH();
  return GSAGE_OK;
}

template <typename T>
int ln_bwd(const NormBwd &n, hipStream_t st) {
  constexpr int V = Tab<T>::V;
  const bool join = n.joined(), nt = norm_streams(n.M, n.F, sizeof(T));
  const NormForm f = norm_form(n.F, V, nt && !join);
  const Ln<T> a{(const T *)n.x, (const T *)n.res, n.w, nullptr, n.M, (int)n.F, n.wdtype, f.row, n.d};
  const Grads<T> d{(const T *)n.g, (const T *)n.gsum, n.mean, n.rstd, (T *)n.gx, (T *)n.gres,
                   n.gw || n.gb ? n.ws : nullptr, n.gw, n.gb};
  int slabs = norm_max_slabs(n.M, n.F);
  if (n.M > 0 && (d.gx || d.gres || d.ws)) {
#define CASE(KIND, V, TPR, K)                                                                          \
  case KIND:                                                                                           \
    slabs = join ? (nt ? ln_bwd_go<T, V, TPR, K, true, true>(a, d, st) : ln_bwd_go<T, V, TPR, K, true, false>(a, d, st))   \
                 : (nt ? ln_bwd_go<T, V, TPR, K, false, true>(a, d, st) : ln_bwd_go<T, V, TPR, K, false, false>(a, d, st)); \
    break;
#define LINE(KIND, V, TPR, K) \
  case KIND: if constexpr (V == 4) slabs = ln_bwd_go<T, V, TPR, K, false, true>(a, d, st); break;
    switch (f.kind) {
      LN_FORMS(CASE, LINE)
      case NORM_B4:
        if constexpr (V == 4)
          slabs = join ? (nt ? ln_bwd_go<T, V, 0, 4, true, true>(a, d, st) : ln_bwd_go<T, V, 0, 4, true, false>(a, d, st))
                       : (nt ? ln_bwd_go<T, V, 0, 4, false, true>(a, d, st) : ln_bwd_go<T, V, 0, 4, false, false>(a, d, st));
        break;
      case NORM_LONG:
        if (d.gx || d.gres)
          hipLaunchKernelGGL(ln_dz_long_k<T>, dim3(gs_grid(n.M, 1, 512)), dim3(1024), 0, st, a, d.g, d.gsum, d.mean, d.rstd,
                             d.gx, d.gres);
        if (d.ws)
          hipLaunchKernelGGL(ln_dw_long_k<T>, dim3((unsigned)((n.F + 256 * V - 1) / (256 * V)), slabs), dim3(256), 0, st, a, d.g, d.mean,
                             d.rstd, d.ws);
    }
#undef CASE
#undef LINE
    GSAGE_CHECK_LAUNCH();
  }
  if (d.ws && (slabs > 0 || n.M == 0)) {
    hipLaunchKernelGGL(ln_slabs_k, dim3((unsigned)((2 * n.F + 15) / 16)), dim3(1024), 0, st, d.ws, slabs, (int)n.F, n.wdtype,
                       d.gw, d.gb);
    GSAGE_CHECK_LAUNCH();
  }
  return GSAGE_OK;
}

template <typename T> int dropout_go(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st) {
  const int64_t threads = n / Tab<T>::V + n % Tab<T>::V;
  for (int64_t begin = 0; begin < threads; begin += (int64_t)MAX_GRID * 256) {
    const int64_t left = (threads - begin + 255) / 256;
    const dim3 grid((unsigned)(left < MAX_GRID ? left : MAX_GRID)), block(256);
    if (norm_large(n, sizeof(T))) hipLaunchKernelGGL((dropout_k<T, true>), grid, block, 0, st, (const T *)x, n, begin, d, (T *)out);
    else hipLaunchKernelGGL((dropout_k<T, false>), grid, block, 0, st, (const T *)x, n, begin, d, (T *)out);
    GSAGE_CHECK_LAUNCH();
  }
  return GSAGE_OK;
}

}  // namespace

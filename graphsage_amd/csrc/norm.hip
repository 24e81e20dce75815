// Layer norm and counter-based dropout, forward and backward, and the two joined with a residual sum.
//
//   z = residual + dropout(x);  y = (z - mean) rstd w + b
//   a = g w;  h = (z - mean) rstd;  dz = rstd (a - mean(a) - h mean(a h)) + grad_sum
//   grad_residual = dz;  grad_x = dropout'(dz);  grad_w = sum_rows g h;  grad_b = sum_rows g
//
// Neither the mask nor z is stored: both are formed again from (seed, index) and from x and residual.
#include <atomic>

#include "gsage_common.h"
#include "gsage_dropout.h"

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
  __device__ __forceinline__ void zero() { w = u32x4{0u, 0u, 0u, 0u}; }
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
  __device__ __forceinline__ void zero() { w = (T)0.f; }
  template <bool NT = false> __device__ __forceinline__ void load(const T *p) { w = *p; }
  __device__ __forceinline__ void open(float (&f)[1]) const { f[0] = (float)w; }
  template <bool NT = false> static __device__ __forceinline__ void store(T *p, const float (&f)[1]) { *p = (T)f[0]; }
};

// ------------------------------------------------------------------ dropout
struct Drop {              // p = 0: no mask
  float p, inv_keep;
  uint64_t seed;
  const int64_t *seed_dev;
  __device__ __forceinline__ uint64_t key() const { return seed_dev ? (uint64_t)*seed_dev : seed; }
};

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

template <typename T, bool NT>
__global__ void __launch_bounds__(256) dropout_k(const T *x, int64_t n, Drop d, T *out) {
  constexpr int V = Tab<T>::V, U = 4;
  const uint64_t key = d.key();
  const uint32_t thr = dropout_threshold(d.p);
  const int64_t nv = n / V, stride = (int64_t)gridDim.x * 256;
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const auto put = [&](const Raw<T, V> &r, int64_t at) {
    float f[V];
    bool kept[V];
    r.open(f);
    draw_vec<V>(kept, (uint64_t)at * V, key, thr, d.p);
    drop_vec<V>(f, kept, d.inv_keep);
    Raw<T, V>::template store<NT>(out + at * V, f);
  };
  for (; i + (U - 1) * stride < nv; i += U * stride) {
    Raw<T, V> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u].template load<NT>(x + (i + u * stride) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) put(r[u], i + u * stride);
  }
  for (; i < nv; i += stride) {
    Raw<T, V> r;
    r.template load<NT>(x + i * V);
    put(r, i);
  }
  if (blockIdx.x == 0 && threadIdx.x < n - nv * V) {      // the last n mod V elements
    const int64_t e = nv * V + threadIdx.x;
    out[e] = (T)(dropout_keep(key, (uint64_t)e, d.p) ? (float)x[e] * d.inv_keep : 0.f);
  }
}

// ------------------------------------------------------------------ sums over the threads of a row
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// over aligned groups of N lanes (8 .. 64), in every lane; all lanes of the wave take part
template <int N> __device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<0xB1>(v);                 // quad_perm: lane ^ 1
  v += dpp<0x4E>(v);                 // quad_perm: lane ^ 2
  v += dpp<0x141>(v);                // row_half_mirror: the other four of eight
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

// V weights from column c on, fp32 or of the tables' type
template <typename T, int V> __device__ __forceinline__ void load_w(const void *w, int wdtype, int c, float (&f)[V]) {
  if (wdtype == GSAGE_F32) {
    const float *p = (const float *)w + c;
    if constexpr (V == 1) f[0] = p[0];
    else {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        float o[4];
        Raw<float, 4> r;
        r.load(p + q);
        r.open(o);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[q + i] = o[i];
      }
    }
  } else {
    Raw<T, V> r;
    r.load((const T *)w + c);
    r.open(f);
  }
}
__device__ __forceinline__ void store_w(void *w, int wdtype, int64_t c, float v) {
  if (wdtype == GSAGE_F32) ((float *)w)[c] = v;
  else if (wdtype == GSAGE_BF16) ((__bf16 *)w)[c] = (__bf16)v;
  else ((_Float16 *)w)[c] = (_Float16)v;
}

template <typename T> struct Ln {
  const T *x, *res;
  const void *w, *b;
  int64_t M;
  int F, wdtype;
  Drop d;
};

// A row takes TPR lanes of a wave (RPB rows a workgroup of four waves), or (TPR = 0) a workgroup of up to MAXW waves.
// Thread t of the row holds K vectors of V columns, a row's threads apart.  Where V does not divide F the last vector is
// moved back to end with the row; its first `lo` elements then belong to the vector before it: both threads form and
// store the same values, the sums count them once.
constexpr int MAXW = 8;
template <int V, int TPR, int K> struct Cols {
  int t, threads, col[K], lo[K];
  bool on[K], full;
  __device__ __forceinline__ Cols(int F) {
    t = TPR ? threadIdx.x % (TPR ? TPR : 1) : threadIdx.x;
    threads = TPR ? TPR : blockDim.x;
    full = F == threads * K * V;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int v = (t + k * threads) * V;
      on[k] = v < F;
      col[k] = v < F - V ? v : F - V;
      lo[k] = v - col[k];
    }
  }
  __device__ __forceinline__ bool live(int k, int i) const { return on[k] && i >= lo[k]; }
  // live elements of wave i of a workgroup's row
  __device__ __forceinline__ int wave_count(int i, int F) const {
    int n = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int left = F - (i * 64 + k * threads) * V;
      n += left < 0 ? 0 : left < 64 * V ? left : 64 * V;
    }
    return n;
  }
};

// The operands of z of one row: loaded a row ahead of their use
template <typename T, int V, int TPR, int K, bool JOIN, bool NT> struct Operands {
  Raw<T, V> x[K], r[JOIN ? K : 1];
  __device__ __forceinline__ void load(const Ln<T> &a, const Cols<V, TPR, K> &c, int64_t row, bool in) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k].zero();
      if (JOIN) r[k].zero();
      if (in && c.on[k]) {
        x[k].template load<NT>(a.x + row * a.F + c.col[k]);
        if (JOIN && a.res) r[k].template load<NT>(a.res + row * a.F + c.col[k]);
      }
    }
  }
  __device__ __forceinline__ void z(const Ln<T> &a, const Cols<V, TPR, K> &c, int64_t row, uint64_t key, uint32_t thr,
                                    float (&z)[K][V], bool (&kept)[K][V]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k].open(z[k]);
      if (JOIN) {
        if (a.d.p > 0.f) {
          draw_vec<V>(kept[k], (uint64_t)(row * a.F + c.col[k]), key, thr, a.d.p);
          drop_vec<V>(z[k], kept[k], a.d.inv_keep);
        }
        if (a.res) {
          float q[V];
          r[k].open(q);
#pragma unroll
          for (int i = 0; i < V; ++i) z[k][i] += q[i];
        }
      }
    }
  }
};

// ------------------------------------------------------------------ forward
template <typename T, int V, int TPR, int K, bool JOIN, bool NT>
__global__ void __launch_bounds__(TPR ? 256 : 64 * MAXW) ln_fwd_k(Ln<T> a, float eps, T *y, T *sum, float *mean, float *rstd) {
  constexpr int RPB = TPR ? 256 / (TPR ? TPR : 1) : 1;
  __shared__ float part[TPR ? 1 : 2][TPR ? 1 : MAXW][2];
  const Cols<V, TPR, K> c(a.F);
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) { w[k][i] = 1.f; b[k][i] = 0.f; }
    if (a.w && c.on[k]) load_w<T, V>(a.w, a.wdtype, c.col[k], w[k]);
    if (a.b && c.on[k]) load_w<T, V>(a.b, a.wdtype, c.col[k], b[k]);
  }
  const uint64_t key = JOIN ? a.d.key() : 0;
  const uint32_t thr = JOIN ? dropout_threshold(a.d.p) : 0;
  const float inv_f = 1.0f / (float)a.F;
  // (workgroup a row) this wave's elements, and those of the wave whose sums this lane puts together
  const int mine = TPR ? 0 : c.wave_count(threadIdx.x >> 6, a.F), 
            other = TPR || threadIdx.x % MAXW >= blockDim.x >> 6 ? 0 : c.wave_count(threadIdx.x % MAXW, a.F);
  const float inv_mine = mine ? 1.0f / (float)mine : 0.f, inv_other = other ? 1.0f / (float)other : 0.f;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + (TPR ? threadIdx.x / (TPR ? TPR : 1) : 0);
  Operands<T, V, TPR, K, JOIN, NT> next;
  next.load(a, c, row, row < a.M);
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.M; r0 += step, row += step, turn ^= 1) {
    float z[K][V];
    bool kept[K][V];
    next.z(a, c, row, key, thr, z, kept);
    next.load(a, c, row + step, row + step < a.M);
    float s = 0.f, q = 0.f, m, var;
    const auto total = [&]() {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s += c.full || c.live(k, i) ? z[k][i] : 0.f;
    };
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
    total();
    if constexpr (TPR != 0) {
      m = lanes_sum<TPR>(s) * inv_f;
      squares(m);
      var = lanes_sum<TPR>(q) * inv_f;
    } else {
      // each wave about its own mean, the waves' (sum, sum of squares about it) then put together: one barrier a row
      // (the slots alternate), and no difference of large sums
      const float sw = lanes_sum<64>(s);
      squares(sw * inv_mine);
      q = lanes_sum<64>(q);
      float(*slot)[2] = part[turn];
      if (gs_lane() == 0) { slot[threadIdx.x >> 6][0] = sw; slot[threadIdx.x >> 6][1] = q; }
      __syncthreads();
      // (waves that are not there have no elements; their slots hold whatever LDS held)
      const float so = other ? slot[threadIdx.x % MAXW][0] : 0.f, qo = other ? slot[threadIdx.x % MAXW][1] : 0.f;
      m = lanes_sum<MAXW>(so) * inv_f;
      const float e = so * inv_other - m;
      var = lanes_sum<MAXW>(fmaf(e * e, (float)other, qo)) * inv_f;
    }
    const float rs = rsqrtf(var + eps);
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

// ------------------------------------------------------------------ backward
// A thread adds up the rows of its columns in two levels, 16 rows and then the sixteens: of thousands of rows in a row
// the fp32 sum would lose some bits.
constexpr int FLUSH = 16;

template <typename T> struct Grads {
  const T *g, *gsum;
  const float *mean, *rstd;
  T *gx, *gres;
  float *ws;               // slabs; NULL: no column sums wanted
  void *gw, *gb;           // written by the kernel itself where one workgroup is the whole grid
};

template <typename T, int V, int TPR, int K, bool JOIN, bool NT>
__global__ void __launch_bounds__(TPR ? 256 : 64 * MAXW) ln_bwd_k(Ln<T> a, Grads<T> d) {
  constexpr int RPB = TPR ? 256 / (TPR ? TPR : 1) : 1;
  __shared__ float part[TPR ? 1 : 2][TPR ? 1 : MAXW][2];
  __shared__ float colsum[TPR ? 4 : 1][TPR ? 2 * TPR * K * V : 1];
  const Cols<V, TPR, K> c(a.F);
  float w[K][V], dw[K][V], db[K][V], dw2[K][V], db2[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) { w[k][i] = 1.f; dw[k][i] = db[k][i] = dw2[k][i] = db2[k][i] = 0.f; }
    if (a.w && c.on[k]) load_w<T, V>(a.w, a.wdtype, c.col[k], w[k]);
  }
  const uint64_t key = JOIN ? a.d.key() : 0;
  const uint32_t thr = JOIN ? dropout_threshold(a.d.p) : 0;
  const float inv_f = 1.0f / (float)a.F;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + (TPR ? threadIdx.x / (TPR ? TPR : 1) : 0);
  Operands<T, V, TPR, K, JOIN, NT> next;
  Raw<T, V> gnext[K], snext[JOIN ? K : 1];
  float mnext = 0.f, rnext = 0.f;
  const auto fetch = [&](int64_t r) {
    const bool in = r < a.M;
    next.load(a, c, r, in);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      gnext[k].zero();
      if (JOIN) snext[k].zero();
      if (in && c.on[k]) {
        gnext[k].template load<NT>(d.g + r * a.F + c.col[k]);
        if (JOIN && d.gsum) snext[k].template load<NT>(d.gsum + r * a.F + c.col[k]);
      }
    }
    mnext = in ? d.mean[r] : 0.f;
    rnext = in ? d.rstd[r] : 0.f;
  };
  const auto flush = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dw2[k][i] += dw[k][i];
        db2[k][i] += db[k][i];
        dw[k][i] = db[k][i] = 0.f;
      }
  };
  fetch(row);
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.M; r0 += step, row += step, ++turn) {
    float h[K][V], gv[K][V], sv[JOIN ? K : 1][V];
    bool kept[K][V];
    next.z(a, c, row, key, thr, h, kept);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      gnext[k].open(gv[k]);
      if (JOIN) snext[k].open(sv[k]);
    }
    const float m = mnext, rs = rnext;
    fetch(row + step);
    if (turn % FLUSH == FLUSH - 1) flush();
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[k][i] = (h[k][i] - m) * rs;
        dw[k][i] = fmaf(gv[k][i], h[k][i], dw[k][i]);
        db[k][i] += gv[k][i];
        gv[k][i] *= w[k][i];
      }
    if (c.full) {
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
    if constexpr (TPR != 0) {
      s1 = lanes_sum<TPR>(s1);
      s2 = lanes_sum<TPR>(s2);
    } else {
      s1 = lanes_sum<64>(s1);
      s2 = lanes_sum<64>(s2);
      float(*slot)[2] = part[turn & 1];
      if (gs_lane() == 0) { slot[threadIdx.x >> 6][0] = s1; slot[threadIdx.x >> 6][1] = s2; }
      __syncthreads();
      const bool there = threadIdx.x % MAXW < blockDim.x >> 6;
      s1 = lanes_sum<MAXW>(there ? slot[threadIdx.x % MAXW][0] : 0.f);
      s2 = lanes_sum<MAXW>(there ? slot[threadIdx.x % MAXW][1] : 0.f);
    }
    s1 *= inv_f;
    s2 *= inv_f;
    if (row < a.M) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!c.on[k]) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          o[i] = rs * fmaf(-h[k][i], s2, gv[k][i] - s1);
          if (JOIN) o[i] += sv[k][i];
        }
        if (JOIN && d.gres) Raw<T, V>::template store<NT>(d.gres + row * a.F + c.col[k], o);
        if (d.gx) {
          if (JOIN && a.d.p > 0.f) drop_vec<V>(o, kept[k], a.d.inv_keep);
          Raw<T, V>::template store<NT>(d.gx + row * a.F + c.col[k], o);
        }
      }
    }
  }
  if (!d.ws) return;
  flush();
  // this workgroup's column sums -> its slab, or the result
  float *slab = d.ws + (int64_t)blockIdx.x * 2 * a.F;
  const auto put = [&](int col, float u, float v) {
    if (gridDim.x > 1) { slab[col] = u; slab[a.F + col] = v; return; }
    if (d.gw) store_w(d.gw, a.wdtype, col, u);
    if (d.gb) store_w(d.gb, a.wdtype, col, v);
  };
  if constexpr (TPR == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c.live(k, i)) put(c.col[k] + i, dw2[k][i], db2[k][i]);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        for (int o = TPR; o < 64; o <<= 1) {
          dw2[k][i] += __shfl_xor(dw2[k][i], o, 64);
          db2[k][i] += __shfl_xor(db2[k][i], o, 64);
        }
        if (gs_lane() < TPR) {
          float *p = colsum[threadIdx.x >> 6] + ((c.t + k * TPR) * V + i) * 2;
          p[0] = dw2[k][i];
          p[1] = db2[k][i];
        }
      }
    __syncthreads();
    if (threadIdx.x < TPR) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c.live(k, i)) {
            float u = 0.f, v = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              u += colsum[q][((c.t + k * TPR) * V + i) * 2];
              v += colsum[q][((c.t + k * TPR) * V + i) * 2 + 1];
            }
            put(c.col[k] + i, u, v);
          }
    }
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

// ------------------------------------------------------------------ rows longer than a workgroup's registers
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

template <typename T> __device__ __forceinline__ float long_z(const Ln<T> &a, int64_t idx, uint64_t key) {
  float v = (float)a.x[idx];
  if (a.d.p > 0.f) v = dropout_keep(key, (uint64_t)idx, a.d.p) ? v * a.d.inv_keep : 0.f;
  return a.res ? (float)a.res[idx] + v : v;
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_long_k(Ln<T> a, float eps, T *y, T *sum, float *mean, float *rstd) {
  const uint64_t key = a.d.key();
  const float inv_f = 1.0f / (float)a.F;
  for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
    const int64_t base = r * a.F;
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < a.F; c += 1024) s += long_z(a, base + c, key);
    const float m = block_sum(s) * inv_f;
    for (int c = threadIdx.x; c < a.F; c += 1024) { const float e = long_z(a, base + c, key) - m; q = fmaf(e, e, q); }
    const float rs = 1.0f / sqrtf(block_sum(q) * inv_f + eps);
    for (int c = threadIdx.x; c < a.F; c += 1024) {
      const float z = long_z(a, base + c, key);
      float w[1] = {1.f}, b[1] = {0.f};
      if (a.w) load_w<T, 1>(a.w, a.wdtype, c, w);
      if (a.b) load_w<T, 1>(a.b, a.wdtype, c, b);
      y[base + c] = (T)fmaf((z - m) * rs, w[0], b[0]);
      if (sum) sum[base + c] = (T)z;
    }
    if (mean && threadIdx.x == 0) { mean[r] = m; rstd[r] = rs; }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_dz_long_k(Ln<T> a, const T *g, const T *gsum, const float *mean,
                                                     const float *rstd, T *gx, T *gres) {
  const uint64_t key = a.d.key();
  const float inv_f = 1.0f / (float)a.F;
  for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
    const int64_t base = r * a.F;
    const float m = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.F; c += 1024) {
      const float h = (long_z(a, base + c, key) - m) * rs;
      float w[1] = {1.f};
      if (a.w) load_w<T, 1>(a.w, a.wdtype, c, w);
      const float e = (float)g[base + c] * w[0];
      s1 += e;
      s2 = fmaf(e, h, s2);
    }
    s1 = block_sum(s1) * inv_f;
    s2 = block_sum(s2) * inv_f;
    for (int c = threadIdx.x; c < a.F; c += 1024) {
      const int64_t i = base + c;
      const float h = (long_z(a, i, key) - m) * rs;
      float w[1] = {1.f};
      if (a.w) load_w<T, 1>(a.w, a.wdtype, c, w);
      const float e = (float)g[i] * w[0];
      float dz = rs * (e - s1 - h * s2);
      if (gsum) dz += (float)gsum[i];
      if (gres) gres[i] = (T)dz;
      if (gx) gx[i] = (T)(a.d.p <= 0.f ? dz : dropout_keep(key, (uint64_t)i, a.d.p) ? dz * a.d.inv_keep : 0.f);
    }
  }
}

// acc + v with the error carried on
__device__ __forceinline__ void add_carry(float &acc, float &carry, float v) {
  const float y = v - carry, t = acc + y;
  carry = (t - acc) - y;
  acc = t;
}

template <typename T>
__global__ void __launch_bounds__(256) ln_dw_long_k(Ln<T> a, const T *g, const float *mean, const float *rstd, float *ws) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.F) return;
  const uint64_t key = a.d.key();
  float dw = 0.f, db = 0.f, dwc = 0.f, dbc = 0.f;
  for (int64_t r = blockIdx.y; r < a.M; r += gridDim.y) {
    const float gv = (float)g[r * a.F + c];
    add_carry(dw, dwc, gv * ((long_z(a, r * a.F + c, key) - mean[r]) * rstd[r]));
    add_carry(db, dbc, gv);
  }
  float *slab = ws + (int64_t)blockIdx.y * 2 * a.F;
  slab[c] = dw;
  slab[a.F + c] = db;
}

// ------------------------------------------------------------------ which kernel
// Lanes a row: as many as it has vectors while they fit a wave, two vectors a lane up to two waves' worth; then a
// workgroup of as many waves as K vectors a thread need.
enum Kind { ONE, R8, R16, R32, R64, R64x2, B1, B2, B4, B8, LONG };
struct Form { Kind kind; int threads, rows; };      // threads of a workgroup, rows it takes at once
Form ln_form(int64_t F, int V, bool backward) {
  if (F < V) return {ONE, 256, 32};
  const int64_t nv = (F + V - 1) / V;
  const auto waves = [&](int k) { return (int)((nv + 64 * k - 1) / (64 * k)) * 64; };
  if (nv <= 8) return {R8, 256, 32};
  if (nv <= 16) return {R16, 256, 16};
  if (nv <= 32) return {R32, 256, 8};
  if (nv <= 64) return {R64, 256, 4};
  if (nv <= 128) return {R64x2, 256, 4};
  if (nv <= 256) return {B1, waves(1), 1};
  if (nv <= 1024) return {B2, waves(2), 1};
  // the backward holds three values and four sums an element: 16 elements a thread at most
  if (nv <= 2048 && (V == 4 || !backward)) return {B4, waves(4), 1};
  if (nv <= 4096 && V == 4 && !backward) return {B8, waves(8), 1};
  return {LONG, 1024, 1};
}
// Workgroups for M rows, at most `cap`, with the same number of turns each (but for the last)
int ln_blocks(int64_t M, int rows, int cap) {
  const int64_t groups = (M + rows - 1) / rows, turns = (groups + cap - 1) / cap;
  return groups ? (int)((groups + turns - 1) / turns) : 0;
}
// Slabs of column sums a backward call writes at most: 1024 workgroups of four waves, fewer of more (their slabs are longer)
int ln_slabs(int64_t M, const Form &f) { return ln_blocks(M, f.rows, f.rows > 1 ? 1024 : f.kind == LONG ? 256 : 131072 / f.threads); }

// Workgroups of this kernel that the GPU holds at once: the rows are dealt out to these, none waits for a place
template <auto KERNEL> int ln_resident(int threads) {
  static std::atomic<int> known[MAXW + 1];
  std::atomic<int> &n = known[threads / 64];
  int blocks = n.load(std::memory_order_relaxed);
  if (blocks == 0) {
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, KERNEL, threads, 0) != hipSuccess || blocks < 1) blocks = 1;
    n.store(blocks, std::memory_order_relaxed);
  }
  return 256 * blocks;
}

// Tables too large for any cache (256 MB behind the L2s) are read and written past them: 10 M x 64 fp32 forward
// 1.09 -> 1.03 ms, backward 1.55 -> 1.51, joined 1.86 -> 1.68 and 3.00 -> 2.89 ms; a 15 MB table loses that way (7.1 ->
// 11.8 us), for the caches serve it.
bool streams(int64_t n, size_t size) { return n * (int64_t)size >= ((int64_t)256 << 20); }

// sizes the kernels' index arithmetic holds for: M F elements counted in int64, columns in int32
constexpr int64_t MAX_F = 1 << 24;
constexpr int64_t MAX_N = (int64_t)1 << 40;

bool bad_dtype(int d) { return d != GSAGE_F32 && d != GSAGE_BF16 && d != GSAGE_F16; }
bool bad_p(float p) { return !(p >= 0.f && p < 1.f); }

template <typename T, int V, int TPR, int K>
void ln_fwd_go(const Ln<T> &a, const Form &f, float eps, T *y, T *sum, float *mean, float *rstd, hipStream_t st) {
  const dim3 block(f.threads);
  const bool join = a.res || a.d.p > 0.f || sum, nt = streams(a.M * a.F, sizeof(T));
#define GO(JOIN, NT)                                                                          \
  hipLaunchKernelGGL((ln_fwd_k<T, V, TPR, K, JOIN, NT>),                                      \
                     dim3(ln_blocks(a.M, f.rows, ln_resident<ln_fwd_k<T, V, TPR, K, JOIN, NT>>(f.threads))), block, 0, st, \
                     a, eps, y, sum, mean, rstd)
  if (join) { if (nt) GO(true, true); else GO(true, false); }
  else { if (nt) GO(false, true); else GO(false, false); }
#undef GO
}

template <typename T>
int ln_fwd(const void *x, const void *res, const void *w, const void *b, int64_t M, int64_t F, int wdtype, float eps,
           const Drop &d, void *y, void *sum, float *mean, float *rstd, hipStream_t st) {
  constexpr int V = Tab<T>::V;
  const Ln<T> a{(const T *)x, (const T *)res, w, b, M, (int)F, wdtype, d};
  const Form f = ln_form(F, V, false);
#define GO(V, TPR, K) ln_fwd_go<T, V, TPR, K>(a, f, eps, (T *)y, (T *)sum, mean, rstd, st); break
  switch (f.kind) {
    case ONE: GO(1, 8, 1);
    case R8: GO(V, 8, 1);
    case R16: GO(V, 16, 1);
    case R32: GO(V, 32, 1);
    case R64: GO(V, 64, 1);
    case R64x2: GO(V, 64, 2);
    case B1: GO(V, 0, 1);
    case B2: GO(V, 0, 2);
    case B4: GO(V, 0, 4);
    case B8: if constexpr (V == 4) { GO(V, 0, 8); } else return GSAGE_ERR_UNSUPPORTED;
    case LONG:
      hipLaunchKernelGGL(ln_fwd_long_k<T>, dim3(gs_grid(M, 1, 512)), dim3(1024), 0, st, a, eps, (T *)y, (T *)sum, mean, rstd);
  }
#undef GO
  GSAGE_CHECK_LAUNCH();
  return GSAGE_OK;
}

// -> the workgroups launched: as many slabs of column sums
template <typename T, int V, int TPR, int K>
int ln_bwd_go(const Ln<T> &a, const Form &f, const Grads<T> &d, hipStream_t st) {
  const dim3 block(f.threads);
  int slabs = ln_slabs(a.M, f);
  const bool join = a.res || a.d.p > 0.f || d.gsum || d.gres, nt = streams(a.M * a.F, sizeof(T));
#define GO(JOIN, NT)                                                                        \
  {                                                                                         \
    const int most = ln_resident<ln_bwd_k<T, V, TPR, K, JOIN, NT>>(f.threads);               \
    if (most < slabs) slabs = ln_blocks(a.M, f.rows, most);                                  \
    hipLaunchKernelGGL((ln_bwd_k<T, V, TPR, K, JOIN, NT>), dim3(slabs), block, 0, st, a, d); \
  }
  if (join) { if (nt) GO(true, true) else GO(true, false) }
  else { if (nt) GO(false, true) else GO(false, false) }
#undef GO
  return slabs;
}

template <typename T>
int ln_bwd(const void *g, const void *gsum, const void *x, const void *res, const void *w, const float *mean,
           const float *rstd, int64_t M, int64_t F, int wdtype, const Drop &drop, void *gx, void *gres, void *gw, void *gb,
           float *ws, hipStream_t st) {
  constexpr int V = Tab<T>::V;
  const Ln<T> a{(const T *)x, (const T *)res, w, nullptr, M, (int)F, wdtype, drop};
  if (!gw && !gb) ws = nullptr;
  const Grads<T> d{(const T *)g, (const T *)gsum, mean, rstd, (T *)gx, (T *)gres, ws, gw, gb};
  const Form f = ln_form(F, V, true);
  int slabs = ln_slabs(M, f);
  if (M > 0 && (gx || gres || ws)) {
#define GO(V, TPR, K) slabs = ln_bwd_go<T, V, TPR, K>(a, f, d, st); break
    switch (f.kind) {
      case ONE: GO(1, 8, 1);
      case R8: GO(V, 8, 1);
      case R16: GO(V, 16, 1);
      case R32: GO(V, 32, 1);
      case R64: GO(V, 64, 1);
      case R64x2: GO(V, 64, 2);
      case B1: GO(V, 0, 1);
      case B2: GO(V, 0, 2);
      case B4: if constexpr (V == 4) { GO(V, 0, 4); } else return GSAGE_ERR_UNSUPPORTED;
      case B8: return GSAGE_ERR_UNSUPPORTED;
      case LONG:
        if (gx || gres)
          hipLaunchKernelGGL(ln_dz_long_k<T>, dim3(gs_grid(M, 1, 512)), dim3(1024), 0, st, a, (const T *)g, (const T *)gsum,
                             mean, rstd, (T *)gx, (T *)gres);
        if (ws)
          hipLaunchKernelGGL(ln_dw_long_k<T>, dim3((unsigned)((F + 255) / 256), slabs), dim3(256), 0, st, a, (const T *)g,
                             mean, rstd, ws);
    }
#undef GO
    GSAGE_CHECK_LAUNCH();
  }
  if (ws && (slabs != 1 || f.kind == LONG)) {
    hipLaunchKernelGGL(ln_slabs_k, dim3((unsigned)((2 * F + 15) / 16)), dim3(1024), 0, st, ws, slabs, (int)F, wdtype, gw, gb);
    GSAGE_CHECK_LAUNCH();
  }
  return GSAGE_OK;
}

template <typename T> void dropout_go(const void *x, int64_t n, const Drop &d, void *out, hipStream_t st) {
  const dim3 grid(gs_grid(n, 256 * 16)), block(256);
  if (streams(n, sizeof(T))) hipLaunchKernelGGL((dropout_k<T, true>), grid, block, 0, st, (const T *)x, n, d, (T *)out);
  else hipLaunchKernelGGL((dropout_k<T, false>), grid, block, 0, st, (const T *)x, n, d, (T *)out);
}

}  // namespace

extern "C" int gsage_dropout(const void *x, int64_t n, int dtype, float p, uint64_t seed, const int64_t *seed_dev,
                             void *out, gsage_stream_t stream) {
  if (n < 0 || bad_dtype(dtype) || bad_p(p)) return GSAGE_ERR_INVALID_ARG;
  if (n == 0) return GSAGE_OK;
  if (!x || !out) return GSAGE_ERR_INVALID_ARG;
  if (n > MAX_N) return GSAGE_ERR_UNSUPPORTED;
  const Drop d{p, 1.0f / (1.0f - p), seed, seed_dev};
  hipStream_t st = gs_stream(stream);
  if (dtype == GSAGE_F32) dropout_go<float>(x, n, d, out, st);
  else if (dtype == GSAGE_BF16) dropout_go<__bf16>(x, n, d, out, st);
  else dropout_go<_Float16>(x, n, d, out, st);
  GSAGE_CHECK_LAUNCH();
  return GSAGE_OK;
}

extern "C" int gsage_layer_norm_fwd(const void *x, const void *residual, const void *weight, const void *bias, int64_t M,
                                    int64_t F, int dtype, int wdtype, float eps, float p, uint64_t seed,
                                    const int64_t *seed_dev, void *y, void *sum, float *mean, float *rstd,
                                    gsage_stream_t stream) {
  if (M < 0 || F <= 0 || bad_dtype(dtype) || bad_p(p) || !(eps >= 0.f)) return GSAGE_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != GSAGE_F32) return GSAGE_ERR_INVALID_ARG;
  if ((mean == nullptr) != (rstd == nullptr)) return GSAGE_ERR_INVALID_ARG;
  if (M == 0) return GSAGE_OK;
  if (!x || !y) return GSAGE_ERR_INVALID_ARG;
  if (F > MAX_F || M > MAX_N / F) return GSAGE_ERR_UNSUPPORTED;
  const Drop d{p, 1.0f / (1.0f - p), seed, seed_dev};
  const auto go = dtype == GSAGE_F32 ? ln_fwd<float> : dtype == GSAGE_BF16 ? ln_fwd<__bf16> : ln_fwd<_Float16>;
  return go(x, residual, weight, bias, M, F, wdtype, eps, d, y, sum, mean, rstd, gs_stream(stream));
}

extern "C" size_t gsage_layer_norm_bwd_workspace_bytes(int64_t M, int64_t F, int dtype) {
  if (M < 0 || F <= 0 || F > MAX_F || bad_dtype(dtype)) return 0;
  const size_t slabs = (size_t)ln_slabs(M, ln_form(F, dtype == GSAGE_F32 ? 4 : 8, true));
  return gs_align_up((slabs ? slabs : 1) * 2 * (size_t)F * sizeof(float), 256);
}

extern "C" int gsage_layer_norm_bwd(const void *grad_y, const void *grad_sum, const void *x, const void *residual,
                                    const void *weight, const float *mean, const float *rstd, int64_t M, int64_t F,
                                    int dtype, int wdtype, float p, uint64_t seed, const int64_t *seed_dev, void *grad_x,
                                    void *grad_residual, void *grad_weight, void *grad_bias, void *ws, size_t ws_bytes,
                                    gsage_stream_t stream) {
  if (M < 0 || F <= 0 || bad_dtype(dtype) || bad_p(p)) return GSAGE_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != GSAGE_F32) return GSAGE_ERR_INVALID_ARG;
  if (F > MAX_F || M > MAX_N / F) return GSAGE_ERR_UNSUPPORTED;
  if (M > 0 && (!grad_y || !x || !mean || !rstd)) return GSAGE_ERR_INVALID_ARG;
  if (grad_weight || grad_bias) {
    if (!ws) return GSAGE_ERR_INVALID_ARG;
    if (ws_bytes < gsage_layer_norm_bwd_workspace_bytes(M, F, dtype)) return GSAGE_ERR_WORKSPACE;
  }
  const Drop d{p, 1.0f / (1.0f - p), seed, seed_dev};
  const auto go = dtype == GSAGE_F32 ? ln_bwd<float> : dtype == GSAGE_BF16 ? ln_bwd<__bf16> : ln_bwd<_Float16>;
  return go(grad_y, grad_sum, x, residual, weight, mean, rstd, M, F, wdtype, d, grad_x, grad_residual, grad_weight,
            grad_bias, (float *)ws, gs_stream(stream));
}

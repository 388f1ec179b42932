// Short causal depthwise convolution over (B, T, D), channels last, with bias and SiLU: forward, backward, one step.
//
//   pre[b,t,c] = bias[c] + sum_k w[c,k] x[b, t-K+1+k, c]        y = act(pre)
// with x before step 0 taken from `state` (B, K-1, D) or 0, and steps at or behind lengths[b] left out (y = 0 there).
//   dpre = dy act'(pre)    dx[t] = sum_j w[j] dpre[t+K-1-j]    dw[j] = sum_{b,t} dpre[t] x[t-K+1+j]    db = sum dpre
//
// Bound by memory: 2 K operations an element against 2 elements moved (forward), 4 moved backward.  A thread owns VEC channels
// (16 bytes; backward of 16-bit types 8) and walks a run of steps with the K-1 last inputs in registers, so that each element is
// read once, plus K-1 of its neighbour's a run; lanes are neighbours in the channels, so a wave reads whole lines.  Four steps
// are fetched together and one group ahead of the arithmetic: a step at a time, the loop waited for memory at each (8 x 2048 x 2048
// bf16: backward 91 us, so 47; forward 34, about 4 TB/s each).  Backward recomputes pre from x instead of keeping it (K multiplications against 2 or 4 bytes an
// element written and read).
#include "elem.h"

#include <type_traits>

namespace {

constexpr int KMAX = 8;

struct ConvArgs {
  const void *x, *w, *bias, *state, *dy;
  const int* lengths;
  void *y, *state_out, *dx;
  float* slab;               // backward: [blocks along the runs][K + 1][D] sums of dw and db
  long sxb, sxt;             // strides of x in elements; y, dy, dx, state are dense
  int B, T, D, run, runs;    // runs of `run` steps each, `runs` of them a sequence
  int act, wf32;
  unsigned gx;               // blocks along the channels; blocks go along them first
};

// AL: every row, and the taps, lie on the access' alignment.  Otherwise accesses of the same width off it, and the last thread of a
// row moves back to the row's last VEC channels: some it shares with its neighbour, who finds and stores the same.
template <bool AL, typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&r)[N]) {
  if constexpr (AL) tb_load_n(p, r);
  else tb_load_u(p, r);
}
template <bool AL, typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float (&r)[N]) {
  if constexpr (AL) tb_store_n(p, r);
  else tb_store_u(p, r);
}
template <bool AL, int VEC>
__device__ __forceinline__ int first_channel(int group, int D) {
  return AL ? group * VEC : min(group * VEC, max(D - VEC, 0));
}

template <typename T, int VEC, bool AL>
__device__ __forceinline__ void load_x(const ConvArgs& a, int b, long t, int len, int K, int c, float (&r)[VEC]) {
  if (t >= 0 && t < len) {
    load_n<AL>(static_cast<const T*>(a.x) + b * a.sxb + t * a.sxt + c, r);
  } else if (t < 0 && a.state && t >= 1 - K) {
    load_n<AL>(static_cast<const T*>(a.state) + ((long)b * (K - 1) + (K - 1 + t)) * a.D + c, r);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r[i] = 0.f;
  }
}

// the taps of VEC channels: K VEC neighbouring values, fetched whole where the channels are (the caller has seen to the
// alignment of w and bias then)
template <typename T, int K, int VEC, bool AL>
__device__ __forceinline__ void load_par(const void* w, const void* bias, int f32, int c, float (&r)[K][VEC], float (&b)[VEC]) {
  float flat[K * VEC];
  if constexpr (VEC == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) flat[k] = tb_load_par<T>(w, (long)c * K + k, f32);
    b[0] = bias ? tb_load_par<T>(bias, c, f32) : 0.f;
  } else {
    if (f32) load_n<AL>(static_cast<const float*>(w) + (long)c * K, flat);
    else load_n<AL>(static_cast<const T*>(w) + (long)c * K, flat);
    if (!bias) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) b[i] = 0.f;
    } else if (f32) load_n<AL>(static_cast<const float*>(bias) + c, b);
    else load_n<AL>(static_cast<const T*>(bias) + c, b);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) r[k][i] = flat[i * K + k];
}

constexpr int GRP = 4;      // steps fetched together; a run is a multiple of it

// GRP rows from step t on, as they lie in memory; rows behind the sequence's steps read another row of it
template <typename T, int VEC, bool AL>
struct Rows {
  typedef std::conditional_t<AL, TbVec<T, VEC>, TbVecU<T, VEC>> Access;
  Access v[GRP];
  __device__ __forceinline__ void fetch(const T* base, long st, int t, int T_) {
#pragma unroll
    for (int i = 0; i < GRP; ++i) v[i] = *reinterpret_cast<const Access*>(base + (long)min(t + i, T_ - 1) * st);
  }
  __device__ __forceinline__ float get(int i, int c, bool on) const { return on ? (float)v[i].v[c] : 0.f; }
};

// block: blockDim.x channel groups of VEC by blockDim.y runs
template <typename T, int K, int VEC, bool AL>
__global__ void __launch_bounds__(256) conv_fwd(ConvArgs a) {
  const int group = blockIdx.x % a.gx * blockDim.x + threadIdx.x, c = first_channel<AL, VEC>(group, a.D);
  const long row = blockIdx.x / a.gx, r = row * blockDim.y + threadIdx.y;
  if ((long)group * VEC >= a.D || r >= (long)a.B * a.runs) return;
  const int b = (int)(r / a.runs), q = (int)(r % a.runs);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const int t0 = q * a.run, t1 = min(t0 + a.run, a.T);
  const T* x = static_cast<const T*>(a.x) + b * a.sxb + c;
  T* y = static_cast<T*>(a.y) + (long)b * a.T * a.D + c;
  if (t0 < t1) {
    Rows<T, VEC, AL> next;
    next.fetch(x, a.sxt, t0, a.T);
    float w[K][VEC], bias[VEC], win[K - 1 + GRP][VEC];
    load_par<T, K, VEC, AL>(a.w, a.bias, a.wf32, c, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load_x<T, VEC, AL>(a, b, (long)t0 - (K - 1) + k, len, K, c, win[k]);
    for (int t = t0; t < t1; t += GRP) {
#pragma unroll
      for (int j = 0; j < GRP; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) win[K - 1 + j][i] = next.get(j, i, t + j < len);
      if (t + GRP < t1) next.fetch(x, a.sxt, t + GRP, a.T);
#pragma unroll
      for (int j = 0; j < GRP; ++j) {
        if (t + j < t1) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float s = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) s = fmaf(w[k][i], win[j + k][i], s);
            if (a.act == TB_ACT_SILU) s = tb_silu(s);
            o[i] = t + j < len ? s : 0.f;
          }
          store_n<AL>(y + (long)(t + j) * a.D, o);
        }
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) win[k][i] = win[k + GRP][i];
    }
  }
  if (a.state_out && q == 0) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float s[VEC];
      load_x<T, VEC, AL>(a, b, (long)len - (K - 1) + k, len, K, c, s);
      store_n<AL>(static_cast<T*>(a.state_out) + ((long)b * (K - 1) + k) * a.D + c, s);
    }
  }
}

template <typename T, int K, int VEC, bool AL>
__global__ void __launch_bounds__(256) conv_bwd(ConvArgs a) {
  __shared__ float red[256][VEC];
  const int group = blockIdx.x % a.gx * blockDim.x + threadIdx.x, c = first_channel<AL, VEC>(group, a.D);
  const long row = blockIdx.x / a.gx, r = row * blockDim.y + threadIdx.y;
  const bool mine = (long)group * VEC < a.D, on = mine && r < (long)a.B * a.runs;
  float dw[K + 1][VEC];
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = 0.f;
  if (on) {
    const int b = (int)(r / a.runs), q = (int)(r % a.runs);
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    const int t0 = q * a.run, t1 = min(t0 + a.run, a.T);
    const T* x = static_cast<const T*>(a.x) + b * a.sxb + c;
    const T* dy = static_cast<const T*>(a.dy) + (long)b * a.T * a.D + c;
    T* dx = static_cast<T*>(a.dx) + (long)b * a.T * a.D + c;
    Rows<T, VEC, AL> nx, ny;
    nx.fetch(x, a.sxt, t0, a.T);
    ny.fetch(dy, a.D, t0, a.T);
    // win[K-1+j]: x of step s + j; dp likewise of dpre
    float w[K][VEC], bias[VEC], win[K - 1 + GRP][VEC], dp[K - 1 + GRP][VEC];
    load_par<T, K, VEC, AL>(a.w, a.bias, a.wf32, c, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      load_x<T, VEC, AL>(a, b, (long)t0 - (K - 1) + k, len, K, c, win[k]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) dp[k][i] = 0.f;
    }
    const int end = t1 + K - 1;               // dx of the run's last steps needs dpre of the next run's first
    for (int s = t0; s < end; s += GRP) {
      float g[GRP][VEC];
#pragma unroll
      for (int j = 0; j < GRP; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          win[K - 1 + j][i] = nx.get(j, i, s + j < len);
          g[j][i] = ny.get(j, i, s + j < len);
        }
      if (s + GRP < end) {
        nx.fetch(x, a.sxt, s + GRP, a.T);
        ny.fetch(dy, a.D, s + GRP, a.T);
      }
#pragma unroll
      for (int j = 0; j < GRP; ++j) {
        const bool own = s + j < t1 && s + j < len;      // the run's own steps, of those that count: their share of dw and db
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float d = g[j][i];
          if (a.act == TB_ACT_SILU) {
            float p = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) p = fmaf(w[k][i], win[j + k][i], p);
            const float sg = tb_sig(p);
            d *= sg * (1.f + p * (1.f - sg));
            d = s + j < len ? d : 0.f;
          }
          dp[K - 1 + j][i] = d;
        }
        if (own) {                            // not 0 times the x of steps before, which may be infinite
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
#pragma unroll
            for (int k = 0; k < K; ++k) dw[k][i] = fmaf(dp[K - 1 + j][i], win[j + k][i], dw[k][i]);
            dw[K][i] += dp[K - 1 + j][i];
          }
        }
        const int t = s + j - (K - 1);        // dx[t] needs dpre[t .. t+K-1] = dp[j .. j+K-1]
        if (t >= t0 && t < t1) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) v = fmaf(w[K - 1 - k][i], dp[j + k][i], v);
            o[i] = t < len ? v : 0.f;
          }
          store_n<AL>(dx + (long)t * a.D, o);
        }
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          win[k][i] = win[k + GRP][i];
          dp[k][i] = dp[k + GRP][i];
        }
    }
  }
  // sums of the block's runs, in the order of the runs
  const int me = threadIdx.y * blockDim.x + threadIdx.x;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) red[me][i] = dw[k][i];
    __syncthreads();
    if (threadIdx.y == 0 && mine) {
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = 0.f;
      for (int j = 0; j < (int)blockDim.y; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] += red[j * blockDim.x + threadIdx.x][i];
      store_n<AL>(a.slab + (row * (K + 1) + k) * a.D + c, o);
    }
    __syncthreads();
  }
}

// dw (D, K), db (D) from the slab's rows, summed in their order by sixteen threads a column
template <typename T>
__global__ void __launch_bounds__(1024) conv_finish(const float* slab, long rows, int K, int D, void* dw, void* db, int wf32) {
  __shared__ float red[16][65];
  const long cols = (long)(K + 1) * D;
  const long col = (long)blockIdx.x * 64 + threadIdx.x;
  float s = 0.f;
  if (col < cols) {
    const long per = (rows + 15) / 16;
    const long r1 = min(rows, (threadIdx.y + 1) * per);
#pragma unroll 4
    for (long r = threadIdx.y * per; r < r1; ++r) s += slab[r * cols + col];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < cols) {
    s = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += red[j][threadIdx.x];
    const int k = (int)(col / D), d = (int)(col % D);
    if (k < K) {
      if (dw) tb_store_par<T>(dw, (long)d * K + k, s, wf32);
    } else if (db) {
      tb_store_par<T>(db, d, s, wf32);
    }
  }
}

struct ConvStepArgs {
  const void *x, *w, *bias;
  void *state, *y;
  long sxb, ssb;     // strides of a row of x and of a row of state
  int B, D, act, wf32;
};

// state (K-1, D) of a row: shifted by one, x appended, in place; a thread reads and writes its own channels only
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_step(ConvStepArgs a) {
  const int groups = a.D / VEC;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)a.B * groups) return;
  const int b = (int)(id / groups), c = (int)(id % groups) * VEC;
  T* st = static_cast<T*>(a.state) + b * a.ssb + c;
  float win[K][VEC], w[K][VEC], bias[VEC], o[VEC];
  load_par<T, K, VEC, true>(a.w, a.bias, a.wf32, c, w, bias);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) tb_load_n(st + (long)k * a.D, win[k]);
  tb_load_n(static_cast<const T*>(a.x) + b * a.sxb + c, win[K - 1]);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float s = bias[i];
#pragma unroll
    for (int k = 0; k < K; ++k) s = fmaf(w[k][i], win[k][i], s);
    o[i] = a.act == TB_ACT_SILU ? tb_silu(s) : s;
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) tb_store_n(st + (long)k * a.D, win[k + 1]);
  tb_store_n(static_cast<T*>(a.y) + (long)b * a.D + c, o);
}

// one instantiation per (type, taps, access): a thread's channels on their alignment, off it, or one by one (fewer channels than
// an access, and the in-place step off the alignment)
enum Access { ALIGNED, OFF, SINGLE };

template <int V16, typename F>
int by_shape(int dtype, int K, Access how, F&& f) {
#define TB_K(T, V, AL)                                                      \
  switch (K) {                                                              \
    case 1: return f.template operator()<T, 1, V, AL>();                    \
    case 2: return f.template operator()<T, 2, V, AL>();                    \
    case 3: return f.template operator()<T, 3, V, AL>();                    \
    case 4: return f.template operator()<T, 4, V, AL>();                    \
    case 5: return f.template operator()<T, 5, V, AL>();                    \
    case 6: return f.template operator()<T, 6, V, AL>();                    \
    case 7: return f.template operator()<T, 7, V, AL>();                    \
    default: return f.template operator()<T, 8, V, AL>();                   \
  }
#define TB_A(T, V)                          \
  {                                         \
    if (how == ALIGNED) TB_K(T, V, true)    \
    if (how == OFF) TB_K(T, V, false)       \
    TB_K(T, 1, true)                        \
  }
  if (dtype == TB_F32) TB_A(float, 4)
  if (dtype == TB_BF16) TB_A(__bf16, V16)
  TB_A(_Float16, V16)
#undef TB_A
#undef TB_K
}

struct FwdLaunch {
  ConvArgs a;
  dim3 grid, block;
  hipStream_t s;
  template <typename T, int K, int V, bool AL>
  int operator()() {
    conv_fwd<T, K, V, AL><<<grid, block, 0, s>>>(a);
    return 0;
  }
};
struct BwdLaunch {
  ConvArgs a;
  dim3 grid, block;
  hipStream_t s;
  template <typename T, int K, int V, bool AL>
  int operator()() {
    conv_bwd<T, K, V, AL><<<grid, block, 0, s>>>(a);
    return 0;
  }
};
struct StepLaunch {
  ConvStepArgs a;
  hipStream_t s;
  template <typename T, int K, int V, bool AL>
  int operator()() {
    const long n = (long)a.B * (a.D / V);
    if constexpr (AL) conv_step<T, K, V><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    return 0;
  }
};

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Plan {
  int vec, bx, by, run, runs;
  long gx, gy;
};

// Steps a run: enough runs to fill the chip (about 2^18 threads), but no fewer than 8 steps (each run reads K-1 steps of its
// neighbour's again) and no more than 64.
Plan plan(int B, int T, int D, int vec) {
  Plan p;
  p.vec = vec;
  const int groups = (D + vec - 1) / vec;
  p.bx = 64;
  while (p.bx > 1 && p.bx / 2 >= groups) p.bx /= 2;
  p.by = 256 / p.bx;
  const long want = ((long)B * T * groups) >> 18;
  p.run = (int)(want < 8 ? 8 : want > 64 ? 64 : want) / GRP * GRP;
  p.runs = (T + p.run - 1) / p.run;
  p.gx = (groups + p.bx - 1) / p.bx;
  p.gy = ((long)B * p.runs + p.by - 1) / p.by;
  return p;
}

int check_common(const char* what, int B, long T, int D, int K, int act, int dtype) {
  if (B < 0 || T < 0 || D < 1) return tb_set_error(TB_ERR_ARG, "%s: bad sizes B=%d T=%ld D=%d", what, B, T, D);
  if (T > TB_STEPS_MAX) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: too many steps in one call", what);
  if (K < 1 || K > KMAX) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: %d taps are not supported (1 to %d)", what, K, KMAX);
  if (act != 0 && act != TB_ACT_SILU) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: activation %d is not supported (none, silu)", what, act);
  if (!tb_dtype_ok(dtype)) return tb_set_error(TB_ERR_ARG, "%s: bad element type %d", what, dtype);
  return TB_OK;
}

bool can_vec(int dtype, int D, long sb, long st, const void* const* p, int n) {
  const int v = dtype == TB_F32 ? 4 : 8;
  if (D % v || sb % v || st % v) return false;
  for (int i = 0; i < n; ++i)
    if (!aligned(p[i])) return false;
  return true;
}

int check_grid(const char* what, const Plan& p) {
  if (!tb_grid_ok(p.gx * p.gy, 256)) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: too many steps in one call", what);
  return TB_OK;
}

}  // namespace

extern "C" {

int tb_conv_fwd(const void* x, long x_batch_stride, long x_step_stride, const void* w, const void* bias, int w_f32,
                const void* state, const int* lengths, void* y, void* state_out, int B, int T, int D, int K, int act, int dtype,
                void* stream) {
  int rc = check_common("conv_fwd", B, T, D, K, act, dtype);
  if (rc) return rc;
  if (B == 0 || (T == 0 && !state_out)) return TB_OK;
  if (!w || (T > 0 && (!x || !y))) return tb_set_error(TB_ERR_ARG, "conv_fwd: null pointer");
  const void* ptrs[] = {x, y, state, state_out, w, bias};
  const int v = dtype == TB_F32 ? 4 : 8;
  const Access how = can_vec(dtype, D, x_batch_stride, x_step_stride, ptrs, 6) ? ALIGNED : D >= v ? OFF : SINGLE;
  const Plan p = plan(B, T > 0 ? T : 1, D, how == SINGLE ? 1 : v);
  rc = check_grid("conv_fwd", p);
  if (rc) return rc;
  ConvArgs a{x, w, bias, state, nullptr, lengths, y, state_out, nullptr, nullptr, x_batch_stride, x_step_stride, B, T, D, p.run,
             p.runs, act, w_f32, (unsigned)p.gx};
  by_shape<8>(dtype, K, how, FwdLaunch{a, dim3((unsigned)(p.gx * p.gy)), dim3(p.bx, p.by), static_cast<hipStream_t>(stream)});
  TB_LAUNCH_CHECK("conv_fwd");
  return TB_OK;
}

size_t tb_conv_bwd_workspace_bytes(int B, int T, int D, int K, int dtype) {
  (void)dtype;
  if (B < 1 || T < 1 || D < 1 || K < 1) return 256;
  // the widest of the two layouts
  const Plan p = plan(B, T, D, 1), q = plan(B, T, D, 4);
  return tb_align_up((size_t)(p.gy > q.gy ? p.gy : q.gy) * (K + 1) * D * 4, 256);
}

int tb_conv_bwd(const void* dy, const void* x, long x_batch_stride, long x_step_stride, const void* w, const void* bias, int w_f32,
                const void* state, const int* lengths, void* dx, void* dw, void* db, int B, int T, int D, int K, int act, int dtype,
                void* ws, size_t ws_bytes, void* stream) {
  int rc = check_common("conv_bwd", B, T, D, K, act, dtype);
  if (rc) return rc;
  if (B < 1 || T < 1) return tb_set_error(TB_ERR_ARG, "conv_bwd: an empty batch has no gradients to form here");
  if (!dy || !x || !w || !dx || !ws) return tb_set_error(TB_ERR_ARG, "conv_bwd: null pointer");
  if (ws_bytes < tb_conv_bwd_workspace_bytes(B, T, D, K, dtype)) return tb_set_error(TB_ERR_WORKSPACE, "conv_bwd: workspace too small");
  const void* ptrs[] = {x, dy, dx, state, w, bias};
  const Access how = can_vec(dtype, D, x_batch_stride, x_step_stride, ptrs, 6) ? ALIGNED : D >= 4 ? OFF : SINGLE;
  const Plan p = plan(B, T, D, how == SINGLE ? 1 : 4);
  rc = check_grid("conv_bwd", p);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  ConvArgs a{x, w, bias, state, dy, lengths, nullptr, nullptr, dx, static_cast<float*>(ws), x_batch_stride, x_step_stride, B, T, D,
             p.run, p.runs, act, w_f32, (unsigned)p.gx};
  by_shape<4>(dtype, K, how, BwdLaunch{a, dim3((unsigned)(p.gx * p.gy)), dim3(p.bx, p.by), s});
  TB_LAUNCH_CHECK("conv_bwd");
  if (dw || db) {
    const long cols = (long)(K + 1) * D;
    const dim3 grid((unsigned)((cols + 63) / 64)), block(64, 16);
    const float* slab = static_cast<const float*>(ws);
    if (dtype == TB_F32) conv_finish<float><<<grid, block, 0, s>>>(slab, p.gy, K, D, dw, db, w_f32);
    else if (dtype == TB_BF16) conv_finish<__bf16><<<grid, block, 0, s>>>(slab, p.gy, K, D, dw, db, w_f32);
    else conv_finish<_Float16><<<grid, block, 0, s>>>(slab, p.gy, K, D, dw, db, w_f32);
    TB_LAUNCH_CHECK("conv_finish");
  }
  return TB_OK;
}

int tb_conv_step(const void* x, long x_batch_stride, void* state, long state_batch_stride, const void* w, const void* bias, int w_f32,
                 void* y, int B, int D, int K, int act, int dtype, void* stream) {
  int rc = check_common("conv_step", B, 1, D, K, act, dtype);
  if (rc) return rc;
  if (B == 0) return TB_OK;
  if (!x || !w || !y || (K > 1 && !state)) return tb_set_error(TB_ERR_ARG, "conv_step: null pointer");
  const void* ptrs[] = {x, y, state, w, bias};
  const bool vec = can_vec(dtype, D, x_batch_stride, state_batch_stride, ptrs, 5);
  if (!tb_grid_ok(((long)B * (vec ? D / (dtype == TB_F32 ? 4 : 8) : D) + 255) / 256, 256))
    return tb_set_error(TB_ERR_UNSUPPORTED, "conv_step: too many rows in one call");
  ConvStepArgs a{x, w, bias, state, y, x_batch_stride, state_batch_stride, B, D, act, w_f32};
  by_shape<8>(dtype, K, vec ? ALIGNED : SINGLE, StepLaunch{a, static_cast<hipStream_t>(stream)});
  TB_LAUNCH_CHECK("conv_step");
  return TB_OK;
}

}  // extern "C"

// Selective state space scan over (B, T, D) with N states a channel: prompts, gradients, one step.
//
//   delta = softplus(dt + bias)   (or dt + bias)          per step and channel
//   h_t   = exp(delta A) h_{t-1} + delta u B_t            per state; A (D, N), B_t / C_t (N) shared by the channels of a group
//   y     = C_t . h_t + D u,   out = y silu(z)
// Backward, with dy = dout silu(z):
//   g_t = C_t dy_t + a_{t+1} g_{t+1},  q = g_t a_t h_{t-1}
//   ddelta = sum_n q A + u sum_n g B,  du = delta sum_n g B + D dy,  dA = sum q delta,  dB_t = sum_c g delta u,
//   dC_t = sum_c dy h,  dD = sum dy u,  dz = dout y silu'(z),  ddt = ddelta sigmoid(dt + bias)
//
// Bound by arithmetic: an exponential (a quarter of the vector rate) and four other operations a state and step forward, as many again and
// nine more backward, against two bytes an element and tensor; where the steps are cut, the first walk comes on top.  Measured, bf16,
// 16 states, gated: 1 x 16384 x 2048 271 us (537 M state steps; the exponentials and operations of both walks alone are 205 at
// the vector units' full rate); 4 x 2048 x 2048 with gradients 468 (vector units busy 80 % of the main backward pass, 88 to 92 % of the
// others).  Layout: a lane owns one channel and S = N/4 of
// its states, four neighbouring lanes a channel, so that the sum over the states is two quad permutes and a block of four
// waves owns 64 neighbouring channels (whole lines of every tensor).  Steps go in tiles: a tile's rows are fetched into
// registers one tile ahead, what does not depend on the state (softplus, the gate's derivative) is computed once per element
// by all lanes and left in LDS in fp32, then each wave walks the tile's steps with its states in registers.
// Where the batch has too few channel blocks for the chip, the steps are cut into chunks: a first pass finds each chunk's own
// end state from zero and the sum of its delta, and the main pass starts every chunk from its true state, which it finds by chaining
// those of the chunks before it (exp(A sum delta) is a chunk's decay).
// States, sums and gradients of parameters are fp32; every output is rounded once.  No atomics: partial sums are added in a
// fixed order.
#include "elem.h"

namespace {

constexpr int CB = 64;          // channels a block
constexpr int YS = CB + 16;     // row length of what four lanes store for four rows at once: they fall on different banks
constexpr int NMAX = 64;
constexpr float LOG2E = 1.4426950408889634f;

// steps a tile of the backward pass.  The states of a tile stay in registers, BWD * S of them, and up to S = 4 as many decays (computed
// again on the way back, with three waves a SIMD instead of two: 16 x 1024 x 2048 bf16 818 us, so 721, and 690 with the
// next tile fetched ahead; beyond, they cost more than they save).  A state is kept in memory every BWD steps.  Backward alone, us, 16 x 1024 x 1024: 32 states in tiles of 16 steps
// bf16 629, fp32 652 (spills), of 8 steps 546, 557, of 8 with the decays kept 597, 671; 8 states fp32 of 32 steps 261, of 16 254.
constexpr int bwd_tile(int S) { return S <= 1 ? 32 : S <= 4 ? 16 : 8; }
template <int S>
struct Tile {
  static constexpr int BWD = bwd_tile(S);
};

struct ScanArgs {
  const void *u, *dt, *z, *Bm, *Cm, *dout;
  const float *A, *Dp, *bias, *h0, *dhT;
  const int* lengths;
  void *out, *du, *ddt, *dz;
  float *hT, *dh0;
  float* ck;               // states at the start of every backward tile: [B][tiles][D][4 S]
  float* cstate;           // chunks: [B][chunks][D][4 S]
  float* csum;             // chunks: [B][chunks][D]
  float* bc;               // backward: [B][G][cblk][T][2][4 S] sums over a block's channels of dB and dC
  float* par;              // backward: [B][chunks][D][4 S + 2] sums over a chunk's steps of dA, dD, dbias
  long sub, sut, sdb, sdt, szb, szt, sob, sot, sBb, sBt, sBg, sCb, sCt, sCg;
  int B, T, D, N, G, Dg;   // Dg channels a group
  int cblk;                // blocks of 64 channels a group
  int chunk, chunks;       // steps a chunk (a multiple of 32), chunks
  int ckt, cktiles;        // steps between kept states (0: none)
  int softplus, vec;
};

// log(1 + e^x).  With w = 1 + e rounded, log(w) e / (w - 1) repairs what the rounding of w lost (w - 1 is exact);
// above 20 the result is x to fp32.
__device__ __forceinline__ float softplus(float x) {
  const float e = tb_exp(x), w = 1.f + e, m = w - 1.f;
  const float l = __builtin_amdgcn_logf(w) * (e / LOG2E) * __builtin_amdgcn_rcpf(m);      // the hardware's log is of base 2
  return x > 20.f ? x : m > 0.f ? l : e;
}

// v or 0, by a mask of all its bits: no branch around what makes v
__device__ __forceinline__ float only(float v, unsigned mask) { return __uint_as_float(__float_as_uint(v) & mask); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += dpp<0xB1>(v);       // lanes 1 0 3 2
  return v + dpp<0x4E>(v); // lanes 2 3 0 1
}

// EPT neighbouring channels of a row as they lie in memory.  The address is always one of the tensor's (the caller clamps the
// row; channels behind the group's last read another), so that nothing branches and all of a tile's loads are under way at
// once: converted and masked as each arrived, they were waited for one after the other.
// VEC: every thread's channels lie on the access' alignment and are all of the group or none; otherwise accesses of the same
// width off it (5 x 1021 x 260 fp32: 25 us, element by element 32), but for the group's last, incomplete thread.
template <int W, int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) Words {
  unsigned v[W];
};
template <typename T, int EPT, bool VEC>
struct Raw {
  static constexpr int WORDS = EPT * sizeof(T) / 4, W = WORDS < 4 ? WORDS : 4;
  typedef Words<W, VEC ? W * 4 : (int)sizeof(T)> Access;
  unsigned v[WORDS];
  __device__ __forceinline__ void fetch(const void* base, long off, int c0, int Dg) {
    const T* p = static_cast<const T*>(base) + off;
    if (VEC || c0 + EPT <= Dg) {
      const unsigned* q = reinterpret_cast<const unsigned*>(p + (VEC && c0 >= Dg ? 0 : c0));
#pragma unroll
      for (int i = 0; i < WORDS; i += W) *reinterpret_cast<TbVec<unsigned, W>*>(v + i) = __builtin_bit_cast(TbVec<unsigned, W>, *reinterpret_cast<const Access*>(q + i));
    } else {
      unsigned e[EPT];
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const T t = p[min(c0 + i, Dg - 1)];
        if constexpr (sizeof(T) == 4) e[i] = __builtin_bit_cast(unsigned, t);
        else e[i] = __builtin_bit_cast(unsigned short, t);
        e[i] = c0 + i < Dg ? e[i] : 0u;
      }
#pragma unroll
      for (int i = 0; i < WORDS; ++i) v[i] = sizeof(T) == 4 ? e[i] : e[i * (4 / sizeof(T))] | e[(i * (4 / sizeof(T)) + 1) % EPT] << 16;
    }
  }
  // rows that do not count, and threads without channels
  __device__ __forceinline__ void mask(bool on, int c0, int Dg, float fill) {
    const bool in = on && c0 < Dg;
    const T f = (T)fill;
    unsigned w;
    if constexpr (sizeof(T) == 4) w = __builtin_bit_cast(unsigned, f);
    else w = __builtin_bit_cast(unsigned short, f) * 0x10001u;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) v[i] = in ? v[i] : w;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, v[i]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(v[i / 2] >> (i & 1) * 16));
  }
};
template <typename T, int EPT, bool VEC>
__device__ __forceinline__ void put(void* base, long off, int c0, int Dg, const float (&r)[EPT]) {
  T* p = static_cast<T*>(base) + off;
  if constexpr (VEC) {
    if (c0 < Dg) tb_store_n(p + c0, r);
  } else if (c0 + EPT <= Dg) {
    tb_store_u(p + c0, r);
  } else {
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (c0 + i < Dg) p[c0 + i] = (T)r[i];
  }
}

struct Where {
  int b, g, cb, chunk, c0, d0, len;   // c0: the block's first channel of its group, d0: of all
};
__device__ __forceinline__ Where where(const ScanArgs& a, int chunks) {
  Where w;
  int id = blockIdx.x;
  w.cb = id % a.cblk; id /= a.cblk;
  w.g = id % a.G; id /= a.G;
  w.chunk = id % chunks;
  w.b = id / chunks;
  w.c0 = w.cb * CB;
  w.d0 = w.g * a.Dg + w.c0;
  w.len = a.lengths ? min(max(a.lengths[w.b], 0), a.T) : a.T;
  return w;
}

// S states of channel d: [d][N] of the caller (count: N), zero behind N
template <int S>
__device__ __forceinline__ void load_state(const float* p, long row, int n0, int N, bool on, float (&h)[S]) {
#pragma unroll
  for (int s = 0; s < S; ++s) h[s] = on && p && n0 + s < N ? p[row * N + n0 + s] : 0.f;
}
template <int S>
__device__ __forceinline__ void store_state(float* p, long row, int n0, int N, bool on, const float (&h)[S]) {
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (on && n0 + s < N) p[row * N + n0 + s] = h[s];
}
// S floats of a row of 4 S
template <int S>
__device__ __forceinline__ void load_row(const float* p, float (&v)[S]) { tb_load_n(p, v); }
template <int S>
__device__ __forceinline__ void store_row(float* p, const float (&v)[S]) { tb_store_n(p, v); }

// rows of B or C of a tile on their way into LDS as fp32, [TT][4 S], zero behind N and where the step is off
template <typename T, int S, int TT>
struct RawRows {
  static constexpr int NP = 4 * S, COUNT = (TT * NP + 255) / 256;
  T v[COUNT];
  __device__ __forceinline__ void fetch(const void* base, long off, long st, int t0, int t1, int N) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int i = threadIdx.x + j * 256, t = max(min(t0 + i / NP, t1 - 1), 0), n = min(i % NP, N - 1);
      v[j] = static_cast<const T*>(base)[off + (long)t * st + n];
    }
  }
  __device__ __forceinline__ void store(float* lds, int t0, int t1, int N) const {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int i = threadIdx.x + j * 256;
      if (TT * NP % 256 == 0 || i < TT * NP) lds[i] = t0 + i / NP < t1 && i % NP < N ? (float)v[j] : 0.f;
    }
  }
};

// the sums over the four lanes of a quad of four steps' values: lane l of the quad gets step l's.  Each exchange adds what is
// left of two values in one instruction behind two selects: nine instructions instead of sixteen and one store instead of four.
__device__ __forceinline__ float quad_sum4(const float (&y)[4], int lane) {
  const bool o = lane & 1, h = lane & 2;
  const float a = (o ? y[1] : y[0]) + dpp<0xB1>(o ? y[0] : y[1]);
  const float b = (o ? y[3] : y[2]) + dpp<0xB1>(o ? y[2] : y[3]);
  return (h ? b : a) + dpp<0x4E>(h ? a : b);
}

// The state that a chunk starts from: the chunks before it (REV: behind it), each with its own end state from zero and the sum of
// its delta, chained from the first (REV: last) one on.  Eight are fetched together: only the products wait for each other.
// A chunk's decay can pass fp32's range where no step's does (a state that grows, or decays from infinity): what does not come out finite
// is chained again with the decay in two factors, and with 0 and infinity kept, as the steps would keep them.
template <int S, bool REV>
__device__ __forceinline__ void chain(const ScanArgs& a, int b, int chunk, long rd, int n0, const float (&A2)[S], float (&h)[S]) {
  constexpr int NP = 4 * S;
  const int count = REV ? a.chunks - 1 - chunk : chunk;
  float first[S];
#pragma unroll
  for (int s = 0; s < S; ++s) first[s] = h[s];
  for (int i = 0; i < count; i += 8) {
    float own[8][S], sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = min(i + j, count - 1);
      const long row = ((long)b * a.chunks + (REV ? a.chunks - 1 - k : k)) * a.D + rd;
      load_row<S>(a.cstate + row * NP + n0, own[j]);
      sum[j] = a.csum[row];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < count)
#pragma unroll
        for (int s = 0; s < S; ++s) h[s] = fmaf(__builtin_amdgcn_exp2f(A2[s] * sum[j]), h[s], own[j][s]);
  }
  bool fine = true;
#pragma unroll
  for (int s = 0; s < S; ++s) fine = fine && fabsf(h[s]) < INFINITY;
  if (__builtin_expect(fine, 1)) return;
#pragma unroll
  for (int s = 0; s < S; ++s) h[s] = first[s];
  for (int k = 0; k < count; ++k) {
    float own[S];
    const long row = ((long)b * a.chunks + (REV ? a.chunks - 1 - k : k)) * a.D + rd;
    load_row<S>(a.cstate + row * NP + n0, own);
    const float sum = a.csum[row];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const float x = A2[s] * sum, e = __builtin_amdgcn_exp2f(x * 0.5f);
      const bool kept = (h[s] == 0.f || fabsf(h[s]) == INFINITY) && fabsf(x) < INFINITY;
      h[s] = (kept ? h[s] : h[s] * e * e) + own[s];
    }
  }
}

// forward.  STATE: only the chunk's end state from zero and its sum of delta (first pass over chunks).
// fp32 is held to four waves a SIMD (4 x 2048 x 2048 x 16 146 us, with three 158); 16-bit types reach them, and are slower held to it
// (1 x 16384 x 2048 x 16 bf16 277 us, 271).
// PART: N is not 4 S, and the states behind it are kept at 0: their products are 0 times what may be infinite.  Kernels of their own, so that
// whole states take no selects (4 x 2048 x 2048 x 11 fp32: forward 144 us without them, 150 with; gradients too 491, 506).
template <typename T, int S, bool STATE, bool VEC, bool PART>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && VEC && S <= 4 ? 4 : 1) scan_fwd(ScanArgs a) {
  constexpr int TT = 32, EPT = 8, NP = 4 * S;
  __shared__ float sD[TT][CB][2];            // delta, delta u
  __shared__ float sB[TT * NP], sC[STATE ? 1 : TT * NP];
  __shared__ float sY[STATE ? 1 : TT][YS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Where w = where(a, STATE ? a.chunks - 1 : a.chunks);
  // the coop part: one step, eight channels a thread
  const int ct = tid / (CB / EPT), cc = (tid % (CB / EPT)) * EPT;
  // the recurrence: channel rc of the block, states n0 .. n0 + S
  const int rc = wave * 16 + (lane >> 2), n0 = (lane & 3) * S;
  const bool ron = w.c0 + rc < a.Dg;
  const long rd = w.d0 + rc;
  const int ts = w.chunk * a.chunk, te = min(ts + a.chunk, a.T);
  const int tv = min(te, w.len);              // steps that count end here

  float A2[S], h[S];
  load_state<S>(a.A, rd, n0, a.N, ron, A2);
#pragma unroll
  for (int s = 0; s < S; ++s) A2[s] *= LOG2E;
  if (STATE) {
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = 0.f;
  } else {
    load_state<S>(a.h0, (long)w.b * a.D + rd, n0, a.N, ron, h);
    if (ron) chain<S, false>(a, w.b, w.chunk, rd, n0, A2, h);
  }
  float bias[EPT], Dp[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const bool on = w.c0 + cc + i < a.Dg;
    bias[i] = on && a.bias ? a.bias[w.d0 + cc + i] : 0.f;
    Dp[i] = !STATE && on && a.Dp ? a.Dp[w.d0 + cc + i] : 0.f;
  }
  const long uo = (long)w.b * a.sub + (long)w.g * a.Dg, dof = (long)w.b * a.sdb + (long)w.g * a.Dg,
             zo = (long)w.b * a.szb + (long)w.g * a.Dg, oo = (long)w.b * a.T * a.D + (long)w.g * a.Dg;
  const long bo = (long)w.b * a.sBb + (long)w.g * a.sBg, co = (long)w.b * a.sCb + (long)w.g * a.sCg;
  const int ch = w.c0 + cc;
  float sum = 0.f;
  Raw<T, EPT, VEC> ru, rd_, rz;
  RawRows<T, S, TT> rB, rC;
  auto load = [&](int t0) {
    const int t = max(min(t0 + ct, tv - 1), 0);
    ru.fetch(a.u, uo + (long)t * a.sut, ch, a.Dg);
    rd_.fetch(a.dt, dof + (long)t * a.sdt, ch, a.Dg);
    if (!STATE && a.z) rz.fetch(a.z, zo + (long)t * a.szt, ch, a.Dg);
    rB.fetch(a.Bm, bo, a.sBt, t0, tv, a.N);
    if (!STATE) rC.fetch(a.Cm, co, a.sCt, t0, tv, a.N);
  };
  const unsigned skip = a.Dp ? ~0u : 0u;
  load(ts);
  for (int t0 = ts; t0 < te; t0 += TT) {
    const int t = t0 + ct;
    const bool on = t < tv;
    float u[EPT], z[EPT];
    // a step that does not count leaves the state as it is: its delta is softplus(-inf) = 0
    ru.mask(on, ch, a.Dg, 0.f);
    if (!STATE && a.z) rz.mask(on, ch, a.Dg, 0.f);
    rd_.mask(on, ch, a.Dg, a.softplus ? -INFINITY : 0.f);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      u[i] = ru.get(i);
      if (!STATE && a.z) z[i] = rz.get(i);
      float d = rd_.get(i) + bias[i];
      if (a.softplus) d = softplus(d);
      else d = on ? d : 0.f;
      sD[ct][cc + i][0] = d;
      sD[ct][cc + i][1] = d * u[i];
      if (!STATE) u[i] = only(u[i], skip);       // no skip term: 0 times u is none where u is infinite
    }
    rB.store(sB, t0, tv, a.N);
    if (!STATE) rC.store(sC, t0, tv, a.N);
    __syncthreads();
    if (t0 + TT < te) load(t0 + TT);           // under way over the walk
    if (!STATE && a.ckt && ron) store_row<S>(a.ck + (((long)w.b * a.cktiles + t0 / a.ckt) * a.D + rd) * NP + n0, h);
#pragma unroll 1
    for (int k = 0; k < TT; k += 4) {
      if (!STATE && Tile<S>::BWD < TT) {       // a backward tile is shorter than this one: its start lies inside
        if (k && a.ckt && k % Tile<S>::BWD == 0 && ron && t0 + k < a.T)
          store_row<S>(a.ck + (((long)w.b * a.cktiles + (t0 + k) / a.ckt) * a.D + rd) * NP + n0, h);
      }
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = sD[k + j][rc][0], x = sD[k + j][rc][1];
        float bv[S], cv[S];
        load_row<S>(sB + (k + j) * NP + n0, bv);
        if (!STATE) load_row<S>(sC + (k + j) * NP + n0, cv);
        y[j] = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float e = __builtin_amdgcn_exp2f(d * A2[s]);
          h[s] = fmaf(e, h[s], x * bv[s]);
          if (PART) h[s] = n0 + s < a.N ? h[s] : 0.f;
          if (!STATE) y[j] = fmaf(h[s], cv[s], y[j]);
        }
        if (STATE) sum += d;
      }
      if (!STATE) sY[k + (lane & 3)][rc] = quad_sum4(y, lane);
    }
    __syncthreads();
    if (!STATE && t < te) {
      float o[EPT];
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        float y = fmaf(Dp[i], u[i], sY[ct][cc + i]);
        if (a.z) y *= tb_silu(z[i]);
        o[i] = on ? y : 0.f;
      }
      put<T, EPT, VEC>(a.out, oo + (long)t * a.D, ch, a.Dg, o);
    }
  }
  if (STATE) {
    const long row = ((long)w.b * a.chunks + w.chunk) * a.D + rd;
    if (ron) store_row<S>(a.cstate + row * NP + n0, h);
    if (ron && (lane & 3) == 0) a.csum[row] = sum;
  } else if (a.hT && w.chunk == a.chunks - 1) {
    store_state<S>(a.hT, (long)w.b * a.D + rd, n0, a.N, ron, h);
  }
}

// v[0..2S) of the wave's sixteen channels (lane bits 2..5) summed: halves are exchanged so that each step adds what is left,
// and every lane ends with S/2 sums (S = 1: one), of v[0..S) in the lower half of the wave and of v[S..2S) in the upper; bit 4 says
// which half of the S, bits 2 and 3 nothing.
template <int S>
__device__ __forceinline__ void channel_sum(float (&v)[2 * S]) {
#pragma unroll
  for (int i = 0; i < S; ++i) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + S]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  constexpr int H = S > 1 ? S / 2 : 1;
#pragma unroll
  for (int i = 0; i < H; ++i) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[S > 1 ? i + H : i]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#pragma unroll
  for (int i = 0; i < H; ++i) {
    v[i] += dpp<0x128>(v[i]);     // rotate the row of sixteen by eight
    v[i] += dpp<0x124>(v[i]);     // and by four
  }
}

// what a lane needs of a step: delta, delta u, dy, and its states' B and C
template <int S>
struct Row {
  float d, x, y, b[S], c[S];
  __device__ __forceinline__ void load(const float* dx, float dy, const float* B, const float* C) {
    d = dx[0];
    x = dx[1];
    y = dy;
    load_row<S>(B, b);
    load_row<S>(C, c);
  }
};

// backward.  STATE: only g in front of the chunk's first step from zero behind its last, and its sum of delta.
template <typename T, int S, bool STATE, bool VEC, bool PART>
__global__ void __launch_bounds__(256, STATE ? 4 : 2) scan_bwd(ScanArgs a) {
  constexpr int TT = STATE ? 32 : Tile<S>::BWD, EPT = TT / 4, NP = 4 * S;
  // The next tile's rows are fetched before the walk, and this one's kept over it, where that spills no registers: 16 x 1024 x 2048
  // of 16 states fp16 532 us (fetched at the tile's start, and again behind the walk), so 500; 16 x 1000 x 1023 of 8 states bf16 343,
  // so 295; 16 states fp32 344, with it 354; 64 states fp32 512, with it 570.
  constexpr bool AHEAD = S < 16 && !(S == 4 && sizeof(T) == 4);
  __shared__ float sD[TT][CB][2], sG[TT][CB];           // delta, delta u; dy
  __shared__ float sB[STATE ? 1 : TT * NP], sC[TT * NP];
  __shared__ float sY[STATE ? 1 : TT][YS], sGB[STATE ? 1 : TT][YS], sGA[STATE ? 1 : TT][YS];
  __shared__ float sP[STATE ? 1 : 4][STATE ? 1 : TT][2 * NP];
  __shared__ float sPar[2][CB];                         // dt_bias, D
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Where w = where(a, STATE ? a.chunks - 1 : a.chunks);
  if (STATE) ++w.chunk;
  const int ct = tid / (CB / EPT), cc = (tid % (CB / EPT)) * EPT;
  const int rc = wave * 16 + (lane >> 2), n0 = (lane & 3) * S;
  const bool ron = w.c0 + rc < a.Dg;
  const long rd = w.d0 + rc;
  const int ts = w.chunk * a.chunk, te = min(ts + a.chunk, a.T), tv = min(te, w.len);

  if (tid < 2 * CB) {
    const float* p = tid < CB ? a.bias : a.Dp;
    sPar[tid / CB][tid % CB] = p && w.c0 + tid % CB < a.Dg ? p[w.d0 + tid % CB] : 0.f;
  }
  float A2[S], g[S], dA[S];
  load_state<S>(a.A, rd, n0, a.N, ron, A2);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    A2[s] = PART && n0 + s >= a.N ? -1.f : A2[s] * LOG2E;      // behind N: an infinite delta decays to 0 (0 times it is NaN)
    dA[s] = 0.f;
    g[s] = 0.f;
  }
  if (!STATE) {
    load_state<S>(a.dhT, (long)w.b * a.D + rd, n0, a.N, ron, g);
    if (ron) chain<S, true>(a, w.b, w.chunk, rd, n0, A2, g);
  }
  float dD[EPT], dbias[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) dD[i] = dbias[i] = 0.f;
  const long gof = (long)w.g * a.Dg;
  const long uo = (long)w.b * a.sub + gof, dof = (long)w.b * a.sdb + gof, zo = (long)w.b * a.szb + gof,
             go = (long)w.b * a.sob + gof, oo = (long)w.b * a.T * a.D + gof;
  const long bo = (long)w.b * a.sBb + (long)w.g * a.sBg, co = (long)w.b * a.sCb + (long)w.g * a.sCg;
  const int ch = w.c0 + cc;
  const unsigned skip = a.Dp ? ~0u : 0u;        // no skip term: 0 times u or dy is none where they are infinite
  float sum = 0.f;
  __syncthreads();

  struct {
    Raw<T, EPT, VEC> u, dt, z, dout;
    RawRows<T, S, TT> B, C;
  } next;
  auto fetch = [&](int t0, auto& r) {
    const int tc = max(min(t0 + ct, tv - 1), 0);
    if (!STATE) r.u.fetch(a.u, uo + (long)tc * a.sut, ch, a.Dg);
    r.dt.fetch(a.dt, dof + (long)tc * a.sdt, ch, a.Dg);
    r.dout.fetch(a.dout, go + (long)tc * a.sot, ch, a.Dg);
    if (a.z) r.z.fetch(a.z, zo + (long)tc * a.szt, ch, a.Dg);
    if (!STATE) r.B.fetch(a.Bm, bo, a.sBt, t0, tv, a.N);
    r.C.fetch(a.Cm, co, a.sCt, t0, tv, a.N);
  };
  for (int t0 = ts + (te - ts - 1) / TT * TT; t0 >= ts; t0 -= TT) {
    const int t = t0 + ct, tc = max(min(t, tv - 1), 0);
    const bool on = t < tv;
    // what the tile's elements give by themselves
    Raw<T, EPT, VEC> ru, rdt, rz, ro;
    {
      RawRows<T, S, TT> rB, rC;
      if (!AHEAD || t0 + TT >= te) fetch(t0, next);
      ru = next.u;
      rdt = next.dt;
      rz = next.z;
      ro = next.dout;
      rB = next.B;
      rC = next.C;
      if (!STATE) ru.mask(on, ch, a.Dg, 0.f);
      rdt.mask(on, ch, a.Dg, a.softplus ? -INFINITY : 0.f);
      ro.mask(on, ch, a.Dg, 0.f);
      if (a.z) rz.mask(on, ch, a.Dg, 0.f);
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        float d = rdt.get(i) + sPar[0][cc + i];
        if (a.softplus) d = softplus(d);
        else d = on ? d : 0.f;
        sD[ct][cc + i][0] = d;
        if (!STATE) sD[ct][cc + i][1] = d * ru.get(i);
        sG[ct][cc + i] = a.z ? ro.get(i) * tb_silu(rz.get(i)) : ro.get(i);
      }
      if (!STATE) rB.store(sB, t0, tv, a.N);
      rC.store(sC, t0, tv, a.N);
    }
    if (AHEAD && t0 > ts) fetch(t0 - TT, next);
    __syncthreads();
    if (STATE) {
#pragma unroll 4
      for (int k = TT - 1; k >= 0; --k) {
        const float d = sD[k][rc][0], y = sG[k][rc];
        float cv[S];
        load_row<S>(sC + k * NP + n0, cv);
        sum += d;
#pragma unroll
        for (int s = 0; s < S; ++s) g[s] = fmaf(cv[s], y, g[s]) * __builtin_amdgcn_exp2f(d * A2[s]);
      }
    } else {
      constexpr bool KEEP = S <= 4;      // each step's decay, too, where registers allow
      const int last = tv - 1 - t0;
      float ea[KEEP ? TT : 1][S];
      float h[TT + 1][S];      // h[k]: the state in front of step k
      if (ron) load_row<S>(a.ck + (((long)w.b * a.cktiles + t0 / TT) * a.D + rd) * NP + n0, h[0]);
      else
#pragma unroll
        for (int s = 0; s < S; ++s) h[0][s] = 0.f;
      if constexpr (PART)
#pragma unroll
        for (int s = 0; s < S; ++s) h[0][s] = n0 + s < a.N ? h[0][s] : 0.f;
      // one step ahead of the arithmetic, and no further: left alone, the compiler keeps all of a tile's rows in registers
      Row<S> r;
      r.load(sD[0][rc], sG[0][rc], sB + n0, sC + n0);
      float q4[4], p4[4];
#pragma unroll
      for (int k = 0; k < TT; ++k) {
        const Row<S> c = r;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (k + 1 < TT) r.load(sD[k + 1][rc], sG[k + 1][rc], sB + (k + 1) * NP + n0, sC + (k + 1) * NP + n0);
        float y = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float e = __builtin_amdgcn_exp2f(c.d * A2[s]);
          if constexpr (KEEP) ea[k][s] = e;
          h[k + 1][s] = fmaf(e, h[k][s], c.x * c.b[s]);
          if constexpr (PART) {
            h[k + 1][s] = n0 + s < a.N ? h[k + 1][s] : 0.f;
            asm volatile("" : "+v"(h[k + 1][s]));          // one value: left alone, the one before the select is kept beside it
          }
          y = fmaf(h[k + 1][s], c.c[s], y);
        }
        asm volatile("" : "+v"(y));
        q4[k & 3] = y;
        if ((k & 3) == 3) sY[k - 3 + (lane & 3)][rc] = quad_sum4(q4, lane);
      }
#pragma unroll
      for (int k = TT - 1; k >= 0; --k) {
        const Row<S> c = r;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (k > 0) r.load(sD[k - 1][rc], sG[k - 1][rc], sB + (k - 1) * NP + n0, sC + (k - 1) * NP + n0);
        float v[2 * S], gB = 0.f, gA = 0.f;
        // the sequence's last step: what the steps behind it added is 0 times the state that they kept, NaN where that is infinite
        if (__builtin_expect(k == last, 0)) {
#pragma unroll
          for (int s = 0; s < S; ++s) {
            dA[s] = 0.f;
            asm volatile("" : "+v"(dA[s]));          // a branch, not a select a step
          }
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
          g[s] = fmaf(c.c[s], c.y, g[s]);
          if constexpr (PART) g[s] = n0 + s < a.N ? g[s] : 0.f;
          v[s] = g[s] * c.x;                       // dB
          v[S + s] = h[k + 1][s] * c.y;            // dC
          gB = fmaf(g[s], c.b[s], gB);
          if constexpr (KEEP) g[s] *= ea[k][s];
          else g[s] *= __builtin_amdgcn_exp2f(c.d * A2[s]);
          float q = g[s] * h[k][s];          // behind N 0: neither factor is infinite there
          if constexpr (PART && S == 16) q = n0 + s < a.N ? q : 0.f;      // for the registers alone (4 x 2048 x 1024 x 40 bf16 1331 us, without 1500)
          gA = fmaf(q, A2[s], gA);                 // of A log2 e: divided out of the sum
          dA[s] = fmaf(q, c.d, dA[s]);
          asm volatile("" : "+v"(g[s]), "+v"(dA[s]));      // here and now: put off, their operands stay in registers
        }
        asm volatile("" : "+v"(gB), "+v"(gA));
        q4[k & 3] = gB;
        p4[k & 3] = gA;
        if ((k & 3) == 0) {
          sGB[k + (lane & 3)][rc] = quad_sum4(q4, lane);
          sGA[k + (lane & 3)][rc] = quad_sum4(p4, lane);
        }
        channel_sum<S>(v);
        constexpr int H = S > 1 ? S / 2 : 1;
        // Lanes that differ in bits 2 and 3 hold and store the same: selecting one of them costs a branch a step (16 x 1024 x 2048
        // bf16 with gradients 861 us, without 813), which pays only where a lane stores many sums (64 states: 202 us, without 227).
        if (S <= 8 || (lane & 12) == 0) {
          float* p = &sP[wave][k][(lane >> 5) * NP + n0 + (S > 1 && (lane & 16) ? H : 0)];
#pragma unroll
          for (int i = 0; i < H; ++i) p[i] = v[i];
        }
      }
      // again, from the caches, where they would take the registers of the walk's states
      if (!AHEAD) {
        ru.fetch(a.u, uo + (long)tc * a.sut, ch, a.Dg);
        rdt.fetch(a.dt, dof + (long)tc * a.sdt, ch, a.Dg);
        if (a.dz) {
          ro.fetch(a.dout, go + (long)tc * a.sot, ch, a.Dg);
          rz.fetch(a.z, zo + (long)tc * a.szt, ch, a.Dg);
        }
      }
    }
    __syncthreads();
    if (!STATE) {
      for (int i = tid; i < TT * 2 * NP; i += 256) {
        const int k = i / (2 * NP), n = i % (2 * NP);
        if (t0 + k < te)
          a.bc[((((long)w.b * a.G + w.g) * a.cblk + w.cb) * a.T + t0 + k) * (2 * NP) + n] =
              t0 + k < tv ? (sP[0][k][n] + sP[1][k][n]) + (sP[2][k][n] + sP[3][k][n]) : 0.f;
      }
      if (t < te) {
        float o[EPT], u[EPT];
        // dy, delta and what the walk left are 0 where a step does not count
        ru.mask(on, ch, a.Dg, 0.f);
        rdt.mask(on, ch, a.Dg, a.softplus ? -INFINITY : 0.f);
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          u[i] = ru.get(i);
          o[i] = fmaf(u[i], sGB[ct][cc + i], sGA[ct][cc + i] * (1.f / LOG2E));
          if (a.softplus) o[i] *= tb_sig(rdt.get(i) + sPar[0][cc + i]);      // d delta / d raw
          o[i] = on ? o[i] : 0.f;
          dbias[i] += o[i];
        }
        if (a.ddt) put<T, EPT, VEC>(a.ddt, oo + (long)t * a.D, ch, a.Dg, o);
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          const float dy = sG[ct][cc + i];
          o[i] = on ? fmaf(sD[ct][cc + i][0], sGB[ct][cc + i], only(sPar[1][cc + i] * dy, skip)) : 0.f;
          dD[i] = fmaf(dy, u[i], dD[i]);
        }
        if (a.du) put<T, EPT, VEC>(a.du, oo + (long)t * a.D, ch, a.Dg, o);
        if (a.dz) {
          ro.mask(on, ch, a.Dg, 0.f);
          rz.mask(on, ch, a.Dg, 0.f);
#pragma unroll
          for (int i = 0; i < EPT; ++i) {
            const float z = rz.get(i), q = tb_sig(z), y = fmaf(sPar[1][cc + i], only(u[i], skip), sY[ct][cc + i]);
            o[i] = on ? ro.get(i) * y * (q * (1.f + z * (1.f - q))) : 0.f;
          }
          put<T, EPT, VEC>(a.dz, oo + (long)t * a.D, ch, a.Dg, o);
        }
      }
      __syncthreads();
    }
  }
  const long row = ((long)w.b * a.chunks + w.chunk) * a.D + rd;
  if (STATE) {
    if (ron) store_row<S>(a.cstate + row * NP + n0, g);
    if (ron && (lane & 3) == 0) a.csum[row] = sum;
    return;
  }
  if (ron) {
#pragma unroll
    for (int s = 0; s < S; ++s) a.par[row * (NP + 2) + n0 + s] = tv > ts ? dA[s] : 0.f;
  }
  if (a.dh0 && w.chunk == 0) store_state<S>(a.dh0, (long)w.b * a.D + rd, n0, a.N, ron, g);
  // dD and dbias: over the block's steps, in their order
  float* f = &sD[0][0][0];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    f[(ct * CB + cc + i) * 2] = dD[i];
    f[(ct * CB + cc + i) * 2 + 1] = dbias[i];
  }
  __syncthreads();
  if (tid < 2 * CB && w.c0 + tid / 2 < a.Dg) {
    float s = 0.f;
    for (int k = 0; k < TT; ++k) s += f[k * CB * 2 + tid];
    a.par[(((long)w.b * a.chunks + w.chunk) * a.D + w.d0 + tid / 2) * (NP + 2) + NP + (tid & 1)] = s;
  }
}

struct FinishArgs {
  const float *par, *bc;
  float *dA, *dD, *dbias;
  void *dB, *dC;
  int rows, B, T, D, N, G, NP, cblk;
  unsigned first;          // blocks of the parameters' sums; behind them those of dB and dC
};

// dA (D, N), dD (D), dbias (D) from the rows of (sequence, chunk), in their order by four threads a value; dB, dC (B, T, G, N) from
// the channel blocks' sums
template <typename T>
__global__ void __launch_bounds__(256) scan_finish(FinishArgs a) {
  __shared__ float red[4][64];
  if (blockIdx.x < a.first) {
    const long cols = (long)a.D * (a.NP + 2), col = (long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int q = threadIdx.x >> 6, per = (a.rows + 3) / 4;
    float s = 0.f;
    if (col < cols) {
      const int r1 = min(a.rows, (q + 1) * per);
#pragma unroll 4
      for (int r = q * per; r < r1; ++r) s += a.par[r * cols + col];
    }
    red[q][threadIdx.x & 63] = s;
    __syncthreads();
    if (q == 0 && col < cols) {
      const int l = threadIdx.x;
      s = (red[0][l] + red[1][l]) + (red[2][l] + red[3][l]);
      const long d = col / (a.NP + 2);
      const int n = (int)(col % (a.NP + 2));
      if (n < a.N) {
        if (a.dA) a.dA[d * a.N + n] = s;
      } else if (n == a.NP) {
        if (a.dD) a.dD[d] = s;
      } else if (n == a.NP + 1) {
        if (a.dbias) a.dbias[d] = s;
      }
    }
    return;
  }
  const long id = (long)(blockIdx.x - a.first) * 256 + threadIdx.x, per = (long)a.T * 2 * a.NP;
  if (id >= (long)a.B * a.G * per) return;
  const long bg = id / per, r = id % per;
  const int n = (int)(r % (2 * a.NP)), t = (int)(r / (2 * a.NP));
  const int half = n >= a.NP, k = n - half * a.NP;
  if (k >= a.N) return;
  float s = 0.f;
#pragma unroll 4
  for (int c = 0; c < a.cblk; ++c) s += a.bc[(bg * a.cblk + c) * per + r];
  void* o = half ? a.dC : a.dB;
  if (o) static_cast<T*>(o)[(((bg / a.G) * a.T + t) * a.G + bg % a.G) * a.N + k] = (T)s;
}

struct StepArgs {
  float* state;
  const void *u, *dt, *z, *Bm, *Cm;
  const float *A, *Dp, *bias;
  void* out;
  long sub, sdb, szb, sBb, sBg, sCb, sCg, ssb;
  int B, D, N, G, Dg, softplus;
  int vec, vecbc;      // whole rows of 4 S states, and of B and C, on 16 bytes
};

// one step: reads and writes each state once.  Lanes as above: four a channel.
template <typename T, int S>
__global__ void __launch_bounds__(256) scan_step(StepArgs a) {
  const int lane = threadIdx.x & 3, n0 = lane * S;
  const long id = (long)blockIdx.x * 64 + (threadIdx.x >> 2);
  const bool on = id < (long)a.B * a.D;
  const int b = on ? (int)(id / a.D) : 0, d = on ? (int)(id % a.D) : 0, g = d / a.Dg;
  float* st = a.state + b * a.ssb + (long)d * a.N;
  float h[S], A[S], bv[S], cv[S];
  const bool whole = a.vec;
  if (whole) {
    tb_load_n(st + n0, h);
    tb_load_n(a.A + (long)d * a.N + n0, A);
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const bool in = n0 + s < a.N;
    if (!whole) {
      h[s] = in ? st[n0 + s] : 0.f;
      A[s] = in ? a.A[(long)d * a.N + n0 + s] : 0.f;
    }
    if (!a.vecbc) {
      bv[s] = in ? (float)static_cast<const T*>(a.Bm)[b * a.sBb + g * a.sBg + n0 + s] : 0.f;
      cv[s] = in ? (float)static_cast<const T*>(a.Cm)[b * a.sCb + g * a.sCg + n0 + s] : 0.f;
    }
  }
  if (a.vecbc) {
    tb_load_n(static_cast<const T*>(a.Bm) + b * a.sBb + g * a.sBg + n0, bv);
    tb_load_n(static_cast<const T*>(a.Cm) + b * a.sCb + g * a.sCg + n0, cv);
  }
  const float u = (float)static_cast<const T*>(a.u)[b * a.sub + d];
  float dl = (float)static_cast<const T*>(a.dt)[b * a.sdb + d] + (a.bias ? a.bias[d] : 0.f);
  if (a.softplus) dl = softplus(dl);
  float y = 0.f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    h[s] = fmaf(__builtin_amdgcn_exp2f(dl * (A[s] * LOG2E)), h[s], dl * u * bv[s]);
    h[s] = n0 + s < a.N ? h[s] : 0.f;          // behind N: 0 times what may be infinite
    y = fmaf(h[s], cv[s], y);
  }
  y = quad_sum(y);
  if (!on) return;
  if (whole) tb_store_n(st + n0, h);
  else
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (n0 + s < a.N) st[n0 + s] = h[s];
  if (lane == 0) {
    if (a.Dp) y = fmaf(a.Dp[d], u, y);
    if (a.z) y *= tb_silu((float)static_cast<const T*>(a.z)[b * a.szb + d]);
    static_cast<T*>(a.out)[(long)b * a.D + d] = (T)y;
  }
}

int states_per_lane(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

template <typename F>
int by_shape(int dtype, int S, F&& f) {
#define TB_S(T)                                                  \
  switch (S) {                                                   \
    case 1: return f.template operator()<T, 1>();                \
    case 2: return f.template operator()<T, 2>();                \
    case 4: return f.template operator()<T, 4>();                \
    case 8: return f.template operator()<T, 8>();                \
    default: return f.template operator()<T, 16>();              \
  }
  if (dtype == TB_F32) TB_S(float)
  if (dtype == TB_BF16) TB_S(__bf16)
  TB_S(_Float16)
#undef TB_S
}

// blocks of scan_finish: the parameters' sums, and those of dB and dC
long finish_blocks_par(const ScanArgs& a, int S) { return ((long)a.D * (4 * S + 2) + 63) / 64; }
long finish_blocks_bc(const ScanArgs& a, int S) { return ((long)a.B * a.G * a.T * 8 * S + 255) / 256; }

struct FwdLaunch {
  ScanArgs a;
  long blocks;       // channel blocks of the batch
  hipStream_t s;
  template <typename T, int S>
  int operator()() {
    // accesses off their alignment serve aligned rows too, but cost time (4 x 2048 x 2048 x 11 fp32 forward 162 us, aligned ones 150);
    // not for 33 to 64 states, whose backward pass they take more registers from
    if (a.N < 4 * S) return a.vec && S < 16 ? run<T, S, S < 16, true>() : run<T, S, false, true>();
    return a.vec ? run<T, S, true, false>() : run<T, S, false, false>();
  }
  template <typename T, int S, bool VEC, bool PART>
  int run() {
    if (a.chunks > 1) scan_fwd<T, S, true, VEC, false><<<(unsigned)(blocks * (a.chunks - 1)), 256, 0, s>>>(a);
    scan_fwd<T, S, false, VEC, PART><<<(unsigned)(blocks * a.chunks), 256, 0, s>>>(a);
    return 0;
  }
};
struct BwdLaunch {
  ScanArgs a;
  long blocks;
  float *dA, *dD, *dbias;
  void *dB, *dC;
  hipStream_t s;
  template <typename T, int S>
  int operator()() {
    if (a.N < 4 * S) return a.vec && S < 16 ? run<T, S, S < 16, true>() : run<T, S, false, true>();
    return a.vec ? run<T, S, true, false>() : run<T, S, false, false>();
  }
  template <typename T, int S, bool VEC, bool PART>
  int run() {
    if (a.chunks > 1) scan_bwd<T, S, true, VEC, false><<<(unsigned)(blocks * (a.chunks - 1)), 256, 0, s>>>(a);
    scan_bwd<T, S, false, VEC, PART><<<(unsigned)(blocks * a.chunks), 256, 0, s>>>(a);
    FinishArgs f{a.par, a.bc, dA, dD, dbias, dB, dC, a.B * a.chunks, a.B, a.T, a.D, a.N, a.G, 4 * S, a.cblk, 0};
    f.first = dA || dD || dbias ? (unsigned)finish_blocks_par(a, S) : 0;
    const unsigned rest = dB || dC ? (unsigned)finish_blocks_bc(a, S) : 0;
    if (f.first + rest) scan_finish<T><<<f.first + rest, 256, 0, s>>>(f);
    return 0;
  }
};
struct StepLaunch {
  StepArgs a;
  hipStream_t s;
  template <typename T, int S>
  int operator()() {
    scan_step<T, S><<<(unsigned)(((long)a.B * a.D + 63) / 64), 256, 0, s>>>(a);
    return 0;
  }
};

// Chunks of the steps.  Cutting them costs a second walk (about 0.9 of the first forward, 0.2 backward), and pays where the channel
// blocks alone leave compute units, or their waves' places, empty: as many chunks as bring four blocks a unit, not for fewer
// than three.  bf16, 2048 channels of 16 states, us forward, and with gradients by the backward pass' chunks:
//   128 blocks (4 x 2048 steps): forward in 4, 6, 8, 12 chunks 183, 155, 143, 152; backward in 4, 6, 8 509, 525, 479
//   256 blocks (8 x 2048): forward whole 288, in three 266, in four 247; backward whole 1084, in two, three, four 906, 973, 883
//   384 blocks (12 x 2048): forward whole 361, in two 380; backward whole 1409, in two 1427
// Chunks of 128 steps at least, of 32 where three quarters of the units would be idle (32 blocks of 512 steps: whole 77 / 261, in four
// 41 / 118, in sixteen 22 / 114; 256 blocks of 128 steps fp32: whole 25 / 111, in four 25 / 113).
void plan(int B, int T, int G, int Dg, int* cblk, int* chunk, int* chunks) {
  *cblk = (Dg + CB - 1) / CB;
  const long blocks = (long)B * G * *cblk, cus = tb_num_cus();
  long n = blocks > 0 ? 4 * cus / blocks : 1;
  if (n < 3) n = 1;
  const long least = blocks * 4 <= cus ? 32 : 128;
  long len = (T + n - 1) / n;
  if (len < least) len = least;
  len = (len + 31) / 32 * 32;
  *chunk = (int)len;
  *chunks = T > 0 ? (int)((T + len - 1) / len) : 1;
}

int check_common(const char* what, int B, long T, int D, int N, int G, int dtype) {
  if (B < 0 || T < 0 || D < 1 || N < 1 || G < 1 || D % G) return tb_set_error(TB_ERR_ARG, "%s: bad sizes B=%d T=%ld D=%d N=%d G=%d", what, B, T, D, N, G);
  if (T > TB_STEPS_MAX) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: too many steps in one call", what);
  if (N > NMAX) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: %d states a channel are not supported (1 to %d)", what, N, NMAX);
  if (!tb_dtype_ok(dtype)) return tb_set_error(TB_ERR_ARG, "%s: bad element type %d", what, dtype);
  return TB_OK;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 16-byte accesses: every row of every tensor starts on 16 bytes, and the channels of a group are whole threads' shares (eight)
bool can_vec(const ScanArgs& a, int dtype) {
  const int v = dtype == TB_F32 ? 4 : 8;
  if (a.Dg % 8 || a.sub % v || a.sut % v || a.sdb % v || a.sdt % v) return false;
  if (a.z && (a.szb % v || a.szt % v)) return false;
  if (a.dout && (a.sob % v || a.sot % v)) return false;
  const void* p[] = {a.u, a.dt, a.z, a.dout, a.out, a.du, a.ddt, a.dz};
  for (const void* q : p)
    if (!aligned(q)) return false;
  return true;
}

struct Sizes {
  size_t cstate, csum, bc, par, total;
};
Sizes sizes(int B, int T, int D, int N, int G, int backward) {
  int cblk, chunk, chunks;
  plan(B, T, G, D / G, &cblk, &chunk, &chunks);
  const size_t NP = 4 * states_per_lane(N);
  Sizes z;
  z.cstate = chunks > 1 ? tb_align_up((size_t)B * chunks * D * NP * 4, 256) : 0;
  z.csum = chunks > 1 ? tb_align_up((size_t)B * chunks * D * 4, 256) : 0;
  z.bc = backward ? tb_align_up((size_t)B * G * cblk * T * 2 * NP * 4, 256) : 0;
  z.par = backward ? tb_align_up((size_t)B * chunks * D * (NP + 2) * 4, 256) : 0;
  z.total = z.cstate + z.csum + z.bc + z.par + 256;
  return z;
}

}  // namespace

extern "C" {

size_t tb_scan_workspace_bytes(int B, int T, int D, int N, int G, int backward) {
  if (B < 1 || T < 1 || D < 1 || N < 1 || N > NMAX || G < 1 || D % G) return 256;
  return sizes(B, T, D, N, G, backward).total;
}

size_t tb_scan_states_bytes(int B, int T, int D, int N) {
  if (B < 1 || T < 1 || D < 1 || N < 1 || N > NMAX) return 0;
  const int S = states_per_lane(N), tt = bwd_tile(S);
  return (size_t)B * ((T + tt - 1) / tt) * D * 4 * S * 4;
}

int tb_scan_fwd(const void* u, const void* dt, const void* z, const void* Bm, const void* Cm, const long* strides, const float* A,
                const float* Dp, const float* dt_bias, int softplus, const float* h0, const int* lengths, void* out, float* hT,
                float* states, int B, int T, int D, int N, int G, int dtype, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_common("scan_fwd", B, T, D, N, G, dtype);
  if (rc) return rc;
  if (B < 1 || T < 1) return tb_set_error(TB_ERR_ARG, "scan_fwd: an empty batch has nothing to scan");
  if (!u || !dt || !Bm || !Cm || !strides || !A || !out || !ws) return tb_set_error(TB_ERR_ARG, "scan_fwd: null pointer");
  const Sizes sz = sizes(B, T, D, N, G, 0);
  if (ws_bytes < sz.total) return tb_set_error(TB_ERR_WORKSPACE, "scan_fwd: workspace too small");
  const int S = states_per_lane(N);
  ScanArgs a{};
  a.u = u; a.dt = dt; a.z = z; a.Bm = Bm; a.Cm = Cm;
  a.A = A; a.Dp = Dp; a.bias = dt_bias; a.h0 = h0; a.lengths = lengths;
  a.out = out; a.hT = hT; a.ck = states;
  const long* q = strides;
  a.sub = q[0]; a.sut = q[1]; a.sdb = q[2]; a.sdt = q[3]; a.szb = q[4]; a.szt = q[5];
  a.sBb = q[6]; a.sBt = q[7]; a.sBg = q[8]; a.sCb = q[9]; a.sCt = q[10]; a.sCg = q[11];
  a.B = B; a.T = T; a.D = D; a.N = N; a.G = G; a.Dg = D / G;
  plan(B, T, G, a.Dg, &a.cblk, &a.chunk, &a.chunks);
  a.softplus = softplus;
  a.ckt = states ? bwd_tile(S) : 0;
  a.cktiles = states ? (T + a.ckt - 1) / a.ckt : 0;
  a.cstate = static_cast<float*>(ws);
  a.csum = reinterpret_cast<float*>(static_cast<char*>(ws) + sz.cstate);
  if (!tb_grid_ok((long)B * G * a.cblk * a.chunks, 256)) return tb_set_error(TB_ERR_UNSUPPORTED, "scan_fwd: too many rows in one call");
  a.vec = can_vec(a, dtype);
  by_shape(dtype, S, FwdLaunch{a, (long)B * G * a.cblk, static_cast<hipStream_t>(stream)});
  TB_LAUNCH_CHECK("scan_fwd");
  return TB_OK;
}

int tb_scan_bwd(const void* dout, const void* u, const void* dt, const void* z, const void* Bm, const void* Cm, const long* strides,
                const float* A, const float* Dp, const float* dt_bias, int softplus, const int* lengths, const float* states,
                const float* dhT, void* du, void* ddt, void* dz, void* dB, void* dC, float* dA, float* dD, float* dbias, float* dh0,
                int B, int T, int D, int N, int G, int dtype, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_common("scan_bwd", B, T, D, N, G, dtype);
  if (rc) return rc;
  if (B < 1 || T < 1) return tb_set_error(TB_ERR_ARG, "scan_bwd: an empty batch has no gradients to form here");
  if (!dout || !u || !dt || !Bm || !Cm || !strides || !A || !states || !ws) return tb_set_error(TB_ERR_ARG, "scan_bwd: null pointer");
  const Sizes sz = sizes(B, T, D, N, G, 1);
  if (ws_bytes < sz.total) return tb_set_error(TB_ERR_WORKSPACE, "scan_bwd: workspace too small");
  const int S = states_per_lane(N);
  ScanArgs a{};
  a.u = u; a.dt = dt; a.z = z; a.Bm = Bm; a.Cm = Cm; a.dout = dout;
  a.A = A; a.Dp = Dp; a.bias = dt_bias; a.dhT = dhT; a.lengths = lengths;
  a.du = du; a.ddt = ddt; a.dz = z ? dz : nullptr; a.dh0 = dh0;
  a.ck = const_cast<float*>(states);
  const long* q = strides;
  a.sub = q[0]; a.sut = q[1]; a.sdb = q[2]; a.sdt = q[3]; a.szb = q[4]; a.szt = q[5];
  a.sBb = q[6]; a.sBt = q[7]; a.sBg = q[8]; a.sCb = q[9]; a.sCt = q[10]; a.sCg = q[11];
  a.sob = q[12]; a.sot = q[13];
  a.B = B; a.T = T; a.D = D; a.N = N; a.G = G; a.Dg = D / G;
  plan(B, T, G, a.Dg, &a.cblk, &a.chunk, &a.chunks);
  a.softplus = softplus;
  a.ckt = bwd_tile(S);
  a.cktiles = (T + a.ckt - 1) / a.ckt;
  char* p = static_cast<char*>(ws);
  a.cstate = reinterpret_cast<float*>(p);
  a.csum = reinterpret_cast<float*>(p + sz.cstate);
  a.bc = reinterpret_cast<float*>(p + sz.cstate + sz.csum);
  a.par = reinterpret_cast<float*>(p + sz.cstate + sz.csum + sz.bc);
  if (!tb_grid_ok((long)B * G * a.cblk * a.chunks, 256) || !tb_grid_ok(finish_blocks_par(a, S) + finish_blocks_bc(a, S), 256))
    return tb_set_error(TB_ERR_UNSUPPORTED, "scan_bwd: too many rows or steps in one call");
  a.vec = can_vec(a, dtype);
  by_shape(dtype, S, BwdLaunch{a, (long)B * G * a.cblk, dA, dD, dbias, dB, dC, static_cast<hipStream_t>(stream)});
  TB_LAUNCH_CHECK("scan_bwd");
  return TB_OK;
}

int tb_scan_step(float* state, long state_batch_stride, const void* u, const void* dt, const void* z, const void* Bm, const void* Cm,
                 const long* strides, const float* A, const float* Dp, const float* dt_bias, int softplus, void* out, int B, int D, int N,
                 int G, int dtype, void* stream) {
  int rc = check_common("scan_step", B, 1, D, N, G, dtype);
  if (rc) return rc;
  if (B == 0) return TB_OK;
  if (!state || !u || !dt || !Bm || !Cm || !strides || !A || !out) return tb_set_error(TB_ERR_ARG, "scan_step: null pointer");
  const long* q = strides;
  StepArgs a{state, u, dt, z, Bm, Cm, A, Dp, dt_bias, out, q[0], q[1], q[2], q[3], q[4], q[5], q[6], state_batch_stride,
             B, D, N, G, D / G, softplus, 0, 0};
  if (!tb_grid_ok(((long)B * D + 63) / 64, 256)) return tb_set_error(TB_ERR_UNSUPPORTED, "scan_step: too many rows in one call");
  const int S = states_per_lane(N), v = dtype == TB_F32 ? 4 : 8;
  a.vec = N == 4 * S && state_batch_stride % 4 == 0 && aligned(state) && aligned(A);
  a.vecbc = N == 4 * S && N % v == 0 && aligned(Bm) && aligned(Cm) && q[3] % v == 0 && q[4] % v == 0 && q[5] % v == 0 && q[6] % v == 0;
  by_shape(dtype, S, StepLaunch{a, static_cast<hipStream_t>(stream)});
  TB_LAUNCH_CHECK("scan_step");
  return TB_OK;
}

}  // extern "C"

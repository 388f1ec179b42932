// Linear with bias, activation and residual: y = act(x W^T + b) + r, its gradients, fp32 / bf16 / fp16.
//
//   z = x W^T + b,  y = act(z) + r        dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = colsum(dz),  dr = dy
//
// One matrix kernel serves all three products: C[m][n] = sum_k P[m][k] Q[n][k] with k running along the rows of both operands,
// which is what a matrix instruction's lanes want (16 neighbouring bytes each).  For dx and dW the operands are written once
// with their axes exchanged (W, x and dz: 2 bytes an element moved against K or M operations on it; fp32 takes dW's as they are);
// the kernel that forms dz = dy act'(z) writes both orders and the column sums of db in its one pass.
// 16-bit operands go through v_mfma_f32_16x16x32, fp32 ones through v_mfma_f32_16x16x4 (exact fp32 products: no splitting
// into 16-bit parts, so infinities and the type's whole range pass).  Sums are fp32, z is kept in fp32 for the gradient (kept in 16 bits it
// would add a second rounding to act').  dz enters the matrix instructions in the operands' type: as it is where that holds it (no
// activation, relu), else, of 16-bit types, in two parts (Halves below), since one rounding of dz alone puts the gradients off by as
// much as their own (4099 x 1000 x 1500 fp16 against 64 bits: 2.93e-4 instead of 2.07e-4) and loses fp16 gradients outside its range.
// Both operands are copied straight to LDS (16 bytes a lane, 64 bytes of a row a tile), tiles ahead of their use; the 16-byte
// pieces of a row change places by the row's low bits, so that the rows a fragment reads fall on different banks.
// Measured (bf16, without activation or residual): 16384 x 8192 x 8192 1948 us, 1.13 PFLOP/s (the library's product 1505 us in turn with it);
// 16384 x 2048 x 8192 491 us (374), with gelu and residual 571 to 590; what bounds the large tiles is LDS (125 of its 128 bytes a
// clock at the matrix instructions' full rate), and behind it the epilogue, which one block a unit leaves uncovered.  Not kept:
// 256 x 128 tiles, two blocks a unit (main loop 507 us against 412 a 2048 of k, LDS bound), 128 x 128 a wave
// (the compiler moves the 256 sums between register files: 219 TFLOP/s), 256 x 128 one block a unit for middle sizes (same).
// Few rows (a batch of single tokens) are bound by reading W once: a kernel without LDS staging whose waves split K.
#include "elem.h"

#include <type_traits>

namespace {

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

__device__ const f32x4 g_zeros[16] = {};     // what pieces behind the end of K are read from

// tanh to a relative error of 2^-20 (measured: 6.0e-7 at most): below 1/4 its series, which leaves out less than 2^-31 of it and rounds
// to 9e-8, where 1 - 2 / (1 + e^2x) cancels
__device__ __forceinline__ float tanh_rel(float x) {
  const float q = x * x;
  const float p = x * (1.f + q * (-0.333333333f + q * (0.133333333f + q * (-0.0539682540f + q * (0.0218694885f + q * -0.00886323553f)))));
  return fabsf(x) < 0.25f ? p : tb_tanh(x);
}
// half of erfc(|z| / sqrt 2): t e^(-z^2/2 + P(t)), t = 1 / (1 + 0.4 x), with P a degree 8 least-maximum fit of
// log(erfc(x) e^(x^2) / t) on 0 <= x < 9.5 (off by 2.2e-7 with its coefficients in fp32): the lower tail keeps a relative precision of
// 2^-20 + 2.5 z^2 2^-24 (the exponent's roundings; measured at z = -1, -9, -13: 6e-7, 8e-6, 1.9e-5), where 1 + erf cancels
__device__ __forceinline__ float half_erfc(float z) {
  const float x = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(0.4f, x, 1.f));
  float p = -0.2059148f;
  p = fmaf(p, t, 0.91647777f);
  p = fmaf(p, t, -1.46799367f);
  p = fmaf(p, t, 0.97708137f);
  p = fmaf(p, t, -0.42703877f);
  p = fmaf(p, t, 0.29283921f);
  p = fmaf(p, t, 0.40185486f);
  p = fmaf(p, t, 1.00138551f);
  p = fmaf(p, t, -1.48869157f);
  return 0.5f * t * tb_exp(fmaf(-x, x, p));
}
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case 1: return tanh_rel(z);
    case 2: return tb_sig(z);
    case 3: return z < 0.f ? 0.f : z;
    case 4: return tb_silu(z);
    case 5: { const float e = half_erfc(z); return z * (z > 0.f ? 1.f - e : e); }
    default: return z;
  }
}
__device__ __forceinline__ float act_grad(float z, int act) {
  switch (act) {
    case 1: { const float y = tanh_rel(z); return 1.f - y * y; }
    case 2: { const float y = tb_sig(z); return y * (1.f - y); }
    case 3: return z > 0.f ? 1.f : 0.f;
    case 4: { const float y = tb_sig(z); return y * (1.f + z * (1.f - y)); }
    case 5: { const float e = half_erfc(z); return (z > 0.f ? 1.f - e : e) + z * 0.39894228f * tb_exp(-0.5f * z * z); }
    default: return 1.f;
  }
}

// 16 bytes of k for each of the sixteen rows of a fragment: lane l holds row l & 15, piece l >> 4 of four
template <typename T>
struct Mfma;
template <>
struct Mfma<__bf16> {
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma<_Float16> {
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma<float> {
  // the four k of a lane's piece in four instructions: the order of k is free as long as both operands keep the same one
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

// dz of 16-bit operands in two values of their type: hi, rounded, and lo, what that left out, together good to 2^-16 (bf16) and
// 2^-21 (fp16).  fp16's range is short at both ends: hi is halved, so that |act'| < 2 cannot push it past the largest value, and lo is
// enlarged, so that it still counts below the smallest.  A product runs over lo first, turns its sums to hi's scale (LO_TO_HI), runs
// over hi and undoes the halving (OUT).
template <typename T>
struct Halves {
  static constexpr bool F16 = std::is_same_v<T, _Float16>;
  static constexpr float HI = F16 ? 0.5f : 1.f, LO = F16 ? 1024.f : 1.f, LO_TO_HI = HI / LO, OUT = 1.f / HI;
  static __device__ __forceinline__ float hi(float v) { return v * HI; }
  static __device__ __forceinline__ float lo(float v) {
    const float h = (float)(T)(v * HI);
    return fabsf(h) < INFINITY ? (v - h * OUT) * LO : 0.f;      // infinities and NaN are hi's alone
  }
};

struct Epi {
  const void *bias, *res;   // element type T, each nullable
  void* y;                  // M x N dense
  float* z;                 // M x N dense, nullable: the pre-activation
  float* slab;              // split k: partial sums [split][M][N] instead of everything above
  long ldr;
  int act;
};

// four neighbouring columns n .. of row m, anywhere in memory; the last ones of a row element by element
template <typename T>
__device__ __forceinline__ void finish4(const Epi& e, int N, long m, int n, float (&o)[4]) {
  const long at = m * N + n;
  if (n + 4 <= N) {
    float q[4];
    if (e.res) tb_load_u(static_cast<const T*>(e.res) + m * e.ldr + n, q);
    if (e.bias) {
      float b[4];
      tb_load_u(static_cast<const T*>(e.bias) + n, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += b[i];
    }
    if (e.z) tb_store_u(e.z + at, o);
    if (e.act)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = act_of(o[i], e.act);
    if (e.res)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += q[i];
    tb_store_u(static_cast<T*>(e.y) + at, o);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i >= N) break;
      float w = o[i];
      if (e.bias) w += (float)static_cast<const T*>(e.bias)[n + i];
      if (e.z) e.z[at + i] = w;
      if (e.act) w = act_of(w, e.act);
      if (e.res) w += (float)static_cast<const T*>(e.res)[m * e.ldr + n + i];
      static_cast<T*>(e.y)[at + i] = (T)w;
    }
  }
}

struct GemmArgs {
  const void *P, *Q;        // P: M rows, Q: N rows; rows start on 16 bytes, K a multiple of 16 bytes
  const void* lo;           // the second part of P, laid out as P is, nullable (Halves)
  long ldp, ldq;
  long M;
  int N, K;
  int tm, tn, splits, per;  // tiles; k tiles a split (with two parts of P: of both, lo's first)
  int width;                // columns an access of the epilogue, of which every row is whole: 8 (16-bit types), 4, 2 or 1
  Epi e;
};

// Tiles of the output in an order that keeps each of the eight dies on neighbouring tiles (consecutive workgroups go to
// different dies, each with its own L2): die x takes the x-th eighth of the tiles, which run down eight rows of tiles at a time.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& im, int& in) {
  const int n = tm * tn, q = n / 8, r = n % 8, x = id % 8, i = id / 8;
  const int at = x < r ? x * (q + 1) + i : r * (q + 1) + (x - r) * q + i;
  const int band = at / (8 * tn), rows = min(8, tm - band * 8), in_band = at - band * 8 * tn;
  im = band * 8 + in_band % rows;
  in = in_band / rows;
}

// The epilogue of rows that are whole pieces of V columns: the residual's pieces are fetched two accesses ahead of their use, the
// activation is chosen once, outside the rows (16384 x 2048 x 8192 with gelu and residual: 685 us, so 585; without both 491, the residual
// alone adds 51, gelu alone 49; four and eight accesses ahead: 606 and 671).
template <typename T, int V>
__device__ __forceinline__ void whole_rows(const GemmArgs& a, const float* own, long m0, int n0, int lane) {
  constexpr int L = 64 / V;      // lanes a row; V rows an access, L accesses
  typedef TbVec<T, V> Piece;
  const Epi& e = a.e;
  const int c = lane % L, n = n0 + c * V;
  if (n >= a.N) return;
  float b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = 0.f;
  if (e.bias) tb_load_n(static_cast<const T*>(e.bias) + n, b);
  const T* res = static_cast<const T*>(e.res) + n;
  auto fetch = [&](int i) {
    const long m = m0 + lane / L + i * V;
    return *reinterpret_cast<const Piece*>(res + (m < a.M ? m : a.M - 1) * e.ldr);
  };
  auto all = [&](auto act) {
    Piece q0{}, q1{};
    if (e.res) {
      q0 = fetch(0);
      q1 = fetch(1);
    }
    auto row = [&](int i, const Piece& q) {
      const int r = lane / L + i * V;
      const long m = m0 + r;
      if (m >= a.M) return;
      float o[V];
      if constexpr (V >= 4) {
#pragma unroll
        for (int k = 0; k < V / 4; ++k) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(own + r * 64 + (((c * (V / 4) + k) ^ (r & 15)) * 4));
#pragma unroll
          for (int j = 0; j < 4; ++j) o[k * 4 + j] = v[j] + b[k * 4 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = own[r * 64 + ((c * V / 4) ^ (r & 15)) * 4 + c * V % 4 + j] + b[j];
      }
      if (e.z) tb_store_n(e.z + m * a.N + n, o);
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = act_of(o[j], act);
      if (e.res) {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += (float)q.v[j];
      }
      tb_store_n(static_cast<T*>(e.y) + m * a.N + n, o);
    };
#pragma unroll 1
    for (int i = 0; i < L; i += 2) {
      const Piece p0 = q0, p1 = q1;
      if (e.res && i + 2 < L) {
        q0 = fetch(i + 2);
        q1 = fetch(i + 3);
      }
      row(i, p0);
      row(i + 1, p1);
    }
  };
  switch (e.act) {
    case 1: all(std::integral_constant<int, 1>{}); break;
    case 2: all(std::integral_constant<int, 2>{}); break;
    case 3: all(std::integral_constant<int, 3>{}); break;
    case 4: all(std::integral_constant<int, 4>{}); break;
    case 5: all(std::integral_constant<int, 5>{}); break;
    default: all(std::integral_constant<int, 0>{});
  }
}

// 64 x 64 sums of a wave, in LDS as gemm leaves them, through the epilogue to memory
template <typename T>
__device__ __forceinline__ void write_block(const GemmArgs& a, const float* own, long m0, int n0, int lane, int part) {
  const Epi& e = a.e;
  auto piece = [&](int r, int c) { return *reinterpret_cast<const f32x4*>(own + r * 64 + ((c ^ (r & 15)) * 4)); };
  if (e.slab) {
    const int c = lane & 15, n = n0 + c * 4;
    if (n >= a.N) return;
#pragma unroll 2
    for (int r = lane >> 4; r < 64; r += 4) {
      const long m = m0 + r;
      if (m >= a.M) break;
      const f32x4 v = piece(r, c);
      float* s = e.slab + ((long)part * a.M + m) * a.N + n;
      if (n + 4 <= a.N) {
        const float o[4] = {v[0], v[1], v[2], v[3]};
        tb_store_u(s, o);
      } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (n + i < a.N) s[i] = v[i];
      }
    }
    return;
  }
  // accesses of 16 bytes off their alignment cost more than smaller ones on theirs (N = 1500 of fp16: 6 us of a 17 us call)
  if (sizeof(T) == 2 && a.width == 8) whole_rows<T, 16 / sizeof(T)>(a, own, m0, n0, lane);
  else if (a.width == 4) whole_rows<T, 4>(a, own, m0, n0, lane);
  else if (a.width == 2) whole_rows<T, 2>(a, own, m0, n0, lane);
  else whole_rows<T, 1>(a, own, m0, n0, lane);
}

// 64 bytes of k a tile, four tiles in LDS: while one tile is multiplied from registers, the next one's fragments are read
// from LDS and the copies of the three behind it are under way.  One barrier a tile: behind it the tile that was just read into
// registers by every wave is free for a new copy, and the next one has landed (the copies still under way are counted, not
// drained).
//
// DOWN (fp32, for dW): k runs down the columns of both operands as they are, P[k][m] and Q[k][n], K rows of M and N columns that are
// whole 16-byte pieces on 16 bytes.  A tile is sixteen rows of BM (BN) columns; a lane takes its k one by one (4 bytes), which the
// fp32 instructions, a quarter of the 16-bit ones' rate a byte, leave time for.  Saves the transposed copies of dz and x
// (65536 x 256 x 256: 345 us of a training step, so 302).
//
// TWO: P comes in two parts, and k runs over all of lo and then over all of P (twice the products; 4099 x 1000 x 1500 fp16 with SiLU and
// gradients: 142 us, with dz rounded once 102).
template <typename T, int BM, int BN, int WM, int WN, bool DOWN, bool TWO>
__device__ __forceinline__ void product(const GemmArgs& a, int tile, int part, char* lds) {
  static_assert(!DOWN || (sizeof(T) == 4 && BM == 128 && BN == 128), "rows of 512 bytes, two a copy");
  static_assert(!TWO || sizeof(T) == 2, "fp32 holds dz as it is");
  constexpr int WAVES = (BM / WM) * (BN / WN), CE = 16 / sizeof(T), BK = 4 * CE;
  constexpr int MF = WM / 16, NF = WN / 16, LP = BM / 16 / WAVES, LQ = BN / 16 / WAVES;
  constexpr int STAGE = (BM + BN) * 64;
  static_assert(LP + LQ == 4, "the counted waits below are for four copies a wave and tile");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int im, in;
  tile_of(tile, a.tm, a.tn, im, in);
  const long m0 = (long)im * BM;
  const int n0 = in * BN;
  const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
  const int kt = (a.K + BK - 1) / BK;                    // k tiles of a part of P
  int kt0 = part * a.per, nt = min(a.per, kt - kt0);      // TWO: set for each part below

  // What this lane copies: row 16 i + lane / 4 of each of its pieces, and of that row's four 16-byte pieces the one whose place
  // in LDS is lane % 4: piece p of row r lies at p ^ (r / 2 % 4), so that eight neighbouring rows fill all banks.
  // DOWN: row 2 i + lane / 32 of the tile's sixteen, of 32 pieces; piece p of row r lies at p ^ (r % 4 * 4), so that the four rows
  // of a read fall on different banks.
  const int lr = DOWN ? lane >> 5 : lane >> 2;
  const int piece = (DOWN ? (lane & 31) : (lane & 3) ^ ((lr >> 1) & 3)) * CE;
  const T* const P = static_cast<const T*>(TWO ? a.lo : a.P);
  const T* pp[LP];
  const T* qp[LQ];
  int pr[LP], qr[LQ];              // DOWN: the row within a tile, or past every K where the columns are behind the last
#pragma unroll
  for (int i = 0; i < LP; ++i) {
    if constexpr (DOWN) {
      const int row = (wave * LP + i) * 2 + lr;
      const long c = m0 + (piece ^ (row & 3) * 16);
      pp[i] = P + (c < a.M ? c : 0) + row * a.ldp;
      pr[i] = c < a.M ? row : 1 << 30;
    } else {
      long r = m0 + (wave * LP + i) * 16 + lr;
      r = r < a.M ? r : a.M - 1;                // rows behind the last: any row, never stored
      pp[i] = P + r * a.ldp + piece;
    }
  }
#pragma unroll
  for (int i = 0; i < LQ; ++i) {
    if constexpr (DOWN) {
      const int row = (wave * LQ + i) * 2 + lr, c = n0 + (piece ^ (row & 3) * 16);
      qp[i] = static_cast<const T*>(a.Q) + (c < a.N ? c : 0) + row * a.ldq;
      qr[i] = c < a.N ? row : 1 << 30;
    } else {
      int r = n0 + (wave * LQ + i) * 16 + lr;
      r = r < a.N ? r : a.N - 1;
      qp[i] = static_cast<const T*>(a.Q) + (long)r * a.ldq + piece;
    }
  }
  // TAIL: the tile may reach behind the end of K, whose pieces come from a row of zeros
  auto copy = [&](int t, auto tail) {
    char* to = lds + (t & 3) * STAGE;
    const long k = (long)(kt0 + t) * BK;
    const bool in_k = !tail || k + piece < a.K;
    const uintptr_t zero = reinterpret_cast<uintptr_t>(g_zeros);
#pragma unroll
    for (int i = 0; i < LP; ++i) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(pp[i] + (DOWN ? k * a.ldp : k));
      __builtin_amdgcn_global_load_lds((gvoid*)((DOWN ? k + pr[i] < a.K : in_k) ? at : zero), (lvoid*)(to + (wave * LP + i) * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < LQ; ++i) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(qp[i] + (DOWN ? k * a.ldq : k));
      __builtin_amdgcn_global_load_lds((gvoid*)((DOWN ? k + qr[i] < a.K : in_k) ? at : zero), (lvoid*)(to + BM * 64 + (wave * LQ + i) * 1024), 16, 0, 0);
    }
  };
  const int place = ((lane >> 4) ^ ((lane >> 1) & 3)) * 16;
  const int po = (wm + (lane & 15)) * 64 + place, qo = BM * 64 + (wn + (lane & 15)) * 64 + place;
  auto read = [&](int t, u32x4 (&fp)[MF], u32x4 (&fq)[NF]) {
    const char* from = lds + (t & 3) * STAGE;
    if constexpr (DOWN) {
      // k = 4 j + lane / 16 of column lane % 16: in the j-th instruction's order of k
      const int row = (lane >> 4) * 512, col = lane & 15, turn = (lane >> 4) * 16;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
          fq[i][j] = *reinterpret_cast<const unsigned*>(from + BM * 64 + j * 2048 + row + (((wn + i * 16) ^ turn) + col) * 4);
#pragma unroll
        for (int i = 0; i < MF; ++i)
          fp[i][j] = *reinterpret_cast<const unsigned*>(from + j * 2048 + row + (((wm + i * 16) ^ turn) + col) * 4);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NF; ++j) fq[j] = *reinterpret_cast<const u32x4*>(from + qo + j * 1024);
#pragma unroll
      for (int i = 0; i < MF; ++i) fp[i] = *reinterpret_cast<const u32x4*>(from + po + i * 1024);
    }
  };

  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 fp[2][MF], fq[2][NF];

  // in front of a barrier: this wave has read tile t into registers, and its copies of tile t + 1 have landed
  auto meet = [&](auto drain) {
    if constexpr (drain) __builtin_amdgcn_s_waitcnt(0x0070);       // vmcnt(0) lgkmcnt(0)
    else __builtin_amdgcn_s_waitcnt(0x0078);                       // vmcnt(8) lgkmcnt(0): two tiles' copies under way
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](const u32x4 (&p)[MF], const u32x4 (&q)[NF]) {
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[i][j] = Mfma<T>::mul(q[j], p[i], acc[i][j]);
    // keeps the products in front of the next barrier (an empty statement; without it they are moved behind it, where
    // they no longer cover the copies and reads)
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) asm volatile("" : "+v"(acc[i][j]));
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto all_tiles = [&] {
    if (nt <= 0) return;
    for (int t = 0; t < 4 && t < nt; ++t) copy(t, yes);
    meet(yes);
    read(0, fp[0], fq[0]);
    int t = 0;
    for (; t + 6 < nt; t += 2) {        // the copies here are of whole tiles
      meet(no);
      copy(t + 4, no);
      read(t + 1, fp[1], fq[1]);
      multiply(fp[0], fq[0]);
      meet(no);
      copy(t + 5, no);
      read(t + 2, fp[0], fq[0]);
      multiply(fp[1], fq[1]);
    }
    for (; t < nt; t += 2) {
      meet(yes);
      if (t + 4 < nt) copy(t + 4, yes);
      if (t + 1 < nt) read(t + 1, fp[1], fq[1]);
      multiply(fp[0], fq[0]);
      if (t + 1 < nt) {
        meet(yes);
        if (t + 5 < nt) copy(t + 5, yes);
        if (t + 2 < nt) read(t + 2, fp[0], fq[0]);
        multiply(fp[1], fq[1]);
      }
    }
  };
  if constexpr (TWO) {
    const int k0 = part * a.per, k1 = min(k0 + a.per, 2 * kt);
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      kt0 = max(k0 - i * kt, 0);
      nt = min(k1 - i * kt, kt) - kt0;
      if (i) {
        __syncthreads();                  // every wave has read lo's last tile: its place is free
#pragma unroll
        for (int j = 0; j < LP; ++j) pp[j] += static_cast<const T*>(a.P) - P;
        if constexpr (Halves<T>::LO_TO_HI != 1.f)
#pragma unroll
          for (int m = 0; m < MF; ++m)
#pragma unroll
            for (int n = 0; n < NF; ++n) acc[m][n] *= Halves<T>::LO_TO_HI;
      }
      all_tiles();
    }
    if constexpr (Halves<T>::OUT != 1.f)
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[m][n] *= Halves<T>::OUT;
  } else {
    all_tiles();
  }
  // A lane holds row lane & 15 and four neighbouring columns of each 16 x 16 piece (Q is the left operand).  They change
  // places through LDS, 64 rows at a time in each wave's own 16 KB, so that every access to memory is of whole rows of
  // the wave's 64 columns; and the epilogue is a short loop: unrolled over the accumulators it was 300 KB of code, whose fetching
  // took longer than the products (K = 2048: 326 of 726 us).
  __syncthreads();
  float* own = reinterpret_cast<float*>(lds + wave * 16384);
  static_assert(WN == 64 && WAVES * 16384 <= 4 * STAGE, "a wave's 64 x 64 block of sums in LDS");
#pragma unroll
  for (int h = 0; h < MF / 4; ++h) {
    asm volatile("" ::: "memory");
    // 16-byte piece c of row r lies at c ^ (r & 15): the sixteen rows of a store fall on different banks
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j)
        *reinterpret_cast<f32x4*>(own + (i * 16 + (lane & 15)) * 64 + (((j * 4 + (lane >> 4)) ^ (lane & 15)) * 4)) = acc[h * 4 + i][j];
    __builtin_amdgcn_s_waitcnt(0xC07F);        // lgkmcnt(0): the block is this wave's own, no barrier
    asm volatile("" ::: "memory");
    write_block<T>(a, own, m0 + wm + h * 64, n0 + wn, lane, part);
  }
}

template <typename T, int BM, int BN, int WM, int WN, bool DOWN, bool TWO>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64, 2) gemm(GemmArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[4 * (BM + BN) * 64];
  product<T, BM, BN, WM, WN, DOWN, TWO>(a, blockIdx.x, blockIdx.y, lds);
}

// Two products in one launch, the first's blocks in front (dW, whose k is long, and dx): neither fills the chip to its end alone.
// With the layouts before them and the finishes behind them in one launch each, a training step of 4099 x 1000 x 1500 fp16, dz in one part, took
// 104 us (launch by launch 121), 1024^3 fp32 92 (106), 145 x 560 x 301 fp16 38 (46).
template <typename T, bool DOWN, bool TWO>
__global__ void __launch_bounds__(256, 2) gemm_pair(GemmArgs a, GemmArgs b, unsigned first) {
  __shared__ __attribute__((aligned(16))) char lds[4 * 256 * 64];
  const bool second = blockIdx.x >= first;
  const int id = blockIdx.x - (second ? first : 0);
  if constexpr (DOWN) {
    const int tiles = second ? b.tm * b.tn : a.tm * a.tn;
    if (second) product<T, 128, 128, 64, 64, false, TWO>(b, id % tiles, id / tiles, lds);
    else product<T, 128, 128, 64, 64, true, TWO>(a, id % tiles, id / tiles, lds);
  } else {
    const GemmArgs c = second ? b : a;
    product<T, 128, 128, 64, 64, false, TWO>(c, id % (c.tm * c.tn), id / (c.tm * c.tn), lds);
  }
}

// the splits' sums and the epilogue: four columns a thread, four threads share a place's splits and are added in their order
template <typename T>
__device__ __forceinline__ void split_sum(const Epi& e, long M, int N, int splits, unsigned block, float (&red)[4][64][4]) {
  const int nq = (N + 3) / 4, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const long id = (long)block * 64 + x;
  const bool on = id < M * nq;
  const long m = on ? id / nq : 0;
  const int n = on ? (int)(id % nq) * 4 : 0;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (on) {
    const int per = (splits + 3) / 4, k1 = min(splits, (y + 1) * per);
    if (n + 4 <= N) {
#pragma unroll 4
      for (int k = y * per; k < k1; ++k) {
        float v[4];
        tb_load_u(e.slab + ((long)k * M + m) * N + n, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += v[i];
      }
    } else {
      for (int k = y * per; k < k1; ++k)
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (n + i < N) s[i] += e.slab[((long)k * M + m) * N + n + i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[y][x][i] = s[i];
  __syncthreads();
  if (y || !on) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = (red[0][x][i] + red[1][x][i]) + (red[2][x][i] + red[3][x][i]);
  finish4<T>(e, N, m, n, s);
}

template <typename T>
__global__ void __launch_bounds__(256) split_finish(Epi e, long M, int N, int splits) {
  __shared__ float red[4][64][4];
  split_sum<T>(e, M, N, splits, blockIdx.x, red);
}

// What the backward pass leaves for the end, in one launch: the split sums of dW and dx, and db from the sums of each 64 rows
// (four columns a block, 64 threads a column, added in a fixed order).
struct EndArgs {
  Epi w, x;
  long Mw, Mx;
  int Nw, Nx, sw, sx;              // rows, columns and parts of each; a part count of one: nothing left to do
  unsigned bw, bx, bb;             // blocks of each
  const float* part;
  long rows;
  int N;
  void* db;
};
template <typename T>
__global__ void __launch_bounds__(256) backward_end(EndArgs a) {
  __shared__ float red[4][64][4];
  if (blockIdx.x < a.bw) {
    split_sum<T>(a.w, a.Mw, a.Nw, a.sw, blockIdx.x, red);
  } else if (blockIdx.x < a.bw + a.bx) {
    split_sum<T>(a.x, a.Mx, a.Nx, a.sx, blockIdx.x - a.bw, red);
  } else {
    const int x = threadIdx.x & 3, y = threadIdx.x >> 2, c = (int)(blockIdx.x - a.bw - a.bx) * 4 + x;
    float s = 0.f;
    if (c < a.N) {
#pragma unroll 8
      for (long r = y; r < a.rows; r += 64) s += a.part[r * a.N + c];
    }
    float(&q)[1024] = reinterpret_cast<float(&)[1024]>(red);
    q[threadIdx.x] = s;
#pragma unroll
    for (int h = 128; h >= 4; h /= 2) {
      __syncthreads();
      if ((int)threadIdx.x < h) q[threadIdx.x] += q[threadIdx.x + h];
    }
    if (threadIdx.x < 4 && c < a.N) static_cast<T*>(a.db)[c] = (T)q[threadIdx.x];
  }
}

struct FewArgs {
  const void *x, *W;
  long ldx, ldw, M;
  int N, K, vec;
  Epi e;
};

template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* row, long k, int K, bool vec, bool on) {
  constexpr int CE = 16 / sizeof(T);
  u32x4 r = (u32x4){0u, 0u, 0u, 0u};
  if (vec) {
    if (on && k < K) r = *reinterpret_cast<const u32x4*>(row + k);
  } else if (on && k + CE <= K) {
    r = __builtin_bit_cast(u32x4, *reinterpret_cast<const TbVecU<T, CE>*>(row + k));
  } else if (on && k < K) {
    TbVec<T, CE> v;
#pragma unroll
    for (int i = 0; i < CE; ++i) v.v[i] = k + i < K ? row[k + i] : (T)0.f;
    r = __builtin_bit_cast(u32x4, v);
  }
  return r;
}

// up to 16 MT rows: a block owns sixteen columns, its waves take turns along K and are summed at the end
template <typename T, int MT, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) gemm_few(FewArgs a) {
  constexpr int CE = 16 / sizeof(T), U = MT == 1 ? 8 : 4, STEP = 4 * CE * U;
  __shared__ f32x4 red[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, piece = (lane >> 4) * CE;
  const int n0 = blockIdx.x * 16;
  const int wr = min(n0 + row, a.N - 1);
  const T* W = static_cast<const T*>(a.W) + (long)wr * a.ldw;
  const T* x[MT];
  bool on[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long m = i * 16 + row;
    on[i] = m < a.M;
    x[i] = static_cast<const T*>(a.x) + (on[i] ? m : 0) * a.ldx;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (long k0 = (long)wave * STEP; k0 < a.K; k0 += WAVES * STEP) {
    u32x4 w[U], v[MT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = load_piece(W, k0 + u * 4 * CE + piece, a.K, a.vec, true);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int u = 0; u < U; ++u) v[i][u] = load_piece(x[i], k0 + u * 4 * CE + piece, a.K, a.vec, on[i]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = Mfma<T>::mul(w[u], v[i][u], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave < MT) {
    f32x4 s = red[0][wave][lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) s += red[k][wave][lane];
    const long m = wave * 16 + row;
    const int n = n0 + (lane >> 4) * 4;
    float o[4] = {s[0], s[1], s[2], s[3]};
    if (m < a.M && n < a.N) finish4<T>(a.e, a.N, m, n, o);
  }
}

// rows copied with their k padded by zeros to whole 16-byte pieces (rows that do not start on 16 bytes): one operand, or both in a launch
template <typename T>
struct Rows {
  const T* src;
  long ld, R;
  T* dst;
};
template <typename T>
__global__ void __launch_bounds__(256) pack_rows(Rows<T> x, Rows<T> w, unsigned first, int C, int Cp) {
  constexpr int CE = 16 / sizeof(T);
  const int per = Cp / CE;
  const bool is_x = blockIdx.x < first;
  const T* src = is_x ? x.src : w.src;
  T* dst = is_x ? x.dst : w.dst;
  const long ld = is_x ? x.ld : w.ld, R = is_x ? x.R : w.R;
  const long id = (long)(blockIdx.x - (is_x ? 0 : first)) * 256 + threadIdx.x;
  if (id >= R * per) return;
  const long r = id / per;
  const int c = (int)(id % per) * CE;
  *reinterpret_cast<u32x4*>(dst + r * Cp + c) = load_piece(src + r * ld, c, C, false, true);
}

// eight neighbouring elements of row r from column c on: zeros behind C and R
template <typename T>
__device__ __forceinline__ void load8(const T* src, long ld, long R, int C, long r, int c, float (&v)[8]) {
  if (r < R && c + 8 <= C) {
    tb_load_u(src + r * ld + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r < R && c + i < C ? (float)src[r * ld + c + i] : 0.f;
  }
}
// row c of the tile's columns r0 + x0 .. + 8, each through f, to dst[c][r], whose rows are Rp long (a multiple of 16 bytes)
template <typename T, typename F>
__device__ __forceinline__ void store_column(const float (&t)[64][65], int c, int x0, T* dst, long Rp, long r0, F&& f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = f(t[x0 + i][c]);
  constexpr int W = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += W) {
    if (r0 + x0 + i < Rp) {
      float w[W];
#pragma unroll
      for (int j = 0; j < W; ++j) w[j] = v[i + j];
      tb_store_n(dst + r0 + x0 + i, w);
    }
  }
}

// dst[c][r] = src[r][c]; dst's rows are padded by zeros to Rp.  64 x 64 a block, 16 bytes an access on both sides.
template <typename T>
struct Across {
  const T* src;
  long ld, R;
  int C;
  T* dst;
  long Rp;
  unsigned blocks;
};
template <typename T>
__device__ __forceinline__ void across_block(const Across<T>& a, unsigned block, float (&t)[64][65]) {
  const unsigned nr = (unsigned)((a.Rp + 63) / 64);
  const long r0 = (long)(block % nr) * 64;
  const int c0 = (int)(block / nr) * 64, x = (threadIdx.x & 7) * 8, y = threadIdx.x >> 3;
#pragma unroll
  for (int i = 0; i < 64; i += 32) {
    float v[8];
    load8(a.src, a.ld, a.R, a.C, r0 + y + i, c0 + x, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) t[y + i][x + j] = v[j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 64; i += 32)
    if (c0 + y + i < a.C) store_column<T>(t, y + i, x, a.dst + (long)(c0 + y + i) * a.Rp, a.Rp, r0, [](float v) { return v; });
}

// dz = dy act'(z) in both orders, each nullable, in one part or two, and the column sums of each 64 rows (fp32, before dz is rounded)
template <typename T>
struct DzArgs {
  const T* dy;
  long ldy;
  const float* z;
  int act, N, Np;
  long M, Mp;
  T *dz, *dzT;
  T *lo, *loT;         // two parts: the second ones, where the first are
  bool two;
  float* part;
  unsigned blocks;
};
template <typename T>
__device__ __forceinline__ void dz_block(const DzArgs<T>& a, unsigned block, float (&t)[64][65], float (&red)[4][64]) {
  const unsigned nr = (unsigned)((a.M + 63) / 64), br = block % nr;
  const long r0 = (long)br * 64;
  const int c0 = (int)(block / nr) * 64, x = (threadIdx.x & 7) * 8, y = threadIdx.x >> 3;
#pragma unroll
  for (int i = 0; i < 64; i += 32) {
    const long r = r0 + y + i;
    float v[8], p[8];
    load8(a.dy, a.ldy, a.M, a.N, r, c0 + x, v);
    if (a.z) {
      load8(a.z, (long)a.N, a.M, a.N, r, c0 + x, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= act_grad(p[j], a.act);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) t[y + i][x + j] = v[j];
    if (a.dz && r < a.M) {
      constexpr int W = 16 / sizeof(T);
      auto put = [&](T* dst, auto&& f) {
#pragma unroll
        for (int k = 0; k < 8; k += W)
          if (c0 + x + k < a.Np) {
            float w[W];
#pragma unroll
            for (int j = 0; j < W; ++j) w[j] = f(v[k + j]);
            tb_store_n(dst + r * a.Np + c0 + x + k, w);
          }
      };
      if (a.two) {
        put(a.dz, [](float q) { return Halves<T>::hi(q); });
        put(a.lo, [](float q) { return Halves<T>::lo(q); });
      } else {
        put(a.dz, [](float q) { return q; });
      }
    }
  }
  __syncthreads();
  if (a.dzT) {
#pragma unroll
    for (int i = 0; i < 64; i += 32)
      if (c0 + y + i < a.N) {
        const long at = (long)(c0 + y + i) * a.Mp;
        if (a.two) {
          store_column<T>(t, y + i, x, a.dzT + at, a.Mp, r0, [](float q) { return Halves<T>::hi(q); });
          store_column<T>(t, y + i, x, a.loT + at, a.Mp, r0, [](float q) { return Halves<T>::lo(q); });
        } else {
          store_column<T>(t, y + i, x, a.dzT + at, a.Mp, r0, [](float q) { return q; });
        }
      }
  }
  if (a.part) {
    const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += t[q * 16 + i][c];
    red[q][c] = s;
    __syncthreads();
    if (q == 0 && c0 + c < a.N) a.part[(long)br * a.N + c0 + c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
  }
}

// what the backward products read, in one launch: dz, W and x with their axes exchanged (each may have no blocks)
template <typename T>
__global__ void __launch_bounds__(256) lay_out(DzArgs<T> z, Across<T> w, Across<T> x) {
  __shared__ float t[64][65];
  __shared__ float red[4][64];
  if (blockIdx.x < z.blocks) dz_block<T>(z, blockIdx.x, t, red);
  else if (blockIdx.x < z.blocks + w.blocks) across_block<T>(w, blockIdx.x - z.blocks, t);
  else across_block<T>(x, blockIdx.x - z.blocks - w.blocks, t);
}

constexpr int FEW = 32;     // rows up to which the kernel for few rows is taken

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Plan {
  bool big;
  int tm, tn, splits, per;
};
// 256 x 256 tiles where they fill the chip, whatever K: 128 x 128 ones (two blocks a unit) move twice the operands and win nothing even
// where prologue and epilogue are most of the time.  K = 64, 128, 256, 512, 1024, 2048, us with 256 (128): 65536 x K x 256 bf16 14 (14), 17 (17), 20 (23),
// 27 (33), 41 (53), 86 (112), fp32 35 (35), 51 (53), 83 (86), 145 (156), 265 (284), 484 (523); 16384 x K x 4096 bf16 45 (45), 53 (53), 66 (70), 93 (98),
// 142 (165), 241 (308).  128 x 128 otherwise; k is split where even those leave units
// idle, into parts of sixteen k tiles (1 KB of a row) at least, of fp32, whose products take longer a byte, of four: 1000 x 1000 x 1000
// fp32 in parts of 16, 8, 4, 2 tiles 33.5, 29.9, 29.6, 29.7 us, 241 x 2048 x 272 24.5, 18.2, 16.4, 16.4; 1024 x 1024 x 1024 bf16
// 16.7, 20.4, 20.4, 20.5.
Plan plan(long M, int N, long K, int esize, bool down = false, int parts = 1) {
  Plan p;
  const long cus = tb_num_cus(), kt = (K * esize + 63) / 64 * parts;
  const long big = ((M + 255) / 256) * ((N + 255) / 256);
  p.big = big >= cus && !down;
  const int b = p.big ? 256 : 128;
  p.tm = (int)((M + b - 1) / b);
  p.tn = (N + b - 1) / b;
  const long tiles = (long)p.tm * p.tn;
  long s = 1;
  if (!p.big && tiles <= cus / 2) {
    s = cus / tiles;
    const int least = esize == 4 ? 4 : 16;
    if (s > kt / least) s = kt / least;
    if (s > 64) s = 64;
    if (s < 1) s = 1;
  }
  p.per = (int)((kt + s - 1) / s);
  p.splits = (int)((kt + p.per - 1) / p.per);
  return p;
}
size_t slab_bytes(long M, int N, long K, int esize, bool down = false, int parts = 1) {
  const Plan p = plan(M, N, K, esize, down, parts);
  return p.splits > 1 ? tb_align_up((size_t)p.splits * M * N * 4, 256) : 0;
}

template <typename T>
GemmArgs gemm_args(const Plan& p, const T* P, long ldp, const T* Q, long ldq, long M, int N, long K, Epi e, float* slab, const T* lo = nullptr) {
  GemmArgs a{P, Q, lo, ldp, ldq, M, N, (int)K, p.tm, p.tn, p.splits, p.per, 16 / (int)sizeof(T), e};
  auto whole = [&](int w) {
    const uintptr_t bytes = w * sizeof(T);
    return N % w == 0 && (!e.res || e.ldr % w == 0) && reinterpret_cast<uintptr_t>(e.y) % bytes == 0 && reinterpret_cast<uintptr_t>(e.res) % bytes == 0 &&
           reinterpret_cast<uintptr_t>(e.bias) % bytes == 0 && reinterpret_cast<uintptr_t>(e.z) % (w < 4 ? w * 4 : 16) == 0;
  };
  while (a.width > 1 && !whole(a.width)) a.width /= 2;
  a.e.slab = p.splits > 1 ? slab : nullptr;
  return a;
}

unsigned split_blocks(const GemmArgs& a) { return a.splits > 1 ? (unsigned)((a.M * ((a.N + 3) / 4) + 63) / 64) : 0; }

template <typename T, bool DOWN>
int launch(const GemmArgs& a, bool big, hipStream_t s) {
  const dim3 grid(a.tm * a.tn, a.splits);
  auto one = [&](auto two) {
    if constexpr (DOWN) gemm<T, 128, 128, 64, 64, true, two><<<grid, 256, 0, s>>>(a);
    else if (big) gemm<T, 256, 256, 128, 64, false, two><<<grid, 512, 0, s>>>(a);
    else gemm<T, 128, 128, 64, 64, false, two><<<grid, 256, 0, s>>>(a);
  };
  if constexpr (sizeof(T) == 2) {
    if (a.lo) one(std::true_type{});
    else one(std::false_type{});
  } else {
    one(std::false_type{});
  }
  TB_LAUNCH_CHECK("linres gemm");
  return TB_OK;
}

// an operand the matrix kernel can copy: rows on 16 bytes, whole 16-byte pieces of k
template <typename T>
bool direct(const void* p, long ld, long K) { return aligned(p) && ld % (16 / (long)sizeof(T)) == 0 && K % (16 / (long)sizeof(T)) == 0; }

long up(long x, int esize) { return (x + 16 / esize - 1) / (16 / esize) * (16 / esize); }

// What a forward call does with its operands and workspace: asked by who sizes the workspace and by the call itself.
struct FwdLayout {
  bool few, pack_x, pack_w;
  long Kp;
  Plan p;
  size_t x, w, slab, total;        // bytes of the copies of x and W, and of the split sums
};
template <typename T>
FwdLayout fwd_layout(const void* x, long ldx, const void* W, long ldw, long M, int K, int N) {
  constexpr int es = sizeof(T);
  FwdLayout l{};
  l.few = M <= FEW;
  l.Kp = up(K, es);
  if (!l.few) {
    l.pack_x = !direct<T>(x, ldx, K);
    l.pack_w = !direct<T>(W, ldw, K);
    l.p = plan(M, N, l.Kp, es);
    l.x = l.pack_x ? tb_align_up((size_t)M * l.Kp * es, 256) : 0;
    l.w = l.pack_w ? tb_align_up((size_t)N * l.Kp * es, 256) : 0;
    l.slab = slab_bytes(M, N, l.Kp, es);
  }
  l.total = l.x + l.w + l.slab + 256;
  return l;
}

template <typename T>
int forward(const T* x, long ldx, const T* W, long ldw, Epi e, long M, int K, int N, char* ws, size_t ws_bytes, hipStream_t s) {
  constexpr int CE = 16 / sizeof(T);
  const FwdLayout l = fwd_layout<T>(x, ldx, W, ldw, M, K, N);
  if (ws_bytes < l.total) return tb_set_error(TB_ERR_WORKSPACE, "linres_fwd: workspace too small");
  if (l.few) {
    FewArgs a{x, W, ldx, ldw, M, N, K, 0, e};
    a.vec = direct<T>(x, ldx, K) && direct<T>(W, ldw, K);
    const unsigned grid = (N + 15) / 16;
    if (M <= 16) gemm_few<T, 1, 8><<<grid, 512, 0, s>>>(a);
    else gemm_few<T, 2, 8><<<grid, 512, 0, s>>>(a);
    TB_LAUNCH_CHECK("linres gemm_few");
    return TB_OK;
  }
  const long Kp = l.Kp;
  T* xp = reinterpret_cast<T*>(ws);
  T* wp = reinterpret_cast<T*>(ws + l.x);
  const long bx = l.pack_x ? (M * (Kp / CE) + 255) / 256 : 0, bw = l.pack_w ? ((long)N * (Kp / CE) + 255) / 256 : 0;
  if (!tb_grid_ok(bx + bw, 256))
    return tb_set_error(TB_ERR_UNSUPPORTED, "linres_fwd: M=%ld K=%d N=%d, off the alignment of 16 bytes, are too many in one call", M, K, N);
  if (bx + bw) {
    pack_rows<T><<<(unsigned)(bx + bw), 256, 0, s>>>(Rows<T>{x, ldx, M, xp}, Rows<T>{W, ldw, N, wp}, (unsigned)bx, K, (int)Kp);
    TB_LAUNCH_CHECK("linres pack");
  }
  if (l.pack_x) {
    x = xp;
    ldx = Kp;
  }
  if (l.pack_w) {
    W = wp;
    ldw = Kp;
  }
  const GemmArgs a = gemm_args<T>(l.p, x, ldx, W, ldw, M, N, Kp, e, reinterpret_cast<float*>(ws + l.x + l.w));
  const int rc = launch<T, false>(a, l.p.big, s);
  if (rc || a.splits == 1) return rc;
  split_finish<T><<<split_blocks(a), 256, 0, s>>>(a.e, M, N, a.splits);
  TB_LAUNCH_CHECK("linres split_finish");
  return TB_OK;
}

// rows of what the backward pass lays out start on whole lines (a row off them costs its copies another line each)
long pitch(long x, int esize) { return (x + 128 / esize - 1) / (128 / esize) * (128 / esize); }

// The same of a backward call: which of dx, dW and db are wanted, and whether there is an activation, decide too.
struct BwdLayout {
  bool as_is, down, across, two;   // dz is dy and can be copied as it lies; dW from dz and x as they are, or from both across; dz in two parts
  long Np, Mp, Kw, Kx;
  Plan pw, px;
  size_t dz, dzT, WT, xT, part, slab_x, slab_w, total;      // bytes; dz and dzT with both parts, one behind the other
};
template <typename T>
BwdLayout bwd_layout(const void* dy, long ldy, const void* x, long ldx, int act, bool dx, bool dW, bool db, long M, int K, int N) {
  constexpr int es = sizeof(T);
  BwdLayout l{};
  l.two = es == 2 && act && act != 3;                   // dy act'(z) of relu is dy or 0: one value holds it
  l.as_is = !act && direct<T>(dy, ldy, N);
  l.down = es == 4 && dW && direct<T>(x, ldx, K);
  l.across = dW && !l.down;
  l.Np = pitch(N, es);
  l.Mp = pitch(M, es);
  l.Kw = l.down ? M : up(M, es);
  l.Kx = up(N, es);
  const int parts = l.two ? 2 : 1;
  l.pw = plan(N, K, l.Kw, es, l.down, parts);
  l.px = plan(M, K, l.Kx, es, false, parts);
  l.dz = !l.as_is && (dx || l.down) ? tb_align_up((size_t)M * l.Np * es, 256) * parts : 0;
  l.dzT = l.across ? tb_align_up((size_t)N * l.Mp * es, 256) * parts : 0;
  l.WT = dx ? tb_align_up((size_t)K * l.Np * es, 256) : 0;
  l.xT = l.across ? tb_align_up((size_t)K * l.Mp * es, 256) : 0;
  l.part = db ? tb_align_up((size_t)((M + 63) / 64) * N * 4, 256) : 0;
  l.slab_x = dx ? slab_bytes(M, K, l.Kx, es, false, parts) : 0;
  l.slab_w = dW ? slab_bytes(N, K, l.Kw, es, l.down, parts) : 0;
  l.total = l.dz + l.dzT + l.WT + l.xT + l.part + l.slab_x + l.slab_w + 256;
  return l;
}

template <typename T>
int backward(const T* dy, long ldy, const T* x, long ldx, const T* W, long ldw, const float* z, int act, T* dx, T* dW, T* db, long M, int K,
             int N, char* ws, size_t ws_bytes, hipStream_t s) {
  const BwdLayout b = bwd_layout<T>(dy, ldy, x, ldx, act, dx, dW, db, M, K, N);
  if (ws_bytes < b.total) return tb_set_error(TB_ERR_WORKSPACE, "linres_bwd: workspace too small");
  const bool two = b.two, as_is = b.as_is, down = b.down, across = b.across;
  size_t used = 0;
  auto take = [&](size_t n) {
    char* p = n ? ws + used : nullptr;
    used += n;
    return p;
  };
  T* const dz = reinterpret_cast<T*>(take(b.dz));
  T* const dzT = reinterpret_cast<T*>(take(b.dzT));
  T* const WT = reinterpret_cast<T*>(take(b.WT));
  T* const xT = reinterpret_cast<T*>(take(b.xT));
  float* const part = reinterpret_cast<float*>(take(b.part));
  float* const slab_x = reinterpret_cast<float*>(take(b.slab_x));
  float* const slab_w = reinterpret_cast<float*>(take(b.slab_w));
  T* const lo = two && dz ? dz + b.dz / 2 / sizeof(T) : nullptr;
  T* const loT = two && dzT ? dzT + b.dzT / 2 / sizeof(T) : nullptr;
  const T* dzr = as_is ? dy : dz;
  const long ldz = as_is ? ldy : b.Np;

  auto tiles = [](long rows, long cols) { return ((rows + 63) / 64) * ((cols + 63) / 64); };
  const long nz = !as_is || across || db ? tiles(M, b.Np) : 0, nw = dx ? tiles(b.Np, K) : 0, nx = across ? tiles(b.Mp, K) : 0;
  if (!tb_grid_ok(nz + nw + nx, 256)) return tb_set_error(TB_ERR_UNSUPPORTED, "linres_bwd: M=%ld K=%d N=%d are too many in one call", M, K, N);
  if (nz + nw + nx) {
    DzArgs<T> az{dy, ldy, z, act, N, (int)b.Np, M, b.Mp, dz, dzT, lo, loT, two, part, (unsigned)nz};
    Across<T> aw{W, ldw, N, K, WT, b.Np, (unsigned)nw}, ax{x, ldx, M, K, xT, b.Mp, (unsigned)nx};
    lay_out<T><<<(unsigned)(nz + nw + nx), 256, 0, s>>>(az, aw, ax);
    TB_LAUNCH_CHECK("linres lay_out");
  }

  const long Kw = b.Kw, Kx = b.Kx;
  const Plan &pw = b.pw, &px = b.px;
  Epi ew{}, ex{};
  ew.y = dW;
  ex.y = dx;
  const GemmArgs gw = down ? gemm_args<T>(pw, dzr, ldz, x, ldx, N, K, Kw, ew, slab_w) : gemm_args<T>(pw, dzT, b.Mp, xT, b.Mp, N, K, Kw, ew, slab_w, loT);
  const GemmArgs gx = gemm_args<T>(px, dzr, ldz, WT, b.Np, M, K, Kx, ex, slab_x, lo);
  const long bw = (long)pw.tm * pw.tn * pw.splits, bx = (long)px.tm * px.tn * px.splits;
  if (dx && dW && !pw.big && !px.big && tb_grid_ok(bw + bx, 256)) {
    if constexpr (sizeof(T) == 4) {
      if (down) gemm_pair<T, true, false><<<(unsigned)(bw + bx), 256, 0, s>>>(gw, gx, (unsigned)bw);
      else gemm_pair<T, false, false><<<(unsigned)(bw + bx), 256, 0, s>>>(gw, gx, (unsigned)bw);
    } else {
      if (two) gemm_pair<T, false, true><<<(unsigned)(bw + bx), 256, 0, s>>>(gw, gx, (unsigned)bw);
      else gemm_pair<T, false, false><<<(unsigned)(bw + bx), 256, 0, s>>>(gw, gx, (unsigned)bw);
    }
    TB_LAUNCH_CHECK("linres gemm_pair");
  } else {
    if (dW) {
      int rc = TB_OK;
      if constexpr (sizeof(T) == 4) rc = down ? launch<T, true>(gw, false, s) : launch<T, false>(gw, pw.big, s);
      else rc = launch<T, false>(gw, pw.big, s);
      if (rc) return rc;
    }
    if (dx) {
      const int rc = launch<T, false>(gx, px.big, s);
      if (rc) return rc;
    }
  }
  EndArgs end{gw.e, gx.e, gw.M, gx.M, gw.N, gx.N, gw.splits, gx.splits, dW ? split_blocks(gw) : 0, dx ? split_blocks(gx) : 0,
              db ? (unsigned)((N + 3) / 4) : 0, part, (M + 63) / 64, N, db};
  if (end.bw + end.bx + end.bb) {
    backward_end<T><<<end.bw + end.bx + end.bb, 256, 0, s>>>(end);
    TB_LAUNCH_CHECK("linres backward_end");
  }
  return TB_OK;
}

int check_common(const char* what, long M, int K, int N, int act, int dtype) {
  if (M < 0 || K < 1 || N < 1) return tb_set_error(TB_ERR_ARG, "%s: bad sizes M=%ld K=%d N=%d", what, M, K, N);
  // Rows below 2^30, because DOWN puts columns that are not there 2^30 rows away; columns and k are 32-bit indexes up to a tile behind their
  // last one, which 4 million leave room for; and the tiles of each product are one launch.
  auto tiles = [](long a, long b) { return ((a + 127) / 128) * ((b + 127) / 128); };
  if (K > 4000000 || N > 4000000 || M > 1000000000L || !tb_grid_ok(tiles(M, N), 256) || !tb_grid_ok(tiles(M, K), 256) || !tb_grid_ok(tiles(N, K), 256))
    return tb_set_error(TB_ERR_UNSUPPORTED, "%s: M=%ld K=%d N=%d are too many in one call", what, M, K, N);
  if (act < 0 || act > TB_ACT_LAST) return tb_set_error(TB_ERR_UNSUPPORTED, "%s: activation %d is not supported", what, act);
  if (!tb_dtype_ok(dtype)) return tb_set_error(TB_ERR_ARG, "%s: bad element type %d", what, dtype);
  return TB_OK;
}

}  // namespace

extern "C" {

// enough for any operands of these sizes: none on 16 bytes, every gradient, an activation
size_t tb_linres_workspace_bytes(long M, int K, int N, int dtype, int backward) {
  if (M < 1 || K < 1 || N < 1 || !tb_dtype_ok(dtype)) return 256;
  const int es = (int)tb_dtype_size(dtype);
  if (!backward) {
    if (M <= FEW) return 256;
    const long Kp = up(K, es);
    return tb_align_up((size_t)M * Kp * es, 256) + tb_align_up((size_t)N * Kp * es, 256) + slab_bytes(M, N, Kp, es) + 256;
  }
  auto most = [&](auto of) {
    size_t m = 0;
    for (int parts = 1; parts <= (es == 2 ? 2 : 1); ++parts) {
      const size_t n = of(parts);
      if (n > m) m = n;
    }
    return m;
  };
  const long Np = pitch(N, es), Mp = pitch(M, es);
  const size_t across = most([&](int q) { return slab_bytes(N, K, up(M, es), es, false, q); }), down = es == 4 ? slab_bytes(N, K, M, es, true) : 0;
  return most([&](int q) { return (tb_align_up((size_t)M * Np * es, 256) + tb_align_up((size_t)N * Mp * es, 256)) * q; }) +
         tb_align_up((size_t)K * Np * es, 256) + tb_align_up((size_t)K * Mp * es, 256) + tb_align_up((size_t)((M + 63) / 64) * N * 4, 256) +
         most([&](int q) { return slab_bytes(M, K, up(N, es), es, false, q); }) + (across > down ? across : down) + 256;
}

size_t tb_linres_fwd_workspace_bytes(const void* x, long x_row_stride, const void* W, long w_row_stride, long M, int K, int N, int dtype) {
  if (M < 1 || K < 1 || N < 1 || !tb_dtype_ok(dtype)) return 256;
  if (dtype == TB_F32) return fwd_layout<float>(x, x_row_stride, W, w_row_stride, M, K, N).total;
  return fwd_layout<_Float16>(x, x_row_stride, W, w_row_stride, M, K, N).total;      // of bf16 too: layouts go by the element's size
}

size_t tb_linres_bwd_workspace_bytes(const void* dy, long dy_row_stride, const void* x, long x_row_stride, int act, int want_dx, int want_dW,
                                     int want_db, long M, int K, int N, int dtype) {
  if (M < 1 || K < 1 || N < 1 || !tb_dtype_ok(dtype)) return 256;
  if (dtype == TB_F32) return bwd_layout<float>(dy, dy_row_stride, x, x_row_stride, act, want_dx, want_dW, want_db, M, K, N).total;
  return bwd_layout<_Float16>(dy, dy_row_stride, x, x_row_stride, act, want_dx, want_dW, want_db, M, K, N).total;
}

int tb_linres_fwd(const void* x, long x_row_stride, const void* W, long w_row_stride, const void* b, const void* residual,
                  long residual_row_stride, void* y, float* z, long M, int K, int N, int act, int dtype, void* ws, size_t ws_bytes,
                  void* stream) {
  int rc = check_common("linres_fwd", M, K, N, act, dtype);
  if (rc) return rc;
  if (M == 0) return TB_OK;
  if (!x || !W || !y || !ws) return tb_set_error(TB_ERR_ARG, "linres_fwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* w = static_cast<char*>(ws);
  Epi e{b, residual, y, z, nullptr, residual_row_stride, act};
  if (dtype == TB_F32) return forward<float>((const float*)x, x_row_stride, (const float*)W, w_row_stride, e, M, K, N, w, ws_bytes, s);
  if (dtype == TB_BF16) return forward<__bf16>((const __bf16*)x, x_row_stride, (const __bf16*)W, w_row_stride, e, M, K, N, w, ws_bytes, s);
  return forward<_Float16>((const _Float16*)x, x_row_stride, (const _Float16*)W, w_row_stride, e, M, K, N, w, ws_bytes, s);
}

int tb_linres_bwd(const void* dy, long dy_row_stride, const void* x, long x_row_stride, const void* W, long w_row_stride, const float* z,
                  int act, void* dx, void* dW, void* db, long M, int K, int N, int dtype, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_common("linres_bwd", M, K, N, act, dtype);
  if (rc) return rc;
  if (M < 1) return tb_set_error(TB_ERR_ARG, "linres_bwd: no rows have no gradients to form here");
  if (!dy || (dx && !W) || (dW && !x) || (act && !z) || !ws) return tb_set_error(TB_ERR_ARG, "linres_bwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* w = static_cast<char*>(ws);
  const float* zz = act ? z : nullptr;
#define TB_BWD(T) \
  return backward<T>((const T*)dy, dy_row_stride, (const T*)x, x_row_stride, (const T*)W, w_row_stride, zz, act, (T*)dx, (T*)dW, (T*)db, M, K, N, w, ws_bytes, s)
  if (dtype == TB_F32) TB_BWD(float);
  if (dtype == TB_BF16) TB_BWD(__bf16);
  TB_BWD(_Float16);
#undef TB_BWD
}

}  // extern "C"

// fw_sequence.hip -- linear attention with a decay per head over rollout columns (include/fwrollout.h):
//
//   k_scan        one wave runs one sequence, head and slice of value columns through time in blocks of C tokens
//   k_scan16      the same on the 16-bit matrix products (bfloat16)
//   k_scan_join   joins the states of time segments when there are few sequences
//   k_token       the single-token form: reads the state once, writes it once (k_token_narrow: fewer than 4 columns)
//
// The mathematics.  With g = exp(log_decay) and S the state before a block of C tokens,
//   out_t = g^(t+1) S^T q_t + sum_{s<=t} g^(t-s) (q_t . k_s) v_s        S <- g^C S + sum_s g^(C-1-s) k_s v_s^T
// and an episode start at x cuts every product whose span crosses it (s < x <= t).  The gradients are the same scan:
//   dq = scan(dout, v, k);  dk = reversed scan(v, dout, q);  dv = reversed scan(k, q, dout)
// with the states transposed where the roles of k and v change, so one kernel serves all four, and the backward
// pass keeps nothing of the forward pass.
#include <algorithm>
#include <type_traits>

#include "fw_seq_common.hpp"

using namespace fwseq;

namespace {

constexpr int MAXDIM = 128;
constexpr int SCAN_WAVES = 4;  // waves per block; each is on its own, with its own share of LDS and no barrier

struct Operand {
  const void* p;
  int64_t st, sn, sh;
};
// Element (n, h, seg, k, v) at p + n sn + h sh + seg sg + (k / 4) k4 + (k % 4) k1 + (v / 4) v4 + (v % 4) v1: a caller's
// [Dk][Dv] or a segment's [Dk / 4][Dv][4] (four keys of a value column together: what a lane holds), either of them as
// it lies or with the roles of k and v exchanged.
struct State {
  float* p;
  int64_t sn, sh, sg;
  int32_t k4, k1, v4, v1;
};
struct Pass {
  Operand q, k, v, o;  // o.p NULL: only the state is wanted
  State in, out;       // p NULL: zeros / not wanted
  int32_t rev;         // runs from the last token to the first
  int32_t Dk, Dv;
};
struct ScanArgs {
  Pass pass[3];
  int32_t n_pass, H, n_slice, n_seg, run_seg;  // segments [0, run_seg) in processing order
  int64_t T, N, seg_len;
  const float* log_decay;
  const uint8_t* starts;
  int64_t starts_st, starts_sn;
  const int32_t* lengths;
  // [n_pass][N][H][n_seg]: what a segment multiplies a state with (a weight too small for float32 is 0, and 0 x inf a NaN as
  // it should be), negative where an episode start cuts it off; or NULL
  float* factor;
};

// What one wave works on: unit = ((n H + h) n_slice + slice) n_pass + pass of segment blockIdx.y, so that the waves of a block
// want the same rows (slices and passes) or neighbouring ones (heads).  They are not in step, and little of that meets in the
// caches: the three backward passes over 2048 x 16 ragged x 16 heads of 64 x 64 bfloat16 read 386 MB, of 427 without any of it.
struct Unit {
  int pass, slice, h, seg;  // seg in processing order
  int64_t n, seg0, seg1, L;  // the segment's tokens [seg0, seg1), of which the first L are live
  __device__ __forceinline__ bool decode(const ScanArgs& A) {
    uint32_t u = blockIdx.x * SCAN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    pass = (int)(u % (uint32_t)A.n_pass);
    u /= (uint32_t)A.n_pass;
    slice = (int)(u % (uint32_t)A.n_slice);
    u /= (uint32_t)A.n_slice;
    h = (int)(u % (uint32_t)A.H);
    n = u / (uint32_t)A.H;
    seg = blockIdx.y;
    if (n >= A.N) return false;
    seg0 = (A.pass[pass].rev ? A.n_seg - 1 - seg : seg) * A.seg_len;
    seg1 = min(seg0 + A.seg_len, A.T);
    int64_t len = A.T;
    if (A.lengths) len = max((int64_t)0, min(A.T, (int64_t)A.lengths[n]));
    L = max((int64_t)0, min(len, seg1) - seg0);
    return true;
  }
};


// D fills the tiles; whole vectors in or out; rows of any length at any address, through registers
enum { FULL, GUARD, ANY };

// Element j of the result on lane x of four is element x of lane j's argument.
template <int CTRL>
__device__ __forceinline__ float quad_perm(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ f32x4 quad_turn(f32x4 y, int x) {
#pragma unroll
  for (int j = 0; j < 4; j += 2) {  // lanes 1 apart
    const float t = quad_perm<0xB1>(x & 1 ? y[j] : y[j + 1]);
    y[j] = x & 1 ? t : y[j];
    y[j + 1] = x & 1 ? y[j + 1] : t;
  }
#pragma unroll
  for (int j = 0; j < 2; j++) {  // lanes 2 apart
    const float t = quad_perm<0x4E>(x & 2 ? y[j] : y[j + 2]);
    y[j] = x & 2 ? t : y[j];
    y[j + 2] = x & 2 ? y[j + 2] : t;
  }
  return y;
}

__device__ __forceinline__ float finite_decay(float ld) { return ld < -1e30f ? -1e30f : ld; }  // g^0 = 1 for g = 0 too
// exp(ld m).  The product's rounding, 2^-24 of an exponent of up to 100, would be an error of the weight: it is carried along.
__device__ __forceinline__ float exponent_rest(float ld, float m) { return fmaf(ld, m, -(ld * m)); }
__device__ __forceinline__ float power_of(float ld, float m) {
  const float x = expf(ld * m);
  return fmaf(x, exponent_rest(ld, m), x);
}

// S becomes g^c S + D, D the sum of what a block adds: near g^c = 1 as S + (S (g^c - 1) + D), rounded once at the size of S, so
// that a long memory does not gather an error per token; below 1/2 with g^c itself, of which g^c - 1 holds too little (at
// g^c = 1e-4, three digits).  One form for both, without a branch: keep is 1 or 0.
struct Decay {
  float keep, by;
  __device__ __forceinline__ void set(float ld, float c) {
    const bool near = ld * c > -0.69f;
    keep = near ? 1.f : 0.f;
    const float x = near ? expm1f(ld * c) : expf(ld * c);
    by = fmaf(keep + x, exponent_rest(ld, c), x);
  }
  __device__ __forceinline__ float operator()(float s, float d) const { return fmaf(s, keep, fmaf(s, by, d)); }
};

// The state as a wave holds it: lane 16 g + r, key column 4 KT g + e, value column dv(f), in S[e % KT][f][e / KT] (WIDE)
// or S[e / 4][f][e % 4].  Four keys move as one access where they lie together.
template <int MODE, bool WIDE, int KT, int VT, typename Col>
__device__ __forceinline__ void load_state(f32x4 (&S)[KT][VT], const State& st, const float* s, int Dk, int Dv, int g,
                                           Col dv) {
  auto set = [&](int e, int f, float x) {
    if (WIDE)
      S[e % KT][f][e / KT] = x;
    else
      S[e / 4][f][e % 4] = x;
  };
  // a segment's state with the roles exchanged: four lanes' columns by four keys lie together, row by row
  if (!WIDE && st.sg && st.v1 == 1) {
    const int x = threadIdx.x & 3;
#pragma unroll
    for (int f = 0; f < VT; f++) {
      const int v4 = MODE == FULL ? dv(f) >> 2 : min(dv(f) >> 2, (Dv - 1) >> 2);
#pragma unroll
      for (int a = 0; a < KT; a++) {
        const int k = 4 * KT * g + 4 * a + x;
        S[a][f] = quad_turn(*(const f32x4*)(s + v4 * st.v4 + (MODE == FULL ? k : min(k, Dk - 1)) * st.k1), x);
      }
    }
    return;
  }
  const bool four = st.k1 == 1 && ((uintptr_t)s | (st.k4 | st.v4 | st.v1) * 4) % 16 == 0;
#pragma unroll
  for (int f = 0; f < VT; f++) {  // outside Dk x Dv: the last row or column, which nothing reads
    const int v = MODE == FULL ? dv(f) : min(dv(f), Dv - 1);
    const float* c = s + (v >> 2) * st.v4 + (v & 3) * st.v1;
    if (four) {
#pragma unroll
      for (int x = 0; x < KT; x++) {
        const int q = MODE == FULL ? KT * g + x : min(KT * g + x, (Dk - 1) >> 2);
        const f32x4 y = *(const f32x4*)(c + q * st.k4);
#pragma unroll
        for (int i = 0; i < 4; i++) set(4 * x + i, f, y[i]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4 * KT; e++) {
        const int k = MODE == FULL ? 4 * KT * g + e : min(4 * KT * g + e, Dk - 1);
        set(e, f, c[(k >> 2) * st.k4 + (k & 3) * st.k1]);
      }
    }
  }
}
template <int MODE, bool WIDE, int KT, int VT, typename Col>
__device__ __forceinline__ void store_state(const f32x4 (&S)[KT][VT], const State& st, float* s, int Dk, int Dv, int g,
                                            Col dv) {
  auto at = [&](int e, int f) { return WIDE ? S[e % KT][f][e / KT] : S[e / 4][f][e % 4]; };
#pragma unroll
  for (int f = 0; f < VT; f++)
    if (MODE == FULL || dv(f) < Dv) {
      float* c = s + (dv(f) >> 2) * st.v4 + (dv(f) & 3) * st.v1;
      if (st.sg) {  // a segment's state
#pragma unroll
        for (int x = 0; x < KT; x++)
          if (MODE == FULL || 4 * (KT * g + x) < Dk)
            *(f32x4*)(c + (KT * g + x) * st.k4) = f32x4{at(4 * x, f), at(4 * x + 1, f), at(4 * x + 2, f), at(4 * x + 3, f)};
      } else {
#pragma unroll
        for (int e = 0; e < 4 * KT; e++) {
          const int k = 4 * KT * g + e;
          if (MODE == FULL || k < Dk) c[(k >> 2) * st.k4 + (k & 3) * st.k1] = at(e, f);
        }
      }
    }
}

// Each active lane copies 16 bytes (or 1) from base + off to its own place behind `lds`: lane x 16 (x 4) bytes.  base and
// lds are the same on all lanes.  There is no result to wait for by register: the reader waits on the count of memory
// operations.  Written as asm because a copy known to the compiler makes it wait for ALL copies before any LDS read; the
// five wait states are those between a VALU write of the base and its use (the compiler does not look into asm).  m0 is a
// register that the compiler never keeps anything in from one statement to the next (it warns where one is said to
// overwrite it), so none is named.
__device__ __forceinline__ uint64_t uniform(const void* p) {
  const uint64_t x = (uint64_t)p;
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}
__device__ __forceinline__ uint32_t lds_address(const char* lds) {
  return __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds);
}
__device__ __forceinline__ void copy16(const void* base, uint32_t off, char* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_address(lds)), "v"(off),
               "s"(uniform(base))
               : "memory");
}
__device__ __forceinline__ void copy1(const void* base, uint32_t off, char* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_ubyte %1, %2" ::"s"(lds_address(lds)), "v"(off),
               "s"(uniform(base))
               : "memory");
}

// the same value, but not known to be: keeps what a rare branch computes from it inside that branch
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

typedef u32x4 __attribute__((aligned(4))) u32x4_any4;
typedef u32x4 __attribute__((aligned(2))) u32x4_any2;

// x is computed here, not later: without it the compiler puts off a block's sums until registers run out
template <bool ON>
__device__ __forceinline__ void pin(f32x4& x) {
  if (ON) asm volatile("" : "+v"(x));
}

// ROWS rows of 16 NT columns in LDS, as 16-byte chunks; chunk c of a row is stored at c ^ turn(row), so that the 16
// lanes that are served together meet in no bank: 16 rows of one chunk, or (TRANSPOSED) 4 rows of 4 half chunks
template <typename T, int NT, int ROWS, bool TRANSPOSED = false>
struct Tile {
  static constexpr int PER = 16 / sizeof(T), CH = 16 * NT / PER, BYTES = ROWS * CH * 16;
  static constexpr int RI = 64 / CH, NI = (ROWS + RI - 1) / RI;  // RI rows per copy instruction
  __device__ static __forceinline__ int turn(int row) {
    if (TRANSPOSED && NT == 4) return (row >> 1 & 1) * 4;
    return (CH >= 16 ? row : row / (16 / CH)) & ((CH < 16 ? CH : 16) - 1);
  }
  __device__ static __forceinline__ int at(int row, int chunk) { return (row * CH + (chunk ^ turn(row))) * 16; }

  // copies the rows of a block of c rows; row u is token u, or c - 1 - u when reversed; rows behind the block repeat
  // its last one.  Chunks outside D are left as they are (zeros).  base: the block's first token.
  template <int MODE, bool WHOLE>
  __device__ static __forceinline__ void fetch(char* lds, const T* base, int64_t st, int D, int c, bool rev, int lane) {
    const int row0 = lane / CH, pc = lane % CH;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int row = i * RI + row0, col = (pc ^ turn(row)) * PER;
      if ((RI <= ROWS || row < ROWS) && (MODE == FULL || col < D)) {
        // uniform base + 32-bit lane offset (the launcher saw that a block's rows fit)
        if constexpr (WHOLE) {  // c = ROWS
          const int first = rev ? ROWS - RI - i * RI : i * RI;
          copy16(base + first * st, ((rev ? RI - 1 - row0 : row0) * (uint32_t)st + col) * (uint32_t)sizeof(T),
                 lds + i * 1024);
        } else {
          const int u = min(row, c - 1);
          copy16(base, ((rev ? c - 1 - u : u) * (uint32_t)st + col) * (uint32_t)sizeof(T), lds + i * 1024);
        }
      }
    }
  }

  // The same rows at any address and of any length, by way of registers: `hold` asks for them, `commit` writes them with
  // zeros behind D.  A row's last chunk is read from where it ends with the row and moved down into place, so nothing
  // outside the row is read.  whole: a row has a chunk at all (base may be some columns into it); else commit reads it by
  // elements.  Addresses are worked out each time: kept, they would take the registers that hold the rows.
  using any16 = std::conditional_t<sizeof(T) == 4, u32x4_any4, u32x4_any2>;
  __device__ static __forceinline__ const T* source(const T* base, int64_t st, int row, int c, bool rev) {
    const int u = min(row, c - 1);
    return base + (int64_t)(rev ? c - 1 - u : u) * st;
  }
  __device__ static __forceinline__ void hold(u32x4 (&held)[NI], const T* base, int64_t st, int D, bool whole, int c,
                                              bool rev, int lane) {
    if (!whole) return;
    lane = here(lane);
    const int row0 = lane / CH, pc = lane % CH;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int row = i * RI + row0, col = (pc ^ turn(row)) * PER;
      held[i] = *(const any16*)(source(base, st, row, c, rev) + min(col, D - PER));
    }
  }
  __device__ static __forceinline__ void commit(char* lds, const u32x4 (&held)[NI], const T* base, int64_t st, int D,
                                                bool whole, int c, bool rev, int lane) {
    lane = here(lane);
    const int row0 = lane / CH, pc = lane % CH;
    if (whole) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int row = i * RI + row0, col = (pc ^ turn(row)) * PER;
        u32x4 v = held[i];
        const int by = (col - min(col, D - PER)) * (int)sizeof(T) * 8;  // bits; 128 and more: outside
        uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
        lo = by & 64 ? hi : lo;
        hi = by & 64 ? 0 : hi;
        lo = lo >> (by & 63) | (hi << 1) << (63 - (by & 63));
        hi >>= by & 63;
        const uint32_t in = by < 128 ? ~0u : 0u;
        v = u32x4{(uint32_t)lo & in, (uint32_t)(lo >> 32) & in, (uint32_t)hi & in, (uint32_t)(hi >> 32) & in};
        if (RI <= ROWS || row < ROWS) *(u32x4*)(lds + (i * 64 + lane) * 16) = v;
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < NI * PER; i++) {
        const int row = i / PER * RI + row0, col = (pc ^ turn(row)) * PER + i % PER;
        const T x = col < D ? source(base, st, row, c, rev)[col] : T{};
        if (RI <= ROWS || row < ROWS) ((T*)(lds + (i / PER * 64 + lane) * 16))[i % PER] = x;
      }
    }
  }

  // the rows from LDS to memory, numbered as in fetch
  template <int MODE>
  __device__ static __forceinline__ void put(const char* lds, T* base, int64_t st, int D, int c, bool rev, int lane) {
    const int row0 = lane / CH, pc = lane % CH;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int row = i * RI + row0, col = (pc ^ turn(row)) * PER;
      if (RI > ROWS && row >= ROWS) continue;
      const Pack<T, PER> v = *(const Pack<T, PER>*)(lds + (i * 64 + lane) * 16);
      if (row < c && (MODE == FULL || col < D)) {
        const int64_t u = rev ? c - 1 - row : row;
        if constexpr (MODE == ANY) {
          T* x = base + u * st + col;
          if (col + PER <= D) {
            *(any16*)x = __builtin_bit_cast(u32x4, v);
          } else {
#pragma unroll
            for (int k = 0; k < PER; k++)
              if (col + k < D) x[k] = v.e[k];
          }
        } else {
          *(Pack<T, PER>*)((char*)base + ((uint32_t)u * (uint32_t)st + col) * (uint32_t)sizeof(T)) = v;
        }
      }
    }
  }
};

__device__ __forceinline__ f32x4 mma(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// One wave; lane = 16 g + r.  Operands of a 16x16x4 product: A row r, B column r, depth g; result: column r, rows
// 4 g + i.  Depths and rows may be numbered at will as long as both operands agree, and the numbering below makes
// every result register the operand register of the product that needs it, so nothing moves between lanes:
//   rows         a block of C = 16 tokens in processing order; depth step j of lane group g is row 4 g + j
//   key columns  4 KT g + e, e = KT i + a: row 4 g + i of state tile a
//   value cols   VT r + f (operand tile f), 4 VT g + VT i + f (result)
// S[a][f] = state tile (k columns a, v columns f); P[i] = weight x (k_s . q_t) for s = 4 g + i, t = r;
// O[f] = out^T: value columns down the rows, tokens along the columns.
// Blocks are copied to LDS by the load unit, NB of them ahead (no registers; the wait is for the oldest alone), in
// processing order, so that a reversed pass is causal too: its rows run from the last token to the first.
//
// float32 runs here because its products have to be float32; float16 because its states leave its range.  A wave owns a
// sequence rather than a block of tokens because the recurrence then never leaves its registers.  Small heads are bound
// by memory: 2048 tokens x 512 x 4 heads of 16 x 16, 285 us, 3790 GB/s (403 us with the loads by way of registers, none
// ahead).  Larger ones are bound by the products, which a padded head wastes: 500 x 250 x 4 heads of 20 x 40 in tiles of
// 32 x 32 and two slices, 96 us, of which 39 % of the products count.
template <typename T, int KT, int VT>
struct Ring {
  using K = Tile<T, KT, 16>;
  using V = Tile<T, VT, 16>;
  static constexpr int BYTES = 2 * K::BYTES + V::BYTES + 64;  // queries, keys, values, episode starts
  static constexpr int ROOM = 20480;                           // a wave's share of LDS: eight waves on a CU
  static constexpr int NB = BYTES * 4 <= ROOM ? 4 : BYTES * 3 <= ROOM ? 3 : BYTES * 2 <= ROOM ? 2 : 1;
};
template <int N>
__device__ __forceinline__ void wait_loads() {  // all but the N newest memory operations are done
  static_assert(N >= 0 && N < 64);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

template <typename T, int KT, int VT, int MODE>
__global__ __launch_bounds__(64 * SCAN_WAVES, KT * VT <= 16 ? 2 : 1) void k_scan(ScanArgs A) {
  constexpr int C = 16, TPL = 4;
  using R = Ring<T, KT, VT>;
  using K = typename R::K;
  using V = typename R::V;
  constexpr int NB = MODE == ANY ? 1 : R::NB;
  constexpr bool LATE = MODE == ANY && KT == 8 && VT == 2;  // no registers to hold the next block's rows beside this one's
  __shared__ alignas(16) char smem[SCAN_WAVES][NB * R::BYTES];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  char* const ring = smem[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
  Unit U;
  if (!U.decode(A)) return;
  const Pass p = A.pass[U.pass];
  const int64_t n = U.n, L = U.L;
  const int h = U.h, seg = U.seg;
  const bool rev = p.rev;
  const int Dk = p.Dk, Dv = p.Dv, v0 = U.slice * 16 * VT;
  const T* qb = (const T*)p.q.p + n * p.q.sn + h * p.q.sh + U.seg0 * p.q.st;
  const T* kb = (const T*)p.k.p + n * p.k.sn + h * p.k.sh + U.seg0 * p.k.st;
  const T* vb = (const T*)p.v.p + n * p.v.sn + h * p.v.sh + U.seg0 * p.v.st + v0;
  T* ob = (T*)p.o.p + n * p.o.sn + h * p.o.sh + U.seg0 * p.o.st + v0;
  const bool want_out = p.o.p != nullptr;
  const uint8_t* xb = A.starts ? A.starts + n * A.starts_sn + U.seg0 * A.starts_st : nullptr;
  const float ld = finite_decay(A.log_decay[h]);
  auto power = [&](int m) { return power_of(ld, (float)m); };

  // rows t0 .. t0 + c - 1 of the segment to a place of the ring: queries, keys and starts, then values
  auto fetch_k = [&](char* to, int64_t t0, int c) {
    auto go = [&](auto whole) {
      constexpr bool W = decltype(whole)::value;
      K::template fetch<MODE, W>(to + K::BYTES, kb + t0 * p.k.st, p.k.st, Dk, c, rev, lane);
      if (want_out) K::template fetch<MODE, W>(to, qb + t0 * p.q.st, p.q.st, Dk, c, rev, lane);
    };
    if (c == C)
      go(std::true_type());
    else
      go(std::false_type());
    if (xb && lane < c)
      copy1(xb + t0 * A.starts_st, (uint32_t)((rev ? c - 1 - lane : lane) * (int)A.starts_st), to + 2 * K::BYTES + V::BYTES);
  };
  auto fetch_v = [&](char* to, int64_t t0, int c) {
    if (c == C)
      V::template fetch<MODE, true>(to + 2 * K::BYTES, vb + t0 * p.v.st, p.v.st, Dv - v0, c, rev, lane);
    else
      V::template fetch<MODE, false>(to + 2 * K::BYTES, vb + t0 * p.v.st, p.v.st, Dv - v0, c, rev, lane);
  };
  if constexpr (MODE == GUARD) {
    for (int i = lane * 16; i < NB * R::BYTES; i += 1024) *(u32x4*)(ring + i) = u32x4{0, 0, 0, 0};
    wait_loads<0>();
  }
  // the first blocks
  int64_t asked = 0;  // tokens whose copy has been asked for
  int ahead = 0, slot = 0;
  auto fill = [&](int64_t from, int blocks, int size) {
    asked = from;
    slot = 0;
    for (ahead = 0; ahead < blocks && asked < L; ahead++) {
      const int c = (int)min((int64_t)size, L - asked);
      fetch_k(ring + ahead * R::BYTES, rev ? L - asked - c : asked, c);
      fetch_v(ring + ahead * R::BYTES, rev ? L - asked - c : asked, c);
      asked += c;
    }
  };
  if constexpr (MODE != ANY) fill(0, NB, C);
  // MODE ANY: one block ahead, in registers
  u32x4 hq[K::NI], hk[K::NI], hv[V::NI];
  uint32_t hx = 0;
  bool held = false;
  auto hold = [&](int64_t t0, int c) __attribute__((always_inline)) {
    constexpr int PER = K::PER;
    K::hold(hk, kb + t0 * p.k.st, p.k.st, Dk, Dk >= PER, c, rev, lane);
    if (want_out) K::hold(hq, qb + t0 * p.q.st, p.q.st, Dk, Dk >= PER, c, rev, lane);
    V::hold(hv, vb + t0 * p.v.st, p.v.st, Dv - v0, Dv >= PER, c, rev, lane);
    const int u = min(lane, c - 1);
    if (xb) hx = lane < c ? xb[(t0 + (rev ? c - 1 - u : u)) * A.starts_st] : 0;
    held = true;
  };
  if (MODE == ANY && L > 0) {
    const int c = (int)min((int64_t)C, L);
    hold(rev ? L - c : 0, c);
  }

  f32x4 S[KT][VT];
#pragma unroll
  for (int a = 0; a < KT; a++)
#pragma unroll
    for (int f = 0; f < VT; f++) S[a][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto column = [&](int f) { return v0 + VT * r + f; };
  if (p.in.p)
    load_state<MODE, true>(S, p.in, p.in.p + n * p.in.sn + h * p.in.sh + seg * p.in.sg, Dk, Dv, g, column);

  // Weights.  A reversed pass carries g x the state of the row before: its first weight is 1, and its final state is
  // the gradient of the initial one.
  const int e = rev ? 0 : 1;
  float wp[4], wi = power(r + e), wu[TPL];
  Decay decay;
  int cur = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) wp[i] = r >= 4 * g + i ? power(r - 4 * g - i) : 0.f;
  bool fresh = false;  // an episode start among the live tokens
  int64_t done = 0;
  int single = 0;  // blocks of one token still to go
  int steady = 0;  // blocks since the last fill
  // memory operations of a block: copies (and the starts'), stores where their number is certain
  constexpr int ND1 = V::NI + K::NI, ND2 = ND1 + K::NI;
  constexpr int NST = MODE == FULL ? V::NI : 0;
  while (done < L) {
    const int c = single ? 1 : (int)min((int64_t)C, L - done);
    const int64_t t0 = rev ? L - done - c : done;
    if constexpr (MODE == ANY) {
      if (!held) hold(t0, c);
      K::commit(ring + K::BYTES, hk, kb + t0 * p.k.st, p.k.st, Dk, Dk >= K::PER, c, rev, lane);
      if (want_out) K::commit(ring, hq, qb + t0 * p.q.st, p.q.st, Dk, Dk >= K::PER, c, rev, lane);
      V::commit(ring + 2 * K::BYTES, hv, vb + t0 * p.v.st, p.v.st, Dv - v0, Dv >= K::PER, c, rev, lane);
    } else {
      if (ahead == 0) {
        wait_loads<0>();
        fill(done, single ? 1 : NB, single ? 1 : C);
        steady = 0;
      }
      // Newer than this block's copies are those of the NB - 1 blocks behind it and, NB blocks after a fill, the stores
      // of the NB - 1 blocks before it.
      if (ahead < NB)
        wait_loads<0>();
      else if (!want_out)
        wait_loads<(NB - 1) * ND1>();
      else if (steady < NB)
        wait_loads<(NB - 1) * ND2>();
      else
        wait_loads<(NB - 1) * (ND2 + NST)>();
    }
    char* const lq = ring + slot * R::BYTES;
    char* const lk = lq + K::BYTES;
    char* const lv = lk + K::BYTES;
    uint32_t M = 0;  // bit u: an episode starts at row u
    if (xb) M = (uint32_t)__ballot(MODE == ANY ? hx != 0 : lane < c && *(const uint8_t*)(lv + V::BYTES + 4 * lane) != 0);
    // A start at row u of a forward pass cuts every span that contains row u but not from it on; in a reversed pass
    // the cut lies behind row u, that is at row u + 1.
    const uint32_t cut = rev ? M << 1 : M;

    f32x4 P{0.f, 0.f, 0.f, 0.f};
    f32x4 O[VT];
#pragma unroll
    for (int f = 0; f < VT; f++) O[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (want_out) {
      // columns 4 KT g .. of row r, in the accesses of 16 bytes (or fewer) that hold them
      constexpr int W = vec_elems<T>(4 * KT);
#pragma unroll
      for (int x = 0; x < 4 * KT; x += W) {
        if (x == 16) asm volatile("" ::: "memory");  // bounds the operands in registers at a time
        const int col = 4 * KT * g + x, byte = (col % K::PER) * (int)sizeof(T), o = K::at(r, col / K::PER) + byte;
        float Q[W], K1[W];
        load_vec<T, W>((const T*)(lq + o), Q);
        load_vec<T, W>((const T*)(lk + o), K1);
#pragma unroll
        for (int y = 0; y < W; y++) {
          P = mma(K1[y], Q[y], P);
#pragma unroll
          for (int f = 0; f < VT; f++) O[f] = mma(S[(x + y) % KT][f][(x + y) / KT], Q[y], O[f]);
        }
      }
    }
    float Vr[TPL][VT], K2[TPL][KT];
    float bad = 0.f;
#pragma unroll
    for (int j = 0; j < TPL; j++) {
      constexpr int WV = vec_elems<T>(VT), WK = vec_elems<T>(KT);
#pragma unroll
      for (int x = 0; x < VT; x += WV)
        load_vec<T, WV>((const T*)(lv + V::at(4 * g + j, (VT * r + x) / V::PER) + (VT * r + x) % V::PER * (int)sizeof(T)), Vr[j] + x);
#pragma unroll
      for (int x = 0; x < KT; x += WK)
        load_vec<T, WK>((const T*)(lk + K::at(4 * g + j, (KT * r + x) / K::PER) + (KT * r + x) % K::PER * (int)sizeof(T)), K2[j] + x);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every read of the block is done: its room is free
    if constexpr (MODE == ANY) asked = done + c;
    const bool more = !single && asked < L;  // a block to copy there; its values after the outputs have used their room
    const int c2 = (int)min((int64_t)C, L - asked);
    const int64_t t2 = rev ? L - asked - c2 : asked;
    if constexpr (MODE == ANY) {
      held = false;
      if (!LATE && more) hold(t2, c2);
    } else {
      if (more) {
        fetch_k(lq, t2, c2);
        asked += c2;
      } else {
        ahead--;
      }
      slot = slot + 1 == NB ? 0 : slot + 1;
      steady++;
    }

#pragma unroll
    for (int j = 0; j < TPL; j++)
#pragma unroll
      for (int f = 0; f < VT; f++) bad += Vr[j][f];
    // A masked product is a product with 0, which keeps a value away only while that value is finite.  A block with an
    // infinity or a NaN among its values is therefore run token by token: nothing is masked then.
    if (c > 1 && __any(!(fabsf(bad) < __builtin_huge_valf()))) {
      single = c;
      ahead = 0;
      held = false;
      continue;
    }
    fresh |= M != 0;
    if (c != cur) {
      cur = c;
      const int g4 = here(4 * g);
#pragma unroll
      for (int j = 0; j < TPL; j++) wu[j] = power(max(c - e - (g4 + j), 0));
      decay.set(ld, (float)c);
    }
    if (M != 0 || c < C) {
      const int g4 = here(4 * g);
#pragma unroll
      for (int j = 0; j < TPL; j++) {
        const bool live = g4 + j < c, open = (cut >> (g4 + j)) >> 1 == 0;
#pragma unroll
        for (int f = 0; f < VT; f++) Vr[j][f] = live ? Vr[j][f] : 0.f;
#pragma unroll
        for (int a = 0; a < KT; a++) K2[j][a] = live && open ? K2[j][a] : 0.f;
      }
    }
    if (want_out) {
#pragma unroll
      for (int f = 0; f < VT; f++) O[f] *= wi;
#pragma unroll
      for (int i = 0; i < 4; i++) P[i] = r >= 4 * g + i ? P[i] * wp[i] : 0.f;  // select, never multiply by 0
      if (M != 0) {
        const int g4 = here(4 * g), rr = here(r);
        if (cut & ((2u << rr) - 1))
#pragma unroll
          for (int f = 0; f < VT; f++) O[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (g4 + i < rr && ((cut >> (g4 + i)) >> 1 & ((1u << (rr - g4 - i)) - 1)) != 0) P[i] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < TPL; j++)
#pragma unroll
        for (int f = 0; f < VT; f++) O[f] = mma(Vr[j][f], P[j], O[f]);
      // through LDS, so that neighbouring lanes store neighbouring columns
      float x[4 * VT];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < VT; f++) x[VT * i + f] = O[f][i];
      constexpr int W = vec_elems<T>(4 * VT);
#pragma unroll
      for (int k = 0; k < 4 * VT; k += W) {
        const int col = 4 * VT * g + k;
        if (MODE != GUARD || col < Dv - v0)  // (the chunks outside stay zeros)
          store_vec<T, W>((T*)(lv + V::at(r, col / V::PER) + col % V::PER * (int)sizeof(T)), x + k);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      V::template put<MODE>(lv, ob + t0 * p.o.st, p.o.st, Dv - v0, c, rev, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (MODE != ANY && more) fetch_v(lq, t2, c2);

    if (M != 0) {
#pragma unroll
      for (int a = 0; a < KT; a++)
#pragma unroll
        for (int f = 0; f < VT; f++) S[a][f] = f32x4{0.f, 0.f, 0.f, 0.f};
      // a block of one token that a reversed pass cuts off behind itself: its value, perhaps an infinity, adds nothing
      if (rev && c == 1)
#pragma unroll
        for (int j = 0; j < TPL; j++)
#pragma unroll
          for (int f = 0; f < VT; f++) Vr[j][f] = 0.f;
    }
#pragma unroll
    for (int a = 0; a < KT; a++) {
      f32x4 D[VT];
#pragma unroll
      for (int f = 0; f < VT; f++) D[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < TPL; j++)
#pragma unroll
        for (int f = 0; f < VT; f++) D[f] = mma(K2[j][a] * wu[j], Vr[j][f], D[f]);
#pragma unroll
      for (int f = 0; f < VT; f++)
#pragma unroll
        for (int i = 0; i < 4; i++) S[a][f][i] = decay(S[a][f][i], D[f][i]);
#pragma unroll
      for (int f = 0; f < VT; f++) pin<KT * VT <= 16>(S[a][f]);
    }
    if constexpr (LATE)
      if (more) hold(t2, c2);
    done += c;
    if (single) single--;
  }

  if (p.out.p && (seg == A.n_seg - 1 || p.out.sg))
    store_state<MODE, true>(S, p.out, p.out.p + n * p.out.sn + h * p.out.sh + seg * p.out.sg, Dk, Dv, g, column);
  if (A.factor && U.slice == 0 && lane == 0)
    A.factor[((U.pass * A.N + n) * A.H + h) * A.n_seg + seg] = fresh ? -1.f : power_of(ld, (float)L);
  if (want_out) {  // rows behind the sequence's end
    for (int i = lane * 16; i < V::BYTES; i += 1024) *(u32x4*)(ring + i) = u32x4{0, 0, 0, 0};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    for (int64_t t = L; t < U.seg1 - U.seg0; t += C)
      V::template put<MODE>(ring, ob + t * p.o.st, p.o.st, Dv - v0, (int)min((int64_t)C, U.seg1 - U.seg0 - t), false, lane);
  }
}

// ------------------------------------------------------------------ bfloat16
// The same scan on the 16x16x32 product of bfloat16, in blocks of C = 32 tokens, the next block's rows copied to LDS
// while a block is computed.
//   rows         key tile z: row 16 z + r; query tile z: row 16 z + r; as depth j = 4 z + i of lane group g: row
//                16 z + 4 g + i -- the result registers of the score product are the operand of the value product
//   key columns  depth 8 s + j of lane group g: 4 KT g + 8 s + j; state tile a: 4 KT g + 4 a + i down its rows
//   value cols   tile f: VC (r >> 2) + 32 (f / 2) + 4 (f % 2) + (r & 3) across, VC = min(4 VT, 8), and so VC g + 32 (f / 2)
//                + 4 (f % 2) + i down: a lane has VC neighbours together
// Operands with tokens as depth (keys and values of the state's product, values of the output's) are read from LDS by
// the transposing read: 4 lanes x 4 columns of one row each become 4 rows x 1 column per lane.
// Products of the inputs are exact in the float32 accumulators.  What is not an input (weighted scores, the state, the
// weighted operand of the state's product) is split into three bfloat16 terms, so that every product is a float32 one: with
// two, terms that cancel leave 2^-16 of their size, and more outputs fall to the neighbouring bfloat16.
//
// 32 tokens a block: the depth of the product, and half as many splits of the state per token as 16.  Measured at 16
// heads of 128 x 128 over 16384 tokens: 108 us of outputs after 63 us of segment states (88 and 57 with two terms and the
// products added to the state one by one; on the float32 products 460 us in all).  In the 108 us the matrix units are busy for
// 30 % of the time and issue 4.0 million products beside 33 million vector instructions, the splits and weights; two waves a
// SIMD hide what they wait for only in part.  Three (the outputs in the values' room), the copies given out between the
// products, and splits by dot products were no faster.
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// a pair of floats as three pairs of bfloat16: 8 bits each, so together exact
__device__ __forceinline__ void split(float x0, float x1, uint32_t& a, uint32_t& b, uint32_t& c) {
  a = pack_bf16(x0, x1);
  x0 -= lo_f32(a);
  x1 -= hi_f32(a);
  b = pack_bf16(x0, x1);
  c = pack_bf16(x0 - lo_f32(b), x1 - hi_f32(b));
}

// Operands from the tiles.  Depth step s of rows 16 z + r: columns 4 NT g + 8 s ..
template <int NT>
__device__ __forceinline__ u32x4 across(const char* lds, int z, int s, int r, int g) {
  using X = Tile<bf16, NT, 32>;
  if constexpr (NT == 1) {
    const u32x2 v = *(const u32x2*)(lds + X::at(16 * z + r, g >> 1) + 8 * (g & 1));
    return u32x4{v[0], v[1], 0, 0};
  } else {
    return *(const u32x4*)(lds + X::at(16 * z + r, NT * g / 2 + s));
  }
}
// tile t with the rows as depth
template <int NT, bool VALUES>
__device__ __forceinline__ u32x4 down(const char* lds, int t, int r, int g) {
  using X = Tile<bf16, NT, 32, VALUES>;
  u32x4 v;
#pragma unroll
  for (int z = 0; z < 2; z++) {
    const int byte = (VALUES && NT == 4 ? 16 * (r & 3) + 64 * (t >> 1) + 8 * (t & 1) : 8 * NT * (r & 3) + 8 * t);
    const int row = 16 * z + 4 * g + (r >> 2);
    const auto x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(lds + X::at(row, byte >> 4) + (byte & 8)));
    const u32x2 y = __builtin_bit_cast(u32x2, x);
    v[2 * z] = y[0];
    v[2 * z + 1] = y[1];
  }
  return v;
}

template <int KT, int VT, int MODE>
__global__ __launch_bounds__(64 * SCAN_WAVES, 2) void k_scan16(ScanArgs A) {
  constexpr int C = 32, NS = KT < 2 ? 1 : KT / 2;
  using K = Tile<bf16, KT, C>;
  using V = Tile<bf16, VT, C, true>;
  constexpr int VC = VT == 1 ? 4 : 8;
  using Out = Tile<bf16, VT, C>;
  __shared__ alignas(16) char smem[SCAN_WAVES][2 * K::BYTES + V::BYTES + Out::BYTES];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  char* const lq = smem[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
  char* const lk = lq + K::BYTES;
  char* const lv = lk + K::BYTES;
  char* const lo_ = lv + V::BYTES;
  Unit U;
  if (!U.decode(A)) return;
  const Pass p = A.pass[U.pass];
  const int64_t n = U.n, L = U.L;
  const int h = U.h, seg = U.seg;
  const bool rev = p.rev;
  const int Dk = p.Dk, Dv = p.Dv, v0 = U.slice * 16 * VT;
  const bf16* qb = (const bf16*)p.q.p + n * p.q.sn + h * p.q.sh + U.seg0 * p.q.st;
  const bf16* kb = (const bf16*)p.k.p + n * p.k.sn + h * p.k.sh + U.seg0 * p.k.st;
  const bf16* vb = (const bf16*)p.v.p + n * p.v.sn + h * p.v.sh + U.seg0 * p.v.st + v0;
  bf16* ob = (bf16*)p.o.p + n * p.o.sn + h * p.o.sh + U.seg0 * p.o.st + v0;
  const bool want_out = p.o.p != nullptr;
  const uint8_t* xb = A.starts ? A.starts + n * A.starts_sn + U.seg0 * A.starts_st : nullptr;
  const float ld = finite_decay(A.log_decay[h]);
  auto power = [&](int m) { return power_of(ld, (float)m); };

  auto fetch = [&](int64_t t0, int c) {
    auto go = [&](auto whole) {
      constexpr bool W = decltype(whole)::value;
      V::template fetch<MODE, W>(lv, vb + t0 * p.v.st, p.v.st, Dv - v0, c, rev, lane);
      K::template fetch<MODE, W>(lk, kb + t0 * p.k.st, p.k.st, Dk, c, rev, lane);
      if (want_out) K::template fetch<MODE, W>(lq, qb + t0 * p.q.st, p.q.st, Dk, c, rev, lane);
    };
    if (c == C)
      go(std::true_type());
    else
      go(std::false_type());
  };
  if constexpr (MODE == GUARD) {
    for (int i = lane * 16; i < 2 * K::BYTES + V::BYTES; i += 1024) *(u32x4*)(lq + i) = u32x4{0, 0, 0, 0};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // MODE ANY: by way of registers
  u32x4 hq[K::NI], hk[K::NI], hv[V::NI];
  auto hold = [&](int64_t t0, int c) __attribute__((always_inline)) {
    constexpr int PER = K::PER;
    V::hold(hv, vb + t0 * p.v.st, p.v.st, Dv - v0, Dv >= PER, c, rev, lane);
    K::hold(hk, kb + t0 * p.k.st, p.k.st, Dk, Dk >= PER, c, rev, lane);
    if (want_out) K::hold(hq, qb + t0 * p.q.st, p.q.st, Dk, Dk >= PER, c, rev, lane);
  };
  auto ask = [&](int64_t t0, int c) __attribute__((always_inline)) {
    if constexpr (MODE == ANY)
      hold(t0, c);
    else
      fetch(t0, c);
  };
  bool loaded = L > 0;
  if (loaded) {
    const int c = (int)min((int64_t)C, L);
    ask(rev ? L - c : 0, c);
  }

  f32x4 S[KT][VT];
#pragma unroll
  for (int a = 0; a < KT; a++)
#pragma unroll
    for (int f = 0; f < VT; f++) S[a][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto column = [&](int f) { return v0 + VC * (r >> 2) + 32 * (f >> 1) + 4 * (f & 1) + (r & 3); };
  if (p.in.p) load_state<MODE, false>(S, p.in, p.in.p + n * p.in.sn + h * p.in.sh + seg * p.in.sg, Dk, Dv, g, column);

  // Weights.  A reversed pass carries g x the state of the row before: its first weight is 1, and its final state is
  // the gradient of the initial one.
  const int e = rev ? 0 : 1;
  float wd[4], wo[4], wi[2], wu[2][4];  // scores on and off the diagonal tile; state out; state in
  Decay decay;
  int cur = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    wd[i] = r >= 4 * g + i ? power(r - 4 * g - i) : 0.f;
    wo[i] = power(16 + r - 4 * g - i);
  }
#pragma unroll
  for (int z = 0; z < 2; z++) wi[z] = power(16 * z + r + e);

  bool fresh = false;  // an episode start among the live tokens
  int64_t done = 0;
  int single = 0;           // blocks of one token still to go

  while (done < L) {
    const int c = single ? 1 : (int)min((int64_t)C, L - done);
    const int64_t t0 = rev ? L - done - c : done;
    if (!loaded) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      ask(t0, c);
    }
    if constexpr (MODE == ANY) {
      V::commit(lv, hv, vb + t0 * p.v.st, p.v.st, Dv - v0, Dv >= K::PER, c, rev, lane);
      K::commit(lk, hk, kb + t0 * p.k.st, p.k.st, Dk, Dk >= K::PER, c, rev, lane);
      if (want_out) K::commit(lq, hq, qb + t0 * p.q.st, p.q.st, Dk, Dk >= K::PER, c, rev, lane);
    }
    uint32_t M = 0;  // bit u: an episode starts at row u
    if (xb) {
      const int u = min(lane, c - 1);
      M = (uint32_t)__ballot(lane < c && xb[(t0 + (rev ? c - 1 - u : u)) * A.starts_st] != 0);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if (c != cur) {
      cur = c;
      const int g4 = here(4 * g);
#pragma unroll
      for (int z = 0; z < 2; z++)
#pragma unroll
        for (int i = 0; i < 4; i++) wu[z][i] = power(max(c - e - (16 * z + g4 + i), 0));
      decay.set(ld, (float)c);
    }

    const f32x4 zero{0.f, 0.f, 0.f, 0.f};
    f32x4 O[VT][2], P[3];  // score tiles (key, query): (0, 0), (0, 1), (1, 1)
    if (want_out) {
#pragma unroll
      for (int z = 0; z < 2; z++)
#pragma unroll
        for (int f = 0; f < VT; f++) O[f][z] = zero;
#pragma unroll
      for (int x = 0; x < 3; x++) P[x] = zero;
#pragma unroll
      for (int s = 0; s < NS; s++) {
        if (s == 2) asm volatile("" ::: "memory");  // bounds the operands in registers at a time
        const u32x4 kf[2] = {across<KT>(lk, 0, s, r, g), across<KT>(lk, 1, s, r, g)};
        const u32x4 qf[2] = {across<KT>(lq, 0, s, r, g), across<KT>(lq, 1, s, r, g)};
        P[0] = mma(kf[0], qf[0], P[0]);
        P[1] = mma(kf[0], qf[1], P[1]);
        P[2] = mma(kf[1], qf[1], P[2]);
#pragma unroll
        for (int f = 0; f < VT; f++) {
          u32x4 t[3] = {};
#pragma unroll
          for (int m = 0; m < (KT < 2 ? 2 : 4); m++) {
            uint32_t y[3];
            split(S[2 * s + m / 2][f][2 * (m & 1)], S[2 * s + m / 2][f][2 * (m & 1) + 1], y[0], y[1], y[2]);
#pragma unroll
            for (int x = 0; x < 3; x++) t[x][m] = y[x];
          }
#pragma unroll
          for (int z = 0; z < 2; z++)
#pragma unroll
            for (int x = 0; x < 3; x++) O[f][z] = mma(t[x], qf[z], O[f][z]);
        }
      }
    }
    u32x4 vf[VT], k2[KT];
#pragma unroll
    for (int f = 0; f < VT; f++) vf[f] = down<VT, true>(lv, f, r, g);
#pragma unroll
    for (int a = 0; a < KT; a++) k2[a] = down<KT, false>(lk, a, r, g);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every read of the block is done: its room is free
    loaded = !single && done + c < L;
    if (loaded) {
      const int c2 = (int)min((int64_t)C, L - done - c);
      ask(rev ? t0 - c2 : t0 + c, c2);
    }
    // Masks.  A start at row u of a forward pass cuts every span that contains row u but not from it on; in a reversed
    // pass the cut lies behind row u, that is at row u + 1.
    const uint64_t cut = rev ? (uint64_t)M << 1 : (uint64_t)M;
    if (M != 0 || c < C) {
      const int g4 = here(4 * g);
#pragma unroll
      for (int z = 0; z < 2; z++)
#pragma unroll
        for (int m = 0; m < 2; m++) {
          const int u = 16 * z + g4 + 2 * m;
          const uint32_t live = (u < c ? 0xffffu : 0u) | (u + 1 < c ? 0xffff0000u : 0u);
          const uint32_t open = ((cut >> u) >> 1 ? 0u : 0xffffu) | ((cut >> (u + 1)) >> 1 ? 0u : 0xffff0000u);
#pragma unroll
          for (int f = 0; f < VT; f++) vf[f][2 * z + m] &= live;
#pragma unroll
          for (int a = 0; a < KT; a++) k2[a][2 * z + m] &= live & open;
        }
    }
    f32x4 bad = zero;
#pragma unroll
    for (int f = 0; f < VT; f++) bad = mma(vf[f], u32x4{0, 0, 0, 0}, bad);  // 0 or NaN
    // A masked product is a product with 0, which keeps a value away only while that value is finite.  A block with an
    // infinity or a NaN among its values is therefore run token by token: nothing is masked then.
    if (c > 1) {
      if (__any(!(bad[0] + bad[1] + bad[2] + bad[3] == 0.f))) {
        single = c;
        loaded = false;
        continue;
      }
    }
    fresh |= M != 0;

    if (want_out) {
#pragma unroll
      for (int z = 0; z < 2; z++)
#pragma unroll
        for (int f = 0; f < VT; f++) O[f][z] *= wi[z];
#pragma unroll
      for (int i = 0; i < 4; i++) {  // select, never multiply by 0
        P[0][i] = r >= 4 * g + i ? P[0][i] * wd[i] : 0.f;
        P[1][i] = P[1][i] * wo[i];
        P[2][i] = r >= 4 * g + i ? P[2][i] * wd[i] : 0.f;
      }
      if (M != 0) {
        const int g4 = here(4 * g), rr = here(r);
#pragma unroll
        for (int z = 0; z < 2; z++)
          if (cut & ((2ull << (16 * z + rr)) - 1))
#pragma unroll
            for (int f = 0; f < VT; f++) O[f][z] = zero;
#pragma unroll
        for (int x = 0; x < 3; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int s = (x == 2 ? 16 : 0) + g4 + i, t = (x == 0 ? 0 : 16) + rr;
            if (s < t && ((cut >> s) >> 1 & ((1ull << (t - s)) - 1)) != 0) P[x][i] = 0.f;
          }
      }
      u32x2 Ps[3][3];  // term, tile
#pragma unroll
      for (int x = 0; x < 3; x++)
#pragma unroll
        for (int m = 0; m < 2; m++) {
          uint32_t t[3];
          split(P[x][2 * m], P[x][2 * m + 1], t[0], t[1], t[2]);
#pragma unroll
          for (int y = 0; y < 3; y++) Ps[y][x][m] = t[y];
        }
#pragma unroll
      for (int f = 0; f < VT; f++)
#pragma unroll
        for (int y = 0; y < 3; y++) {
          O[f][0] = mma(vf[f], u32x4{Ps[y][0][0], Ps[y][0][1], 0, 0}, O[f][0]);
          O[f][1] = mma(vf[f], u32x4{Ps[y][1][0], Ps[y][1][1], Ps[y][2][0], Ps[y][2][1]}, O[f][1]);
        }
      // through LDS, so that neighbouring lanes store neighbouring columns
#pragma unroll
      for (int z = 0; z < 2; z++) {
        uint32_t x[2 * VT];
#pragma unroll
        for (int f = 0; f < VT; f++)
#pragma unroll
          for (int m = 0; m < 2; m++) x[2 * f + m] = pack_bf16(O[f][z][2 * m], O[f][z][2 * m + 1]);
        if constexpr (VT == 1) {
          *(u32x2*)(lo_ + Out::at(16 * z + r, g >> 1) + 8 * (g & 1)) = u32x2{x[0], x[1]};
        } else {
#pragma unroll
          for (int k = 0; k < VT / 2; k++)
            *(u32x4*)(lo_ + Out::at(16 * z + r, g + 4 * k)) = u32x4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      Out::template put<MODE>(lo_, ob + t0 * p.o.st, p.o.st, Dv - v0, c, rev, lane);
    }

    if (M != 0) {
#pragma unroll
      for (int a = 0; a < KT; a++)
#pragma unroll
        for (int f = 0; f < VT; f++) S[a][f] = f32x4{0.f, 0.f, 0.f, 0.f};
      // a block of one token that a reversed pass cuts off behind itself: its value, perhaps an infinity, adds nothing
      if (rev && c == 1)
#pragma unroll
        for (int f = 0; f < VT; f++) vf[f] = u32x4{0, 0, 0, 0};
    }
    // the weights go to the operand of fewer tiles
    auto weigh = [&](u32x4 x, u32x4(&t)[3]) {
#pragma unroll
      for (int m = 0; m < 4; m++) {
        uint32_t y[3];
        split(lo_f32(x[m]) * wu[m / 2][2 * (m & 1)], hi_f32(x[m]) * wu[m / 2][2 * (m & 1) + 1], y[0], y[1], y[2]);
#pragma unroll
        for (int i = 0; i < 3; i++) t[i][m] = y[i];
      }
    };
    u32x4 t[3];
    if constexpr (KT < VT) {
#pragma unroll
      for (int a = 0; a < KT; a++) {
        f32x4 D[VT];
        weigh(k2[a], t);
#pragma unroll
        for (int x = 0; x < 3; x++)
#pragma unroll
          for (int f = 0; f < VT; f++) D[f] = mma(t[x], vf[f], x ? D[f] : zero);
#pragma unroll
        for (int f = 0; f < VT; f++)
#pragma unroll
          for (int i = 0; i < 4; i++) S[a][f][i] = decay(S[a][f][i], D[f][i]);
      }
    } else {
      constexpr int AT = KT < 2 ? KT : 2;  // tiles at a time
#pragma unroll
      for (int f = 0; f < VT; f++) {
        weigh(vf[f], t);
#pragma unroll
        for (int a0 = 0; a0 < KT; a0 += AT) {
          f32x4 D[AT];
#pragma unroll
          for (int x = 0; x < 3; x++)
#pragma unroll
            for (int a = 0; a < AT; a++) D[a] = mma(k2[a0 + a], t[x], x ? D[a] : zero);
#pragma unroll
          for (int a = 0; a < AT; a++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[a0 + a][f][i] = decay(S[a0 + a][f][i], D[a][i]);
#pragma unroll
          for (int a = 0; a < AT; a++) pin<true>(S[a0 + a][f]);
        }
      }
    }
    done += c;
    if (single) single--;
  }
  if (p.out.p && (seg == A.n_seg - 1 || p.out.sg))
    store_state<MODE, false>(S, p.out, p.out.p + n * p.out.sn + h * p.out.sh + seg * p.out.sg, Dk, Dv, g, column);
  if (A.factor && U.slice == 0 && lane == 0)
    A.factor[((U.pass * A.N + n) * A.H + h) * A.n_seg + seg] = fresh ? -1.f : power_of(ld, (float)L);
  if (want_out) {  // rows behind the sequence's end
#pragma unroll
    for (int i = 0; i < Out::NI; i++) *(u32x4*)(lo_ + (i * 64 + lane) * 16) = u32x4{0, 0, 0, 0};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    for (int64_t t = L; t < U.seg1 - U.seg0; t += C)
      Out::template put<MODE>(lo_, ob + t * p.o.st, p.o.st, Dv - v0, (int)min((int64_t)C, U.seg1 - U.seg0 - t), false, lane);
  }
}

// ws[seg] holds what segment seg adds to a state; rewritten as the state that enters segment seg:
//   c_0 = in;  c_{s+1} = factor_s c_s + ws_s  (factor_s negative: ws_s alone)
// One thread per four keys of a value column; the loads of all segments are independent of the recurrence.  Bound by
// memory: 32 segments of 16 heads of 128 x 128, 34 MB in and out, 14 us.
struct JoinArgs {
  State in[2];  // p NULL: zeros
  float* ws;    // [dirs][N][H][n_seg][ceil(Dk / 4)][Dv][4]
  const float* factor;
  int64_t N;
  int32_t dirs, H, n_seg, Dk, Dv;
};
__global__ __launch_bounds__(256) void k_scan_join(JoinArgs A) {
  const uint32_t E = (uint32_t)((A.Dk + 3) / 4 * A.Dv), x = blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = x / E, e = x - row * E;  // row = (dir N + n) H + h
  if (row >= (uint32_t)(A.dirs * A.N * A.H)) return;
  const uint32_t h = row % (uint32_t)A.H, n = row / (uint32_t)A.H % (uint32_t)A.N;
  const State& in = A.in[row / (uint32_t)A.H / (uint32_t)A.N];
  f32x4 c{0.f, 0.f, 0.f, 0.f};
  if (in.p) {
    const int k4 = (int)(e / A.Dv), v = (int)(e % A.Dv);
    const float* s = in.p + n * in.sn + h * in.sh + k4 * in.k4 + (v >> 2) * in.v4 + (v & 3) * in.v1;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (4 * k4 + i < A.Dk) c[i] = s[i * in.k1];
  }
  f32x4* w = (f32x4*)A.ws + (int64_t)row * A.n_seg * E + e;
  const float* f = A.factor + (int64_t)row * A.n_seg;
  constexpr int PF = 8;
  for (int s0 = 0; s0 < A.n_seg; s0 += PF) {
    f32x4 add[PF];
    float fac[PF];
#pragma unroll
    for (int k = 0; k < PF; k++)
      if (s0 + k < A.n_seg - 1) {  // the last segment adds to nothing
        add[k] = w[(int64_t)(s0 + k) * E];
        fac[k] = f[s0 + k];
      }
#pragma unroll
    for (int k = 0; k < PF; k++)
      if (s0 + k < A.n_seg) {
        w[(int64_t)(s0 + k) * E] = c;
        if (s0 + k < A.n_seg - 1)
#pragma unroll
          for (int i = 0; i < 4; i++) c[i] = fac[k] < 0.f ? add[k][i] : fmaf(fac[k], c[i], add[k][i]);
      }
  }
}

// ------------------------------------------------------------------ the single-token form
struct TokenArgs {
  Operand q, k, v, o;
  const float* log_decay;
  const uint8_t* starts;
  int64_t starts_sn, N;
  const float* in;
  float* out;
  int32_t H, Dk, Dv;
};

// Bound by the state, read once and written once.  A wave takes B pairs (n, h); nv lanes cover a state row in vectors of
// 4, 64 / nv rows an access, and four accesses are in flight before the first is used (65536 x 4 x 16 x 16: one access
// is a whole state, so B = 4).  Where 4 does not divide a row its last vector begins earlier and shares columns with the
// one before: both lanes compute and store the same values there.  Rows then begin at any multiple of 4 bytes, which
// the load unit takes (2165 x 12 of 116 x 41: 4670 GB/s; by elements 2770).
// The state of a row that starts afresh is read all the same: waiting for its flag first would cost every row a memory
// round trip.
// VEC: v and out are read and written in vectors too.
// SPLIT: a block's four waves share one pair's rows, where there are too few pairs to fill the card.
// STREAM: the states are larger than the last-level cache and pass it by.  Rows of whole vectors only: without the cache
// the parts of a memory line that two accesses write do not meet (116 x 41: 4050 GB/s with it).
typedef f32x4 __attribute__((aligned(4))) f32x4_any;  // at any element
template <typename T, bool VEC, int B, bool SPLIT, bool STREAM>
__global__ __launch_bounds__(256) void k_token(TokenArgs A, int nv, int rows, int magic) {
  static_assert(!SPLIT || B == 1);
  constexpr int R = 4 / B;
  __shared__ float part[SPLIT ? 4 : 1][SPLIT ? MAXDIM : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const uint32_t units = (uint32_t)(A.N * A.H);
  const uint32_t u0 = SPLIT ? blockIdx.x : (blockIdx.x * 4 + wave) * B;
  if (u0 >= units) return;
  const int rr = lane * magic >> 16;  // lane / nv
  const int c = VEC ? (lane - rr * nv) * 4 : min((lane - rr * nv) * 4, A.Dv - 4);
  const bool on = rr < rows;
  const int E = A.Dk * A.Dv;
  const T *q[B], *k[B], *v[B];
  T* o[B];
  float vv[B][4], acc[B][4], ld[B];
  Decay decay[B];
  bool start[B];
  {
    uint32_t n = u0 / (uint32_t)A.H, h = u0 - n * (uint32_t)A.H;
#pragma unroll
    for (int b = 0; b < B; b++) {
      q[b] = (const T*)A.q.p + n * A.q.sn + h * A.q.sh;
      k[b] = (const T*)A.k.p + n * A.k.sn + h * A.k.sh;
      v[b] = (const T*)A.v.p + n * A.v.sn + h * A.v.sh;
      o[b] = (T*)A.o.p + n * A.o.sn + h * A.o.sh;
      start[b] = A.starts && A.starts[n * A.starts_sn] != 0;
      ld[b] = A.log_decay[h];
      if (u0 + b + 1 < units) {  // (the last pair again, where the wave has more places than there are pairs)
        h = h + 1 == (uint32_t)A.H ? 0 : h + 1;
        n += h == 0;
      }
    }
  }
  const float* in0 = A.in + (int64_t)u0 * E;
  float* out0 = A.out + (int64_t)u0 * E;
  const int live = (int)min(units - u0, (uint32_t)B);
  const int first = SPLIT ? wave * R * rows + rr : rr, step = (SPLIT ? 4 : 1) * R * rows;
#pragma unroll
  for (int b = 0; b < B; b++)
#pragma unroll
    for (int x = 0; x < 4; x++) acc[b][x] = 0.f;
  for (int d0 = first; d0 < A.Dk; d0 += step) {
    f32x4 s[B][R];
    float kd[B][R], qd[B][R];
#pragma unroll
    for (int b = 0; b < B; b++)
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int d = min(d0 + i * rows, A.Dk - 1);
        const f32x4_any* from = (const f32x4_any*)(in0 + min(b, live - 1) * E + d * A.Dv + c);
        s[b][i] = STREAM ? __builtin_nontemporal_load(from) : *from;
        kd[b][i] = to_f32(k[b][d]);
        qd[b][i] = to_f32(q[b][d]);
      }
    if (d0 == first)
#pragma unroll
      for (int b = 0; b < B; b++) {
        if constexpr (VEC) {
          load_vec<T, 4>(v[b] + c, vv[b]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; x++) vv[b][x] = to_f32(v[b][c + x]);
        }
      }
    if (d0 == first) {  // the pairs' decays, one per lane, at the price of one
      float x = ld[0];
#pragma unroll
      for (int b = 1; b < B; b++) x = lane % B == b ? ld[b] : x;
      Decay mine;
      mine.set(finite_decay(x), 1.f);
#pragma unroll
      for (int b = 0; b < B; b++) {
        decay[b].keep = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine.keep), b));
        decay[b].by = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine.by), b));
      }
    }
#pragma unroll
    for (int b = 0; b < B; b++)
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int d = d0 + i * rows;
        if (d < A.Dk && on && b < live) {
#pragma unroll
          for (int x = 0; x < 4; x++) {
            s[b][i][x] = decay[b](start[b] ? 0.f : s[b][i][x], kd[b][i] * vv[b][x]);
            acc[b][x] = fmaf(qd[b][i], s[b][i][x], acc[b][x]);
          }
          f32x4_any* so = (f32x4_any*)(out0 + b * E + d * A.Dv + c);
          if (STREAM)
            __builtin_nontemporal_store(s[b][i], so);
          else
            *so = s[b][i];
        }
      }
  }
#pragma unroll
  for (int b = 0; b < B; b++) {
    // the rows' shares, in a fixed order, to row 0
    for (int r = rows; r > 1; r = (r + 1) >> 1) {
      const int half = (r + 1) >> 1;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const float y = __shfl(acc[b][x], lane + half * nv);
        acc[b][x] += rr < r - half ? y : 0.f;
      }
    }
    if constexpr (SPLIT) {  // the waves' shares, in their order
      if (rr == 0)
#pragma unroll
        for (int x = 0; x < 4; x++) part[wave][c + x] = acc[b][x];
      __syncthreads();
      if (wave != 0) return;
      if (rr == 0)
#pragma unroll
        for (int x = 0; x < 4; x++) acc[b][x] = ((part[0][c + x] + part[1][c + x]) + part[2][c + x]) + part[3][c + x];
    }
    if (rr == 0 && b < live) {
      if constexpr (VEC) {
        store_vec<T, 4>(o[b] + c, acc[b]);
      } else {
#pragma unroll
        for (int x = 0; x < 4; x++) o[b][c + x] = from_f32<T>(acc[b][x]);
      }
    }
  }
}

// Rows of fewer than 4 columns: a wave per pair, a lane per key.
template <typename T>
__global__ __launch_bounds__(256) void k_token_narrow(TokenArgs A) {
  const uint32_t units = (uint32_t)(A.N * A.H), u = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (u >= units) return;
  const int lane = threadIdx.x & 63;
  const uint32_t n = u / (uint32_t)A.H, h = u - n * (uint32_t)A.H;
  const T* q = (const T*)A.q.p + n * A.q.sn + h * A.q.sh;
  const T* k = (const T*)A.k.p + n * A.k.sn + h * A.k.sh;
  const T* v = (const T*)A.v.p + n * A.v.sn + h * A.v.sh;
  T* o = (T*)A.o.p + n * A.o.sn + h * A.o.sh;
  const bool start = A.starts && A.starts[n * A.starts_sn] != 0;
  Decay decay;
  decay.set(finite_decay(A.log_decay[h]), 1.f);
  const int64_t at = (int64_t)u * A.Dk * A.Dv;
  for (int c = 0; c < A.Dv; c++) {
    const float vc = to_f32(v[c]);
    float acc = 0.f;
    for (int d = lane; d < A.Dk; d += 64) {
      const float s = A.in[at + d * A.Dv + c];
      const float y = decay(start ? 0.f : s, to_f32(k[d]) * vc);
      A.out[at + d * A.Dv + c] = y;
      acc = fmaf(to_f32(q[d]), y, acc);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) acc += __shfl_xor(acc, m);
    if (lane == 0) o[c] = from_f32<T>(acc);
  }
}

// ------------------------------------------------------------------ host side
int tiles(int d) { return d <= 16 ? 1 : d <= 32 ? 2 : d <= 64 ? 4 : 8; }
// value tiles of one wave: the state is KT x VT tiles of registers
int slice_tiles(int dtype, int Dk, int Dv, int most) {
  return std::min({most, tiles(Dv), dtype == FW_DT_BF16 && tiles(Dk) == 8 ? 2 : 4});
}
int slices(int dtype, int Dk, int Dv, int most) {
  const int cols = 16 * slice_tiles(dtype, Dk, Dv, most);
  return (Dv + cols - 1) / cols;
}

// Time segments: with few waves the card is not full, so the time axis is cut, at the price of reading k and v twice and
// of a state per segment.  SEG_WAVES is two waves per SIMD; the backward pass runs three passes at once and wants fewer.
// Two segments cost more than they bring unless all their waves have a SIMD each (measured, us; 1000 waves of 500 tokens, 20 x
// 40 float32: 1 segment 108 forward and 243 backward, 2 segments 132 and 279; 400 waves of 512, 32 x 32 float32, backward: 1
// segment 84, 2: 104, 4: 106; 256 waves of 2048, 64 x 64 bfloat16: forward 4 segments 120, 8: 111, backward 4 segments 224,
// 8: 242).
constexpr int SEG_WAVES = 2048;
constexpr int SEG_MIN = 128;  // tokens
struct Plan {
  int64_t seg_len;
  int n_seg;
};
Plan plan(int dtype, int64_t T, int64_t N, int H, int Dk, int Dv, bool backward) {
  const int64_t waves = std::max<int64_t>(1, N * H * slices(dtype, Dk, Dv, 4));
  const int64_t segs = std::min<int64_t>((backward ? SEG_WAVES / 2 : SEG_WAVES) / waves, T / SEG_MIN);
  if (segs < 2 || (segs == 2 && (backward ? 3 : 1) * 2 * waves > SEG_WAVES / 2)) return {std::max<int64_t>(T, 1), 1};
  const int64_t len = ((T + segs - 1) / segs + 31) / 32 * 32;
  return {len, (int)((T + len - 1) / len)};
}
int quads(int Dk) { return (Dk + 3) / 4 * 4; }
// a state per segment and what a segment multiplies a state with; the backward pass has two directions of them
size_t plan_floats(const Plan& pl, int dirs, int64_t N, int H, int Dk, int Dv) {
  if (pl.n_seg < 2) return 0;
  return (size_t)dirs * N * H * pl.n_seg * ((size_t)quads(Dk) * Dv + 1);
}

template <typename T>
bool aligned(const Operand& o, int D) {
  const int per16 = 16 / sizeof(T);
  // (a block's rows, 16 of 4 or 2 bytes or 32 of 2, are addressed by 32-bit offsets)
  return D % per16 == 0 && (uintptr_t)o.p % 16 == 0 && o.st % per16 == 0 && o.sn % per16 == 0 && o.sh % per16 == 0 &&
         o.st >= 0 && o.st <= (int64_t)1 << 26;
}

template <typename T, int KT, int VT>
int launch_mode(const ScanArgs& A, int mode, hipStream_t s) {
  const int64_t units = A.n_pass * (int64_t)A.n_slice * A.H * A.N;
  const int64_t blocks = (units + SCAN_WAVES - 1) / SCAN_WAVES;
  if (blocks > UINT32_MAX / (64 * SCAN_WAVES))  // threads of a launch
    return fw::set_error(FW_E_INVALID, "linear attention: too many sequences for one call");
  const dim3 grid((unsigned)blocks, A.run_seg), block(64 * SCAN_WAVES);
  auto kernel = [&](auto m) {
    constexpr int MODE = decltype(m)::value;
    if constexpr (std::is_same_v<T, bf16>)
      return k_scan16<KT, VT, MODE>;
    else
      return k_scan<T, KT, VT, MODE>;
  };
  if (mode == FULL)
    hipLaunchKernelGGL(kernel(std::integral_constant<int, FULL>()), grid, block, 0, s, A);
  else if (mode == GUARD)
    hipLaunchKernelGGL(kernel(std::integral_constant<int, GUARD>()), grid, block, 0, s, A);
  else
    hipLaunchKernelGGL(kernel(std::integral_constant<int, ANY>()), grid, block, 0, s, A);
  FW_HIP(hipGetLastError());
  return FW_OK;
}

template <typename T>
int launch_scan(ScanArgs A, int kt, int vt, hipStream_t s) {
  int mode = FULL;
  for (int i = 0; i < A.n_pass; i++) {
    const Pass& p = A.pass[i];
    bool vec = aligned<T>(p.q, p.Dk) && aligned<T>(p.k, p.Dk) && aligned<T>(p.v, p.Dv) && aligned<T>(p.o, p.Dv);
    mode = std::max<int>(mode, !vec ? ANY : p.Dk == 16 * kt && p.Dv % (16 * vt) == 0 ? FULL : GUARD);
  }
  switch (kt * 8 + vt) {
#define FW_CASE(K, V) \
  case K * 8 + V: return launch_mode<T, K, V>(A, mode, s)
    FW_CASE(1, 1); FW_CASE(1, 2); FW_CASE(1, 4);
    FW_CASE(2, 1); FW_CASE(2, 2); FW_CASE(2, 4);
    FW_CASE(4, 1); FW_CASE(4, 2); FW_CASE(4, 4);
    FW_CASE(8, 1); FW_CASE(8, 2);
    case 8 * 8 + 4:
      if constexpr (!std::is_same_v<T, bf16>) return launch_mode<T, 8, 4>(A, mode, s);
#undef FW_CASE
  }
  return fw::set_error(FW_E_INVALID, "linear attention: head sizes 1..128");
}

// Passes of equal tiles and slices go in one launch.
// Where there is one segment, a wave takes fewer value columns as long as each wave has a SIMD to itself (two waves a SIMD
// with two tiles of float32 products, which are further from the memory's rate): its blocks are shorter and the scores
// are computed once more per slice.  100 tokens of 4 heads of 64 x 64 bfloat16, one tile against four: 12 against
// 19 us; 500 x 250 x 4 heads of 20 x 40 float32, two against four: 96 against 107; 500 x 420 x 4 heads of 20 x 20 float32, one
// (3360 waves) against two: 133 against 97.
int launch_passes(int dtype, ScanArgs A, const Pass* pass, int n_pass, hipStream_t s) {
  for (int i = 0; i < n_pass; i += A.n_pass) {
    const int kt = tiles(pass[i].Dk);
    auto alike = [&](const Pass& p, int most) {
      return tiles(p.Dk) == kt && slice_tiles(dtype, p.Dk, p.Dv, most) == slice_tiles(dtype, pass[i].Dk, pass[i].Dv, most) &&
             slices(dtype, p.Dk, p.Dv, most) == slices(dtype, pass[i].Dk, pass[i].Dv, most);
    };
    int most = A.n_seg > 1 ? 4 : 1;
    for (;; most *= 2) {
      A.n_slice = slices(dtype, pass[i].Dk, pass[i].Dv, most);
      A.n_pass = 0;
      for (int j = i; j < n_pass && alike(pass[j], most); j++) A.pass[A.n_pass++] = pass[j];
      const int64_t limit = most == 2 && dtype != FW_DT_BF16 ? SEG_WAVES : SEG_WAVES / 2;
      if (most == 4 || A.N * A.H * A.n_pass * A.n_slice <= limit) break;
    }
    const int vt = slice_tiles(dtype, pass[i].Dk, pass[i].Dv, most);
    const int rc = dtype == FW_DT_F32    ? launch_scan<float>(A, kt, vt, s)
                   : dtype == FW_DT_BF16 ? launch_scan<bf16>(A, kt, vt, s)
                                         : launch_scan<f16>(A, kt, vt, s);
    if (rc) return rc;
  }
  return FW_OK;
}

// The states that enter the segments, for each of `dirs` directions: what the segments add (add[d]: keys and values
// alone), joined along time from in[d].  Leaves them in ws (see segments()).
int segment_states(int dtype, ScanArgs A, const Pass* add, const State* in, int dirs, float* ws, hipStream_t s) {
  const int Dk = add[0].Dk, Dv = add[0].Dv;
  const int64_t E = (int64_t)quads(Dk) * Dv;
  A.factor = ws + dirs * A.N * A.H * A.n_seg * E;
  A.run_seg = A.n_seg - 1;  // the last segment adds to nothing
  if (int rc = launch_passes(dtype, A, add, dirs, s)) return rc;
  JoinArgs J{};
  for (int d = 0; d < dirs; d++) J.in[d] = in[d];
  J.ws = ws;
  J.factor = A.factor;
  J.N = A.N;
  J.dirs = dirs;
  J.H = A.H;
  J.n_seg = A.n_seg;
  J.Dk = Dk;
  J.Dv = Dv;
  const int64_t blocks = (dirs * A.N * A.H * E / 4 + 255) / 256;  // N H < SEG_WAVES
  hipLaunchKernelGGL(k_scan_join, dim3((unsigned)blocks), dim3(256), 0, s, J);
  FW_HIP(hipGetLastError());
  return FW_OK;
}

int check(const fw_linattn* a, const char* who) {
  auto bad = [&](const char* m) { return fw::set_error(FW_E_INVALID, std::string(who) + ": " + m); };
  if (!a) return bad("NULL arguments");
  if (a->T < 0 || a->N < 0 || a->H < 1) return bad("T and N must be >= 0, H >= 1");
  if (a->Dk < 1 || a->Dk > MAXDIM || a->Dv < 1 || a->Dv > MAXDIM) return bad("head sizes must be 1..128");
  if (a->dtype < FW_DT_F32 || a->dtype > FW_DT_F16) return bad("dtype must be float32, bfloat16 or float16");
  if (a->T > 0 && a->N > 0 && (!a->q.p || !a->k.p || !a->v.p)) return bad("NULL q, k or v");
  if (!a->log_decay) return bad("NULL log_decay");
  if (a->N > INT32_MAX / a->H) return bad("too many sequences for one call");
  if (a->starts && (a->starts_st < 0 || a->starts_st >= (int64_t)1 << 26)) return bad("starts_st must be 0..2^26 - 1");
  return FW_OK;
}
bool room(const fw_linattn* a, bool backward) {
  const size_t need = fw_linattn_workspace_bytes(a->T, a->N, a->H, a->Dk, a->Dv, a->dtype, backward);
  return need == 0 || (a->workspace && a->workspace_bytes >= need && (uintptr_t)a->workspace % 16 == 0);
}
// the strides of single tokens, sequences and heads mean nothing and are not to cost an operand its alignment
Operand in(const fw_linattn* a, const fw_seq_tensor& t) {
  return {t.p, a->T > 1 ? t.st : 0, a->N > 1 ? t.sn : 0, a->H > 1 ? t.sh : 0};
}
Operand in(const fw_seq_tensor& t) { return {t.p, t.st, t.sn, t.sh}; }
ScanArgs base(const fw_linattn* a, const Plan& pl) {
  ScanArgs A{};
  A.H = a->H;
  A.T = a->T;
  A.N = a->N;
  A.seg_len = pl.seg_len;
  A.n_seg = A.run_seg = pl.n_seg;
  A.log_decay = a->log_decay;
  A.starts = a->starts;
  A.starts_st = a->starts_st;
  A.starts_sn = a->starts_sn;
  A.lengths = a->lengths;
  return A;
}
State straight(const fw_linattn* a, const float* p) {
  const int64_t E = (int64_t)a->Dk * a->Dv;
  return {const_cast<float*>(p), a->H * E, E, 0, 4 * a->Dv, a->Dv, 4, 1};
}
State turned(State s) {
  std::swap(s.k4, s.v4);
  std::swap(s.k1, s.v1);
  return s;
}
State segments(const fw_linattn* a, float* ws, int dir, int n_seg) {
  const int64_t E = (int64_t)quads(a->Dk) * a->Dv;
  return {ws + dir * a->N * a->H * n_seg * E, a->H * n_seg * E, n_seg * E, E, 4 * a->Dv, 1, 16, 4};
}

}  // namespace

extern "C" {

size_t fw_linattn_workspace_bytes(int64_t T, int64_t N, int32_t H, int32_t Dk, int32_t Dv, int32_t dtype, int32_t backward) {
  if (T < 1 || N < 1 || H < 1 || Dk < 1 || Dk > MAXDIM || Dv < 1 || Dv > MAXDIM) return 0;
  return sizeof(float) * plan_floats(plan(dtype, T, N, H, Dk, Dv, backward), backward ? 2 : 1, N, H, Dk, Dv);
}

int fw_linattn_forward(const fw_linattn* a, void* stream) {
  if (int rc = check(a, "fw_linattn_forward")) return rc;
  if (a->N == 0) return FW_OK;
  if (a->T > 0 && !a->out.p) return fw::set_error(FW_E_INVALID, "fw_linattn_forward: NULL out");
  const Plan pl = plan(a->dtype, a->T, a->N, a->H, a->Dk, a->Dv, false);
  if (!room(a, false)) return fw::set_error(FW_E_INVALID, "fw_linattn_forward: workspace too small or not 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  float* ws = (float*)a->workspace;
  const ScanArgs A = base(a, pl);
  Pass p{in(a, a->q), in(a, a->k), in(a, a->v), in(a, a->out), straight(a, a->state_in), straight(a, a->state_out), 0, a->Dk, a->Dv};
  if (pl.n_seg > 1) {
    const State seg = segments(a, ws, 0, pl.n_seg);
    const Pass add{p.q, p.k, p.v, Operand{}, State{}, seg, 0, a->Dk, a->Dv};
    if (int rc = segment_states(a->dtype, A, &add, &p.in, 1, ws, s)) return rc;
    p.in = seg;
  }
  return launch_passes(a->dtype, A, &p, 1, s);
}

int fw_linattn_backward(const fw_linattn* a, void* stream) {
  if (int rc = check(a, "fw_linattn_backward")) return rc;
  if (a->N == 0) return FW_OK;
  if (a->T > 0 && (!a->dout.p || !a->dq.p || !a->dk.p || !a->dv.p))
    return fw::set_error(FW_E_INVALID, "fw_linattn_backward: NULL dout, dq, dk or dv");
  const Plan pl = plan(a->dtype, a->T, a->N, a->H, a->Dk, a->Dv, true);
  if (!room(a, true)) return fw::set_error(FW_E_INVALID, "fw_linattn_backward: workspace too small or not 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  float* ws = (float*)a->workspace;
  const ScanArgs A = base(a, pl);
  State S = straight(a, a->state_in), R = straight(a, a->dstate);  // forward states; reversed ones
  if (pl.n_seg > 1) {
    const State in_[2] = {S, R};
    S = segments(a, ws, 0, pl.n_seg);
    R = segments(a, ws, 1, pl.n_seg);
    const Pass add[2] = {{in(a, a->q), in(a, a->k), in(a, a->v), Operand{}, State{}, S, 0, a->Dk, a->Dv},
                         {in(a, a->k), in(a, a->q), in(a, a->dout), Operand{}, State{}, R, 1, a->Dk, a->Dv}};
    if (int rc = segment_states(a->dtype, A, add, in_, 2, ws, s)) return rc;
  }
  const Pass main[3] = {
      {in(a, a->dout), in(a, a->v), in(a, a->k), in(a, a->dq), turned(S), State{}, 0, a->Dv, a->Dk},
      {in(a, a->v), in(a, a->dout), in(a, a->q), in(a, a->dk), turned(R), State{}, 1, a->Dv, a->Dk},
      {in(a, a->k), in(a, a->q), in(a, a->dout), in(a, a->dv), R, straight(a, a->dstate_in), 1, a->Dk, a->Dv}};
  return launch_passes(a->dtype, A, main, 3, s);
}

int fw_linattn_step(const fw_linattn_token* a, void* stream_) {
  auto bad = [&](const char* m) { return fw::set_error(FW_E_INVALID, std::string("fw_linattn_step: ") + m); };
  if (!a) return bad("NULL arguments");
  if (a->N < 0 || a->H < 1) return bad("N must be >= 0, H >= 1");
  if (a->Dk < 1 || a->Dk > MAXDIM || a->Dv < 1 || a->Dv > MAXDIM) return bad("head sizes must be 1..128");
  if (a->dtype < FW_DT_F32 || a->dtype > FW_DT_F16) return bad("dtype must be float32, bfloat16 or float16");
  if (a->N == 0) return FW_OK;
  if (!a->q.p || !a->k.p || !a->v.p || !a->out.p || !a->log_decay || !a->state || !a->state_out) return bad("NULL buffer");
  if ((uintptr_t)a->state % 16 || (uintptr_t)a->state_out % 16) return bad("states must be 16-byte aligned");
  TokenArgs A{in(a->q), in(a->k), in(a->v), in(a->out), a->log_decay, a->starts, a->starts_sn, a->N,
              a->state, a->state_out, a->H, a->Dk, a->Dv};
  if (a->N > INT32_MAX / a->H) return bad("too many sequences for one call");
  const int64_t units = a->N * a->H;
  const int nv = (a->Dv + 3) / 4, rows = 64 / nv;
  auto fours = [&](const fw_seq_tensor& t) {
    return (uintptr_t)t.p % (a->dtype == FW_DT_F32 ? 16 : 8) == 0 && t.sn % 4 == 0 && t.sh % 4 == 0;
  };
  const bool vec = a->Dv % 4 == 0 && fours(a->v) && fours(a->out);
  // Measured in float32: split against not, 128 pairs of 128 x 128: 6.8 against 14.9 us, 1024 pairs: 23 against 28;
  // stream against not, 537 MB of states: 5290 against 4700 GB/s, 134 MB: 4970 against 6050 (it is 256 MB of cache).
  const int accesses = (a->Dk + rows - 1) / rows;  // of one state
  const bool narrow = a->Dv < 4, split = !narrow && accesses >= 8 && units <= 2048;
  const bool stream = !split && a->Dv % 4 == 0 && units * a->Dk * a->Dv * 4 >= (int64_t)192 << 20;
  const int B = narrow ? 1 : accesses == 1 ? 4 : accesses == 2 ? 2 : 1;
  const int64_t blocks = split ? units : (units + 4 * B - 1) / (4 * B);
  if (blocks > UINT32_MAX / 256) return bad("too many sequences for one call");  // threads of a launch
  const dim3 grid((unsigned)blocks), block(256);
  hipStream_t s = (hipStream_t)stream_;
#define FW_TOKEN_V(T, V, B_, SP)                                                       \
  if (stream)                                                                          \
    hipLaunchKernelGGL((k_token<T, V, B_, SP, !SP>), grid, block, 0, s, A, nv, rows, 65536 / nv + 1); \
  else                                                                                 \
    hipLaunchKernelGGL((k_token<T, V, B_, SP, false>), grid, block, 0, s, A, nv, rows, 65536 / nv + 1)
#define FW_TOKEN_K(T, B_, SP)                                                          \
  if (vec) {                                                                           \
    FW_TOKEN_V(T, true, B_, SP);                                                       \
  } else {                                                                             \
    FW_TOKEN_V(T, false, B_, SP);                                                      \
  }
#define FW_TOKEN(T)                                                                    \
  if (narrow) {                                                                        \
    hipLaunchKernelGGL((k_token_narrow<T>), grid, block, 0, s, A);                     \
  } else if (split) {                                                                  \
    FW_TOKEN_K(T, 1, true);                                                            \
  } else if (B == 4) {                                                                 \
    FW_TOKEN_K(T, 4, false);                                                           \
  } else if (B == 2) {                                                                 \
    FW_TOKEN_K(T, 2, false);                                                           \
  } else {                                                                             \
    FW_TOKEN_K(T, 1, false);                                                           \
  }
  if (a->dtype == FW_DT_F32) {
    FW_TOKEN(float);
  } else if (a->dtype == FW_DT_BF16) {
    FW_TOKEN(bf16);
  } else {
    FW_TOKEN(f16);
  }
#undef FW_TOKEN
#undef FW_TOKEN_K
#undef FW_TOKEN_V
  FW_HIP(hipGetLastError());
  return FW_OK;
}

}  // extern "C"

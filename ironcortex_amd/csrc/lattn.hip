// Linear attention with a decay for each head, over sequences (chunked) and for single positions (recurrent):
//   S_t = e^{-r} S_{t-1} + k_t v_t^T,   o_t = scale * q_t^T S_t.
//
// Chunks of C = 64 positions.  With S the state at a chunk's border and i, j positions inside the chunk,
//   o_i = e^{-r(i+1)} q_i^T S + sum_{j <= i} e^{-r(i-j)} (q_i . k_j) v_j,    S' = e^{-rC} S + sum_j e^{-r(C-1-j)} k_j v_j^T:
// four matrix products on the matrix cores, every exponent of e^{-r} a non-negative count (no quotients of decays).
//
// The backward is the same map three more times:
//   dq = (q, k, v) := (dout, v, k) with the transposed state;
//   dv = (k, q, scale dout) and dk = (v, dout, scale q), both from the last position to the first, starting from the
//   gradient of the final state; dstate is where that reversed recurrence ends.
// So ONE kernel serves the forward (one pass) and the backward (three).  Against a kernel that forms all three gradients of a
// chunk at once it multiplies 12 tiles instead of 10, and needs neither the state at every chunk's border in memory nor two
// states in registers.  Gradients of shared key / value heads: a workgroup takes their query heads in turn and keeps the sum
// in fp32 rows that only its own lanes touch (against a partial gradient for each query head and a joining launch: 14 us less
// of a forward and backward of 8 x 4096 positions, 8 / 4 bf16 heads of 128, and half the workspace).
// d rate: -d o / d rate weighs every pair by its lag.  The dq pass carries the lag-weighted state L = sum lag e^{-r lag}
// k v^T next to S, and sums q_i . (lag-weighted dq_i): every term counted once with its own lag, where a difference of
// position-weighted q . dq and k . dk would cancel to T times the rounding error.
//
// Work split: a workgroup owns (sequence, head, segment of chunks); a wave 16 (or 32) of the value columns, with its slice
// of the state in the accumulator registers, in the layout that the next product takes as its operand (16x16 tiles: lane
// l holds rows 4 (l / 16) + 0..3 of column l % 16, and as an operand k-indices 4 (l / 16) + 0..3 of row / column l % 16).
// Several segments per sequence only where sequences and heads do not fill the chip.  Their launches, in order: the sums of
// all segments but the last (k_lattn_sums), the start states by a scan over them (k_lattn_scan), the pass itself (k_lattn).
// The sums read k and v a second time; folding the scan into the pass's prologue was slower than its launch.
//
// Measured (microseconds; floors are the rows' bytes at the 4.76 TB/s of a large copy and the products at the 153 / 1201
// TFLOP/s of large fp32 / bf16 matrix products):
//   one document of 65536 positions, 8 bf16 heads of 128: sums 74 (3.6 TB/s), scan 18, pass 209 (2.6 TB/s); floor 113, and
//     169 with k and v read twice.  Of the pass's time the matrix instructions are busy for 28%, vector arithmetic for 41%, 35%
//     of its waves' time waits (LDS round trips between the barriers, rows from memory).  Four waves a SIMD instead of two (one column tile a wave, 128 registers) spill: 240 us, when operands of two parts
//     took 163.  K and V without bank conflicts in the products of rows (a third of the LDS time has them) cost a register that
//     is not there.
//   forward and backward of 8 x 4096 positions, 8 / 4 bf16 heads of 128: forward 38 + 28 + 105; backward sums 92, scan 28, dq
//     and d rate 190 (matrix 29%, vector 45%, waves waiting 41%, 222 MB), dk and dv 249 (22%, 38%, 46%, 484 MB), d rate's sum 5.
//   forward and backward of 16 x 1024 positions, 4 fp32 heads of 64: forward 14 + 10 + 27; backward 31 + 10 + 51 + 54 + 4; the
//     products alone take 54 at the fp32 rate, and 2 chunks a workgroup leave half of a pass to its ends.
// Registers: a pass of 128 channels fills all 256, with a few in scratch memory (vector / scalar ones the compiler reports: bf16
// forward 2 / 51, dk and dv of shared heads 8 / 166, dq with d rate 2 / 75; fp32 and fp16 up to 9 / 154).
//
// fp16 rows take the fp32 kernels: products of rows would be exact on 16-bit matrix instructions of their type, but the state,
// P and the decayed values leave its range (65504, and below 2^-24), and bf16 parts would have to be cut from the rows as well.
//
// Exactness: sums are formed where they are small and added to the state or the row once (an fp32 matrix instruction rounds after
// every product), a carried state is rounded once or twice a chunk.  Mean square errors of the sizes above: states 1.0e-7 to
// 1.3e-7, fp32 rows 1.9e-7, 4e-4 of the bf16 values rounded otherwise than the exact ones, d rate 1.5e-7 (bf16), 2.0e-7 (fp16) and
// 2.4e-7 (fp32) of the root of its terms' squares; a plain evaluation in fp32 has 1.5e-7, 2.1e-7 and 3e-7 to 6e-7.
#include <type_traits>

#include "ic_types.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
constexpr int kC = 64;
constexpr int64_t kMaxStride = 1 << 22;  // elements from position to position
constexpr int64_t kMaxHeads = 1 << 22;   // sequences * heads (a launch has fewer than 2^32 threads)

struct Mat {  // rows [B,heads,T,D] of one of q, k, v, dout, ...
  void* p;
  int64_t sb, sh, st;
  int32_t group;  // query heads that share one of its heads
  int32_t vec;    // 16-byte accesses are allowed
};

struct Span {
  int32_t nseg, cps;        // segments of a sequence, chunks of a segment
};

struct Pass {               // one application of the map
  Mat q, k, v, out, x;      // x: the rows that the lag-weighted output is multiplied with (d rate)
  Span sp;
  int32_t G;                // query heads whose outputs are one output (gradients of shared heads): a workgroup takes them in turn,
  float* part;              // keeping the sum so far in fp32 rows [B,H/G,T,Db] that only its own lanes touch
  int32_t Da, Db;           // channels of q / k rows and of v / out rows
  int32_t rev;              // positions from the last valid one down
  float oscale, vscale;
  const float* init;        // start state: element (b*H + h) * Dk*Dv + a*ia + b*ib, or NULL: zero
  int32_t ia, ib;
  float* fin;               // end state, laid out like init, or NULL
  int32_t fin_decay;        // the end state takes one more e^{-r} (gradient of the incoming state)
  const float* seg;         // start states of the segments [B*H][nseg][nst][.] with the strides sga, sgb; NULL: one segment
  int32_t sga, sgb, nst;
  const float* gfin;        // gradient of the end state (lag-weighted: d rate), laid out like init, or NULL
  double* dr;               // [B*H][nseg] partial sums of d rate, or NULL
};

struct Sums {               // segment sums of one state
  Mat k, v;
  Span sp;
  int32_t Da, Db, rev;
  float vscale;
  float* seg;
};

struct Geo {
  int32_t B, H, T;
  const float* rate;
  const int32_t* valid_len;
};

struct PassArgs {
  Geo g;
  Pass p[3];
};
struct SumArgs {
  Geo g;
  Sums s[2];
};

__device__ __forceinline__ int valid_of(const Geo& g, int b) {
  if (!g.valid_len) return g.T;
  const int n = g.valid_len[b];
  return n < 0 ? 0 : n < g.T ? n : g.T;
}

// e^{-rate * n}, n >= 0; n = 0 is 1 for every rate
__device__ __forceinline__ float decay(float l2, int n) { return n == 0 ? 1.f : exp2f(l2 * (float)n); }
// A state carried over n positions: e^{-rate n} x, as x + (e^{-rate n} - 1) x where more than half of it stays.  The factor itself,
// rounded next to 1 and applied at every chunk, would leave a slowly decaying state off by that rounding times the number of
// chunks; where little stays, the sum would cancel.
struct Carry {
  float keep, loss;  // 1 and e^{-rate n} - 1, or e^{-rate n} and 0
};
__device__ __forceinline__ Carry carry_of(float rate, int n) {
  const float x = n == 0 ? 0.f : -rate * (float)n, loss = expm1f(x);
  Carry c;
  c.keep = loss > -0.5f ? 1.f : expf(x);
  c.loss = loss > -0.5f ? loss : 0.f;
  return c;
}
__device__ __forceinline__ Carry uniform(Carry c) {  // the same in all lanes: in scalar registers
  c.keep = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(c.keep)));
  c.loss = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(c.loss)));
  return c;
}
// The state carried plus what is new, and with n > 0 positions of lag the lag-weighted one, e^{-rate n} (l + n x) plus what is new:
// the small terms first, so that the sum is rounded once at the state's size.  (What is lost is formed from a finite number: an
// infinite state stays one.)
__device__ __forceinline__ float carried(float x, Carry c, float more) {
  return fmaf(c.keep, x, fmaf(c.loss, __builtin_amdgcn_fmed3f(x, -3.402823466e38f, 3.402823466e38f), more));
}
__device__ __forceinline__ float carried(float x, Carry c) { return fmaf(c.loss, __builtin_amdgcn_fmed3f(x, -3.402823466e38f, 3.402823466e38f), c.keep * x); }
__device__ __forceinline__ v4f carried(const v4f& x, Carry c) { return v4f{carried(x[0], c), carried(x[1], c), carried(x[2], c), carried(x[3], c)}; }
__device__ __forceinline__ float carried_lag(float l, float x, Carry c, int n, float more) { return carried(l, c, fmaf((float)n * (c.keep + c.loss), x, more)); }
__device__ __forceinline__ v4f carried(const v4f& x, Carry c, const v4f& more) {
  v4f y;
#pragma unroll
  for (int v = 0; v < 4; ++v) y[v] = carried(x[v], c, more[v]);
  return y;
}
__device__ __forceinline__ v4f carried_lag(const v4f& l, const v4f& x, Carry c, int n, const v4f& more) {
  v4f y;
#pragma unroll
  for (int v = 0; v < 4; ++v) y[v] = carried_lag(l[v], x[v], c, n, more[v]);
  return y;
}
// a + f b
__device__ __forceinline__ v4f fma4(float f, const v4f& b, const v4f& a) {
  v4f y;
#pragma unroll
  for (int v = 0; v < 4; ++v) y[v] = fmaf(f, b[v], a[v]);
  return y;
}

template <typename T>
__device__ __forceinline__ const T* row_base(const Mat& m, int b, int h) {
  return (const T*)m.p + (int64_t)b * m.sb + (int64_t)(h / m.group) * m.sh;
}

// Rows of one matrix as a workgroup reads them: 16-byte pieces, RT rows at a time.  A chunk's address is uniform, base
// positions times `step` behind `src`; a lane's place in the chunk is fixed (a 32-bit byte offset: 64 rows span less than 2^31
// bytes, checked on the host).  In a reversed pass step < 0 and src is 63 rows below the first position's, so that the lanes'
// offsets count down and stay positive.  Pieces stay in registers until their tile is free (fetch, then put).
__device__ __forceinline__ const char* chunk_src(const char* rows, int64_t st, int n, int rev) { return rows + (rev ? (int64_t)(n - kC) * st : 0); }
template <typename T, int DP, int NTH>
struct RowsF {
  static constexpr int VE = 16 / (int)sizeof(T), PER = DP / VE, RT = NTH / PER, NP = kC / RT;
  const char* src;
  int64_t step;
  uint32_t off;        // this lane's piece of row threadIdx / PER
  int32_t D;
  bool rev, vec, whole;  // whole: (uniform) 16-byte accesses, no lane outside the row
  __device__ __forceinline__ void open(const Mat& m, int b, int h, int D_, int n, int rev_) {
    const int64_t st = m.st * (int)sizeof(T);
    rev = rev_;
    src = chunk_src((const char*)row_base<T>(m, b, h), st, n, rev);
    step = rev ? -st : st;
    D = D_;
    vec = m.vec;
    whole = vec && D == DP;
    const int r = threadIdx.x / PER, c = (threadIdx.x % PER) * VE;
    off = (uint32_t)((rev ? kC - 1 - r : r) * (int32_t)st + c * (int)sizeof(T));
  }
  // rows [base, base + cnt) (virtual positions); others read as zero.  WHOLE: a whole chunk and `whole`
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(uint4 (&x)[NP], int base, int cnt) const {
    const char* at = src + base * step;
    if constexpr (WHOLE) {
#pragma unroll
      for (int j = 0; j < NP; ++j, at += RT * step) x[j] = *reinterpret_cast<const uint4*>(at + off);
      return;
    }
    const int r = threadIdx.x / PER, c = (threadIdx.x % PER) * VE;
#pragma unroll
    for (int j = 0; j < NP; ++j, at += RT * step) {
      x[j] = make_uint4(0, 0, 0, 0);
      if (c < D && r + RT * j < cnt) {
        if (vec) {
          x[j] = *reinterpret_cast<const uint4*>(at + off);
        } else {  // element by element; columns behind the row read its first one and count as zero
          const T* e = (const T*)(at + off);
          T y[VE];
#pragma unroll
          for (int u = 0; u < VE; ++u) {
            const T v = e[c + u < D ? u : 0];
            y[u] = c + u < D ? v : ic_from_f<T>(0.f);
          }
          x[j] = *reinterpret_cast<uint4*>(y);
        }
      }
    }
  }
  static __device__ __forceinline__ void put(float (*dst)[DP + 4], const uint4 (&x)[NP]) {
    const int r = threadIdx.x / PER, c = (threadIdx.x % PER) * VE;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      T e[VE];
      *reinterpret_cast<uint4*>(e) = x[j];
#pragma unroll
      for (int u = 0; u < VE; u += 4)
        *reinterpret_cast<float4*>(&dst[r + RT * j][c + u]) = make_float4(ic_to_f(e[u]), ic_to_f(e[u + 1]), ic_to_f(e[u + 2]), ic_to_f(e[u + 3]));
    }
  }
};
// The value columns of a wave, as operands: element [16 s + q4 + u][col], straight from memory (16 lanes side by side)
template <typename T>
struct ColsF {
  const char* src;
  int64_t step;
  uint32_t off;
  int32_t row0;  // bytes from the chunk's address to virtual row 0
  int32_t q4;
  bool in, whole;
  __device__ __forceinline__ void open(const Mat& m, int b, int h, int D, int n, int rev, int col, int q4_, int DP) {
    const int64_t st = m.st * (int)sizeof(T);
    src = chunk_src((const char*)row_base<T>(m, b, h), st, n, rev);
    step = rev ? -st : st;
    in = col < D;
    whole = D == DP;
    q4 = q4_;
    row0 = (rev ? kC - 1 : 0) * (int32_t)st + (in ? col : 0) * (int)sizeof(T);
    off = (uint32_t)(row0 + q4 * (int32_t)step);
  }
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(v4f (&x)[4], int base, int cnt) const {
    const char* at = src + base * step;
    if constexpr (WHOLE) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int u = 0; u < 4; ++u) x[s][u] = ic_to_f(*reinterpret_cast<const T*>(at + (16 * s + u) * step + off));
      return;
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = 16 * s + q4 + u;
        const bool ok = in && j < cnt;
        const float v = ic_to_f(*reinterpret_cast<const T*>(at + row0 + (ok ? j : 0) * step));
        x[s][u] = ok ? v : 0.f;
      }
  }
};

__device__ __forceinline__ v4f mma(float a, float b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// sum over 16 k-indices: a, b hold k = 4 (lane / 16) + 0..3
__device__ __forceinline__ v4f mma16(v4f a, v4f b, v4f c) {
#pragma unroll
  for (int u = 0; u < 4; ++u) c = mma(a[u], b[u], c);
  return c;
}
__device__ __forceinline__ v4f ld4(const float* p) { return *reinterpret_cast<const v4f*>(p); }

// table[0], table[-1], ...: together and for every lane (left alone, the compiler puts each behind a branch of its own where
// only some lanes use it, and waits for each)
__device__ __forceinline__ void load_decays(float (&d)[4], const float* table) {
#pragma unroll
  for (int v = 0; v < 4; ++v) d[v] = table[-v];
  asm volatile("" : "+v"(d[0]), "+v"(d[1]), "+v"(d[2]), "+v"(d[3]));
}

template <int DP>
struct Lds {
  float Ks[kC][DP + 4];  // (padded rows: 16-byte reads of 16 rows and 4-byte reads of 4 rows spread over the banks)
  float Qs[kC][DP + 4];
  float Ps[kC][kC + 4];
  float dec[2 * kC + 1], dev[2 * kC + 1];  // dec[kC + lag] = e^{-r lag}, 0 for lag < 0; dev = dec * vscale
  double red[DP / 16];
  Carry whole;  // over a chunk
};
template <int DP>
struct LdsSums {
  float Ks[kC][DP + 4];
  float dec[2 * kC + 1], dev[2 * kC + 1];
};

// A wave's slice of a state: elements (16 t + q4 + v, col) at a * ia + b * ib of src.  Out of range: zero, read at a clamped
// address and without a branch, so that all loads are in flight together.
template <int NT>
__device__ __forceinline__ void load_state(v4f (&S)[NT], const float* src, int ia, int ib, int Da, int Db, int col, int q4) {
  const bool in = col < Db;
  const float* at = src + (size_t)(in ? col : 0) * ib;
  if (Da == 16 * NT) {  // (uniform: no row left out)
    at += (size_t)q4 * ia;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float x = at[(size_t)(16 * t + v) * ia];
        S[t][v] = in ? x : 0.f;
      }
    return;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int a = 16 * t + q4 + v;
      const float x = at[(size_t)(a < Da ? a : 0) * ia];
      S[t][v] = in && a < Da ? x : 0.f;
    }
}
template <int NT>
__device__ __forceinline__ void store_state(const v4f (&S)[NT], float* dst, int ia, int ib, int Da, int Db, int col, int q4, float f) {
  if (col >= Db) return;
  float* at = dst + (size_t)col * ib;
  if (Da == 16 * NT) {
    at += (size_t)q4 * ia;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) at[(size_t)(16 * t + v) * ia] = S[t][v] * f;
    return;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int a = 16 * t + q4 + v;
      if (a < Da) at[(size_t)a * ia] = S[t][v] * f;
    }
}
template <int NT>
__device__ __forceinline__ double dot_state(const v4f (&S)[NT], const float* src, int ia, int ib, int Da, int Db, int col, int q4) {
  v4f G[NT];
  load_state(G, src, ia, ib, Da, Db, col, q4);
  double d = 0.0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 4; ++v) d += (double)S[t][v] * (double)G[t][v];
  return d;
}
// the end of a segment: its sums, or (last segment) the end state and its share of d rate; d rate's partial sum.
template <bool LAG, int NT, int NL>
__device__ __forceinline__ void write_sums(const Sums* sm, const v4f (&S)[NT], const v4f (&L)[NL], size_t dd, int Da, int Db, int col, int q4, int bh, int seg) {
  float* dst = sm->seg + ((size_t)bh * sm->sp.nseg + seg) * (LAG ? 2 : 1) * dd;
  store_state(S, dst, Db, 1, Da, Db, col, q4, 1.f);
  if constexpr (LAG) store_state(L, dst + dd, Db, 1, Da, Db, col, q4, 1.f);
}
template <bool LAG, int NT, int NL>
__device__ __forceinline__ double write_end(const Pass* p, const v4f (&S)[NT], const v4f (&L)[NL], size_t dd, int Da, int Db, int col, int q4, int bh, int seg, int n, float l2) {
  double dr = 0.0;
  if (seg != p->sp.nseg - 1) return dr;
  if (p->fin) store_state(S, p->fin + (size_t)bh * dd, p->ia, p->ib, Da, Db, col, q4, p->fin_decay && n > 0 ? decay(l2, 1) : 1.f);
  if constexpr (LAG) {
    if (p->gfin) dr -= dot_state(L, p->gfin + (size_t)bh * dd, p->ia, p->ib, Da, Db, col, q4);
  }
  return dr;
}
// four columns of a shared output: the sum of the heads so far comes from, or goes to, the fp32 rows
__device__ __forceinline__ v4f add_part(const Pass* p, v4f o, int64_t at, int gi, int c0, int D) {
  float* part = p->part + at;
  if (D % 4 == 0) {
    if (gi > 0) o += ld4(part);
    if (gi < p->G - 1) *reinterpret_cast<v4f*>(part) = o;
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (c0 + v >= D) continue;
      if (gi > 0) o[v] += part[v];
      if (gi < p->G - 1) part[v] = o[v];
    }
  }
  return o;
}
template <typename T>
__device__ __forceinline__ void store_row4(char* row, const v4f& o) {
  union { T e[4]; uint4 u4; uint2 u2; } x;
#pragma unroll
  for (int v = 0; v < 4; ++v) x.e[v] = ic_from_f<T>(o[v]);
  if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(row) = x.u4;
  else *reinterpret_cast<uint2*>(row) = x.u2;
}
template <int NW>
__device__ __forceinline__ void write_drate(const Pass* p, double* red, double dr, int bh, int seg) {
  for (int o = 32; o; o >>= 1) dr += __shfl_xor(dr, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = dr;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < NW; ++i) t += red[i];
    p->dr[(size_t)bh * p->sp.nseg + seg] = t;
  }
}

// O += v P^T for the tile on the diagonal, one position at a time and without what lies above: for values that are not all
// finite
__device__ __forceinline__ void add_diagonal(v4f& O, const v4f& v, const v4f& P, int c, int q4) {
#pragma unroll 1
  for (int j0 = 0; j0 < 16; j0 += 4)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const v4f o = mma(q4 == j0 ? v[u] : 0.f, P[u], O);
      if (j0 + u <= c) O = o;
    }
}

template <typename T, int DP, bool LAG, bool SUMS, bool SHARED, typename LDS>
__device__ __forceinline__ void lattn_body(const Geo& g, const Pass* p, const Sums* sm, LDS& lds, int b, int h, int seg) {
  constexpr int NT = DP * 4, NW = DP / 16, KS = DP / 16, MT = (10 + NW - 1) / NW;
  using R = RowsF<T, DP, NT>;
  auto& Ks = lds.Ks;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, q4 = (lane >> 4) * 4;
  const int bh = b * g.H + h;
  const Span sp = SUMS ? sm->sp : p->sp;
  const int n = valid_of(g, b), T_ = g.T;
  const float rate = g.rate[h], l2 = -rate * 1.44269504088896340736f;
  const int Da = SUMS ? sm->Da : p->Da, Db = SUMS ? sm->Db : p->Db;
  const int rev = SUMS ? sm->rev : p->rev;
  const float vscale = SUMS ? sm->vscale : p->vscale, oscale = SUMS ? 1.f : p->oscale;
  const int col = 16 * w + c;  // this lane's value column
  R rk, rq;
  ColsF<T> cv;
  rk.open(SUMS ? sm->k : p->k, b, h, Da, n, rev);
  cv.open(SUMS ? sm->v : p->v, b, h, Db, n, rev, col, q4, DP);
  if constexpr (!SUMS) rq.open(p->q, b, h, Da, n, rev);
  for (int i = threadIdx.x; i < 2 * kC + 1; i += NT) {
    const float d = i < kC ? 0.f : decay(l2, i - kC);
    lds.dec[i] = d;
    lds.dev[i] = d * vscale;
  }
  if constexpr (!SUMS) {
    if (threadIdx.x == 0) lds.whole = carry_of(rate, kC);
  }
  const int NC = (T_ + kC - 1) / kC;
  const int ch0 = seg * sp.cps, ch1 = ch0 + sp.cps < NC ? ch0 + sp.cps : NC;
  const int nend = ch1 * kC < n ? ch1 * kC : n;  // the segment's end
  const size_t dd = (size_t)Da * Db;

  v4f S[KS], L[LAG ? KS : 1];
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    S[t] = v4f{0.f, 0.f, 0.f, 0.f};
    if constexpr (LAG) L[t] = S[t];
  }
  if constexpr (!SUMS) {
    const float* s0 = p->seg ? p->seg + ((size_t)bh * sp.nseg + seg) * p->nst * dd : p->init ? p->init + (size_t)bh * dd : nullptr;
    const int ia = p->seg ? p->sga : p->ia, ib = p->seg ? p->sgb : p->ib;
    if (s0) {
      load_state(S, s0, ia, ib, Da, Db, col, q4);
      if constexpr (LAG) {
        if (p->seg) load_state(L, s0 + dd, ia, ib, Da, Db, col, q4);
      }
    }
  }
  const int b0 = 16 * w + q4;  // this lane's four columns of an output row
  char* out = nullptr;
  int64_t ost = 0, xst = 0;
  uint32_t ooff = 0;
  bool ovec = false, owhole = false;  // (uniform) 16- or 8-byte stores are allowed; no lane outside the row either
  const T* x0 = nullptr;
  if constexpr (!SUMS) {
    ost = p->out.st * (int)sizeof(T);
    out = (char*)const_cast<T*>(row_base<T>(p->out, b, h));
    ooff = (uint32_t)((rev ? kC - 1 - c : c) * (int32_t)ost + b0 * (int)sizeof(T));
    ovec = p->out.vec;
    owhole = ovec && Db == DP;
    if constexpr (LAG) {
      xst = p->x.st;
      x0 = row_base<T>(p->x, b, h);
    }
  }
  double dr = 0.0;
  uint4 fk[R::NP], fq[SUMS ? 1 : R::NP];
  v4f vf[4];
  // one branch for all rows: behind a join of two paths the next loads wait for those in flight
  const bool all = rk.whole && cv.whole && (SUMS || rq.whole);
  auto fetch_as = [&](auto WHOLE, int base, int cnt) {
    rk.template fetch<WHOLE.value>(fk, base, cnt);
    if constexpr (!SUMS) rq.template fetch<WHOLE.value>(fq, base, cnt);
    cv.template fetch<WHOLE.value>(vf, base, cnt);
  };
  auto fetch = [&](int base) {
    if (n - base >= kC && all) fetch_as(std::true_type(), base, kC);
    else fetch_as(std::false_type(), base, n - base < kC ? n - base : kC);
  };
  if (ch0 * kC < n) fetch(ch0 * kC);
  for (int ch = ch0; ch < ch1; ++ch) {
    const int base = ch * kC;
    const int cnt = n - base < 0 ? 0 : n - base < kC ? n - base : kC;
    if (SUMS && cnt == 0) break;
    const int off = rev && ch == 0 ? 1 : 0;  // (the gradient of the final state enters without a step of decay)
    v4f O[4], v0[4];
    float drc = 0.f;
    if (cnt > 0) {
      R::put(Ks, fk);
      if constexpr (!SUMS) R::put(lds.Qs, fq);
#pragma unroll
      for (int s = 0; s < 4; ++s) v0[s] = vf[s];
      __syncthreads();
      if (ch + 1 < ch1 && base + kC < n) fetch(base + kC);
      if constexpr (!SUMS) {
        auto& Ps = lds.Ps;
        auto& Qs = lds.Qs;
        bool finite = true;  // (0 * a value that is not would reach the rows in front of its own)
        if constexpr (!LAG && !SHARED) {
          float bad = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int u = 0; u < 4; ++u) bad = fmaf(v0[s][u], 0.f, bad);
          finite = __all(bad == 0.f);
        }
        v4f E[LAG ? 4 : 1];
        // P[i][j] = e^{-r(i-j)} q_i . k_j for the ten 16x16 tiles with a j <= i, formed transposed (rows j)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int t = w + i * NW;
          if (t >= 10) break;
          const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
          v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < KS; ++s) acc = mma16(ld4(&Ks[16 * jt + c][16 * s + q4]), ld4(&Qs[16 * it + c][16 * s + q4]), acc);
          const int lag0 = 16 * (it - jt) + c - q4;
          float d[4];
          load_decays(d, &lds.dev[kC + lag0]);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            acc[v] = lag0 >= v ? acc[v] * (d[v] * oscale) : 0.f;  // (a select: what lies above the diagonal may be infinite)
          }
          *reinterpret_cast<v4f*>(&Ps[16 * it + c][16 * jt + q4]) = acc;
        }
        // what the state at the chunk's border adds
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          O[it] = v4f{0.f, 0.f, 0.f, 0.f};
          if constexpr (LAG) E[it] = O[it];
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const v4f bq = ld4(&Qs[16 * it + c][16 * s + q4]);
            O[it] = mma16(S[s], bq, O[it]);
            if constexpr (LAG) E[it] = mma16(L[s], bq, E[it]);
          }
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const float f = lds.dec[kC + 16 * it + c + 1 - off] * oscale;
          O[it] = f * O[it];
          if constexpr (LAG) E[it] = fma4((float)(16 * it + c + 1), O[it], f * E[it]);
        }
        __syncthreads();
        if (!finite) {
#pragma unroll
          for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int s = 0; s <= it; ++s) {
              const v4f bp = ld4(&Ps[16 * it + c][16 * s + q4]);
              if (s < it) O[it] = mma16(v0[s], bp, O[it]);
              else add_diagonal(O[it], v0[s], bp, c, q4);
            }
        } else
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          v4f o = v4f{0.f, 0.f, 0.f, 0.f};  // (a sum of its own: see the state's below)
#pragma unroll
          for (int s = 0; s <= it; ++s) {
            v4f bp = ld4(&Ps[16 * it + c][16 * s + q4]);
            o = mma16(v0[s], bp, o);
            if constexpr (LAG) {
#pragma unroll
              for (int u = 0; u < 4; ++u) bp[u] *= (float)(16 * (it - s) + c - q4 - u);  // (0 above the diagonal stays 0)
              E[it] = mma16(v0[s], bp, E[it]);
            }
          }
          O[it] += o;
        }
        if constexpr (LAG) {
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int i = 16 * it + c;
            const T* x = x0 + (base + (i < cnt ? i : 0)) * xst;  // (the lag-weighted pass is no reversed one)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float xv = ic_to_f(x[16 * w + q4 + v < Db ? 16 * w + q4 + v : 0]);
              drc = i < cnt && 16 * w + q4 + v < Db ? fmaf(E[it][v], xv, drc) : drc;
            }
          }
          dr -= (double)drc;
        }
      }
    }
    if constexpr (!SUMS) {
      if (!SHARED && cnt == kC && owhole) {
        const int64_t step = rev ? -ost : ost;
        char* at = const_cast<char*>(chunk_src(out, ost, n, rev)) + base * step;
#pragma unroll
        for (int it = 0; it < 4; ++it, at += 16 * step) store_row4<T>(at + ooff, O[it]);
      } else {
        const int gi = SHARED ? h % p->G : 0;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int i = base + 16 * it + c;
          if (i >= T_ || b0 >= Db) continue;
          const bool live = i < n;
          const int64_t t = rev && live ? n - 1 - i : i;
          v4f o = live ? O[it] : v4f{0.f, 0.f, 0.f, 0.f};
          if constexpr (SHARED) {
            o = add_part(p, o, ((int64_t)(bh / p->G) * T_ + t) * Db + b0, gi, b0, Db);
            if (gi < p->G - 1) continue;
          }
          char* row = out + t * ost + b0 * (int)sizeof(T);
          if (ovec) {
            store_row4<T>(row, o);
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (b0 + v < Db) ((T*)row)[v] = ic_from_f<T>(o[v]);
          }
        }
      }
    }
    if (cnt > 0) {  // the state behind the chunk; a segment's sums weigh every position from the segment's end, with no carry
      const int left = SUMS ? nend - base - cnt : 0;
      const float ahead = SUMS ? decay(l2, left) : 1.f;
      Carry over{};
      if constexpr (!SUMS) over = cnt - off == kC ? lds.whole : carry_of(rate, cnt - off);
      constexpr int HS = LAG && DP == 128 ? 1 : 2;
      // A half chunk's own sum first, then one addition: a matrix instruction rounds after each of its products, and added to the
      // state one by one each of the chunk's 64 would be rounded at the state's size (1024 positions of slow decay: state off by
      // 5.1e-7 in the mean square, so 1.4e-7).
#pragma unroll
      for (int s0 = 0; s0 < 4; s0 += HS) {
        v4f vw[HS];
#pragma unroll
        for (int s = 0; s < HS; ++s) {
          float d[4];
          load_decays(d, &lds.dev[kC + cnt - 1 - q4 - 16 * (s0 + s)]);
#pragma unroll
          for (int u = 0; u < 4; ++u) vw[s][u] = v0[s0 + s][u] * (SUMS ? d[u] * ahead : d[u]);
        }
#pragma unroll
        for (int t = 0; t < KS; ++t) {
          v4f ds = v4f{0.f, 0.f, 0.f, 0.f}, dl = ds;
#pragma unroll
          for (int s = 0; s < HS; ++s) {
            v4f ak;
#pragma unroll
            for (int u = 0; u < 4; ++u) ak[u] = Ks[16 * (s0 + s) + q4 + u][16 * t + c];
            ds = mma16(ak, vw[s], ds);
            if constexpr (LAG) {
              v4f vl;
#pragma unroll
              for (int u = 0; u < 4; ++u) vl[u] = vw[s][u] * (float)(left + cnt - 1 - q4 - 16 * (s0 + s) - u);  // (0 behind the last valid position)
              dl = mma16(ak, vl, dl);
            }
          }
          if constexpr (LAG) L[t] = SUMS || s0 ? L[t] + dl : carried_lag(L[t], S[t], over, cnt, dl);
          S[t] = SUMS || s0 ? S[t] + ds : carried(S[t], over, ds);
        }
      }
      __syncthreads();
    }
  }
  if constexpr (SUMS) {
    write_sums<LAG>(sm, S, L, dd, Da, Db, col, q4, bh, seg);
  } else {
    dr += write_end<LAG>(p, S, L, dd, Da, Db, col, q4, bh, seg, n, l2);
    if constexpr (LAG) write_drate<NW>(p, lds.red, dr, bh, seg);
  }
}

// ------------------------------------------------------------------------------------------------ bf16 rows
// Rows that allow 16-byte accesses (others take the body above).
// The same map on bf16 matrix instructions (16x16x32: sixteen times the fp32 rate).  Products of rows (q . k) are exact
// there.  Operands that are computed in fp32 -- the decayed products P, the state, the decay-weighted values -- are split
// into three bf16 parts (x = x1 + x2 + x3, each the rounded rest of the one before, 8 bits apiece), all of fp32's 24 bits.  Two
// parts are 13% faster (wide training pass of the figures above: 564 us), but 16 bits are fewer than the sums' 24: 3e-3 of the bf16
// results were rounded otherwise than the exact ones, states off by 2.4e-6.
// Rows lie in LDS as they come; column operands (k^T, v^T) are read with the transposing LDS load
// (16 lanes x 8 bytes of four rows -> four rows of one column per lane).  A 32-deep operand of a lane is therefore k-indices
// 4 q .. 4 q + 3 of either 16-row half, on both sides of a product; products of rows use contiguous eights instead.
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
constexpr int kParts = 3;
// P in LDS, three parts: rows of 32 positions in the upper half (the others lie above the diagonal), of 64 in the lower; 16 bytes
// of padding a row
constexpr int kPn = 32 * (32 + 8) + 32 * (64 + 8);
__device__ __forceinline__ int p_row(int i) { return i < 32 ? 40 * i : 72 * i - 1024; }

// padding: 32 bytes a row spread the 8 rows of a transposing read over the 64 banks, 16 bytes the 16 rows of a 16-byte read
template <int W>
struct RowTile {
  uint16_t r[kC][W];
};
template <int DP, bool LAG>
struct Lds16 {
  RowTile<DP + 16> K, V;
  RowTile<DP + 8> Q;
  RowTile<LAG ? DP + 8 : 1> X;
  uint16_t P[kParts][kPn];
  float dec[2 * kC + 1], dev[2 * kC + 1];  // dec[kC + lag] = e^{-r lag}, 0 for lag < 0; dev = dec * vscale
  double red[DP / 16];
  Carry whole;  // over a chunk
};
template <int DP>
struct LdsSums16 {
  RowTile<DP + 16> K, V;
  float dec[2 * kC + 1], dev[2 * kC + 1];
};

__device__ __forceinline__ v4f mma32(b8 a, b8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ b8 lds16(const uint16_t* p) { return *reinterpret_cast<const b8*>(p); }
__device__ __forceinline__ b8 lds8x2(const uint16_t* p) {  // k-indices p[0..3] and p[16..19]
  union { uint64_t u[2]; b8 b; } x;
  x.u[0] = *reinterpret_cast<const uint64_t*>(p);
  x.u[1] = *reinterpret_cast<const uint64_t*>(p + 16);
  return x.b;
}
// rows [r0, r0 + 32) of column c0 + lane % 16: k-indices 4 (lane / 16) + 0..3 of either half
template <int W>
__device__ __forceinline__ b8 lds_col(const uint16_t (*t)[W], int r0, int c0, int lane) {
  const int c = lane & 15, q = lane >> 4;
  const uint16_t* p = &t[r0 + 4 * q + (c >> 2)][c0 + 4 * (c & 3)];
  union { s4v s[2]; b8 b; } x;
  x.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)p);
  x.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(p + 16 * W));
  return x.b;
}
// two values' bf16 parts; take2: x keeps the rest
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2)); }
__device__ __forceinline__ uint32_t take2(float& a, float& b) {
  const uint32_t u = pack2(a, b);
  a -= __uint_as_float(u << 16);
  b -= __uint_as_float(u & 0xffff0000u);
  return u;
}
template <int N>
__device__ __forceinline__ void split(float (&x)[8], b8 (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    union { uint32_t u[4]; b8 b; } y;
#pragma unroll
    for (int u = 0; u < 4; ++u) y.u[u] = i + 1 < N ? take2(x[2 * u], x[2 * u + 1]) : pack2(x[2 * u], x[2 * u + 1]);
    out[i] = y.b;
  }
}
template <int N>
__device__ __forceinline__ void split(const v4f& a, const v4f& b, b8 (&out)[N]) {
  float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  split(x, out);
}

// four consecutive columns of an output row
__device__ __forceinline__ void store4(char* row, const v4f& o) {
  *reinterpret_cast<uint2*>(row) = make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
}

// RowsF for bf16 tiles that stay bf16 (16-byte accesses only)
template <int DP, int CW>
struct Rows {
  static constexpr int RT = 32 / CW, NP = 2 * CW;  // rows at a time, times
  const char* src;
  int64_t step;
  uint32_t off;  // this lane's piece of row threadIdx / (DP / 8)
  bool live;     // inside the row
  bool whole;    // (uniform) every lane is
  __device__ __forceinline__ void open(const Mat& m, int b, int h, int D, int n, int rev) {
    constexpr int PER = DP / 8;
    const int64_t st = m.st * 2;
    src = chunk_src((const char*)row_base<uint16_t>(m, b, h), st, n, rev);
    step = rev ? -st : st;
    const int r = threadIdx.x / PER, c = (threadIdx.x % PER) * 8;
    live = c < D;
    whole = D == DP;
    off = (uint32_t)((rev ? kC - 1 - r : r) * (int32_t)st + c * 2);
  }
  // rows [base, base + cnt) (virtual positions); others read as zero.  WHOLE: a whole chunk and `whole`
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(uint4 (&x)[NP], int base, int cnt) const {
    const int r = threadIdx.x / (DP / 8);
    const char* at = src + base * step;
    if constexpr (WHOLE) {  // (no lane left out)
#pragma unroll
      for (int j = 0; j < NP; ++j, at += RT * step) x[j] = *reinterpret_cast<const uint4*>(at + off);
      return;
    }
#pragma unroll
    for (int j = 0; j < NP; ++j, at += RT * step) {
      x[j] = make_uint4(0, 0, 0, 0);
      if (live && r + RT * j < cnt) x[j] = *reinterpret_cast<const uint4*>(at + off);
    }
  }
  template <int W>
  static __device__ __forceinline__ void put(RowTile<W>& dst, const uint4 (&x)[NP]) {
    constexpr int PER = DP / 8;
#pragma unroll
    for (int j = 0; j < NP; ++j) *reinterpret_cast<uint4*>(&dst.r[threadIdx.x / PER + RT * j][(threadIdx.x % PER) * 8]) = x[j];
  }
};

// O += P v by elements and without the products above the diagonal: for the chunks whose values are not all finite
template <int CW, int W>
__device__ __forceinline__ void add_rows_at_or_before(v4f (&O)[CW][4], const uint16_t (*P)[kPn], const uint16_t (*V)[W], int cnt, int c, int b0) {
#pragma unroll 1
  for (int j = 0; j < cnt; ++j) {
    const int at = 32 * (j >> 5) + 8 * ((j >> 2) & 3) + 4 * ((j >> 4) & 1) + (j & 3);
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int i = 16 * it + c;
      if (j > i) continue;
      const int e = p_row(i) + at;
      const float pj = __uint_as_float((uint32_t)P[0][e] << 16) + (__uint_as_float((uint32_t)P[1][e] << 16) + __uint_as_float((uint32_t)P[2][e] << 16));
#pragma unroll
      for (int k = 0; k < CW; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) O[k][it][v] = fmaf(pj, __uint_as_float((uint32_t)V[j][b0 + 16 * k + v] << 16), O[k][it][v]);
    }
  }
}

// A wave owns CW tiles of 16 value columns; a workgroup has DP / (16 CW) waves.
template <int DP, int CW, bool LAG, bool SUMS, bool SHARED, typename LDS>
__device__ __forceinline__ void lattn_body16(const Geo& g, const Pass* p, const Sums* sm, LDS& lds, int b, int h, int seg) {
  constexpr int NW = DP / (16 * CW), NT = DP / 16, KS = DP / 32, MT = (10 + NW - 1) / NW;
  using R = Rows<DP, CW>;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, q4 = (lane >> 4) * 4;
  const int bh = b * g.H + h;
  const Span sp = SUMS ? sm->sp : p->sp;
  const int n = valid_of(g, b), T = g.T;
  const float rate = g.rate[h], l2 = -rate * 1.44269504088896340736f;
  const int Da = SUMS ? sm->Da : p->Da, Db = SUMS ? sm->Db : p->Db;
  const int rev = SUMS ? sm->rev : p->rev;
  const float vscale = SUMS ? sm->vscale : p->vscale, oscale = SUMS ? 1.f : p->oscale;
  R rk, rv, rq, rx;
  rk.open(SUMS ? sm->k : p->k, b, h, Da, n, rev);
  rv.open(SUMS ? sm->v : p->v, b, h, Db, n, rev);
  if constexpr (!SUMS) rq.open(p->q, b, h, Da, n, rev);
  if constexpr (!SUMS && LAG) rx.open(p->x, b, h, Db, n, rev);
  for (int i = threadIdx.x; i < 2 * kC + 1; i += 64 * NW) {
    const float d = i < kC ? 0.f : decay(l2, i - kC);
    lds.dec[i] = d;
    lds.dev[i] = d * vscale;
  }
  if constexpr (!SUMS) {
    if (threadIdx.x == 0) lds.whole = carry_of(rate, kC);
  }
  const int col0 = 16 * CW * w;  // this wave's columns
  const int NC = (T + kC - 1) / kC;
  const int ch0 = seg * sp.cps, ch1 = ch0 + sp.cps < NC ? ch0 + sp.cps : NC;
  const int nend = ch1 * kC < n ? ch1 * kC : n;  // the segment's end
  const size_t dd = (size_t)Da * Db;

  v4f S[CW][NT], L[LAG ? CW : 1][LAG ? NT : 1];
#pragma unroll
  for (int k = 0; k < CW; ++k)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      S[k][t] = v4f{0.f, 0.f, 0.f, 0.f};
      if (LAG) L[k][t] = S[k][t];
    }
  char* out = nullptr;
  int64_t ost = 0;
  uint32_t ooff = 0;
  if constexpr (!SUMS) {
    ost = p->out.st * 2;
    out = (char*)p->out.p + ((int64_t)b * p->out.sb + (int64_t)(h / p->out.group) * p->out.sh) * 2;
    ooff = (uint32_t)((rev ? kC - 1 - c : c) * (int32_t)ost + (col0 + q4) * 2);
    const float* s0 = p->seg ? p->seg + ((size_t)bh * sp.nseg + seg) * p->nst * dd : p->init ? p->init + (size_t)bh * dd : nullptr;
    const int ia = p->seg ? p->sga : p->ia, ib = p->seg ? p->sgb : p->ib;
    if (s0) {
#pragma unroll
      for (int k = 0; k < CW; ++k) {
        load_state(S[k], s0, ia, ib, Da, Db, col0 + 16 * k + c, q4);
        if constexpr (LAG) {
          if (p->seg) load_state(L[k], s0 + dd, ia, ib, Da, Db, col0 + 16 * k + c, q4);
        }
      }
    }
    // the two 16x16 tiles of P above the diagonal that a 32-deep product reads stay zero
    for (int i = threadIdx.x; i < 128; i += 64 * NW) {
      const int it = (i >> 6) << 1, r = i & 15, at = 32 * (it >> 1) + 8 * ((i >> 4) & 3) + 4;
#pragma unroll
      for (int k = 0; k < kParts; ++k) *reinterpret_cast<uint64_t*>(&lds.P[k][p_row(16 * it + r) + at]) = 0;
    }
  }
  double dr = 0.0;
  uint4 fk[R::NP], fv[R::NP], fq[SUMS ? 1 : R::NP], fx[!SUMS && LAG ? R::NP : 1];
  // one branch for all rows: behind a join of two paths the next loads wait for those in flight
  const bool all = rk.whole && rv.whole;
  auto fetch_as = [&](auto WHOLE, int base, int cnt) {
    rk.template fetch<WHOLE.value>(fk, base, cnt);
    rv.template fetch<WHOLE.value>(fv, base, cnt);
    if constexpr (!SUMS) rq.template fetch<WHOLE.value>(fq, base, cnt);
    if constexpr (!SUMS && LAG) rx.template fetch<WHOLE.value>(fx, base, cnt);
  };
  auto fetch = [&](int base) {
    if (n - base >= kC && all) fetch_as(std::true_type(), base, kC);
    else fetch_as(std::false_type(), base, n - base < kC ? n - base : kC);
  };
  if (ch0 * kC < n) fetch(ch0 * kC);
  for (int ch = ch0; ch < ch1; ++ch) {
    const int base = ch * kC;
    const int cnt = n - base < 0 ? 0 : n - base < kC ? n - base : kC;
    if (SUMS && cnt == 0) break;
    const int off = rev && ch == 0 ? 1 : 0;  // (the gradient of the final state enters without a step of decay)
    v4f O[CW][4];
    b8 vf[CW][2];
    if (cnt > 0) {
      R::put(lds.K, fk);
      R::put(lds.V, fv);
      if constexpr (!SUMS) R::put(lds.Q, fq);
      if constexpr (!SUMS && LAG) R::put(lds.X, fx);
      __syncthreads();
      if (ch + 1 < ch1 && base + kC < n) fetch(base + kC);
#pragma unroll
      for (int k = 0; k < CW; ++k)
#pragma unroll
        for (int s = 0; s < 2; ++s) vf[k][s] = lds_col(lds.V.r, 32 * s, col0 + 16 * k, lane);
      if constexpr (!SUMS) {
        float drc = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int t = w + i * NW;
          if (t >= 10) break;
          const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
          v4f acc = v4f{0.f, 0.f, 0.f, 0.f}, ax = acc;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            acc = mma32(lds16(&lds.K.r[16 * jt + c][32 * s + 2 * q4]), lds16(&lds.Q.r[16 * it + c][32 * s + 2 * q4]), acc);
            if constexpr (LAG) ax = mma32(lds16(&lds.V.r[16 * jt + c][32 * s + 2 * q4]), lds16(&lds.X.r[16 * it + c][32 * s + 2 * q4]), ax);
          }
          float x[4];
          const int lag0 = 16 * (it - jt) + c - q4;
          float d[4];
          load_decays(d, &lds.dev[kC + lag0]);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            x[v] = lag0 >= v ? acc[v] * (d[v] * oscale) : 0.f;  // (a select: what lies above the diagonal may be infinite)
            if constexpr (LAG) drc = lag0 > v ? fmaf((float)(lag0 - v) * x[v], ax[v], drc) : drc;
          }
          const int at = p_row(16 * it + c) + 32 * (jt >> 1) + 2 * q4 + 4 * (jt & 1);  // the order in which a 32-deep operand of P is read
#pragma unroll
          for (int k = 0; k < kParts; ++k) {
            uint2 y;
            y.x = k + 1 < kParts ? take2(x[0], x[1]) : pack2(x[0], x[1]);
            y.y = k + 1 < kParts ? take2(x[2], x[3]) : pack2(x[2], x[3]);
            *reinterpret_cast<uint2*>(&lds.P[k][at]) = y;
          }
        }
        v4f E[LAG ? CW : 1][4];
#pragma unroll
        for (int k = 0; k < CW; ++k)
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            O[k][it] = v4f{0.f, 0.f, 0.f, 0.f};
            if constexpr (LAG) E[k][it] = O[k][it];
          }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          b8 sp[CW][kParts], lp[LAG ? CW : 1][kParts];
#pragma unroll
          for (int k = 0; k < CW; ++k) {
            split(S[k][2 * s], S[k][2 * s + 1], sp[k]);
            if constexpr (LAG) split(L[k][2 * s], L[k][2 * s + 1], lp[k]);
          }
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const b8 bq = lds8x2(&lds.Q.r[16 * it + c][32 * s + q4]);
#pragma unroll
            for (int i = 0; i < kParts; ++i)
#pragma unroll
              for (int k = 0; k < CW; ++k) {
                O[k][it] = mma32(sp[k][i], bq, O[k][it]);
                if constexpr (LAG) E[k][it] = mma32(lp[k][i], bq, E[k][it]);
              }
          }
        }
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const float f = lds.dec[kC + 16 * it + c + 1 - off] * oscale;
#pragma unroll
          for (int k = 0; k < CW; ++k) {
            O[k][it] = f * O[k][it];
            if constexpr (LAG) {  // what the lag-weighted state adds to d rate
              E[k][it] = fma4((float)(16 * it + c + 1), O[k][it], f * E[k][it]);
              const uint16_t* x = &lds.X.r[16 * it + c][col0 + 16 * k + q4];
#pragma unroll
              for (int v = 0; v < 4; ++v) drc = fmaf(E[k][it][v], __uint_as_float((uint32_t)x[v] << 16), drc);
            }
          }
        }
        if (LAG) dr -= (double)drc;
        bool finite = true;  // (0 * a value that is not would reach the rows in front of its own)
        if constexpr (!LAG && !SHARED) {
          float bad = 0.f;
#pragma unroll
          for (int k = 0; k < CW; ++k)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int u = 0; u < 4; ++u) bad = __builtin_amdgcn_fdot2_f32_bf16((b2){vf[k][s][2 * u], vf[k][s][2 * u + 1]}, (b2){(__bf16)0.f, (__bf16)0.f}, bad, false);
          finite = __all(bad == 0.f);
        }
        __syncthreads();
        if (!finite) {
          add_rows_at_or_before(O, lds.P, lds.V.r, cnt, c, col0 + q4);
        } else
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
          for (int s = 0; s <= it / 2; ++s) {
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
              const b8 bp = lds16(&lds.P[i][p_row(16 * it + c) + 32 * s + 2 * q4]);
#pragma unroll
              for (int k = 0; k < CW; ++k) O[k][it] = mma32(vf[k][s], bp, O[k][it]);
            }
          }
      }
    }
    if constexpr (!SUMS) {
      if constexpr (SHARED) {  // the sum of the heads so far in fp32 rows
        const int gi = h % p->G;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int i = base + 16 * it + c;
          const bool live = i < n;
          const int64_t t = rev && live ? n - 1 - i : i;
#pragma unroll
          for (int k = 0; k < CW; ++k) {
            const int b0 = col0 + 16 * k + q4;
            if (i >= T || b0 >= Db) continue;
            const v4f o = add_part(p, live ? O[k][it] : v4f{0.f, 0.f, 0.f, 0.f}, ((int64_t)(bh / p->G) * T + t) * Db + b0, gi, b0, Db);
            if (gi == p->G - 1) store4(out + t * ost + b0 * 2, o);
          }
        }
      } else if (cnt == kC && rv.whole) {  // a whole chunk
        const int64_t step = rev ? -ost : ost;
        char* at = const_cast<char*>(chunk_src(out, ost, n, rev)) + base * step;
#pragma unroll
        for (int it = 0; it < 4; ++it, at += 16 * step)
#pragma unroll
          for (int k = 0; k < CW; ++k) store4(at + ooff + 32 * k, O[k][it]);
      } else {
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int i = base + 16 * it + c;
          const bool live = i < n;
          char* at = out + (rev && live ? n - 1 - i : i) * ost + (col0 + q4) * 2;
#pragma unroll
          for (int k = 0; k < CW; ++k) {
            if (!live) O[k][it] = v4f{0.f, 0.f, 0.f, 0.f};
            if (i < T && col0 + 16 * k + q4 < Db) store4(at + 32 * k, O[k][it]);
          }
        }
      }
    }
    if (cnt > 0) {  // the state behind the chunk; a segment's sums weigh every position from the segment's end, with no carry
      const int left = SUMS ? nend - base - cnt : 0;
      const float ahead = SUMS ? decay(l2, left) : 1.f;
      Carry over{};
      if constexpr (!SUMS) over = cnt - off == kC ? lds.whole : carry_of(rate, cnt - off);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        b8 vp[CW][kParts], lp[LAG ? CW : 1][kParts];
        const float* dl = &lds.dev[kC + cnt - 1 - q4 - 51];  // (51: the largest position of this lane's values)
#pragma unroll
        for (int k = 0; k < CW; ++k) {
          float x[8], y[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int j = 32 * s + 16 * (u >> 2) + (u & 3);
            x[u] = (float)vf[k][s][u] * (SUMS ? dl[51 - j] * ahead : dl[51 - j]);
            if constexpr (LAG) y[u] = x[u] * (float)(left + cnt - 1 - q4 - j);  // (0 behind the last valid position)
          }
          split(x, vp[k]);
          if constexpr (LAG) split(y, lp[k]);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const b8 ak = lds_col(lds.K.r, 32 * s, 16 * t, lane);
#pragma unroll
          for (int k = 0; k < CW; ++k) {  // (a half chunk's own sum first, as for fp32 rows)
            v4f ds = v4f{0.f, 0.f, 0.f, 0.f}, dl = ds;
#pragma unroll
            for (int i = kParts - 1; i >= 0; --i) {
              ds = mma32(ak, vp[k][i], ds);
              if constexpr (LAG) dl = mma32(ak, lp[k][i], dl);
            }
            if constexpr (LAG) L[k][t] = SUMS || s ? L[k][t] + dl : carried_lag(L[k][t], S[k][t], over, cnt, dl);
            if (SUMS || s) S[k][t] += ds;
            else if (CW == 1) S[k][t] = carried(S[k][t], over, ds);
            else S[k][t] = carried(S[k][t], over) + ds;  // (in one sum the two tiles a wave spill: a pass of 302 instead of 202 us)
          }
        }
      }
      __syncthreads();
    }
  }
  if constexpr (SUMS) {
#pragma unroll
    for (int k = 0; k < CW; ++k) write_sums<LAG>(sm, S[k], L[LAG ? k : 0], dd, Da, Db, col0 + 16 * k + c, q4, bh, seg);
  } else {
#pragma unroll
    for (int k = 0; k < CW; ++k) dr += write_end<LAG>(p, S[k], L[LAG ? k : 0], dd, Da, Db, col0 + 16 * k + c, q4, bh, seg, n, l2);
    if constexpr (LAG) write_drate<NW>(p, lds.red, dr, bh, seg);
  }
}

// bf16 rows, 128 channels: two column tiles a wave, so that 4 waves own the columns and two workgroups fit a compute unit
// (77 KB of LDS, <= 256 registers): the one's barriers under the other's products.  One tile a wave where the lag-weighted
// state doubles the registers.
template <int DP, bool LAG, bool W16>
constexpr int cw_of() { return W16 && DP == 128 && !LAG ? 2 : 1; }

// LAG: the pass that carries the lag-weighted state, a launch of its own (its registers and LDS would bound the others).
template <typename T, int DP, bool LAG, bool W16, bool SHARED>
__global__ __launch_bounds__((DP * 4 / cw_of<DP, LAG, W16>()), (DP == 64 && !LAG ? 3 : 2)) void k_lattn(PassArgs a) {
  __shared__ __align__(16) std::conditional_t<W16, Lds16<DP, LAG>, Lds<DP>> lds;
  const Pass* p = &a.p[blockIdx.y];
  const int seg = blockIdx.x % p->sp.nseg, u = blockIdx.x / p->sp.nseg;
  auto body = [&](int b, int h) __attribute__((always_inline)) {
    if constexpr (W16) lattn_body16<DP, cw_of<DP, LAG, W16>(), LAG, false, SHARED>(a.g, p, nullptr, lds, b, h, seg);
    else lattn_body<T, DP, LAG, false, SHARED>(a.g, p, nullptr, lds, b, h, seg);
  };
  if constexpr (SHARED) {
    const int U = a.g.H / p->G, b = u / U;
    for (int gi = 0; gi < p->G; ++gi) body(b, (u - b * U) * p->G + gi);
  } else {
    const int b = u / a.g.H;
    if (b < a.g.B) body(b, u - b * a.g.H);  // (a launch is as wide as its widest pass)
  }
}
// (the last segment's sum is not needed)
template <typename T, int DP, bool LAG, bool W16>
__global__ __launch_bounds__(DP * 4) void k_lattn_sums(SumArgs a) {
  __shared__ __align__(16) std::conditional_t<W16, LdsSums16<DP>, LdsSums<DP>> lds;
  const Sums& z = a.s[blockIdx.y];
  const int n = z.sp.nseg - 1;
  if ((int)blockIdx.x >= a.g.B * a.g.H * n) return;
  const int seg = blockIdx.x % n, bh = blockIdx.x / n, b = bh / a.g.H, h = bh - b * a.g.H;
  if constexpr (W16) {
    if (LAG && blockIdx.y == 0) lattn_body16<DP, 1, LAG, true, false>(a.g, nullptr, &z, lds, b, h, seg);
    else lattn_body16<DP, 1, false, true, false>(a.g, nullptr, &z, lds, b, h, seg);
  } else {
    if (LAG && blockIdx.y == 0) lattn_body<T, DP, LAG, true, false>(a.g, nullptr, &z, lds, b, h, seg);
    else lattn_body<T, DP, false, true, false>(a.g, nullptr, &z, lds, b, h, seg);
  }
}

// segment sums -> start states: seg[s] <- state in front of segment s.  A thread owns an element of a state; memory-bound but for
// the ends of its chain (64 segments of 8 heads of 128 x 128: 67 MB in 17 us, 3.9 TB/s; with eight sums in flight 7 us more).
struct ScanState {
  Span sp;
  float* seg;
  const float* init;
  int32_t Da, Db, ia, ib, lag, rev;
};
struct ScanArgs {
  Geo g;
  ScanState s[2];
};
__global__ __launch_bounds__(256) void k_lattn_scan(ScanArgs a) {
  const ScanState& z = a.s[blockIdx.z];
  const int dd = z.Da * z.Db, e = blockIdx.y * 256 + threadIdx.x, bh = blockIdx.x;
  if (e >= dd || z.sp.nseg <= 1) return;
  const int b = bh / a.g.H, h = bh - b * a.g.H, n = valid_of(a.g, b), len = z.sp.cps * kC;
  const float rate = a.g.rate[h];
  const int nst = z.lag ? 2 : 1;
  float* at = z.seg + (size_t)bh * z.sp.nseg * nst * dd + e;
  float S = z.init ? z.init[(size_t)bh * dd + (size_t)(e / z.Db) * z.ia + (size_t)(e % z.Db) * z.ib] : 0.f, L = 0.f;
  const size_t next = (size_t)nst * dd;
  constexpr int U = 16;  // sums in flight: the chain of states would wait for each of them in turn otherwise
  // segments in front of the one that the sequence ends in, that one, and those behind it; in a reversed pass the first position
  // takes no decay
  const int p = n / len, r = n - p * len;
  const Carry none{1.f, 0.f}, whole = uniform(carry_of(rate, len));
  Carry first = whole, part = none;
  if (z.rev) first = uniform(carry_of(rate, len - 1));
  if (r > 0 && p < z.sp.nseg - 1) part = uniform(carry_of(rate, z.rev && p == 0 ? r - 1 : r));  // (nothing starts behind the last one)
  for (int s0 = 0; s0 < z.sp.nseg; s0 += U, at += U * next) {
    float ls[U], ll[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool more = s0 + u + 1 < z.sp.nseg;  // (the last segment's sum is not formed)
      ls[u] = more ? at[u * next] : 0.f;
      ll[u] = more && z.lag ? at[u * next + dd] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u;
      if (s < z.sp.nseg) {
        const int cnt = s < p ? len : s == p ? r : 0;
        at[u * next] = S;
        if (z.lag) at[u * next + dd] = L;
        const Carry over = s < p ? (s == 0 ? first : whole) : s == p ? part : none;
        L = carried_lag(L, S, over, cnt, ll[u]);
        S = carried(S, over, ls[u]);
      }
    }
  }
}

// d rate of a head: over sequences and segments, in 64 bits
__global__ __launch_bounds__(64) void k_lattn_drate(const double* part, float* drate, int B, int H, int nseg) {
  const int h = blockIdx.x;
  double v = 0.0;
  for (int i = threadIdx.x; i < B * nseg; i += 64) v += part[((size_t)(i / nseg) * H + h) * nseg + i % nseg];
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  if (threadIdx.x == 0) drate[h] = (float)v;
}

// One position.  Memory-bound: the state is read and written once (256 sequences, 16 heads of 128 x 128: 537 MB in 114 us, 4.7 TB/s,
// a large copy's rate; a call for 4 heads of 64 x 64 costs its launch, 11 us).  A workgroup owns (sequence, head, 32 value columns):
// 8 lanes x 4 columns, 32 rows of threads over the key channels; the output's sum over them goes through LDS.
constexpr int kStepRows = 32;
template <typename T>
__global__ __launch_bounds__(256) void k_lattn_step(ic_lattn_step_args a) {
  __shared__ float red[kStepRows][33];
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hk);
  const int r = threadIdx.x >> 3, c0 = blockIdx.y * 32 + (threadIdx.x & 7) * 4;
  T* out = (T*)a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
  const int oc = blockIdx.y * 32 + threadIdx.x;
  if (a.active && !a.active[b]) {
    if (threadIdx.x < 32 && oc < a.Dv) out[oc] = ic_from_f<T>(0.f);
    return;
  }
  const T* Q = (const T*)a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh;
  const T* K = (const T*)a.k + (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh;
  const T* V = (const T*)a.v + (int64_t)b * a.v_sb + (int64_t)hk * a.v_sh;
  float* S = a.state + (size_t)bh * a.Dk * a.Dv;
  const float dec = expf(-a.rate[h]);
  float v[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = c0 + u < a.Dv ? ic_to_f(V[c0 + u]) : 0.f;
  const bool vec = a.Dv % 4 == 0 && ((uintptr_t)a.state & 15) == 0;
  for (int k = r; k < a.Dk; k += kStepRows) {
    const float kk = ic_to_f(K[k]), qq = ic_to_f(Q[k]);
    float* row = S + (size_t)k * a.Dv;
    if (vec) {
      if (c0 < a.Dv) {
        v4f x = ld4(row + c0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          x[u] = fmaf(kk, v[u], dec * x[u]);
          o[u] = fmaf(qq, x[u], o[u]);
        }
        *reinterpret_cast<v4f*>(row + c0) = x;
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u < a.Dv) {
          const float x = fmaf(kk, v[u], dec * row[c0 + u]);
          row[c0 + u] = x;
          o[u] = fmaf(qq, x, o[u]);
        }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) red[r][(threadIdx.x & 7) * 4 + u] = o[u];
  __syncthreads();
  if (threadIdx.x < 32 && oc < a.Dv) {
    float s[kStepRows];  // (in pairs: five roundings on a term's path, one after the other 32)
#pragma unroll
    for (int i = 0; i < kStepRows; ++i) s[i] = red[i][threadIdx.x];
#pragma unroll
    for (int w = kStepRows / 2; w; w /= 2)
#pragma unroll
      for (int i = 0; i < w; ++i) s[i] += s[i + w];
    out[oc] = ic_from_f<T>(s[0] * a.scale);
  }
}

// ------------------------------------------------------------------------------------------------------------- host
int check_lattn(const ic_lattn_args* a, const char* who) {
  IC_REQUIRE(a != nullptr, "%s: NULL args", who);
  IC_REQUIRE(a->B >= 1 && a->H >= 1 && a->T >= 1, "%s: B=%d H=%d T=%d", who, a->B, a->H, a->T);
  IC_REQUIRE(a->Hk >= 1 && a->H % a->Hk == 0, "%s: H=%d is no multiple of Hk=%d", who, a->H, a->Hk);
  IC_REQUIRE((int64_t)a->B * a->H <= kMaxHeads, "%s: B*H=%lld (at most 2^22)", who, (long long)a->B * a->H);
  IC_REQUIRE(a->T <= (1 << 30), "%s: T=%d (at most 2^30)", who, a->T);
  IC_REQUIRE(a->Dk >= 1 && a->Dk <= 128 && a->Dv >= 1 && a->Dv <= 128, "%s: Dk=%d Dv=%d (need 1 .. 128)", who, a->Dk, a->Dv);
  IC_REQUIRE(ic_dt_ok(a->dtype), "%s: dtype=%d", who, a->dtype);
  return IC_OK;
}

// 64 rows of a matrix lie within 2^31 bytes behind the first one (the kernels' offsets inside a chunk, unsigned)
int check_stride(int64_t st, const char* who, const char* n) {
  IC_REQUIRE(st >= 0 && st < kMaxStride, "%s: %s has %lld elements from position to position (0 to below %lld)", who, n, (long long)st, (long long)kMaxStride);
  return IC_OK;
}

int pad_of(const ic_lattn_args* a) {
  const int d = a->Dk > a->Dv ? a->Dk : a->Dv;
  return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}

// Segments of a sequence: the number for which the last of the launch's workgroups ends first, counted in chunks.  A chip of
// 256 compute units holds `slots` workgroups at a time (LDS and registers: see the kernels); every round of them takes the
// chunks of a segment and about one more (start state, first loads), and with more than one segment their sums come first,
// at 0.4 of a chunk's time each.  (One sequence of 1024 chunks and 8 heads, 512 slots: 64 segments, 17 + 8.4 chunks against
// 1025; 64 sequences and heads of 16 chunks, 768 slots: 8 segments of 2, 3 + 2.8 chunks against 17.)
Span span_of(int T, int64_t have, int slots) {
  Span g;
  const int NC = ic_ceil_div(T, kC);
  double best = 0.0;
  g.nseg = 1;
  g.cps = NC;
  const int64_t most = (2 * slots + have - 1) / have;
  for (int ns = 1, cps = NC; ns <= most; ns = ic_ceil_div(NC, --cps)) {  // each number of chunks that differs in its segments
    cps = ic_ceil_div(NC, ns);
    const double rounds = (double)((have * ns + slots - 1) / slots);
    const double cost = rounds * (cps + 1.0) + (ns > 1 ? 0.4 * rounds * cps + 2.0 : 0.0);
    if (ns == 1 || cost < best) {
      best = cost;
      g.nseg = ns;
      g.cps = cps;
    }
    if (cps == 1) break;
  }
  return g;
}
// Workgroups at a time: 32 channels 40 KB of LDS, 64 channels 53 KB and 168 registers (256 with the lag-weighted state), 128
// channels 75 KB and 256 registers for bf16 rows, 86 KB for others.  (bf16 rows that take the fp32 kernels for want of
// 16-byte accesses are planned like the rest of their type.)
int slots_of(const ic_lattn_args* a, bool lag) {
  const int dp = pad_of(a);
  return 256 * (dp == 32 ? 4 : dp == 64 ? (lag ? 2 : 3) : a->dtype == IC_DT_BF16 && !lag ? 2 : 1);
}
Span span_fwd(const ic_lattn_args* a) { return span_of(a->T, (int64_t)a->B * a->H, slots_of(a, false)); }
// the dq pass, and the dv and dk passes, whose workgroups take all query heads of a key head
Span span_q(const ic_lattn_args* a, bool lag) { return span_of(a->T, (int64_t)a->B * a->H, slots_of(a, lag)); }
Span span_kv(const ic_lattn_args* a) { return span_of(a->T, 2 * (int64_t)a->B * a->Hk, slots_of(a, false)); }

Geo geo_of(const ic_lattn_args* a) {
  Geo g;
  g.B = a->B; g.H = a->H; g.T = a->T;
  g.rate = a->rate;
  g.valid_len = a->valid_len;
  return g;
}

Mat mat(const void* p, int64_t sb, int64_t sh, int64_t st, int group, int D, int esz) {
  Mat m;
  m.p = const_cast<void*>(p);
  m.sb = sb; m.sh = sh; m.st = st;
  m.group = group;
  const int ve = 16 / esz;
  m.vec = ((uintptr_t)p & 15) == 0 && D % ve == 0 && sb % ve == 0 && sh % ve == 0 && st % ve == 0;
  return m;
}

// floats of workspace: the segments' states (backward: the forward state and, for d rate, its lag-weighted companion, and the
// reversed state), partial sums of d rate (doubles), sums of shared heads' gradients
int64_t ws_floats(const ic_lattn_args* a, int backward) {
  const int64_t bh = (int64_t)a->B * a->H, dd = (int64_t)a->Dk * a->Dv;
  if (!backward) {
    const int ns = span_fwd(a).nseg;
    return ns > 1 ? bh * ns * dd : 0;
  }
  int64_t n = 0;
  for (int lag = 0; lag < 2; ++lag) {  // (whether d rate is wanted is the call's matter, not the sizes')
    const int ns = span_q(a, lag).nseg;
    const int64_t m = (lag ? 2 * bh * ns : 0) + (ns > 1 ? bh * ns * dd * (lag ? 2 : 1) : 0);
    n = n > m ? n : m;
  }
  const int nr = span_kv(a).nseg;
  n += (nr > 1 ? bh * nr * dd : 0) + 2;
  if (a->H != a->Hk) n += (int64_t)a->B * a->Hk * a->T * (a->Dk + a->Dv) + 8;
  return n;
}

}  // namespace

#define IC_LATTN_T(dt, wide, BODY)                                                   \
  do {                                                                               \
    if ((dt) == IC_DT_F32) { [[maybe_unused]] constexpr bool W16 = false; BODY(float) }               \
    else if ((dt) == IC_DT_BF16 && (wide)) { [[maybe_unused]] constexpr bool W16 = true; BODY(ic_bf16) } \
    else if ((dt) == IC_DT_BF16) { [[maybe_unused]] constexpr bool W16 = false; BODY(ic_bf16) }       \
    else { [[maybe_unused]] constexpr bool W16 = false; BODY(ic_f16) }                                \
  } while (0)
#define IC_LATTN_DP(dp, T, BODY)                                \
  if ((dp) == 32) { constexpr int DP = 32; BODY(T, DP); }       \
  else if ((dp) == 64) { constexpr int DP = 64; BODY(T, DP); }  \
  else { constexpr int DP = 128; BODY(T, DP); }

extern "C" int ic_lattn_ws(const ic_lattn_args* a, int32_t backward, int64_t* floats) {
  int rc = check_lattn(a, "ic_lattn_ws");
  if (rc) return rc;
  IC_REQUIRE(floats != nullptr, "ic_lattn_ws: NULL pointer");
  *floats = ws_floats(a, backward);
  return IC_OK;
}

extern "C" int ic_lattn_fwd(const ic_lattn_args* a, ic_stream_t stream) {
  int rc = check_lattn(a, "ic_lattn_fwd");
  if (rc) return rc;
  IC_REQUIRE(a->q && a->k && a->v && a->rate && a->out, "ic_lattn_fwd: NULL tensor pointer");
  IC_REQUIRE(!a->state_out || a->state_out != a->state, "ic_lattn_fwd: state_out is state");
  IC_REQUIRE(a->ws || ws_floats(a, 0) == 0, "ic_lattn_fwd: NULL workspace");
  if ((rc = check_stride(a->q_st, "ic_lattn_fwd", "q")) || (rc = check_stride(a->k_st, "ic_lattn_fwd", "k")) ||
      (rc = check_stride(a->v_st, "ic_lattn_fwd", "v")) || (rc = check_stride(a->o_st, "ic_lattn_fwd", "out"))) return rc;
  const Geo g = geo_of(a);
  const Span sp = span_fwd(a);
  const int esz = ic_dt_size(a->dtype), G = a->H / a->Hk, dp = pad_of(a), bh = a->B * a->H;
  hipStream_t st = (hipStream_t)stream;
  const Mat q = mat(a->q, a->q_sb, a->q_sh, a->q_st, 1, a->Dk, esz), k = mat(a->k, a->k_sb, a->k_sh, a->k_st, G, a->Dk, esz);
  const Mat v = mat(a->v, a->v_sb, a->v_sh, a->v_st, G, a->Dv, esz), o = mat(a->out, a->o_sb, a->o_sh, a->o_st, 1, a->Dv, esz);
  const bool wide = a->dtype == IC_DT_BF16 && q.vec && k.vec && v.vec && o.vec;
  if (sp.nseg > 1) {
    SumArgs s{};
    s.g = g;
    s.s[0] = Sums{k, v, sp, a->Dk, a->Dv, 0, 1.f, a->ws};
#define IC_BODY(T, DP) IC_TIMED(IC_KID_lattn_sums, st, hipLaunchKernelGGL((k_lattn_sums<T, DP, false, W16>), dim3(bh * (sp.nseg - 1)), dim3(DP * 4), 0, st, s))
#define IC_BODY_T(T) IC_LATTN_DP(dp, T, IC_BODY)
    IC_LATTN_T(a->dtype, wide, IC_BODY_T);
#undef IC_BODY
    IC_LAUNCH_CHECK("ic_lattn_fwd");
    ScanArgs sc{};
    sc.g = g;
    sc.s[0] = ScanState{sp, a->ws, a->state, a->Dk, a->Dv, a->Dv, 1, 0, 0};
    IC_TIMED(IC_KID_lattn_scan, st, hipLaunchKernelGGL(k_lattn_scan, dim3(bh, ic_ceil_div(a->Dk * a->Dv, 256), 1), dim3(256), 0, st, sc));
    IC_LAUNCH_CHECK("ic_lattn_fwd");
  }
  PassArgs p{};
  p.g = g;
  Pass& f = p.p[0];
  f.q = q; f.k = k; f.v = v; f.out = o;
  f.sp = sp; f.G = 1;
  f.Da = a->Dk; f.Db = a->Dv;
  f.oscale = a->scale; f.vscale = 1.f;
  f.init = a->state; f.ia = a->Dv; f.ib = 1;
  f.fin = a->state_out;
  if (sp.nseg > 1) { f.seg = a->ws; f.sga = a->Dv; f.sgb = 1; f.nst = 1; }
#define IC_BODY(T, DP) IC_TIMED(IC_KID_lattn_fwd, st, hipLaunchKernelGGL((k_lattn<T, DP, false, W16, false>), dim3(bh * sp.nseg), dim3(DP * 4 / cw_of<DP, false, W16>()), 0, st, p))
  IC_LATTN_T(a->dtype, wide, IC_BODY_T);
#undef IC_BODY
  IC_LAUNCH_CHECK("ic_lattn_fwd");
  return IC_OK;
}

extern "C" int ic_lattn_bwd(const ic_lattn_bwd_args* ba, ic_stream_t stream) {
  IC_REQUIRE(ba != nullptr, "ic_lattn_bwd: NULL args");
  const ic_lattn_args* a = &ba->f;
  int rc = check_lattn(a, "ic_lattn_bwd");
  if (rc) return rc;
  IC_REQUIRE(a->q && a->k && a->v && a->rate && ba->dout && ba->dq && ba->dk && ba->dv, "ic_lattn_bwd: NULL tensor pointer");
  IC_REQUIRE(!ba->dstate || ba->dstate != ba->dstate_out, "ic_lattn_bwd: dstate is dstate_out");
  IC_REQUIRE(a->ws && ((uintptr_t)a->ws & 7) == 0, "ic_lattn_bwd: the workspace is NULL or not on 8 bytes");
  if ((rc = check_stride(a->q_st, "ic_lattn_bwd", "q")) || (rc = check_stride(a->k_st, "ic_lattn_bwd", "k")) ||
      (rc = check_stride(a->v_st, "ic_lattn_bwd", "v")) || (rc = check_stride(ba->do_st, "ic_lattn_bwd", "dout")) ||
      (rc = check_stride(ba->dq_st, "ic_lattn_bwd", "dq")) || (rc = check_stride(ba->dk_st, "ic_lattn_bwd", "dk")) ||
      (rc = check_stride(ba->dv_st, "ic_lattn_bwd", "dv"))) return rc;
  const bool lag = ba->drate != nullptr;
  const Geo g = geo_of(a);
  const Span sq = span_q(a, lag), skv = span_kv(a);
  const int esz = ic_dt_size(a->dtype), G = a->H / a->Hk, dp = pad_of(a), bh = a->B * a->H, bk = a->B * a->Hk, Dk = a->Dk, Dv = a->Dv;
  const int64_t dd = (int64_t)Dk * Dv;
  hipStream_t st = (hipStream_t)stream;
  const Mat q = mat(a->q, a->q_sb, a->q_sh, a->q_st, 1, Dk, esz), k = mat(a->k, a->k_sb, a->k_sh, a->k_st, G, Dk, esz);
  const Mat v = mat(a->v, a->v_sb, a->v_sh, a->v_st, G, Dv, esz), o = mat(ba->dout, ba->do_sb, ba->do_sh, ba->do_st, 1, Dv, esz);
  const Mat dk = mat(ba->dk, ba->dk_sb, ba->dk_sh, ba->dk_st, G, Dk, esz), dv = mat(ba->dv, ba->dv_sb, ba->dv_sh, ba->dv_st, G, Dv, esz);
  const Mat dq = mat(ba->dq, ba->dq_sb, ba->dq_sh, ba->dq_st, 1, Dk, esz);
  const bool wide = a->dtype == IC_DT_BF16 && q.vec && k.vec && v.vec && o.vec && dq.vec && dk.vec && dv.vec;
  const int nst = lag ? 2 : 1;
  double* dr = (double*)a->ws;
  float* seg_s = a->ws + (lag ? 2 * (int64_t)bh * sq.nseg : 0);                 // S (and L): transposed, [Dv][Dk]
  float* seg_r = seg_s + (sq.nseg > 1 ? (int64_t)bh * sq.nseg * dd * nst : 0);  // the reversed state, [Dk][Dv]
  float* part_k = seg_r + (skv.nseg > 1 ? (int64_t)bh * skv.nseg * dd : 0);
  part_k += -((uintptr_t)part_k / 4) & 3;  // (rows on 16 bytes)
  float* part_v = part_k + (((int64_t)bk * a->T * Dk + 3) & ~(int64_t)3);
  const int nmax = sq.nseg > skv.nseg ? sq.nseg : skv.nseg;
  if (nmax > 1) {
    SumArgs s{};
    s.g = g;
    s.s[0] = Sums{v, k, sq, Dv, Dk, 0, 1.f, seg_s};
    s.s[1] = Sums{q, o, skv, Dk, Dv, 1, a->scale, seg_r};
#define IC_SUMS(T, DP, LAG) IC_TIMED(IC_KID_lattn_sums, st, hipLaunchKernelGGL((k_lattn_sums<T, DP, LAG, W16>), dim3(bh * (nmax - 1), 2), dim3(DP * 4), 0, st, s))
#define IC_BODY(T, DP)                    \
  if (lag) { IC_SUMS(T, DP, true); }      \
  else { IC_SUMS(T, DP, false); }
    IC_LATTN_T(a->dtype, wide, IC_BODY_T);
#undef IC_BODY
#undef IC_SUMS
    IC_LAUNCH_CHECK("ic_lattn_bwd");
    ScanArgs sc{};
    sc.g = g;
    sc.s[0] = ScanState{sq, seg_s, a->state, Dv, Dk, 1, Dv, lag, 0};
    sc.s[1] = ScanState{skv, seg_r, ba->dstate_out, Dk, Dv, Dv, 1, 0, 1};
    IC_TIMED(IC_KID_lattn_scan, st, hipLaunchKernelGGL(k_lattn_scan, dim3(bh, ic_ceil_div(Dk * Dv, 256), 2), dim3(256), 0, st, sc));
    IC_LAUNCH_CHECK("ic_lattn_bwd");
  }
  PassArgs p{};
  p.g = g;
  Pass& pq = p.p[0];  // dq
  pq.q = o; pq.k = v; pq.v = k; pq.x = q;
  pq.out = dq;
  pq.sp = sq; pq.G = 1;
  pq.Da = Dv; pq.Db = Dk;
  pq.oscale = a->scale; pq.vscale = 1.f;
  pq.init = a->state; pq.ia = 1; pq.ib = Dv;
  pq.gfin = ba->dstate_out;
  pq.dr = dr;
  Pass& pv = p.p[1];  // dv
  pv.q = k; pv.k = q; pv.v = o; pv.out = dv;
  pv.sp = skv; pv.G = G; pv.part = part_v;
  pv.Da = Dk; pv.Db = Dv;
  pv.rev = 1;
  pv.oscale = 1.f; pv.vscale = a->scale;
  pv.init = ba->dstate_out; pv.ia = Dv; pv.ib = 1;
  pv.fin = ba->dstate; pv.fin_decay = 1;
  Pass& pk = p.p[2];  // dk
  pk.q = v; pk.k = o; pk.v = q; pk.out = dk;
  pk.sp = skv; pk.G = G; pk.part = part_k;
  pk.Da = Dv; pk.Db = Dk;
  pk.rev = 1;
  pk.oscale = 1.f; pk.vscale = a->scale;
  pk.init = ba->dstate_out; pk.ia = 1; pk.ib = Dv;
  if (sq.nseg > 1) { pq.seg = seg_s; pq.sga = Dk; pq.sgb = 1; pq.nst = nst; }
  if (skv.nseg > 1) {
    pv.seg = seg_r; pv.sga = Dv; pv.sgb = 1; pv.nst = 1;
    pk.seg = seg_r; pk.sga = 1; pk.sgb = Dv; pk.nst = 1;
  }
  const int nq = bh * sq.nseg, nkv = bk * skv.nseg;
  PassArgs pkv = p;
  pkv.p[0] = p.p[1];
  pkv.p[1] = p.p[2];
#define IC_LATTN_BWD(T, DP, LAG, SHARED, GRID, ARGS) \
  IC_TIMED(IC_KID_lattn_bwd, st, hipLaunchKernelGGL((k_lattn<T, DP, LAG, W16, SHARED>), GRID, dim3(DP * 4 / cw_of<DP, LAG, W16>()), 0, st, ARGS))
#define IC_BODY(T, DP)                                                           \
  if (!lag && G == 1) {                                                          \
    IC_LATTN_BWD(T, DP, false, false, dim3(nq > nkv ? nq : nkv, 3), p);          \
  } else {                                                                       \
    if (lag) { IC_LATTN_BWD(T, DP, true, false, dim3(nq), p); }                  \
    else { IC_LATTN_BWD(T, DP, false, false, dim3(nq), p); }                     \
    if (G == 1) { IC_LATTN_BWD(T, DP, false, false, dim3(nkv, 2), pkv); }        \
    else { IC_LATTN_BWD(T, DP, false, true, dim3(nkv, 2), pkv); }                \
  }
  IC_LATTN_T(a->dtype, wide, IC_BODY_T);
#undef IC_BODY
#undef IC_LATTN_BWD
  IC_LAUNCH_CHECK("ic_lattn_bwd");
  if (lag) {
    IC_TIMED(IC_KID_lattn_drate, st, hipLaunchKernelGGL(k_lattn_drate, dim3(a->H), dim3(64), 0, st, dr, ba->drate, a->B, a->H, sq.nseg));
    IC_LAUNCH_CHECK("ic_lattn_bwd");
  }
  return IC_OK;
}

extern "C" int ic_lattn_step(const ic_lattn_step_args* a, ic_stream_t stream) {
  IC_REQUIRE(a != nullptr, "ic_lattn_step: NULL args");
  IC_REQUIRE(a->B >= 1 && a->H >= 1 && (int64_t)a->B * a->H < (1ll << 24), "ic_lattn_step: B=%d H=%d (fewer than 2^24 together)", a->B, a->H);
  IC_REQUIRE(a->Hk >= 1 && a->H % a->Hk == 0, "ic_lattn_step: H=%d is no multiple of Hk=%d", a->H, a->Hk);
  IC_REQUIRE(a->Dk >= 1 && a->Dk <= 1024 && a->Dv >= 1 && a->Dv <= 1024, "ic_lattn_step: Dk=%d Dv=%d (need 1 .. 1024)", a->Dk, a->Dv);
  IC_REQUIRE(ic_dt_ok(a->dtype), "ic_lattn_step: dtype=%d", a->dtype);
  IC_REQUIRE(a->q && a->k && a->v && a->rate && a->state && a->out, "ic_lattn_step: NULL tensor pointer");
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(a->B * a->H, ic_ceil_div(a->Dv, 32));
#define IC_BODY(T) IC_TIMED(IC_KID_lattn_step, st, hipLaunchKernelGGL(k_lattn_step<T>, grid, dim3(256), 0, st, *a));
  IC_LATTN_T(a->dtype, false, IC_BODY);
#undef IC_BODY
  IC_LAUNCH_CHECK("ic_lattn_step");
  return IC_OK;
}

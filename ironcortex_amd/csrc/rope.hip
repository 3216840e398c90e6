// Rotary positions of queries and keys, alone or behind an RMSNorm of every head's row (reference iron_rope.py:49-66,
// utils.py:33-35), forward and backward.
//
// Memory-bound: a row is read once and written once (backward with norms: x and g read, gx written), the angles belong
// to a token and are shared by all its heads.  So a group of lanes owns a TOKEN: it forms (or loads) the cos / sin of its
// channel pairs once and walks over the heads of q or of k with them.  A lane holds NP pairs, two 16-byte vectors of a
// row in either layout; the norm's sum runs over the group's lanes with shuffles.  Rows whose width, alignment or
// strides do not allow 16-byte accesses take the same kernel with one lane per pair and single-element accesses.
//
// Measured (bytes read and written once / time; a large copy reaches 4.76 TB/s): rotation of 131072 positions of 8 + 2 bf16
// heads of 128 channels, half of each turned, 671 MB in 136 us = 4.9 TB/s; norms and rotation, forward and backward, of
// 32768 positions of 16 + 4 bf16 heads of 128, 839 MB in 190 us = 4.4 TB/s; 16 x 266 positions of 4 + 4 fp32 heads of 64,
// forward and backward, 9 + 9 us, where the call and the autograd engine around them take 110.
#include "ic_types.h"

namespace {

constexpr int kThreads = 256;
constexpr int kParts = 1024;  // workgroups of the backward with norms: one partial sum of gw each
constexpr int kAnyNP = 4;     // pairs per lane of the single-element form: 64 lanes x 4 = rows up to 512 channels

// how a lane's pairs lie in a row
enum { M_INTER = 0, M_HALF = 1, M_ANY = 2 };
template <typename T, int MODE>
struct Own {
  static constexpr int NP = MODE == M_ANY ? kAnyNP : 16 / (int)sizeof(T);
};

// slot of pair i of lane l
template <int MODE, int NP>
__device__ __forceinline__ int slot_of(int l, int i) { return MODE == M_ANY ? l + 64 * i : l * NP + i; }
// channels of a slot: the m rotated pairs first, then the rest of the row in twos
__device__ __forceinline__ void slot_channels(int s, int m, int layout, int& a, int& b) {
  const bool half = layout == IC_ROPE_HALF && s < m;
  a = half ? s : 2 * s;
  b = half ? s + m : 2 * s + 1;
}

template <typename T, int MODE, int NP>
__device__ __forceinline__ void load_pairs(const T* row, int l, int D, int m, int layout, float (&a)[NP], float (&b)[NP]) {
  if constexpr (MODE == M_ANY) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int ca, cb;
      slot_channels(slot_of<MODE, NP>(l, i), m, layout, ca, cb);
      a[i] = ca < D ? ic_to_f(row[ca]) : 0.f;
      b[i] = cb < D ? ic_to_f(row[cb]) : 0.f;
    }
  } else {
    const int s0 = l * NP;
    const bool live = 2 * s0 < D;
    const bool half = MODE == M_HALF && s0 < m;
    const int c0 = half ? s0 : 2 * s0, c1 = half ? s0 + m : 2 * s0 + NP;
    uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
    if (live) {
      u0 = *reinterpret_cast<const uint4*>(row + c0);
      u1 = *reinterpret_cast<const uint4*>(row + c1);
    }
    T e[2 * NP];
    *reinterpret_cast<uint4*>(e) = u0;
    *reinterpret_cast<uint4*>(e + NP) = u1;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      a[i] = ic_to_f(half ? e[i] : e[2 * i]);
      b[i] = ic_to_f(half ? e[NP + i] : e[2 * i + 1]);
    }
  }
}

template <typename T, int MODE, int NP, bool PAST = false>  // PAST: past the caches
__device__ __forceinline__ void store_pairs(T* row, int l, int D, int m, int layout, const float (&a)[NP], const float (&b)[NP]) {
  if constexpr (MODE == M_ANY) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int ca, cb;
      slot_channels(slot_of<MODE, NP>(l, i), m, layout, ca, cb);
      if (ca < D) row[ca] = ic_from_f<T>(a[i]);
      if (cb < D) row[cb] = ic_from_f<T>(b[i]);
    }
  } else {
    const int s0 = l * NP;
    if (2 * s0 >= D) return;
    const bool half = MODE == M_HALF && s0 < m;
    const int c0 = half ? s0 : 2 * s0, c1 = half ? s0 + m : 2 * s0 + NP;
    T e[2 * NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const T va = ic_from_f<T>(a[i]), vb = ic_from_f<T>(b[i]);
      if (half) { e[i] = va; e[NP + i] = vb; }
      else { e[2 * i] = va; e[2 * i + 1] = vb; }
    }
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    u4* d0 = reinterpret_cast<u4*>(row + c0);
    u4* d1 = reinterpret_cast<u4*>(row + c1);
    if constexpr (PAST) {
      __builtin_nontemporal_store(*reinterpret_cast<u4*>(e), d0);
      __builtin_nontemporal_store(*reinterpret_cast<u4*>(e + NP), d1);
    } else {
      *d0 = *reinterpret_cast<u4*>(e);
      *d1 = *reinterpret_cast<u4*>(e + NP);
    }
  }
}

// cos / sin of position * freq: the angle in turns in 64 bits, reduced there to an eighth of a turn around the nearest
// quarter, so that the 32-bit functions see |x| <= 1/4 (of half turns) exactly to 2^-25
__device__ __forceinline__ void far_sincos(double turns, float& c, float& s) {
  const double fr = turns - rint(turns);  // exact
  const double q = rint(4.0 * fr);        // quarter: -2 .. 2
  const float d = (float)(4.0 * fr - q);  // in quarters, |d| <= 1/2
  float s0, c0;
  sincospif(0.5f * d, &s0, &c0);
  const int n = (int)q & 3;
  c = n == 0 ? c0 : n == 1 ? -s0 : n == 2 ? -c0 : s0;
  s = n == 0 ? s0 : n == 1 ? c0 : n == 2 ? -s0 : -c0;
}

template <int MODE, int NP>
__device__ __forceinline__ void token_angles(const ic_rope_args& a, int b, int t, int l, float (&c)[NP], float (&s)[NP]) {
  const float sign = a.inverse ? -1.f : 1.f;
  double pos = 0.0;
  if (!a.cos) {
    const int64_t at = (int64_t)b * a.pos_sb + t;
    pos = !a.positions ? (double)t : a.pos64 ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int j = slot_of<MODE, NP>(l, i);
    c[i] = 1.f;
    s[i] = 0.f;
    if (j < a.m) {
      if (a.cos) {
        const int64_t at = (int64_t)b * a.cs_sb + (int64_t)t * a.m + j;
        c[i] = a.cos[at];
        s[i] = a.sin[at];
      } else {
        const double f = a.freq64 ? ((const double*)a.freqs)[j] : (double)((const float*)a.freqs)[j];
        far_sincos(pos * f * 0.15915494309189533577, c[i], s[i]);
      }
      c[i] *= a.scale;
      s[i] *= sign * a.scale;
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int G) {
  for (int o = G >> 1; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct RopePlan {
  int G;       // lanes of a token (a power of two, divides 64)
  int hc;      // heads a lane group walks over
  int nq, nk;  // head chunks of q and of k: blockIdx.y < nq is a chunk of q
  int past;    // outputs that no cache holds until they are read are written past the caches
};

template <typename T, int MODE, bool NORM, bool PAST>
__global__ __launch_bounds__(kThreads) void k_rope_fwd(ic_rope_args a, RopePlan p) {
  constexpr int NP = Own<T, MODE>::NP;
  constexpr int UH = 2;  // rows in flight
  const int l = threadIdx.x & (p.G - 1);
  const int per = kThreads / p.G;
  const int64_t tok = (int64_t)blockIdx.x * per + threadIdx.x / p.G;
  const bool isq = (int)blockIdx.y < p.nq;
  const ic_rope_rows& r = isq ? a.q : a.k;
  const int h0 = (isq ? blockIdx.y : blockIdx.y - p.nq) * p.hc;
  const int h1 = h0 + p.hc < r.H ? h0 + p.hc : r.H;
  if (tok >= (int64_t)a.B * a.T) return;  // (whole lane groups: the shuffles below stay inside one)
  const int b = (int)(tok / a.T), t = (int)(tok - (int64_t)b * a.T);
  const T* X = (const T*)r.x + (int64_t)b * r.x_sb + (int64_t)t * r.x_st;
  T* Y = (T*)r.y + (int64_t)b * r.y_sb + (int64_t)t * r.y_st;
  float xa[UH][NP], xb[UH][NP], wa[NP], wb[NP], c[NP], s[NP];
#pragma unroll
  for (int u = 0; u < UH; ++u)
    if (h0 + u < h1) load_pairs<T, MODE, NP>(X + (int64_t)(h0 + u) * r.x_sh, l, a.D, a.m, a.layout, xa[u], xb[u]);
  token_angles<MODE, NP>(a, b, t, l, c, s);
  if (NORM) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int ca, cb;
      slot_channels(slot_of<MODE, NP>(l, i), a.m, a.layout, ca, cb);
      wa[i] = ca < a.D ? ic_load_dt(r.w, r.w_dtype, ca) : 0.f;
      wb[i] = cb < a.D ? ic_load_dt(r.w, r.w_dtype, cb) : 0.f;
    }
  }
  for (int h = h0; h < h1; h += UH) {
#pragma unroll
    for (int u = 0; u < UH; ++u) {
      if (h + u >= h1) continue;
      float ya[NP], yb[NP];
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) ss = fmaf(xa[u][i], xa[u][i], fmaf(xb[u][i], xb[u][i], ss));
        const float inv = 1.0f / sqrtf(group_sum(ss, p.G) / (float)a.D + a.eps);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          xa[u][i] = xa[u][i] * inv * wa[i];
          xb[u][i] = xb[u][i] * inv * wb[i];
        }
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const bool rot = slot_of<MODE, NP>(l, i) < a.m;
        ya[i] = rot ? xa[u][i] * c[i] - xb[u][i] * s[i] : xa[u][i];
        yb[i] = rot ? xa[u][i] * s[i] + xb[u][i] * c[i] : xb[u][i];
      }
      store_pairs<T, MODE, NP, PAST>(Y + (int64_t)(h + u) * r.y_sh, l, a.D, a.m, a.layout, ya, yb);
    }
#pragma unroll
    for (int u = 0; u < UH; ++u)
      if (h + UH + u < h1) load_pairs<T, MODE, NP>(X + (int64_t)(h + UH + u) * r.x_sh, l, a.D, a.m, a.layout, xa[u], xb[u]);
  }
}

// Backward with norms: u = w xhat, xhat = x inv; with h = R^T g:  gw = sum h xhat,  gx = inv (w h - xhat mean(w h xhat)).
// A workgroup walks over tokens (grid stride), so that gw leaves it as ONE partial sum per channel.
template <typename T, int MODE, bool PAST>
__global__ __launch_bounds__(kThreads) void k_rope_norm_bwd(ic_rope_bwd_args ba, RopePlan p) {
  constexpr int NP = Own<T, MODE>::NP;
  __shared__ float red[kThreads / 64][512];
  const ic_rope_args& a = ba.f;
  const int l = threadIdx.x & (p.G - 1);
  const int per = kThreads / p.G;
  const bool isq = (int)blockIdx.y < p.nq;
  const ic_rope_rows& r = isq ? a.q : a.k;
  const ic_rope_grad& g = isq ? ba.q : ba.k;
  const int h0 = (isq ? blockIdx.y : blockIdx.y - p.nq) * p.hc;
  const int h1 = h0 + p.hc < r.H ? h0 + p.hc : r.H;
  float wa[NP], wb[NP], da[NP], db[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    int ca, cb;
    slot_channels(slot_of<MODE, NP>(l, i), a.m, a.layout, ca, cb);
    wa[i] = ca < a.D ? ic_load_dt(r.w, r.w_dtype, ca) : 0.f;
    wb[i] = cb < a.D ? ic_load_dt(r.w, r.w_dtype, cb) : 0.f;
    da[i] = db[i] = 0.f;
  }
  const int64_t ntok = (int64_t)a.B * a.T;
  for (int64_t tok = (int64_t)blockIdx.x * per + threadIdx.x / p.G; tok < ntok; tok += (int64_t)gridDim.x * per) {
    const int b = (int)(tok / a.T), t = (int)(tok - (int64_t)b * a.T);
    const T* X = (const T*)r.x + (int64_t)b * r.x_sb + (int64_t)t * r.x_st;
    const T* Gr = (const T*)g.g + (int64_t)b * g.g_sb + (int64_t)t * g.g_st;
    T* GX = (T*)g.gx + (int64_t)b * g.gx_sb + (int64_t)t * g.gx_st;
    float c[NP], s[NP];
    token_angles<MODE, NP>(a, b, t, l, c, s);
    for (int h = h0; h < h1; ++h) {
      float xa[NP], xb[NP], ga[NP], gb[NP];
      load_pairs<T, MODE, NP>(X + (int64_t)h * r.x_sh, l, a.D, a.m, a.layout, xa, xb);
      load_pairs<T, MODE, NP>(Gr + (int64_t)h * g.g_sh, l, a.D, a.m, a.layout, ga, gb);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const bool rot = slot_of<MODE, NP>(l, i) < a.m;
        const float ha = rot ? ga[i] * c[i] + gb[i] * s[i] : ga[i];
        const float hb = rot ? gb[i] * c[i] - ga[i] * s[i] : gb[i];
        ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
        ga[i] = ha;
        gb[i] = hb;
        dot = fmaf(wa[i] * ha, xa[i], fmaf(wb[i] * hb, xb[i], dot));
      }
      for (int o = p.G >> 1; o; o >>= 1) {
        ss += __shfl_xor(ss, o, 64);
        dot += __shfl_xor(dot, o, 64);
      }
      const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
      const float mean = dot * inv / (float)a.D;  // mean(w h xhat)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float na = xa[i] * inv, nb = xb[i] * inv;
        da[i] = fmaf(ga[i], na, da[i]);
        db[i] = fmaf(gb[i], nb, db[i]);
        ga[i] = inv * (wa[i] * ga[i] - na * mean);
        gb[i] = inv * (wb[i] * gb[i] - nb * mean);
      }
      store_pairs<T, MODE, NP, PAST>(GX + (int64_t)h * g.gx_sh, l, a.D, a.m, a.layout, ga, gb);
    }
  }
  // the workgroup's sum of each channel, in a fixed order: lane groups of a wave, then the four waves
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    for (int o = p.G; o < 64; o <<= 1) {
      da[i] += __shfl_xor(da[i], o, 64);
      db[i] += __shfl_xor(db[i], o, 64);
    }
    int ca, cb;
    slot_channels(slot_of<MODE, NP>(l, i), a.m, a.layout, ca, cb);
    if ((threadIdx.x & 63) < p.G) {
      if (ca < a.D) red[wave][ca] = da[i];
      if (cb < a.D) red[wave][cb] = db[i];
    }
  }
  __syncthreads();
  float* part = ba.part + ((size_t)(blockIdx.y * gridDim.x + blockIdx.x)) * a.D;
  for (int j = threadIdx.x; j < a.D; j += kThreads) part[j] = (red[0][j] + red[1][j]) + (red[2][j] + red[3][j]);
}

// gw[j] = sum of the partial sums of channel j: 64 channels per workgroup, 16 rows of threads over the parts
__global__ __launch_bounds__(1024) void k_rope_gw(ic_rope_bwd_args ba, int nq, int nk, int gx) {
  __shared__ float red[16][64];
  const int D = ba.f.D;
  const bool isq = blockIdx.y == 0;
  const int j = blockIdx.x * 64 + (threadIdx.x & 63), row = threadIdx.x >> 6;
  const int n = (isq ? nq : nk) * gx;
  const float* part = ba.part + (isq ? 0 : (size_t)nq * gx * D);
  float v = 0.f;
  if (j < D) {
    int i = row;
    for (; i + 48 < n; i += 64) {
      const float v0 = part[(size_t)i * D + j], v1 = part[(size_t)(i + 16) * D + j];
      const float v2 = part[(size_t)(i + 32) * D + j], v3 = part[(size_t)(i + 48) * D + j];
      v += (v0 + v1) + (v2 + v3);
    }
    for (; i < n; i += 16) v += part[(size_t)i * D + j];
  }
  red[row][threadIdx.x & 63] = v;
  __syncthreads();
  if (row == 0 && j < D) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += red[i][threadIdx.x];
    const ic_rope_rows& r = isq ? ba.f.q : ba.f.k;
    ic_store_dt(isq ? ba.q.gw : ba.k.gw, r.w_dtype, j, v);
  }
}

int check_rows(const ic_rope_rows& r, const char* who, const char* n) {
  IC_REQUIRE(r.H >= 1 && r.H <= 65535, "%s: %s has H=%d (need 1 .. 65535)", who, n, r.H);
  IC_REQUIRE(r.x != nullptr, "%s: NULL pointer to %s", who, n);
  IC_REQUIRE(!r.w || ic_dt_ok(r.w_dtype), "%s: %s has w_dtype=%d", who, n, r.w_dtype);
  return IC_OK;
}

int check_rope(const ic_rope_args* a, const char* who) {
  IC_REQUIRE(a != nullptr, "%s: NULL args", who);
  IC_REQUIRE(a->B >= 1 && a->T >= 1 && (int64_t)a->B * a->T < (1ll << 31), "%s: B=%d T=%d", who, a->B, a->T);
  IC_REQUIRE(a->D >= 1 && a->D <= 512, "%s: D=%d (need 1 .. 512)", who, a->D);
  IC_REQUIRE(a->m >= 0 && 2 * a->m <= a->D, "%s: m=%d pairs do not fit D=%d channels", who, a->m, a->D);
  IC_REQUIRE(ic_dt_ok(a->dtype), "%s: dtype=%d", who, a->dtype);
  IC_REQUIRE(a->layout == IC_ROPE_INTERLEAVED || a->layout == IC_ROPE_HALF, "%s: layout=%d", who, a->layout);
  IC_REQUIRE((a->cos == nullptr) == (a->sin == nullptr), "%s: cos and sin come together", who);
  IC_REQUIRE(a->m == 0 || a->cos || a->freqs, "%s: neither cos / sin nor freqs", who);
  IC_REQUIRE(!(a->cos && a->freqs), "%s: both cos / sin and freqs", who);
  int rc = check_rows(a->q, who, "q");
  if (rc) return rc;
  if (a->k.H != 0) {
    rc = check_rows(a->k, who, "k");
    if (rc) return rc;
    IC_REQUIRE((a->q.w == nullptr) == (a->k.w == nullptr), "%s: a norm weight for one of q and k only", who);
  }
  return IC_OK;
}

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool on16(int64_t stride, int esz) { return (stride * esz) % 16 == 0; }

// 16-byte form: whole vectors of pairs on either side of the rotated part, rows that start on 16 bytes
bool vec_ok(const ic_rope_args& a) {
  const int NP = 16 / ic_dt_size(a.dtype);
  return a.D % (2 * NP) == 0 && a.m % NP == 0;
}
bool vec_rows(const void* p, int64_t sb, int64_t sh, int64_t st, int esz) {
  return on16(p) && on16(sb, esz) && on16(sh, esz) && on16(st, esz);
}

// lanes per token and heads per lane group.  A group that walks over all heads forms its angles once; with few tokens the
// heads are spread over more groups instead, until the launch has 4 workgroups for each of the 256 compute units.
RopePlan plan_of(const ic_rope_args& a, int mode, bool limit_blocks, int* gx) {
  RopePlan p;
  const int NP = 16 / ic_dt_size(a.dtype);
  p.G = 64;
  if (mode != M_ANY) {
    const int lanes = a.D / (2 * NP);
    for (p.G = 1; p.G < lanes; p.G *= 2) {}
  }
  const int per = kThreads / p.G;
  const int64_t blocks = ((int64_t)a.B * a.T + per - 1) / per;
  const int hmax = a.q.H > a.k.H ? a.q.H : a.k.H;
  p.hc = hmax;
  while (p.hc > 1 && blocks * (ic_ceil_div(a.q.H, p.hc) + ic_ceil_div(a.k.H, p.hc)) < 1024) p.hc = (p.hc + 1) / 2;
  p.nq = ic_ceil_div(a.q.H, p.hc);
  p.nk = ic_ceil_div(a.k.H, p.hc);
  // Outputs of more than half of the 256 MB cache, with norms: a pass forward and backward over 32768 positions of 16 + 4
  // heads of 128 bf16 channels (168 MB a tensor) takes 192 us with them past the caches, 205 us through them, 206 us with
  // only the backward's past them; without norms (a copy's pattern) 147 against 141 us, so not there.
  p.past = a.q.w && (int64_t)a.B * a.T * (a.q.H + a.k.H) * a.D * ic_dt_size(a.dtype) > (128 << 20);
  int64_t n = blocks;
  if (limit_blocks) {  // (heads enough to fill kParts on their own: one token column of workgroups walks over all tokens)
    const int64_t most = kParts / (p.nq + p.nk);
    if (n > most) n = most;
  }
  *gx = (int)n;
  return p;
}

}  // namespace

#define IC_ROPE_MODES(T, mode, BODY)                                    \
  do {                                                                  \
    if ((mode) == M_INTER) { constexpr int MODE = M_INTER; BODY(T); }   \
    else if ((mode) == M_HALF) { constexpr int MODE = M_HALF; BODY(T); } \
    else { constexpr int MODE = M_ANY; BODY(T); }                       \
  } while (0)
#define IC_ROPE_DISPATCH(dt, mode, BODY)                                \
  do {                                                                  \
    if ((dt) == IC_DT_F32) IC_ROPE_MODES(float, mode, BODY);            \
    else if ((dt) == IC_DT_BF16) IC_ROPE_MODES(ic_bf16, mode, BODY);    \
    else IC_ROPE_MODES(ic_f16, mode, BODY);                             \
  } while (0)

extern "C" int ic_rope_parts(void) { return kParts; }

extern "C" int ic_rope_fwd(const ic_rope_args* a, ic_stream_t stream) {
  int rc = check_rope(a, "ic_rope_fwd");
  if (rc) return rc;
  IC_REQUIRE(a->q.y && (a->k.H == 0 || a->k.y), "ic_rope_fwd: NULL output pointer");
  IC_REQUIRE(!(a->inverse && a->q.w), "ic_rope_fwd: inverse with a norm");
  const int esz = ic_dt_size(a->dtype);
  auto rows_ok = [&](const ic_rope_rows& r) {
    return vec_rows(r.x, r.x_sb, r.x_sh, r.x_st, esz) && vec_rows(r.y, r.y_sb, r.y_sh, r.y_st, esz);
  };
  const bool vec = vec_ok(*a) && rows_ok(a->q) && (a->k.H == 0 || rows_ok(a->k));
  const int mode = !vec ? M_ANY : a->layout == IC_ROPE_HALF ? M_HALF : M_INTER;
  int gx;
  const RopePlan p = plan_of(*a, mode, false, &gx);
  IC_REQUIRE(gx < (1 << 24), "ic_rope_fwd: B=%d T=%d (a launch has fewer than 2^32 threads)", a->B, a->T);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(gx, p.nq + p.nk);
#define IC_ROPE_FWD(T, NORM, PAST) IC_TIMED(IC_KID_rope_fwd, st, hipLaunchKernelGGL((k_rope_fwd<T, MODE, NORM, PAST>), grid, dim3(kThreads), 0, st, *a, p))
#define IC_BODY(T)                                     \
  if (!a->q.w) { IC_ROPE_FWD(T, false, false); }       \
  else if (p.past) { IC_ROPE_FWD(T, true, true); }     \
  else { IC_ROPE_FWD(T, true, false); }
  IC_ROPE_DISPATCH(a->dtype, mode, IC_BODY);
#undef IC_BODY
#undef IC_ROPE_FWD
  IC_LAUNCH_CHECK("ic_rope_fwd");
  return IC_OK;
}

extern "C" int ic_rope_bwd(const ic_rope_bwd_args* b, ic_stream_t stream) {
  IC_REQUIRE(b != nullptr, "ic_rope_bwd: NULL args");
  const ic_rope_args* a = &b->f;
  int rc = check_rope(a, "ic_rope_bwd");
  if (rc) return rc;
  IC_REQUIRE(a->q.w != nullptr, "ic_rope_bwd: no norm weight (without norms: ic_rope_fwd with inverse = 1)");
  IC_REQUIRE(!a->inverse, "ic_rope_bwd: inverse");
  IC_REQUIRE(a->q.H + a->k.H <= kParts, "ic_rope_bwd: %d + %d heads (at most %d)", a->q.H, a->k.H, kParts);
  IC_REQUIRE(b->part && b->q.g && b->q.gx && b->q.gw, "ic_rope_bwd: NULL pointer");
  IC_REQUIRE(a->k.H == 0 || (b->k.g && b->k.gx && b->k.gw), "ic_rope_bwd: NULL pointer to k's gradients");
  const int esz = ic_dt_size(a->dtype);
  auto rows_ok = [&](const ic_rope_rows& r, const ic_rope_grad& g) {
    return vec_rows(r.x, r.x_sb, r.x_sh, r.x_st, esz) && vec_rows(g.g, g.g_sb, g.g_sh, g.g_st, esz) &&
           vec_rows(g.gx, g.gx_sb, g.gx_sh, g.gx_st, esz);
  };
  const bool vec = vec_ok(*a) && rows_ok(a->q, b->q) && (a->k.H == 0 || rows_ok(a->k, b->k));
  const int mode = !vec ? M_ANY : a->layout == IC_ROPE_HALF ? M_HALF : M_INTER;
  int gx;
  const RopePlan p = plan_of(*a, mode, true, &gx);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(gx, p.nq + p.nk);
#define IC_BODY(T)                                                                                                            \
  if (p.past) IC_TIMED(IC_KID_rope_bwd, st, hipLaunchKernelGGL((k_rope_norm_bwd<T, MODE, true>), grid, dim3(kThreads), 0, st, *b, p)); \
  else IC_TIMED(IC_KID_rope_bwd, st, hipLaunchKernelGGL((k_rope_norm_bwd<T, MODE, false>), grid, dim3(kThreads), 0, st, *b, p))
  IC_ROPE_DISPATCH(a->dtype, mode, IC_BODY);
#undef IC_BODY
  IC_LAUNCH_CHECK("ic_rope_bwd");
  IC_TIMED(IC_KID_rope_bwd, st, hipLaunchKernelGGL(k_rope_gw, dim3(ic_ceil_div(a->D, 64), p.nk ? 2 : 1), dim3(1024), 0, st, *b, p.nq, p.nk, gx));
  IC_LAUNCH_CHECK("ic_rope_bwd");
  return IC_OK;
}

// Shared pieces of the shared-prefix decode attention: how a step's work is cut into key tiles and dealt
// out to the CTAs, where the partial results lie, the q/k head norm and rotation, and the parameters.
//
// Work. The keys of a step are cut into tiles of KT rows: first the prefix, per (key/value head, tile of RT
// query rows) an item of ceil(P / KT) tiles — query row i = r*g + h of a head, all requests together —, then
// the own rows, per (request, key/value head) an item of ceil(n / KT) tiles. All tiles in one row, item
// after item, are split evenly over G = min(grid, N) CTAs (floor(N*c/G) .. floor(N*(c+1)/G)): every CTA
// moves the same number of bytes whatever the lengths are, and an item is cut only where a CTA's share
// ends. The part of an item that one CTA does is a segment; it leaves one partial (running max, sum,
// unnormalised output) per query row. Along the row of tiles the pair (CTA, item) never steps back in
// either and moves in one at least, so CTA + item numbers a segment's place in the workspace uniquely.
// The lengths are read on the device, so one captured graph serves every step.
#pragma once

#include "sk_common.cuh"

namespace sk {
namespace shared {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxRequests = 1024;
constexpr int kMaxGroup = 8;

struct Params {
  const void* Kp;
  const void* Vp;
  long long prefix_head_stride, prefix_row_stride;
  void* Kc;
  void* Vc;
  long long request_stride, head_stride, row_stride;
  float* mass;
  long long mass_request_stride, mass_head_stride;
  const float* rope;
  const long long* pos;
  const long long* rows;
  const void* qkv;
  const float* qn;
  const float* kn;
  void* out;
  long long qkv_stride, out_stride;
  int R, nq, nkv, g, P, max_len, rope_len;
  int qkv_bf16, out_bf16;
  float eps, q_scale;  // softmax scale * log2(e): scores come out in the log2 domain
  int* cum;            // [R + 1] own tiles of the requests before r, per head (written by CTA 0)
  float* po;           // prefix partials [CTA + item][RT][hd]; ml [..][RT][2]
  float* pml;
  float* oo;           // own partials [CTA + item][OL][hd]; ml [..][OL][2]
  float* oml;
  float* sc;           // log2-domain scores of the own rows [R][nq][sc_stride] (mass only)
  long long sc_stride;
  int* err;
};

// How one of the two main kernels cuts the work: key rows per tile, query rows per prefix item, CTAs,
// partial rows per query head that an own segment leaves (one per quarter of a tile's keys where the
// four warps of the tensor-core kernel each keep their own running maximum).
template <int KT_, int RT_, int G_, int OQ_>
struct CutOf {
  static constexpr int KT = KT_, RT = RT_, G = G_, OQ = OQ_;
};
using CutSimt = CutOf<64, 16, 296, 1>;  // CUDA cores: two CTAs on each of 148 SMs

__host__ __device__ inline long long align_up(long long x, long long a) { return (x + a - 1) / a * a; }

struct WsLayout {
  long long cum, po, pml, oo, oml, sc, sc_stride, bytes;
};
template <class Cut>
__host__ inline WsLayout ws_layout(int R, int nq, int nkv, int hd, int P, int max_len, bool mass) {
  const long long g = nq / nkv, items_p = P > 0 ? (long long)nkv * ((R * g + Cut::RT - 1) / Cut::RT) : 0;
  const long long slots_p = P > 0 ? items_p + Cut::G : 0, slots_o = (long long)R * nkv + Cut::G;
  WsLayout w;
  long long at = 0;
  auto take = [&](long long n) {
    const long long p = at;
    at = align_up(at + n, 256);
    return p;
  };
  w.cum = take((long long)(R + 1) * 4);
  w.po = take(slots_p * Cut::RT * hd * 4);
  w.pml = take(slots_p * Cut::RT * 8);
  w.oo = take(slots_o * Cut::OQ * g * hd * 4);
  w.oml = take(slots_o * Cut::OQ * g * 8);
  w.sc_stride = align_up(max_len, 128);
  w.sc = take(mass ? (long long)R * nq * w.sc_stride * 4 : 0);
  w.bytes = at;
  return w;
}

// Own rows of request r before this step, -1 if the slot is idle (or out of range: *bad).
__device__ __forceinline__ int own_rows(const Params& p, int r, bool* bad) {
  const long long pos = p.pos[r];
  if (pos < 0) return -1;
  const long long n = p.rows ? p.rows[r] : pos - p.P;
  if (pos >= p.rope_len || n < 0 || n >= p.max_len) {
    *bad = true;
    return -1;
  }
  return (int)n;
}

// One warp: cum_s[r] = own tiles per head of the requests before r (cum_s[R]: of all), and whether any
// request is live; records positions out of range. Sixteen requests' lengths are in flight per lane pair
// of loads, so a server of 64 pays for one trip to L2.
template <int KT>
__device__ __forceinline__ bool scan_tiles(const Params& p, int* cum_s, bool report) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  bool any = false, bad = false;
  for (int r0 = 0; r0 < p.R; r0 += 32) {
    const int r = r0 + lane;
    const int n = r < p.R ? own_rows(p, r, &bad) : -1;
    any |= n >= 0;
    int x = n > 0 ? (n + KT - 1) / KT : 0;
    const int own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (r < p.R) cum_s[r] = base + x - own;
    base += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) cum_s[p.R] = base;
  if (report && bad) set_dev_error(p.err, SK_DEVERR_POS_RANGE);
  return __any_sync(0xffffffffu, any);
}

// The row of tiles of one step.
struct Tiles {
  int tp;             // tiles of a prefix item
  int nrt;            // prefix items per head
  long long n_prefix; // tiles of all prefix items
  long long n;        // all tiles
  int G;              // CTAs with work: min(grid, n), so that none between two of an item's is without a part
};
template <class Cut>
__device__ __forceinline__ Tiles tiles_of(const Params& p, int own_tiles, bool any) {
  Tiles t;
  t.tp = any ? (p.P + Cut::KT - 1) / Cut::KT : 0;
  t.nrt = (p.R * p.g + Cut::RT - 1) / Cut::RT;
  t.n_prefix = (long long)t.tp * t.nrt * p.nkv;
  t.n = t.n_prefix + (long long)own_tiles * p.nkv;
  t.G = (int)min((long long)Cut::G, t.n);
  return t;
}
__device__ __forceinline__ long long share_begin(const Tiles& t, int c) { return c < t.G ? t.n * c / t.G : t.n; }
__device__ __forceinline__ int share_of(const Tiles& t, long long tile) {  // the CTA whose share holds `tile`
  return (int)(((tile + 1) * t.G - 1) / t.n);
}

// The part of one item that a CTA does.
struct Segment {
  bool prefix;
  int item;     // prefix: kvh * nrt + rt; own: r * nkv + kvh
  int kvh, r;   // r: request (own), or the tile of query rows (prefix)
  int t0, t1;   // tiles of the item
  int n_keys;   // rows of the item (prefix: P; own: n)
};
// The segment that starts at `tile`, ending at `end` at the latest. cum: the scan of scan_tiles.
template <class Cut>
__device__ __forceinline__ Segment segment_at(const Params& p, const Tiles& t, const int* cum, long long tile,
                                              long long end) {
  Segment s;
  if (tile < t.n_prefix) {
    s.prefix = true;
    s.item = (int)(tile / t.tp);
    s.kvh = s.item / t.nrt;
    s.r = s.item - s.kvh * t.nrt;
    s.t0 = (int)(tile - (long long)s.item * t.tp);
    s.t1 = (int)min((long long)t.tp, s.t0 + (end - tile));
    s.n_keys = p.P;
    return s;
  }
  const long long o = tile - t.n_prefix;
  int lo = 0, hi = p.R;  // the last r with cum[r] * nkv <= o (and tiles of its own)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long long)cum[mid] * p.nkv <= o)
      lo = mid;
    else
      hi = mid;
  }
  const int tr = cum[lo + 1] - cum[lo];
  const int in_r = (int)(o - (long long)cum[lo] * p.nkv);
  s.prefix = false;
  s.r = lo;
  s.kvh = in_r / tr;
  s.item = lo * p.nkv + s.kvh;
  s.t0 = in_r - s.kvh * tr;
  s.t1 = (int)min((long long)tr, s.t0 + (end - tile));
  bool bad = false;
  s.n_keys = own_rows(p, lo, &bad);
  return s;
}

// E consecutive floats, E 2 or 4, aligned to their size.
template <int E>
__device__ __forceinline__ void load_vec(const float* p, float (&x)[E]) {
  if constexpr (E == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    static_assert(E == 2, "2 or 4");
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x, x[1] = v.y;
  }
}
template <int E>
__device__ __forceinline__ void store_vec(float* p, const float (&x)[E]) {
  if constexpr (E == 4)
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
}

// ---- head rows ------------------------------------------------------------------------------------
// One warp holds a head row of HD elements, HD / 32 consecutive ones per lane; an element's partner in the
// rotate-half rotation (d and d + HD/2) is then in lane ^ 16 at the same place.
template <int HD>
__device__ __forceinline__ void load_row(const void* base, long long at, int is_bf16, float (&x)[HD / 32]) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  if (is_bf16) {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(base) + at + lane * E;
    uint32_t w[E / 2];
    if constexpr (E == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x;
      w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      x[2 * e] = __uint_as_float(w[e] << 16);
      x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
    load_vec<E>(reinterpret_cast<const float*>(base) + at + lane * E, x);
  }
}
// RMS norm (x w) and rotation of a head row in fp32, the reference's order of operations
// (qwen3/kernels.py:354-380); `turn` = the rope table's row of the position.
template <int HD>
__device__ __forceinline__ void norm_rotate(float (&x)[HD / 32], const float* w, const float* turn, float eps) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) ss += x[e] * x[e];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss / HD + eps);
  float wv[E], c[E], s[E];
  load_vec<E>(w + lane * E, wv);
  load_vec<E>(turn + (lane & 15) * E, c);
  load_vec<E>(turn + HD / 2 + (lane & 15) * E, s);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = x[e] * inv * wv[e];
    const float other = __shfl_xor_sync(0xffffffffu, y, 16);
    x[e] = y * c[e] + (lane < 16 ? -other : other) * s[e];
  }
}

}  // namespace shared
}  // namespace sk

// Key tiles of the shared-prefix decode attention on the sm_100a tensor cores (bf16 caches). The work split
// and the workspace are described in shared_decode.cuh.
//
// One persistent CTA per SM walks its share of 128-key tiles:
//   warp 8 (a lane)   TMA producer: K and V tiles into two rings.
//   warp 9 (a lane)   the score products, into tensor-memory buffer S[i % 2].
//   warp 10 (a lane)  the value products, into O[segment % 2].
//   warp 11           the scan of the lengths at the start.
//   warps 0-3         softmax.
//   warps 4-7         the query rows of the next segment (norm, rotation, split, into shared memory) and the
//                     partials of the last one out of tensor memory, both while the segment between runs.
//
// Two forms of the products, by the segment's query rows n (measured per 128-key tile, head size 128, fp32
// out, when nothing waits for memory):
//   n <= 32  S^T = K·Q^T and O^T = V^T·P^T: M = 128 are the tile's keys (the head's elements), N the query
//            rows, hi and lo terms side by side (16 columns for up to 8 rows, 64 for up to 32). Thread j of the
//            softmax owns key j of the tile; P^T goes to shared memory; the running maximum is shared by the
//            128 threads and moved only when a score exceeds it by 2^8, so a tile costs one vote. Nearly all
//            own rows (g <= 8 query heads per key) run here: a 128-row operand for 2 rows would be 1/64 full.
//   n > 32   S = Q·K^T and O = P·V: M = 128 are the query rows, thread r owns row r; P stays in tensor memory.
//
// Rounding. K and V are bf16 already. q = hi + lo in bf16 leaves 2^-16 of q at most, and costs one more
// product per tile, which runs while memory is waited for; with a single bf16 term a score of 10 is off by
// 0.02. The weights P are rounded to bf16 where the output is (2^-8 either way); P_SPLIT (fp32 outputs) adds
// their rest as a second bf16 term. The running sum is of the unrounded weights, in fp32.
#include <type_traits>

#include "shared_decode.cuh"

namespace sk {
namespace shared {

constexpr int kThreadsTc = 384;
constexpr int kWarpQo = 4, kWarpProducer = 8, kWarpS = 9, kWarpPv = 10, kWarpScan = 11;
// Launched at 128 registers a thread (49152, which leaves room on the SM for a CTA of the joining kernel, 16384):
// softmax 168, query/output 128, the others 88.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 168, kQoRegs = 128, kControlRegs = 88;
static_assert(128 * (kSoftmaxRegs + kQoRegs + kControlRegs) <= kThreadsTc * kLaunchRegs, "register split over budget");
constexpr float kRescale = 8.0f;  // O is rescaled when the running max grows by more than 2^8; exact either way

template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Where the row, head and request coordinates of a cache go in its tensor map, whose dimensions are sorted by
// stride.
struct MapOrder {
  int row, head, req;  // 0..2: dimension 1 + that
};

template <int HD>
struct SmemTc {
  static constexpr int NSK = HD == 128 ? 2 : 4, NSV = HD == 128 ? 2 : 4;
  static constexpr int NCH = HD / 64;
  static constexpr int Q_BYTES = 128 * HD * 2, KV_BYTES = 128 * HD * 2;
  // Query area. n > 32: hi rows, then lo rows [128][hd]. n <= 32: two buffers of 64 rows (hi, then lo), then
  // two of P^T [64 rows][128 keys] (weights, then their rests); 64-element chunks 8 KB apart.
  static constexpr int QT_BYTES = 64 * HD * 2, PT_BYTES = 64 * 128 * 2;
  static constexpr int OFF_Q = 0, OFF_PT = 2 * QT_BYTES;
  static constexpr int Q_AREA = 2 * QT_BYTES + 2 * PT_BYTES;
  static_assert(Q_AREA >= 2 * Q_BYTES, "the query area holds either form");
  // V before K: at hd = 64 the V^T operand (M = 128) reads 16 KB past its tile, into lanes that are not used
  static constexpr int OFF_V = OFF_Q + Q_AREA;
  static constexpr int OFF_K = OFF_V + NSV * KV_BYTES;
  static constexpr int OFF_ML = OFF_K + NSK * KV_BYTES;  // [2] n > 32: [128] (max, sum); else sums [4][32], max [32]
  static constexpr int OFF_MX = OFF_ML + 2 * 128 * 8;    // [4][32] maxima of the warps, [32] running, [32] factors
  static constexpr int OFF_BAR = OFF_MX + 6 * 32 * 4;
  static constexpr int NBAR = 2 * NSK + 2 * NSV + 16;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;    // tensor-memory base, whether there is a segment
  static constexpr int OFF_TILES = OFF_MISC + 16;
  static constexpr int OFF_SEG = OFF_TILES + 32;
  static constexpr int OFF_LENS = OFF_SEG + 32;
  static_assert(sizeof(Tiles) <= 32 && sizeof(Segments) <= 32, "their places in shared memory");
  static __host__ __device__ int bytes(int R) { return OFF_LENS + Lens::bytes(R); }
  static_assert(OFF_LENS + (3 * kMaxRequests + 1) * 4 <= 232448, "shared memory over the 227 KB per-CTA limit");
};

struct TcArgs {
  Params p;
  MapOrder order;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_part(float x, uint32_t packed, int half) {  // x less its bf16 term
  return x - __uint_as_float(half ? (packed & 0xffff0000u) : (packed << 16));
}
// 16 tensor-memory columns of this warp's lanes.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 16 tensor-memory columns of this warp's lanes into registers, and back.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
template <int N>  // N a multiple of 16
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float (&v)[N]) {
  if constexpr (N % 32 == 0) {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_ld32(taddr + c, v + c);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 16) tmem_ld16(taddr + c, v + c);
  }
}
template <int N>
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 16) tmem_st16(taddr + c, *reinterpret_cast<const uint32_t(*)[16]>(v + c));
}
// Whether any of the 128 softmax threads says so (named barrier 1).
__device__ __forceinline__ bool any_of_128(bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"((uint32_t)x)
      : "memory");
  return y != 0;
}
// Sum or maximum over the warp of each of H values per lane (H a power of two up to 32), by halves: lane l
// returns that of value l * H / 32.
template <int H, class Op>
__device__ __forceinline__ float warp_reduce(float (&x)[H], Op op) {
  const int lane = threadIdx.x & 31;
  int off = 16;
#pragma unroll
  for (int m = H; m > 1; m >>= 1, off >>= 1) {
    const bool upper = lane & off;
#pragma unroll
    for (int i = 0; i < m / 2; ++i) {
      const float send = upper ? x[i] : x[i + m / 2], keep = upper ? x[i + m / 2] : x[i];
      x[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, off));
    }
  }
#pragma unroll
  for (; off > 0; off >>= 1) x[0] = op(x[0], __shfl_xor_sync(0xffffffffu, x[0], off));
  return x[0];
}

// Query rows of a segment, and the columns' half width of its transposed form: 8 or 32 (0: the other form).
__device__ __forceinline__ int rows_of(const Params& p, const Segments& s) {
  return s.prefix ? min(CutTc::RT, p.R * p.g - s.r * CutTc::RT) : p.g;
}
__device__ __forceinline__ int form_of(int n) { return n <= 8 ? 8 : n <= 32 ? 32 : 0; }

template <int HD, bool P_SPLIT>
__global__ void __maxnreg__(kLaunchRegs)
    tiles_tc_kernel(const __grid_constant__ CUtensorMap tmKp, const __grid_constant__ CUtensorMap tmVp,
                    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ TcArgs args) {
  using S = SmemTc<HD>;
  constexpr int NSK = S::NSK, NSV = S::NSV, NCH = S::NCH, E = HD / 32;
  const Params& p = args.p;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {  // uniform, before any barrier: report and leave
    if (threadIdx.x == 0) set_dev_error(p.err, SK_DEVERR_TIMEOUT);
    return;
  }
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint64_t* k_empty = k_full + NSK;
  uint64_t* v_full = k_empty + NSK;
  uint64_t* v_empty = v_full + NSV;
  uint64_t* s_full = v_empty + NSV;   // [tile & 1] S computed
  uint64_t* p_full = s_full + 2;      // [tile & 1] P written (128 arrivals)
  uint64_t* o_done = p_full + 2;      // [tile & 1] P·V complete
  uint64_t* q_full = o_done + 2;      // [segment & 1] query rows in place (128 arrivals)
  uint64_t* sq_done = q_full + 2;     // [segment & 1] every S of the segment complete
  uint64_t* so_full = sq_done + 2;    // [segment & 1] every P·V complete
  uint64_t* ml_full = so_full + 2;    // [segment & 1] (max, sum) written (128 arrivals)
  uint64_t* o_free = ml_full + 2;     // [segment & 1] output and (max, sum) read (128 arrivals)
  float2* ml_s = reinterpret_cast<float2*>(smem + S::OFF_ML);
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + S::OFF_MISC);
  const Lens ls(smem + S::OFF_LENS, p.R);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NSK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < NSV; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 128), mbar_init(&o_done[i], 1);
      mbar_init(&q_full[i], 128), mbar_init(&sq_done[i], 1), mbar_init(&so_full[i], 1);
      mbar_init(&ml_full[i], 128), mbar_init(&o_free[i], 128);
    }
    fence_mbar_init();
  }
  if (warp == kWarpProducer && lane == 0) {
    if (p.P > 0) {
      tma_prefetch_desc(&tmKp);
      tma_prefetch_desc(&tmVp);
    }
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == kWarpS) {
    tmem_alloc(misc, 512);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch_dependents();
  if (warp == kWarpScan) {
    const bool any = scan_tiles<CutTc::KT>(p, ls, c == 0);
    __syncwarp();
    if (lane == 0) {
      const Tiles tl = tiles_of<CutTc>(p, ls.cum[p.R], any);
      Segments sg;
      misc[1] = sg.first(p, tl, ls, c);
      *reinterpret_cast<Tiles*>(smem + S::OFF_TILES) = tl;
      *reinterpret_cast<Segments*>(smem + S::OFF_SEG) = sg;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0], tS = tmem, tO = tmem + 256;  // S0 S1 | O0 O1, 128 columns each; P over S
  const Tiles tl = *reinterpret_cast<const Tiles*>(smem + S::OFF_TILES);
  Segments sg = *reinterpret_cast<const Segments*>(smem + S::OFF_SEG);
  bool more = misc[1];

  // The eight working warps keep step with one another (votes, warp-wide loads): a thread whose wait ran out
  // (the error word then says so) goes on to the end without waiting, its results void, rather than leaving.
  bool dead = false;
  auto wait = [&](uint64_t* bar, int phase) {
    if (!dead) dead = !mbar_wait(bar, phase & 1, p.err);
    __syncwarp();
  };

  if (warp >= 8) {
    setmaxnreg_dec<kControlRegs>();
    if (warp == kWarpProducer && lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      int i = 0;
      bool ok = true;
      auto load = [&](uint8_t* dst, const CUtensorMap* mp, const CUtensorMap* mo, uint64_t* bar, int row) {
        mbar_arrive_expect_tx(bar, S::KV_BYTES);
        if (sg.prefix) {
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch) tma_load_3d(dst + ch * 16384, mp, bar, ch * 64, row, sg.kvh);
        } else {
          const MapOrder& o = args.order;
          const int y = o.row == 0 ? row : o.head == 0 ? sg.kvh : sg.r;
          const int z = o.row == 1 ? row : o.head == 1 ? sg.kvh : sg.r;
          const int w = o.row == 2 ? row : o.head == 2 ? sg.kvh : sg.r;
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch) tma_load_4d(dst + ch * 16384, mo, bar, ch * 64, y, z, w);
        }
      };
      for (; more && ok; more = sg.next(p, tl, ls)) {
        for (int t = sg.t0; t < sg.t1; ++t, ++i) {
          const int k = i % NSK, v = i % NSV;
          if (i >= NSK && !(ok = mbar_wait(&k_empty[k], (i / NSK - 1) & 1, p.err))) break;
          load(smem + S::OFF_K + k * S::KV_BYTES, &tmKp, &tmK, &k_full[k], t * CutTc::KT);
          if (i >= NSV && !(ok = mbar_wait(&v_empty[v], (i / NSV - 1) & 1, p.err))) {
            mbar_wait(&k_full[k], (i / NSK) & 1, p.err);  // the copy in flight
            break;
          }
          load(smem + S::OFF_V + v * S::KV_BYTES, &tmVp, &tmV, &v_full[v], t * CutTc::KT);
        }
      }
      // shared memory stays until every copy has landed (on the normal path they all have)
      for (int j = max(0, i - NSK); j < i; ++j) mbar_wait(&k_full[j % NSK], (j / NSK) & 1, p.err);
      for (int j = max(0, i - NSV); j < i; ++j) mbar_wait(&v_full[j % NSV], (j / NSV) & 1, p.err);
    } else if (warp == kWarpS && lane == 0) {
      // ---------------------------------------------------------------- S = Q·K^T
      const uint32_t aQ = sbase + S::OFF_Q, aK = sbase + S::OFF_K;
      int i = 0, seg = 0;
      bool ok = true;
      for (; more && ok; more = sg.next(p, tl, ls), ++seg) {
        const int form = form_of(rows_of(p, sg));
        const uint32_t id = form == 0 ? idesc_bf16_f32(128, 128, 0, 0)
                            : form == 8 ? idesc_bf16_f32(128, 16, 0, 0) : idesc_bf16_f32(128, 64, 0, 0);
        if (!(ok = mbar_wait(&q_full[seg & 1], (seg >> 1) & 1, p.err))) break;
        for (int t = sg.t0; t < sg.t1; ++t, ++i) {
          const int w = i & 1, k = i % NSK;
          if (!(ok = mbar_wait(&k_full[k], (i / NSK) & 1, p.err))) break;
          // the value product of tile i - 2 has read its P, which overlays this buffer or was made from it
          if (i >= 2 && !(ok = mbar_wait(&o_done[w], ((i - 2) >> 1) & 1, p.err))) break;
          tc_fence_after();
          const uint32_t kb = aK + k * S::KV_BYTES;
          if (form == 0) {
#pragma unroll
            for (int term = 0; term < 2; ++term)
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk) {
                const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                tc_mma_ss(tS + w * 128, smem_desc_sw128(aQ + term * S::Q_BYTES + off, 16, 1024),
                          smem_desc_sw128(kb + off, 16, 1024), id, term > 0 || kk > 0);
              }
          } else {
            const uint32_t qb = aQ + (seg & 1) * S::QT_BYTES;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              tc_mma_ss(tS + w * 128, smem_desc_sw128(kb + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                        smem_desc_sw128(qb + (kk >> 2) * 8192 + (kk & 3) * 32, 16, 1024), id, kk > 0);
          }
          tc_commit(&s_full[w]);
          tc_commit(&k_empty[k]);
        }
        if (ok) tc_commit(&sq_done[seg & 1]);
      }
    } else if (warp == kWarpPv && lane == 0) {
      // ---------------------------------------------------------------- O += P·V
      const uint32_t aV = sbase + S::OFF_V, aP = sbase + S::OFF_PT;
      int i = 0, seg = 0;
      bool ok = true;
      for (; more && ok; more = sg.next(p, tl, ls), ++seg) {
        const int form = form_of(rows_of(p, sg));
        const uint32_t id = form == 0 ? idesc_bf16_f32(128, HD, 0, 1)
                            : form == 8 ? idesc_bf16_f32(128, 16, 1, 0)
                            : P_SPLIT ? idesc_bf16_f32(128, 64, 1, 0) : idesc_bf16_f32(128, 32, 1, 0);
        const uint32_t oc = tO + (seg & 1) * 128;
        if (seg >= 2 && !(ok = mbar_wait(&o_free[seg & 1], ((seg - 2) >> 1) & 1, p.err))) break;
        for (int t = sg.t0; t < sg.t1; ++t, ++i) {
          const int w = i & 1, v = i % NSV;
          if (!(ok = mbar_wait(&v_full[v], (i / NSV) & 1, p.err))) break;
          if (!(ok = mbar_wait(&p_full[w], (i >> 1) & 1, p.err))) break;
          tc_fence_after();
          const uint32_t vb = aV + v * S::KV_BYTES;
          if (form == 0) {
#pragma unroll
            for (int term = 0; term < (P_SPLIT ? 2 : 1); ++term)
#pragma unroll
              for (int kk = 0; kk < 8; ++kk)
                tc_mma_ts(oc, tS + w * 128 + (kk >> 1) * 32 + (kk & 1) * 8 + term * 16,
                          smem_desc_sw128(vb + kk * 2048, 16384, 1024), id,
                          t > sg.t0 || term > 0 || kk > 0);
          } else {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc_mma_ss(oc, smem_desc_sw128(vb + kk * 2048, 16384, 1024),
                        smem_desc_sw128(aP + w * S::PT_BYTES + (kk >> 2) * 8192 + (kk & 3) * 32, 16, 1024), id,
                        t > sg.t0 || kk > 0);
          }
          tc_commit(&o_done[w]);
          tc_commit(&v_empty[v]);
        }
        if (ok) tc_commit(&so_full[seg & 1]);
      }
    }
  } else if (warp >= kWarpQo) {
    // ------------------------------------------------------------------ query rows and partials
    setmaxnreg_dec<kQoRegs>();
    const int q = warp & 3;  // this warp's quarter of the lanes
    uint8_t* Qs = smem + S::OFF_Q;
    auto prepare = [&](const Segments& s, int seg) {
      const int n = rows_of(p, s), form = form_of(n);
      // rows q, q + 4, ...: kRowsAhead of them at a time, so that a batch pays for one trip to memory
      constexpr int kRowsAhead = 4;
      for (int i0 = q; i0 < n; i0 += 4 * kRowsAhead) {
        float x[kRowsAhead][E];
        int r[kRowsAhead];
#pragma unroll
        for (int b = 0; b < kRowsAhead; ++b) {
          const int i = min(i0 + 4 * b, n - 1), row = s.prefix ? s.r * CutTc::RT + i : i;
          r[b] = s.prefix ? (int)((uint32_t)row / p.g) : s.r;
          load_row<HD>(p.qkv, r[b] * p.qkv_stride + (long long)(s.kvh * p.g + row - (s.prefix ? r[b] * p.g : 0)) * HD,
                       p.qkv_bf16, x[b]);
        }
        norm_rotate_rows<HD, kRowsAhead>(x, r, ls.pos, p.qn, p.rope, p.eps);
#pragma unroll
        for (int b = 0; b < kRowsAhead; ++b) {
          const int i = i0 + 4 * b;
          if (i >= n) break;
          uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            const float u = x[b][2 * e] * p.q_scale, v = x[b][2 * e + 1] * p.q_scale;
            hi[e] = pack_bf16(u, v);
            lo[e] = pack_bf16(lo_part(u, hi[e], 0), lo_part(v, hi[e], 1));
          }
          // element d: 64-element chunk d / 64, 16-byte unit (d % 64) / 8 exclusive-or the row's low bits
          const int d = lane * E, unit = (d & 63) >> 3, chunk = d >> 6;
          const int at_hi = form == 0 ? chunk * 16384 + i * 128 + ((unit ^ (i & 7)) << 4)
                                      : (seg & 1) * S::QT_BYTES + chunk * 8192 + i * 128 + ((unit ^ (i & 7)) << 4);
          const int at_lo = at_hi + (form == 0 ? S::Q_BYTES : form * 128);  // form rows on: the same low bits
          if (SK_INB(at_hi >= 0 && at_lo + 16 <= S::Q_AREA, p.err)) {
            if constexpr (E == 4) {
              *reinterpret_cast<uint2*>(Qs + at_hi + (d & 7) * 2) = make_uint2(hi[0], hi[1]);
              *reinterpret_cast<uint2*>(Qs + at_lo + (d & 7) * 2) = make_uint2(lo[0], lo[1]);
            } else {
              *reinterpret_cast<uint32_t*>(Qs + at_hi + (d & 7) * 2) = hi[0];
              *reinterpret_cast<uint32_t*>(Qs + at_lo + (d & 7) * 2) = lo[0];
            }
          }
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&q_full[seg & 1]);
    };
    if (more) prepare(sg, 0);
    for (int seg = 0; more; ++seg) {
      const int n = rows_of(p, sg), form = form_of(n);
      Segments nx = sg;
      const bool another = nx.next(p, tl, ls);
      if (another) {
        // Small segments alternate between two buffers. Rows of the large form fill the area: every product
        // of the segment before that reads it (the values' too, if that one is small) comes first.
        const int nf = form_of(rows_of(p, nx));
        if (form == 0) wait(&sq_done[seg & 1], seg >> 1);
        if (form != 0 && nf == 0) wait(&so_full[seg & 1], seg >> 1);
        prepare(nx, seg + 1);
      }
      wait(&so_full[seg & 1], seg >> 1);
      wait(&ml_full[seg & 1], seg >> 1);
      tc_fence_after();
      const long long slot = (long long)c + sg.item;
      const long long row0 = sg.prefix ? slot * CutTc::RT : slot * p.g;  // first partial row
      float* o = (sg.prefix ? p.po : p.oo) + row0 * HD;
      float2* ml = reinterpret_cast<float2*>(sg.prefix ? p.pml : p.oml) + row0;
      const uint32_t oc = tO + (seg & 1) * 128 + ((uint32_t)(32 * q) << 16);
      const int l = 32 * q + lane;
      if (form == 0) {
        if (32 * q < n) {
#pragma unroll
          for (int ch = 0; ch < HD / 32; ++ch) {
            float v[32];
            tmem_ld32(oc + ch * 32, v);
            tmem_wait_ld();
            if (l < n) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(o + l * HD + ch * 32 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
          }
          if (l < n) ml[l] = ml_s[(seg & 1) * 128 + l];
        }
      } else {
        auto columns = [&](auto half) {  // lane l holds element l of every row
          constexpr int N = decltype(half)::value;
          if (32 * q < HD) {
            float v[2 * N];  // weights' part, then their rests'
            tmem_ld_cols(oc, v);
            tmem_wait_ld();
#pragma unroll
            for (int h = 0; h < N; ++h)
              if (h < n) o[h * HD + l] = P_SPLIT ? v[h] + v[N + h] : v[h];
          }
        };
        if (form == 8)
          columns(std::integral_constant<int, 8>());
        else
          columns(std::integral_constant<int, 32>());
        const float* st = reinterpret_cast<const float*>(ml_s + (seg & 1) * 128);
        if (l < n) ml[l] = make_float2(st[128 + l], (st[l] + st[32 + l]) + (st[64 + l] + st[96 + l]));
      }
      tc_fence_before();
      mbar_arrive(&o_free[seg & 1]);
      sg = nx;
      more = another;
    }
  } else {
    // ------------------------------------------------------------------ softmax
    setmaxnreg_inc<kSoftmaxRegs>();
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const int j = threadIdx.x;  // the key of a tile (n <= 32) or the query row (n > 32) of this thread
    float* mx_s = reinterpret_cast<float*>(smem + S::OFF_MX);
    float *m_s = mx_s + 128, *a_s = m_s + 32;
    int i = 0, seg = 0;
    // Rows past the request's last: P is zero there, but what the cache holds may be NaN (past a prefix's end
    // the copy has already put zeros).
    auto clear_tail = [&](int nk) {
      const int v = i % NSV;
      wait(&v_full[v], i / NSV);
      uint8_t* Vt = smem + S::OFF_V + v * S::KV_BYTES;
      for (int u = j; u < (CutTc::KT - nk) * 8; u += 128)
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch)
          if (SK_INB(nk * 8 + u < 1024, p.err))
            *reinterpret_cast<uint4*>(Vt + ch * 16384 + nk * 128 + u * 16) = make_uint4(0, 0, 0, 0);
    };
    // n <= 32 query rows: N the half width of the columns, H >= n rows computed
    auto by_keys = [&](auto half, auto rows, int n) {
      constexpr int N = decltype(half)::value, H = decltype(rows)::value;
      float l[H] = {};
      const uint32_t o_at = tO + (seg & 1) * 128 + lane_off;
      float* sc = !sg.prefix && p.mass ? p.sc + ((long long)sg.r * p.nq + sg.kvh * p.g) * p.sc_stride + j : nullptr;
      for (int t = sg.t0; t < sg.t1; ++t, ++i) {
        const int w = i & 1, nk = min(CutTc::KT, sg.n_keys - t * CutTc::KT);
        wait(&s_full[w], i >> 1);
        tc_fence_after();
        float x[H];
        {
          float raw[2 * N];
          tmem_ld_cols(tS + w * 128 + lane_off, raw);
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < H; ++h) x[h] = j < nk && h < n ? raw[h] + raw[N + h] : -INFINITY;
        }
        bool over = t == sg.t0;
        if (t > sg.t0) {
#pragma unroll
          for (int h = 0; h < H; ++h) over |= x[h] > m_s[h] + kRescale;
        }
        if (sc) {
#pragma unroll
          for (int h = 0; h < (H < kMaxGroup ? H : kMaxGroup); ++h)
            if (h < n) sc[h * p.sc_stride + (long long)t * CutTc::KT] = x[h];
        }
        if (any_of_128(over)) {
          float y[H];
#pragma unroll
          for (int h = 0; h < H; ++h) y[h] = x[h];
          const float top = warp_reduce<H>(y, [](float a, float b) { return fmaxf(a, b); });
          if (lane % (32 / H) == 0) mx_s[warp * 32 + lane / (32 / H)] = top;
          named_bar_sync(2, 128);
          if (j < H) {
            const float old = t > sg.t0 ? m_s[j] : -INFINITY;
            const float to = fmaxf(fmaxf(fmaxf(mx_s[j], mx_s[32 + j]), fmaxf(mx_s[64 + j], mx_s[96 + j])), old);
            a_s[j] = to == -INFINITY ? 1.f : ex2_approx(old - to);
            m_s[j] = to;
          }
          named_bar_sync(2, 128);
          if (t > sg.t0) {
#pragma unroll
            for (int h = 0; h < H; ++h) l[h] *= a_s[h];
            wait(&o_done[(i - 1) & 1], (i - 1) >> 1);
            tc_fence_after();
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {  // the weights' columns and their rests'
              float v[N < 16 ? 16 : N];
              tmem_ld_cols(o_at + part * N, v);
              tmem_wait_ld();
#pragma unroll
              for (int h = 0; h < H; ++h) {
                v[h] *= a_s[h];
                if (N < 16) v[N + h] *= a_s[h];
              }
              tmem_st_cols(o_at + part * N, v);
              if (N < 16) break;  // both at once
            }
            tmem_wait_st();
            tc_fence_before();
          }
        }
        uint8_t* Pt = smem + S::OFF_PT + w * S::PT_BYTES + (j >> 6) * 8192 + (j & 7) * 2;
        const int unit = (j & 63) >> 3;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float top = m_s[h], y = ex2_approx(x[h] - (top == -INFINITY ? 0.f : top));
          l[h] += y;
          const __nv_bfloat16 b = __float2bfloat16_rn(y);
          const int at = h * 128 + ((unit ^ (h & 7)) << 4);  // N rows on: the same low bits
          *reinterpret_cast<__nv_bfloat16*>(Pt + at) = b;
          if (P_SPLIT) *reinterpret_cast<__nv_bfloat16*>(Pt + at + N * 128) = __float2bfloat16_rn(y - __bfloat162float(b));
        }
        if (nk < CutTc::KT && !sg.prefix) clear_tail(nk);
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
      }
      if (seg >= 2) wait(&o_free[seg & 1], (seg - 2) >> 1);
      float* st = reinterpret_cast<float*>(ml_s + (seg & 1) * 128);
      if (j < H) st[128 + j] = m_s[j];
      const float sum = warp_reduce<H>(l, [](float a, float b) { return a + b; });
      if (lane % (32 / H) == 0) st[warp * 32 + lane / (32 / H)] = sum;
      mbar_arrive(&ml_full[seg & 1]);
    };
    // n > 32 query rows, one per thread. A tile's scores are read twice, a quarter of the columns at a time,
    // for the maximum and for the weights, which go back over the quarter they came from (16 columns of bf16
    // pairs, 16 of their rests): in registers a row would take 128.
    auto by_rows = [&](int n) {
      const bool any = warp * 32 < n;
      const uint32_t o_at = tO + (seg & 1) * 128 + lane_off;
      float m_run = -INFINITY, l_run = 0.f;
      for (int t = sg.t0; t < sg.t1; ++t, ++i) {
        const int w = i & 1, nk = min(CutTc::KT, sg.n_keys - t * CutTc::KT);
        const uint32_t s_at = tS + w * 128 + lane_off;
        wait(&s_full[w], i >> 1);
        tc_fence_after();
        if (any) {
          float m_new = m_run;
#pragma unroll 1
          for (int u = 0; u < 4; u += 2) {
            float x[64];
            tmem_ld_cols(s_at + u * 32, x);
            tmem_wait_ld();
            if (nk < CutTc::KT) {
#pragma unroll
              for (int e = 0; e < 64; ++e) x[e] = u * 32 + e < nk ? x[e] : -INFINITY;
            }
            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
              m0 = max3(m0, x[e], x[e + 1]);
              m1 = max3(m1, x[e + 2], x[e + 3]);
            }
            m_new = max3(m_new, m0, m1);
          }
          if (__any_sync(0xffffffffu, m_new > m_run + kRescale)) {  // O and the sum of this warp's rows
            const float alpha = m_new == -INFINITY ? 1.f : ex2_approx(m_run - m_new);
            if (t > sg.t0) {
              wait(&o_done[(i - 1) & 1], (i - 1) >> 1);
              tc_fence_after();
#pragma unroll 1
              for (int ch = 0; ch < HD / 32; ++ch) {
                float v[32];
                tmem_ld32(o_at + ch * 32, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] *= alpha;
                tmem_st32(o_at + ch * 32, v);
              }
              tmem_wait_st();
            }
            l_run *= alpha;
            m_run = m_new;
          }
          const float use = m_run == -INFINITY ? 0.f : m_run;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll 1
          for (int u = 0; u < 4; u += 2) {
            float x[64];
            tmem_ld_cols(s_at + u * 32, x);
            tmem_wait_ld();
            if (nk < CutTc::KT) {
#pragma unroll
              for (int e = 0; e < 64; ++e) x[e] = u * 32 + e < nk ? x[e] : -INFINITY;
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              uint32_t hi[16], lo[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float a = ex2_approx(x[32 * v + 2 * e] - use), b = ex2_approx(x[32 * v + 2 * e + 1] - use);
                l0 += a;
                l1 += b;
                hi[e] = pack_bf16(a, b);
                if (P_SPLIT) lo[e] = pack_bf16(lo_part(a, hi[e], 0), lo_part(b, hi[e], 1));
              }
              tmem_st16(s_at + (u + v) * 32, hi);
              if (P_SPLIT) tmem_st16(s_at + (u + v) * 32 + 16, lo);
            }
          }
          l_run += l0 + l1;
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&p_full[w]);
      }
      if (seg >= 2) wait(&o_free[seg & 1], (seg - 2) >> 1);
      ml_s[(seg & 1) * 128 + j] = make_float2(m_run, l_run);
      mbar_arrive(&ml_full[seg & 1]);
    };
    for (; more; more = sg.next(p, tl, ls), ++seg) {
      const int n = rows_of(p, sg), form = form_of(n);
      if (form == 0)
        by_rows(n);
      else if (n <= 2)
        by_keys(std::integral_constant<int, 8>(), std::integral_constant<int, 2>(), n);
      else if (form == 8)
        by_keys(std::integral_constant<int, 8>(), std::integral_constant<int, 8>(), n);
      else
        by_keys(std::integral_constant<int, 32>(), std::integral_constant<int, 32>(), n);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- host -----------------------------------------------------------------------------------------
// K and V of the requests' own caches as (hd, then row, head and request by ascending stride), boxes of 128
// rows x 64 elements; dimensions of one entry last, at the largest stride.
static bool own_map(CUtensorMap* m, const void* base, const Params& p, int hd, MapOrder* order) {
  struct Dim {
    long long stride;
    int n, box, which;
  } d[3] = {{p.row_stride, p.max_len, CutTc::KT, 0}, {p.head_stride, p.nkv, 1, 1}, {p.request_stride, p.R, 1, 2}};
  long long top = hd;
  for (Dim& x : d)
    if (x.n > 1 && x.stride > top) top = x.stride;
  for (Dim& x : d)
    if (x.n == 1) x.stride = top;
  auto before = [](const Dim& a, const Dim& b) { return a.stride < b.stride || (a.stride == b.stride && a.n > 1 && b.n == 1); };
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (before(d[j + 1], d[j])) {
        const Dim x = d[j];
        d[j] = d[j + 1];
        d[j + 1] = x;
      }
  cuuint64_t dims[4] = {(cuuint64_t)hd}, str[3];
  cuuint32_t box[4] = {64};
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = (cuuint64_t)d[i].n;
    str[i] = (cuuint64_t)d[i].stride * 2;
    box[i + 1] = (cuuint32_t)d[i].box;
    (d[i].which == 0 ? order->row : d[i].which == 1 ? order->head : order->req) = i;
  }
  return sk_make_map_bf16(m, base, 4, dims, str, box);
}
static bool prefix_map(CUtensorMap* m, const void* base, const Params& p, int hd) {
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)p.P, (cuuint64_t)p.nkv};
  const long long hs = p.nkv > 1 ? p.prefix_head_stride : p.prefix_row_stride;
  cuuint64_t str[2] = {(cuuint64_t)p.prefix_row_stride * 2, (cuuint64_t)hs * 2};
  cuuint32_t box[3] = {64, CutTc::KT, 1};
  return sk_make_map_bf16(m, base, 3, dims, str, box);
}

template <int HD, bool P_SPLIT>
static int launch(const Params& p, cudaStream_t st) {
  CUtensorMap kp, vp, k, v;
  TcArgs a;
  a.p = p;
  if (!own_map(&k, p.Kc, p, HD, &a.order) || !own_map(&v, p.Vc, p, HD, &a.order)) return SK_ERR_CUDA;
  if (p.P > 0) {
    if (!prefix_map(&kp, p.Kp, p, HD) || !prefix_map(&vp, p.Vp, p, HD)) return SK_ERR_CUDA;
  } else {
    kp = k;  // never read
    vp = v;
  }
  const int smem = SmemTc<HD>::bytes(p.R);
  if (cudaFuncSetAttribute(tiles_tc_kernel<HD, P_SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
      cudaSuccess)
    return SK_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CutTc::G);
  cfg.blockDim = dim3(kThreadsTc);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tiles_tc_kernel<HD, P_SPLIT>, kp, vp, k, v, a) == cudaSuccess ? SK_OK : SK_ERR_CUDA;
}

int launch_tiles_tc(const Params& p, int hd, bool p_split, cudaStream_t st) {
  if (hd == 128) return p_split ? launch<128, true>(p, st) : launch<128, false>(p, st);
  return p_split ? launch<64, true>(p, st) : launch<64, false>(p, st);
}

}  // namespace shared
}  // namespace sk

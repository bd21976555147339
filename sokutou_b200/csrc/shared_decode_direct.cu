// Shared-prefix decode attention in one launch, for steps where the prefix is short or the requests are few:
// every (request, key/value head) reads prefix and own rows for itself (the prefix comes from L2 after the
// first). A cluster of CTAs per (request, head), all rows dealt out to its warps in batches:
//
//   A row is loaded as 16 bytes per lane, so a row takes W = 8, 16 or 32 lanes and one load of a warp covers
//   32 / W rows; kLoads loads of K and of V make a batch, and the next batch is in flight while one is worked
//   on. Scores: every lane multiplies its elements for all g heads, then one butterfly leaves each sum in
//   one lane (each of the W lanes of a row group ends with g * kLoads / W of them), which exponentiates it;
//   the weights go back to the group by shuffles for P·V. The running maximum is the warp's and moves only
//   when a score exceeds it by 2^8. Warps are joined through shared memory, CTAs through the cluster's.
//
// All fp32: q is not rounded, K and V as stored. What bounds it: the loads in flight, 16 warps of 4 KB (K and V
// of 8 rows of 128) and their successors per SM.
#include "shared_decode.cuh"

namespace sk {
namespace shared {

constexpr int kDirThreads = 256, kDirWarps = kDirThreads / 32, kMaxCluster = 8;

template <typename T>
struct Pair;  // two neighbouring elements of a 16-byte load
template <>
struct Pair<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float2 get(const uint4& v, int i) {
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float rnd(float f) { return __bfloat162float(__float2bfloat16_rn(f)); }
  static __device__ __forceinline__ __nv_bfloat16 st(float f) { return __float2bfloat16_rn(f); }
};
template <>
struct Pair<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float2 get(const uint4& v, int i) {
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float rnd(float f) { return f; }
  static __device__ __forceinline__ float st(float f) { return f; }
};

__device__ __forceinline__ float warp_sum32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {  // read once by this CTA
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_remote(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Lanes per row, rows per load, loads per batch.
template <typename T, int HD, int GP>
struct DirectCfg {
  static constexpr int E = Pair<T>::E, W = HD / E, RPL = 32 / W;
  static constexpr int kLoads = 4;
  static constexpr int kRows = kLoads * RPL;     // rows of a batch
  static constexpr int NV = kLoads * GP;         // sums per row group
  static constexpr int VK = NV > W ? NV / W : 1; // of which a lane keeps this many
  static constexpr int REP = NV < W ? W / NV : 1;  // lanes that hold the same one
  static constexpr bool kAhead = GP <= 2;        // the next batch in registers
};

template <typename T, int HD, int GP>
__global__ void __launch_bounds__(kDirThreads, GP <= 4 ? 2 : 1) direct_kernel(const Params p, int cluster) {
  using C = DirectCfg<T, HD, GP>;
  constexpr int E = C::E, W = C::W, RPL = C::RPL, NL = C::kLoads, NV = C::NV, VK = C::VK, REP = C::REP, EL = HD / 32;
  __shared__ __align__(16) float q_s[GP][HD];
  __shared__ __align__(16) float kv_s[2][HD];              // the new token's k and v as the cache holds them
  __shared__ __align__(16) float red_s[kDirWarps][GP][HD];
  __shared__ float2 ml_s[kDirWarps][GP];
  __shared__ __align__(16) float o_s[GP][HD];              // the CTA's partial (read by the cluster)
  __shared__ float2 oml_s[GP];
  __shared__ float snew_s[GP], M_s[GP], iL_s[GP];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % W, grp = lane / W;
  const int item = blockIdx.x / cluster, rank = blockIdx.x % cluster;  // clusters are consecutive CTAs
  const int r = item / p.nkv, kvh = item - r * p.nkv, g = p.g;

  griddep_wait();
  griddep_launch_dependents();
  const long long pos64 = p.pos[r], own64 = p.rows ? p.rows[r] : pos64 - p.P;
  RawRow<HD> raw[1];  // warps 0 .. g-1: q rows; g: k; g + 1: v (several per warp where g + 2 > 8)
  raw[0].load(p.qkv, r * p.qkv_stride + (long long)(w < g ? kvh * g + w : w == g ? p.nq + kvh : p.nq + p.nkv + kvh) * HD,
              p.qkv_bf16);
  const bool idle = pos64 < 0, bad = !idle && (pos64 >= p.rope_len || own64 < 0 || own64 >= p.max_len);
  if (idle || bad) {  // uniform over the cluster
    if (bad && rank == 0 && kvh == 0 && threadIdx.x == 0) set_dev_error(p.err, SK_DEVERR_POS_RANGE);
    return;
  }
  const int n = (int)own64, P = p.P, N = P + n;
  const int pos = (int)pos64;
  const char* Kp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.Kp) + kvh * p.prefix_head_stride) + sub * 16;
  const char* Vp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.Vp) + kvh * p.prefix_head_stride) + sub * 16;
  const long long own_at = r * p.request_stride + kvh * p.head_stride;
  const char* Kc = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.Kc) + own_at) + sub * 16;
  const char* Vc = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.Vc) + own_at) + sub * 16;
  const int batches = (N + C::kRows - 1) / C::kRows, stride = cluster * kDirWarps;

  uint4 k[NL], v[NL];
  auto load = [&](int b, uint4 (&kk)[NL], uint4 (&vv)[NL]) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int j = b * C::kRows + i * RPL + grp;
      const bool own = j >= P;
      const long long at = (own ? (j - P) * p.row_stride : j * p.prefix_row_stride) * (long long)sizeof(T);
      kk[i] = vv[i] = make_uint4(0, 0, 0, 0);
      if (j < N) {
        kk[i] = ld_stream((own ? Kc : Kp) + at);
        vv[i] = ld_stream((own ? Vc : Vp) + at);
      }
    }
  };
  const int b0 = rank * kDirWarps + w;
  if (b0 < batches) load(b0, k, v);

  // q, and the new token's k and v
  for (int x = w; x < g + 2; x += kDirWarps) {
    if (x != w)
      raw[0].load(p.qkv, r * p.qkv_stride + (long long)(x < g ? kvh * g + x : x == g ? p.nq + kvh : p.nq + p.nkv + kvh) * HD,
                  p.qkv_bf16);
    float y[1][EL];
    if (x <= g) {
      const int ps[1] = {pos};
      norm_rotate_rows<HD, 1>(y, raw, p.qkv_bf16, ps, x < g ? p.qn : p.kn, p.rope, p.eps);
#pragma unroll
      for (int e = 0; e < EL; ++e) y[0][e] = x < g ? y[0][e] * p.q_scale : Pair<T>::rnd(y[0][e]);
      store_vec<EL>((x < g ? q_s[x] : kv_s[0]) + lane * EL, y[0]);
    } else {
      raw[0].values(p.qkv_bf16, y[0]);
#pragma unroll
      for (int e = 0; e < EL; ++e) y[0][e] = Pair<T>::rnd(y[0][e]);
      store_vec<EL>(kv_s[1] + lane * EL, y[0]);
    }
    if (rank == 0 && x >= g) {  // appended as own row n
      T* dst = reinterpret_cast<T*>(x == g ? p.Kc : p.Vc) + own_at + n * p.row_stride + lane * EL;
#pragma unroll
      for (int e = 0; e < EL; ++e) dst[e] = Pair<T>::st(y[0][e]);
    }
  }
  __syncthreads();

  float m[GP], l[VK] = {};
  float2 acc[GP][E / 2] = {};
#pragma unroll
  for (int h = 0; h < GP; ++h) m[h] = -INFINITY;
  float2 q[C::kAhead ? GP : 1][E / 2];
  if (C::kAhead) {
#pragma unroll
    for (int h = 0; h < GP; ++h)
#pragma unroll
      for (int e = 0; e < E / 2; ++e)
        q[C::kAhead ? h : 0][e] = h < g ? *reinterpret_cast<const float2*>(q_s[h] + sub * E + 2 * e) : make_float2(0.f, 0.f);
  }
  // value x = row slot * GP + head of a row group is kept by the lane (or the REP lanes) that sub / REP = x / VK
  const int x0 = sub / REP * VK;
  // the new token is the first partial of warp 0 of the cluster's first CTA, its weight 1 in the sum that
  // row slot 0 has for the head
  if (rank == 0 && w == 0) {
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      if (h >= g) break;
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < EL; ++e) d += q_s[h][lane * EL + e] * kv_s[0][lane * EL + e];
      m[h] = warp_sum32(d);
      if (lane == 0) snew_s[h] = m[h];
      if (grp == 0) {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) acc[h][e] = *reinterpret_cast<const float2*>(kv_s[1] + sub * E + 2 * e);
      }
    }
    if (grp == 0 && sub % REP == 0) {
#pragma unroll
      for (int c = 0; c < VK; ++c) l[c] = x0 + c < g ? 1.f : 0.f;
    }
  }

  for (int b = b0; b < batches; b += stride) {
    uint4 kn[NL], vn[NL];
    if (C::kAhead && b + stride < batches) load(b + stride, kn, vn);
    float s[NV];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        float2 d = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const float2 qq = C::kAhead ? q[C::kAhead ? h : 0][e] : *reinterpret_cast<const float2*>(q_s[h] + sub * E + 2 * e);
          d = __ffma2_rn(Pair<T>::get(k[i], e), qq, d);
        }
        s[i * GP + h] = d.x + d.y;
      }
    }
    {  // sum over the W lanes of a row, each sum left in one lane (or REP)
      int off = W / 2;
#pragma unroll
      for (int c = NV; c > VK; c >>= 1, off >>= 1) {
        const bool upper = sub & off;
#pragma unroll
        for (int i = 0; i < c / 2; ++i) {
          const float send = upper ? s[i] : s[i + c / 2], keep = upper ? s[i + c / 2] : s[i];
          s[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
        }
      }
#pragma unroll
      for (; off > 0; off >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
    }
    bool over = false;
    float mo[VK];
#pragma unroll
    for (int c = 0; c < VK; ++c) {
      const int x = x0 + c, h = x % GP, j = b * C::kRows + x / GP * RPL + grp;
      if (j >= N || h >= g) s[c] = -INFINITY;
      mo[c] = m[0];
#pragma unroll
      for (int y = 1; y < GP; ++y) mo[c] = y == h ? m[y] : mo[c];
      over |= s[c] > mo[c] + 8.0f;
      if (p.mass && j >= P && j < N && h < g && (REP == 1 || sub % REP == 0))
        p.sc[((long long)r * p.nq + kvh * g + h) * p.sc_stride + (j - P)] = s[c];
    }
    if (__any_sync(0xffffffffu, over)) {
      float a[GP];
#pragma unroll
      for (int y = 0; y < GP; ++y) {
        float t = -INFINITY;
#pragma unroll
        for (int c = 0; c < VK; ++c) t = (x0 + c) % GP == y ? fmaxf(t, s[c]) : t;
        t = fmaxf(m[y], redux_max(t));
        a[y] = t == -INFINITY ? 1.f : ex2_approx(m[y] - t);
        m[y] = t;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) acc[y][e] = __fmul2_rn(acc[y][e], make_float2(a[y], a[y]));
      }
#pragma unroll
      for (int c = 0; c < VK; ++c) {
        const int h = (x0 + c) % GP;
        float f = a[0];
        mo[c] = m[0];
#pragma unroll
        for (int y = 1; y < GP; ++y) f = y == h ? a[y] : f, mo[c] = y == h ? m[y] : mo[c];
        l[c] *= f;
      }
    }
#pragma unroll
    for (int c = 0; c < VK; ++c) {
      s[c] = ex2_approx(s[c] - (mo[c] == -INFINITY ? 0.f : mo[c]));
      l[c] += s[c];
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const int x = i * GP + h;
        const float pr = __shfl_sync(0xffffffffu, s[x % VK], (lane & ~(W - 1)) | (x / VK * REP));
        const float2 pp = make_float2(pr, pr);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) acc[h][e] = __ffma2_rn(Pair<T>::get(v[i], e), pp, acc[h][e]);
      }
    }
    if (C::kAhead) {
#pragma unroll
      for (int i = 0; i < NL; ++i) k[i] = kn[i], v[i] = vn[i];
    } else if (b + stride < batches) {
      load(b + stride, k, v);
    }
  }

  // the warp's partial: sums over its row groups and, of the weights, its lanes
#pragma unroll
  for (int h = 0; h < GP; ++h) {
    float t = 0.f;
#pragma unroll
    for (int c = 0; c < VK; ++c) t += (x0 + c) % GP == h && (REP == 1 || sub % REP == 0) ? l[c] : 0.f;
    t = warp_sum32(t);
#pragma unroll
    for (int e = 0; e < E / 2; ++e)
#pragma unroll
      for (int o = W; o < 32; o <<= 1) {
        acc[h][e].x += __shfl_xor_sync(0xffffffffu, acc[h][e].x, o);
        acc[h][e].y += __shfl_xor_sync(0xffffffffu, acc[h][e].y, o);
      }
    __syncwarp();
    if (lane == 0) ml_s[w][h] = make_float2(m[h], t);
    if (grp == 0) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) *reinterpret_cast<float2*>(red_s[w][h] + sub * E + 2 * e) = acc[h][e];
    }
  }
  __syncthreads();
  // the CTA's
  for (int x = threadIdx.x; x < g * HD; x += kDirThreads) {
    const int h = x / HD, d = x % HD;
    float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
    for (int y = 0; y < kDirWarps; ++y) M = fmaxf(M, ml_s[y][h].x);
#pragma unroll
    for (int y = 0; y < kDirWarps; ++y) {
      const float a = ex2_approx(ml_s[y][h].x - (M == -INFINITY ? 0.f : M));
      L += a * ml_s[y][h].y;
      o += a * red_s[y][h][d];
    }
    o_s[h][d] = o;
    if (d == 0) oml_s[h] = make_float2(M, L);
  }
  __syncthreads();
  if (cluster > 1) {
    cluster_arrive();
    cluster_wait();
  }
  // out: element x by CTA x % cluster ... each CTA a run of them
  const int total = g * HD, per = (total + cluster - 1) / cluster;
  for (int x = rank * per + threadIdx.x; x < min(total, (rank + 1) * per); x += kDirThreads) {
    const int h = x / HD, d = x % HD;
    float2 ml[kMaxCluster];
    float part[kMaxCluster];
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {  // all in flight at once
      ml[c] = make_float2(-INFINITY, 0.f);
      part[c] = 0.f;
      if (c < cluster) {
        ml[c] = make_float2(ld_remote(mapa(&oml_s[h].x, c)), ld_remote(mapa(&oml_s[h].y, c)));
        part[c] = ld_remote(mapa(&o_s[h][d], c));
      }
    }
    float M = ml[0].x, L = 0.f, o = 0.f;
#pragma unroll
    for (int c = 1; c < kMaxCluster; ++c) M = fmaxf(M, ml[c].x);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      const float a = c < cluster ? ex2_approx(ml[c].x - M) : 0.f;
      L += a * ml[c].y;
      o += a * part[c];
    }
    const long long at = r * p.out_stride + (long long)kvh * g * HD + x;
    if (p.out_bf16)
      reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o / L);
    else
      reinterpret_cast<float*>(p.out)[at] = o / L;
  }
  if (p.mass) {
    if (threadIdx.x < g) {
      const int h = threadIdx.x;
      float2 ml[kMaxCluster];
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        ml[c] = c < cluster ? make_float2(ld_remote(mapa(&oml_s[h].x, c)), ld_remote(mapa(&oml_s[h].y, c)))
                            : make_float2(-INFINITY, 0.f);
      float M = ml[0].x, L = 0.f;
#pragma unroll
      for (int c = 1; c < kMaxCluster; ++c) M = fmaxf(M, ml[c].x);
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) L += c < cluster ? ex2_approx(ml[c].x - M) * ml[c].y : 0.f;
      M_s[h] = M;
      iL_s[h] = 1.f / L;
    }
    __syncthreads();
    // the rows whose scores this CTA's warps have written
    float* mass = p.mass + r * p.mass_request_stride + kvh * p.mass_head_stride;
    const float* sc = p.sc + ((long long)r * p.nq + kvh * g) * p.sc_stride;
    for (int b = b0; b < batches; b += stride) {
      const int j = b * C::kRows + lane - P;
      if (lane < C::kRows && j >= 0 && j < n) {
        float a = 0.f;
        for (int h = 0; h < g; ++h) a += ex2_approx(__ldcg(sc + h * p.sc_stride + j) - M_s[h]) * iL_s[h];
        mass[j] += a;
      }
    }
    if (rank == 0 && threadIdx.x == 0) {
      float a = 0.f;
      for (int h = 0; h < g; ++h) a += ex2_approx(snew_s[h] - M_s[h]) * iL_s[h];
      mass[n] = a;
    }
  }
  if (cluster > 1) {  // no CTA leaves while another reads its partial
    cluster_arrive();
    cluster_wait();
  }
}

// ---- host -----------------------------------------------------------------------------------------
template <typename T, int HD, int GP>
static int launch(const Params& p, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.R * p.nkv * cluster));
  cfg.blockDim = dim3(kDirThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, direct_kernel<T, HD, GP>, p, cluster) == cudaSuccess ? SK_OK : SK_ERR_CUDA;
}
template <typename T, int HD>
static int launch_group(const Params& p, int cluster, cudaStream_t st) {
  if (p.g == 1) return launch<T, HD, 1>(p, cluster, st);
  if (p.g == 2) return launch<T, HD, 2>(p, cluster, st);
  if (p.g <= 4) return launch<T, HD, 4>(p, cluster, st);
  return launch<T, HD, 8>(p, cluster, st);
}

int launch_direct(const Params& p, int hd, int cache_dtype, cudaStream_t st) {
  // CTAs per (request, head): as many as keep the grid within two CTAs per SM and give every warp a batch
  const int rows = cache_dtype == SK_BF16 ? (hd == 128 ? 8 : 16) : (hd == 128 ? 4 : 8);
  int cluster = 1;
  while (cluster < kMaxCluster && (long long)p.R * p.nkv * cluster * 2 <= 296 &&
         (long long)(p.P + p.max_len) > (long long)cluster * kDirWarps * rows)
    cluster *= 2;
  if (cache_dtype == SK_BF16)
    return hd == 128 ? launch_group<__nv_bfloat16, 128>(p, cluster, st) : launch_group<__nv_bfloat16, 64>(p, cluster, st);
  return hd == 128 ? launch_group<float, 128>(p, cluster, st) : launch_group<float, 64>(p, cluster, st);
}

}  // namespace shared
}  // namespace sk

// Key/value caches brought down to a budget of rows by accumulated attention weight.
//
// Two kernels. `select`: one CTA per cache (layer, request, head) finds the smallest mass that still fits
// the budget by radix selection — 11, 11 and 10 bits of the order-preserving integer image of the float
// from the top, a histogram each, so three reads of the masses whatever the budget — and lists the kept
// rows in order, one pass that counts and one that writes. `move`: gathers the listed rows of K, V and mass.
//
// In place a kept row never moves up (its new index is at most its old one), so a CTA that owns a column
// slice of a cache can walk the list from the front in batches: a batch's rows are all in registers before
// any of them is written, and a later batch reads only rows past everything written so far. Slices are
// independent, which is where the parallelism comes from. Into another buffer whole rows are copied.
#include "sk_common.cuh"

namespace sk {
namespace evict {

struct Params {
  const uint8_t* K;
  const uint8_t* V;
  const float* mass;
  long long kv[4], ms[3];       // byte strides of K and V (layer, request, head, row); element strides of mass
  uint8_t* Ko;
  uint8_t* Vo;
  float* mo;
  long long kvo[4], mso[3];
  const long long* rows;
  long long* rows_out;
  int* cnt;                     // [R] rows read once (-1: idle), so that rows_out may be rows
  int* list;                    // [N * R * nkv][keep] kept rows in order
  int N, R, nkv, row_bytes, max_len, keep, first, recent;
  int* err;
};

__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Order-preserving image of a mass: a > b as numbers iff key(a) > key(b); NaN below everything, -0 = +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 + 0 = +0
  return (b >> 31) ? ~b : (b | 0x80000000u);
}

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32, kBins = 2048;

__global__ void __launch_bounds__(kSelThreads) select_kernel(const Params p) {
  __shared__ int hist[kBins];
  __shared__ int warp_tot[kSelWarps][2];
  __shared__ int found_bin, found_above;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int head = blockIdx.x, kvh = head % p.nkv, r = (head / p.nkv) % p.R, layer = head / (p.nkv * p.R);
  griddep_wait();
  griddep_launch_dependents();
  const long long n64 = p.rows[r];
  const int n = n64 < 0 || n64 > p.max_len ? -1 : (int)n64;
  if (t == 0 && kvh == 0 && layer == 0) {
    p.cnt[r] = n;
    if (n64 > p.max_len) set_dev_error(p.err, SK_DEVERR_POS_RANGE);
  }
  if (n <= p.keep) return;
  const float* mass = p.mass + layer * p.ms[0] + r * p.ms[1] + kvh * p.ms[2];
  const int a = p.first, z = n - p.recent;      // candidates [a, z)
  int need = p.keep - p.first - p.recent;       // of which this many stay (fewer than there are)

  uint32_t prefix = 0, known = 0;  // the threshold key's leading bits so far and which they are
  if (need > 0) {
    const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = t; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j = a + t; j < z; j += kSelThreads) {
        const uint32_t k = key_of(mass[j]);
        if ((k & known) == prefix) atomicAdd(&hist[(k >> shifts[pass]) & ((1u << widths[pass]) - 1)], 1);
      }
      __syncthreads();
      // the bin, from the top, in which the count reaches `need`: thread t sums bins 4t .. 4t+3 reversed
      constexpr int B = kBins / kSelThreads;
      int own[B], sum = 0;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        own[b] = hist[kBins - 1 - (t * B + b)];
        sum += own[b];
      }
      int x = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) warp_tot[w][0] = x;
      __syncthreads();
      int above = x - sum;
      for (int i = 0; i < w; ++i) above += warp_tot[i][0];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (above < need && above + own[b] >= need) {
          found_bin = kBins - 1 - (t * B + b);
          found_above = above;
        }
        above += own[b];
      }
      __syncthreads();
      need -= found_above;
      prefix |= (uint32_t)found_bin << shifts[pass];
      known |= ((1u << widths[pass]) - 1) << shifts[pass];
    }
  }
  // kept: first, recent, keys above the threshold `prefix`, and the first `need` of those equal to it.
  // Each warp takes a run of rows: count, add up the warps before, write.
  const bool none = p.keep == p.first + p.recent;
  const int run = ((n + kSelWarps - 1) / kSelWarps + 31) & ~31, j0 = w * run, j1 = min(n, j0 + run);
  int* list = p.list + (long long)head * p.keep;
  int sure = 0, ties = 0;
#pragma unroll 1
  for (int write = 0; write < 2; ++write) {
    for (int j = j0; j < j1; j += 32) {
      const int i = j + lane;
      const bool end = i < j1 && (i < a || i >= z);
      const uint32_t k = i < j1 && !end && !none ? key_of(mass[i]) : 0u;
      const bool mid = i < j1 && !end && !none;
      const bool s = end || (mid && k > prefix), e = mid && k == prefix;
      const uint32_t bs = __ballot_sync(0xffffffffu, s), be = __ballot_sync(0xffffffffu, e);
      if (write) {
        const uint32_t below = (1u << lane) - 1;
        const int eb = ties + __popc(be & below);
        if (s || (e && eb < need)) list[sure + __popc(bs & below) + min(eb, need)] = i;
      }
      sure += __popc(bs);
      ties += __popc(be);
    }
    if (write) break;
    if (lane == 0) {
      warp_tot[w][0] = sure;
      warp_tot[w][1] = ties;
    }
    __syncthreads();
    sure = ties = 0;
    for (int i = 0; i < w; ++i) {
      sure += warp_tot[i][0];
      ties += warp_tot[i][1];
    }
  }
}

constexpr int kMoveThreads = 256, kBatch = 8;

// In place: CTA (cache, K or V, column slice of SLICE bytes).
template <int SLICE>
__global__ void __launch_bounds__(kMoveThreads) move_in_place_kernel(const Params p) {
  constexpr int U = SLICE / 16, RPP = kMoveThreads / U;  // 16-byte units per row, rows per pass
  const int t = threadIdx.x, head = blockIdx.x;
  const int kvh = head % p.nkv, r = (head / p.nkv) % p.R, layer = head / (p.nkv * p.R);
  const int slices = p.row_bytes / SLICE, which = blockIdx.y / slices, slice = blockIdx.y % slices;
  griddep_wait();
  griddep_launch_dependents();
  const int n = p.cnt[r];
  if (t == 0 && blockIdx.y == 0 && kvh == 0 && layer == 0)
    p.rows_out[r] = n > p.keep ? (long long)p.keep : p.rows[r];
  if (n <= p.keep) return;
  const int* list = p.list + (long long)head * p.keep;
  uint8_t* base = (which ? p.Vo : p.Ko) + layer * p.kv[0] + r * p.kv[1] + kvh * p.kv[2] + slice * SLICE + (t % U) * 16;
  for (int d0 = 0; d0 < p.keep; d0 += RPP * kBatch) {
    uint4 v[kBatch];
    int src[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int d = d0 + i * RPP + t / U;
      src[i] = d < p.keep ? list[d] : d;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int d = d0 + i * RPP + t / U;
      if (src[i] != d) v[i] = *reinterpret_cast<const uint4*>(base + src[i] * p.kv[3]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int d = d0 + i * RPP + t / U;
      if (src[i] != d) *reinterpret_cast<uint4*>(base + d * p.kv[3]) = v[i];
    }
  }
  if (blockIdx.y != 0) return;
  float* mass = p.mo + layer * p.ms[0] + r * p.ms[1] + kvh * p.ms[2];
  for (int d0 = 0; d0 < p.keep; d0 += kMoveThreads * kBatch) {
    float v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int d = d0 + i * kMoveThreads + t;
      v[i] = d < p.keep ? mass[list[d]] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int d = d0 + i * kMoveThreads + t;
      if (d < p.keep) mass[d] = v[i];
    }
  }
}

// Into another buffer: CTA (cache, K or V, chunk of kCopyRows rows), whole rows.
constexpr int kCopyRows = 128;

__global__ void __launch_bounds__(kMoveThreads) move_copy_kernel(const Params p) {
  const int t = threadIdx.x, head = blockIdx.x;
  const int kvh = head % p.nkv, r = (head / p.nkv) % p.R, layer = head / (p.nkv * p.R);
  const int which = blockIdx.y & 1, d0 = (int)(blockIdx.y >> 1) * kCopyRows;
  griddep_wait();
  griddep_launch_dependents();
  const int n = p.cnt[r];
  if (t == 0 && blockIdx.y == 0 && kvh == 0 && layer == 0)
    p.rows_out[r] = n > p.keep ? (long long)p.keep : p.rows[r];
  const int m = min(n, p.keep), d1 = min(m, d0 + kCopyRows);
  if (d0 >= m) return;
  const bool all = n <= p.keep;
  const int* list = p.list + (long long)head * p.keep;
  const int U = p.row_bytes / 16;
  const uint8_t* src = (which ? p.V : p.K) + layer * p.kv[0] + r * p.kv[1] + kvh * p.kv[2];
  uint8_t* dst = (which ? p.Vo : p.Ko) + layer * p.kvo[0] + r * p.kvo[1] + kvh * p.kvo[2];
  for (int i0 = 0; i0 < (d1 - d0) * U; i0 += kMoveThreads * kBatch) {
    uint4 v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kMoveThreads + t, d = d0 + i / U;
      if (d < d1) v[b] = __ldcs(reinterpret_cast<const uint4*>(src + (all ? d : list[d]) * p.kv[3] + (i % U) * 16));
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kMoveThreads + t, d = d0 + i / U;
      if (d < d1) *reinterpret_cast<uint4*>(dst + d * p.kvo[3] + (i % U) * 16) = v[b];
    }
  }
  if (which == 0)
    for (int d = d0 + t; d < d1; d += kMoveThreads)
      p.mo[layer * p.mso[0] + r * p.mso[1] + kvh * p.mso[2] + d] =
          p.mass[layer * p.ms[0] + r * p.ms[1] + kvh * p.ms[2] + (all ? d : list[d])];
}

static int check_sizes(const SkCacheEvict* d) {
  if (!d) return SK_ERR_INVALID_ARG;
  if (d->cache_dtype != SK_BF16 && d->cache_dtype != SK_F32) return SK_ERR_UNSUPPORTED;
  if (d->hd != 64 && d->hd != 128) return SK_ERR_UNSUPPORTED;
  if (d->N < 1 || d->R < 1 || d->nkv < 1 || d->max_len < 1 || d->max_len_out < 1) return SK_ERR_INVALID_ARG;
  if (d->keep < 1 || d->keep > d->max_len || d->keep > d->max_len_out || d->first < 0 || d->recent < 0 ||
      (long long)d->first + d->recent > d->keep)
    return SK_ERR_INVALID_ARG;
  if ((long long)d->N * d->R * d->nkv > 0x7fffffffLL || d->max_len > (1 << 21)) return SK_ERR_UNSUPPORTED;
  return SK_OK;
}
// The address range of a buffer of these extents and strides (bytes).
struct Range {
  uintptr_t lo, hi;
};
static Range range_of(const void* p, const SkCacheEvict* d, int max_len, const long long* stride, int esz, int row) {
  long long last = 0;
  const int extent[3] = {d->N, d->R, d->nkv};
  for (int i = 0; i < 3; ++i) last += (extent[i] - 1) * stride[i];
  last += (max_len - 1) * (row > 4 ? stride[3] : 1);
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return {a, a + (uintptr_t)(last * esz + row)};
}
static long long cnt_bytes(const SkCacheEvict* d) { return ((long long)d->R * 4 + 255) / 256 * 256; }

}  // namespace evict
}  // namespace sk

extern "C" size_t sk_cache_evict_workspace_bytes(const SkCacheEvict* d) {
  using namespace sk::evict;
  if (check_sizes(d) != SK_OK) return 0;
  return (size_t)(cnt_bytes(d) + (long long)d->N * d->R * d->nkv * d->keep * 4);
}

extern "C" int sk_cache_evict(const SkCacheEvict* d, void* stream) {
  using namespace sk::evict;
  const int rc = check_sizes(d);
  if (rc != SK_OK) return rc;
  if (!d->K || !d->V || !d->mass || !d->K_out || !d->V_out || !d->mass_out || !d->rows || !d->rows_out)
    return SK_ERR_INVALID_ARG;
  const int esz = d->cache_dtype == SK_BF16 ? 2 : 4, per16 = 16 / esz;
  const uintptr_t all = reinterpret_cast<uintptr_t>(d->K) | reinterpret_cast<uintptr_t>(d->V) |
                        reinterpret_cast<uintptr_t>(d->K_out) | reinterpret_cast<uintptr_t>(d->V_out);
  if (all & 15) return SK_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(d->mass) | reinterpret_cast<uintptr_t>(d->mass_out)) & 3) return SK_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(d->rows) | reinterpret_cast<uintptr_t>(d->rows_out)) & 7) return SK_ERR_INVALID_ARG;
  const int extent[4] = {d->N, d->R, d->nkv, d->max_len};
  bool same = true;
  for (int i = 0; i < 4; ++i) {
    if (extent[i] == 1) continue;
    if (d->kv_stride[i] < d->hd || d->kv_stride[i] % per16 || d->kv_out_stride[i] < d->hd || d->kv_out_stride[i] % per16)
      return SK_ERR_INVALID_ARG;
    if (i < 3 && (d->mass_stride[i] < 1 || d->mass_out_stride[i] < 1)) return SK_ERR_INVALID_ARG;
    same = same && d->kv_stride[i] == d->kv_out_stride[i] && (i == 3 || d->mass_stride[i] == d->mass_out_stride[i]);
  }
  const bool in_place = d->K == d->K_out;
  // in place: all three the source itself, laid out alike
  if (in_place != (d->V == d->V_out) || in_place != (d->mass == d->mass_out) || (in_place && !same))
    return SK_ERR_INVALID_ARG;
  if (!in_place) {
    const int row = d->hd * esz;
    const Range from[3] = {range_of(d->K, d, d->max_len, d->kv_stride, esz, row),
                           range_of(d->V, d, d->max_len, d->kv_stride, esz, row),
                           range_of(d->mass, d, d->max_len, d->mass_stride, 4, 4)};
    const Range to[3] = {range_of(d->K_out, d, d->max_len_out, d->kv_out_stride, esz, row),
                         range_of(d->V_out, d, d->max_len_out, d->kv_out_stride, esz, row),
                         range_of(d->mass_out, d, d->max_len_out, d->mass_out_stride, 4, 4)};
    for (const Range& a : from)
      for (const Range& b : to)
        if (a.lo < b.hi && b.lo < a.hi) return SK_ERR_INVALID_ARG;
  }
  if (!d->workspace || (reinterpret_cast<uintptr_t>(d->workspace) & 255) ||
      d->ws_bytes < sk_cache_evict_workspace_bytes(d))
    return SK_ERR_WORKSPACE;
  const int dev = sk_check_device();
  if (dev != SK_OK) return dev;

  Params p = {};
  p.K = reinterpret_cast<const uint8_t*>(d->K), p.V = reinterpret_cast<const uint8_t*>(d->V), p.mass = d->mass;
  p.Ko = reinterpret_cast<uint8_t*>(d->K_out), p.Vo = reinterpret_cast<uint8_t*>(d->V_out), p.mo = d->mass_out;
  for (int i = 0; i < 4; ++i) p.kv[i] = d->kv_stride[i] * esz, p.kvo[i] = d->kv_out_stride[i] * esz;
  for (int i = 0; i < 3; ++i) p.ms[i] = d->mass_stride[i], p.mso[i] = d->mass_out_stride[i];
  p.rows = d->rows, p.rows_out = d->rows_out;
  p.cnt = reinterpret_cast<int*>(d->workspace);
  p.list = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(d->workspace) + cnt_bytes(d));
  p.N = d->N, p.R = d->R, p.nkv = d->nkv, p.row_bytes = d->hd * esz, p.max_len = d->max_len;
  p.keep = d->keep, p.first = d->first, p.recent = d->recent;
  p.err = sk_error_word_ptr();
  if (!p.err) return SK_ERR_CUDA;
  const unsigned heads = (unsigned)(d->N * d->R * d->nkv);

  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.gridDim = dim3(heads);
  cfg.blockDim = dim3(kSelThreads);
  if (cudaLaunchKernelEx(&cfg, select_kernel, p) != cudaSuccess) return SK_ERR_CUDA;
  cfg.blockDim = dim3(kMoveThreads);
  constexpr int kSlice = 64;
  if (in_place) {
    cfg.gridDim = dim3(heads, (unsigned)(2 * (p.row_bytes / kSlice)));
    return cudaLaunchKernelEx(&cfg, move_in_place_kernel<kSlice>, p) == cudaSuccess ? SK_OK : SK_ERR_CUDA;
  }
  cfg.gridDim = dim3(heads, (unsigned)(2 * ((d->keep + kCopyRows - 1) / kCopyRows)));
  return cudaLaunchKernelEx(&cfg, move_copy_kernel, p) == cudaSuccess ? SK_OK : SK_ERR_CUDA;
}

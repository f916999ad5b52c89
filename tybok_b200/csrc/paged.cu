// The paged cache of keys and values: which pages a step takes (page_plan), and what goes into them (head_norm_rope_store).
//
// A cache is a pool of pages [P][G][page][D] (any strides); request b's key j lies in page table[b][j / page] at row
// j % page, so requests of different lengths share one pool and nothing is padded to the longest.  A slot is
// page number * page size + row.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/tybok_b200.h"
#include "host_util.h"
#include "ptx.cuh"

namespace tb {

// ------------------------------------------------------------------------------------------------ page plan
// With held = ceil(len / page), a finished request's pages go back (its row starts anew at length 0), and a request that grows to
// total = len + new takes ceil(total / page) - held pages.  Both are prefix sums over the requests: the i-th page that
// comes back lies at free[count + i] of the stack, the i-th that is taken comes from free[count + R - 1 - i] (R pages came back).
// Every CTA makes the sums itself (a few thousand lengths out of L2), so CTAs share nothing: functional calls spread over as
// many as the copies and tokens need, without a barrier; calls in place run as one cluster that meets once, between
// reading the old state and writing the new.
// Bound by latency: the launch, the lengths, the scan, one table entry, the stores.
struct PlanParams {
  const int* lens;
  const int* fresh;           // new tokens per request
  const uint8_t* finished;    // or NULL
  const int* table;
  const int* stack;
  const int* count;
  int *table_out, *stack_out, *count_out, *lens_out;
  int *cu, *pos, *slots, *missing;
  int B, W, P, T, page_shift, in_place, pdl;
};

constexpr int PLAN_MAX_REQUESTS = 8192;

// Largest i in [0, n) with start[i] <= x, for start[0] = 0 <= x < start[n].
__device__ __forceinline__ int plan_find(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ long long plan_pages(long long tokens, int shift) { return (tokens + (1ll << shift) - 1) >> shift; }

__global__ void __launch_bounds__(1024) page_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  __shared__ long long warp_sum[3][32];
  __shared__ int bad_any;
  int* back = plan_smem;             // [B + 1] pages that came back before request b
  int* more = back + p.B + 1;        // [B + 1] pages taken before request b
  int* cu = more + p.B + 1;          // [B + 1] tokens before request b
  int* base = cu + p.B + 1;          // [B] length that the new tokens follow
  const int tid = threadIdx.x, n = blockDim.x, lane = tid & 31, warp = tid >> 5;
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  if (tid == 0) bad_any = 0;
  __syncthreads();
  const int count = *p.count;
  // sums of each thread's requests, then over the threads; 64 bits, so that no length overflows them before it is refused
  const int per = (p.B + n - 1) / n, b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  long long sb = 0, sm = 0, sn = 0;
  bool bad = count < 0 || count > p.P;
  for (int b = b0; b < b1; ++b) {
    const long long len = p.lens[b], add = p.fresh[b];
    const bool gone = p.finished && p.finished[b];
    const long long held = plan_pages(len, p.page_shift), need = plan_pages((gone ? 0 : len) + add, p.page_shift);
    bad = bad || len < 0 || add < 0 || held > p.W || need > p.W;
    back[b] = static_cast<int>(gone ? held : 0);
    more[b] = static_cast<int>(need - (gone ? 0 : held));
    cu[b] = static_cast<int>(add);
    base[b] = static_cast<int>(gone ? 0 : len);
    sb += gone ? held : 0;
    sm += need - (gone ? 0 : held);
    sn += add;
  }
  long long xb = sb, xm = sm, xn = sn;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long tb_ = __shfl_up_sync(0xffffffffu, xb, o), tm = __shfl_up_sync(0xffffffffu, xm, o), tn = __shfl_up_sync(0xffffffffu, xn, o);
    if (lane >= o) {
      xb += tb_;
      xm += tm;
      xn += tn;
    }
  }
  if (lane == 31) {
    warp_sum[0][warp] = xb;
    warp_sum[1][warp] = xm;
    warp_sum[2][warp] = xn;
  }
  if (bad) bad_any = 1;
  __syncthreads();
  long long ob = 0, om = 0, on = 0, R = 0, N = 0, tokens = 0;
  for (int w = 0; w < (n >> 5); ++w) {
    if (w == warp) {
      ob = R;
      om = N;
      on = tokens;
    }
    R += warp_sum[0][w];
    N += warp_sum[1][w];
    tokens += warp_sum[2][w];
  }
  const bool refused = bad_any || tokens > p.T || count + R > p.P;
  const int missing = refused ? -1 : static_cast<int>(max(0ll, N - count - R));
  const bool ok = missing == 0;
  ob += xb - sb;
  om += xm - sm;
  on += xn - sn;
  for (int b = b0; b < b1; ++b) {
    const int vb = back[b], vm = more[b], vn = cu[b];
    back[b] = static_cast<int>(ob);
    more[b] = static_cast<int>(om);
    cu[b] = static_cast<int>(on);
    ob += vb;
    om += vm;
    on += vn;
  }
  if (tid == 0) {
    back[p.B] = static_cast<int>(R);
    more[p.B] = static_cast<int>(N);
    cu[p.B] = static_cast<int>(tokens);
  }
  __syncthreads();

  const int g0 = blockIdx.x * n + tid, gn = gridDim.x * n;
  const int nback = ok ? static_cast<int>(R) : 0, nmore = ok ? static_cast<int>(N) : 0;
  auto back_page = [&](int i) {  // the i-th page that comes back
    const int b = plan_find(back, p.B, i);
    return p.table[static_cast<long long>(b) * p.W + i - back[b]];
  };
  if (p.in_place) {
    for (int i = g0; i < nback; i += gn) p.stack_out[count + i] = back_page(i);
    __syncthreads();
    cluster_sync_all();  // the old state has been read, the stack is whole
  } else {
    for (int i = g0; i < p.P; i += gn) p.stack_out[i] = i >= count && i < count + nback ? back_page(i - count) : p.stack[i];
    for (long long i = g0; i < static_cast<long long>(p.B) * p.W; i += gn) {
      const int b = static_cast<int>(i / p.W), j = static_cast<int>(i - static_cast<long long>(b) * p.W);
      const int keep = static_cast<int>(plan_pages(base[b], p.page_shift));
      if (!ok || j < keep || j >= keep + more[b + 1] - more[b]) p.table_out[i] = p.table[i];
    }
  }
  auto taken = [&](int x) {  // the x-th page that is taken
    const int i = count + nback - 1 - x;
    if (p.in_place) return __ldcg(p.stack_out + i);
    return i < count ? p.stack[i] : back_page(i - count);
  };
  for (int x = g0; x < nmore; x += gn) {
    const int b = plan_find(more, p.B, x);
    p.table_out[static_cast<long long>(b) * p.W + plan_pages(base[b], p.page_shift) + x - more[b]] = taken(x);
  }
  const int page = 1 << p.page_shift, real = ok ? cu[p.B] : 0;
  for (int t = g0; t < p.T; t += gn) {
    int at = 0, slot = -1;
    if (t < real) {
      const int b = plan_find(cu, p.B, t);
      at = base[b] + t - cu[b];
      const int j = at >> p.page_shift, keep = static_cast<int>(plan_pages(base[b], p.page_shift));
      const int number = j < keep ? p.table[static_cast<long long>(b) * p.W + j] : taken(more[b] + j - keep);
      slot = number * page + (at & (page - 1));
    }
    p.pos[t] = at;
    p.slots[t] = slot;
  }
  for (int b = g0; b <= p.B; b += gn) p.cu[b] = ok ? cu[b] : 0;
  for (int b = g0; b < p.B; b += gn) {
    if (ok) p.lens_out[b] = base[b] + cu[b + 1] - cu[b];
    else if (!p.in_place) p.lens_out[b] = p.lens[b];
  }
  if (g0 == 0) {
    *p.count_out = count + nback - nmore;
    *p.missing = missing;
  }
}

// ------------------------------------------------------------------------------------- head norms, rotation, store
// Per token and head of a packed projection row [q heads | k heads | v heads]:
//   y = x / sqrt(mean(x^2) + eps) * w  (q and k; fp32 over the head's D channels, each with its own weight or none),
//   (a, b) -> (a cos - b sin, b cos + a sin) for the rotated pairs, i and i + R / 2, or 2i and 2i + 1 (paired), of the
//   first R channels, angles by position from a table; one rounding to bf16 at the end.
// q goes to rows [T][H*D], k and the untouched v to their slots; a row without a slot (negative) stores neither.
// D / 8 lanes hold a head, eight channels each; the partners of the half-way rotation lie D / 16 lanes away (R = D) and come by
// shuffle before the norm, whose factor the whole head shares.  A warp takes four such loads at once.
// Bound by memory: every byte is read once and written once.
struct HeadNormParams {
  const __nv_bfloat16* src;
  long long ld;
  const int* pos;
  const int* slots;
  const float* cos;  // [max_pos][R / 2]
  const float* sin;
  const float* wq;   // [D] or NULL
  const float* wk;
  __nv_bfloat16* q_out;
  __nv_bfloat16* kp;
  __nv_bfloat16* vp;
  long long k_page, k_head, k_row, v_page, v_head, v_row;  // strides in elements
  int T, H, G, rot, max_pos, page_shift, num_slots, paired;
  float eps;
  int* status;
  int pdl;
};
constexpr int HN_THREADS = 128;
constexpr int HN_LOADS = 4;

__device__ __forceinline__ void hn_unpack(const uint4& v, float (&x)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __bfloat1622float2(h[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}

template <int D>
__global__ void __launch_bounds__(HN_THREADS) head_norm_rope_store_kernel(const HeadNormParams p) {
  constexpr int TEAM = D / 8, PER_LOAD = 32 / TEAM, HEADS = PER_LOAD * HN_LOADS;  // heads of a warp
  const int lane = threadIdx.x & 31, l = lane % TEAM, sub = lane / TEAM;
  const int all = p.H + 2 * p.G, chunks = (all + HEADS - 1) / HEADS;
  const long long w = (static_cast<long long>(blockIdx.x) * HN_THREADS + threadIdx.x) >> 5;
  const long long t = w / chunks;
  const int h0 = static_cast<int>(w - t * chunks) * HEADS + sub;
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  if (t >= p.T) return;
  const __nv_bfloat16* row = p.src + t * p.ld + l * 8;
  uint4 raw[HN_LOADS];
#pragma unroll
  for (int i = 0; i < HN_LOADS; ++i) {
    const int h = h0 + i * PER_LOAD;
    raw[i] = h < all ? *reinterpret_cast<const uint4*>(row + static_cast<long long>(h) * D) : uint4{};
  }
  const int pos = p.pos[t], slot = p.slots[t];
  const bool pos_ok = pos >= 0 && pos < p.max_pos, stored = slot >= 0 && slot < p.num_slots;
  if (lane == 0 && (!pos_ok || slot >= p.num_slots) && p.status) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
  // this lane's angles: of its eight channels' pairs (the same for every head of the token)
  const int c0 = l * 8, half = p.rot >> 1;
  const bool turned = c0 < p.rot, first = c0 < half;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (turned && pos_ok) {
    const long long at = static_cast<long long>(pos) * half;
    if (p.paired) {
      const float4 c = *reinterpret_cast<const float4*>(p.cos + at + (c0 >> 1)), s = *reinterpret_cast<const float4*>(p.sin + at + (c0 >> 1));
      const float c4[4] = {c.x, c.y, c.z, c.w}, s4[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = c4[e >> 1];
        sn[e] = (e & 1) ? s4[e >> 1] : -s4[e >> 1];
      }
    } else {
      const int i0 = first ? c0 : c0 - half;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 c = reinterpret_cast<const float4*>(p.cos + at + i0)[j], s = reinterpret_cast<const float4*>(p.sin + at + i0)[j];
        const float c4[4] = {c.x, c.y, c.z, c.w}, s4[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cs[4 * j + e] = c4[e];
          sn[4 * j + e] = first ? -s4[e] : s4[e];
        }
      }
    }
  }
  const int away = p.paired || !turned ? 0 : first ? (half >> 3) : -(half >> 3);  // lanes to the partner
  const long long page = stored ? slot >> p.page_shift : 0, off = stored ? slot & ((1 << p.page_shift) - 1) : 0;
#pragma unroll
  for (int i = 0; i < HN_LOADS; ++i) {
    const int h = h0 + i * PER_LOAD;
    const bool is_q = h < p.H, is_k = h >= p.H && h < p.H + p.G;
    uint4 other;
    other.x = __shfl_sync(0xffffffffu, raw[i].x, lane + away);
    other.y = __shfl_sync(0xffffffffu, raw[i].y, lane + away);
    other.z = __shfl_sync(0xffffffffu, raw[i].z, lane + away);
    other.w = __shfl_sync(0xffffffffu, raw[i].w, lane + away);
    float x[8], y[8];
    hn_unpack(raw[i], x);
    hn_unpack(other, y);
    const float* weight = is_q ? p.wq : p.wk;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (is_q || is_k) {
      if (weight) {
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 a = reinterpret_cast<const float4*>(weight + c0)[j], b = reinterpret_cast<const float4*>(weight + c0 + away * 8)[j];
          const float a4[4] = {a.x, a.y, a.z, a.w}, b4[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[4 * j + e] = x[4 * j + e] * r * a4[e];
            y[4 * j + e] = y[4 * j + e] * r * b4[e];
          }
        }
      }
      uint4 packed;
      __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&packed);
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = turned ? x[e] * cs[e] + (p.paired ? x[e ^ 1] : y[e]) * sn[e] : x[e];
#pragma unroll
      for (int j = 0; j < 4; ++j) o2[j] = __floats2bfloat162_rn(z[2 * j], z[2 * j + 1]);
      if (is_q) *reinterpret_cast<uint4*>(p.q_out + (t * p.H + h) * D + c0) = pos_ok ? packed : uint4{};
      else if (stored && pos_ok) *reinterpret_cast<uint4*>(p.kp + page * p.k_page + (h - p.H) * p.k_head + off * p.k_row + c0) = packed;
    } else if (h < all && stored && pos_ok) {
      *reinterpret_cast<uint4*>(p.vp + page * p.v_page + (h - p.H - p.G) * p.v_head + off * p.v_row + c0) = raw[i];
    }
  }
}

static int page_shift_of(int page) {
  if (page < 16 || (page & (page - 1))) return -1;
  int s = 4;
  while ((1 << s) != page) ++s;
  return s;
}

}  // namespace tb

extern "C" {

int tybok_page_plan(const int* key_lens, const int* new_lens, const void* finished, const int* block_table, const int* free_pages,
                    const int* free_count, int* key_lens_out, int* block_table_out, int* free_pages_out, int* free_count_out,
                    int* cu_tokens, int* pos, int* slots, int* missing, int B, int table_width, int num_pages, int tokens,
                    int page_size, void* stream) {
  using namespace tb;
  if (!key_lens || !new_lens || !block_table || !free_pages || !free_count || !key_lens_out || !block_table_out || !free_pages_out ||
      !free_count_out || !cu_tokens || !missing || (tokens > 0 && (!pos || !slots)))
    return host::fail(TYBOK_ERR_ARG, "page_plan: null pointer argument");
  const int shift = page_shift_of(page_size);
  if (shift < 0) return host::fail(TYBOK_ERR_ARG, "page_plan: the page size must be a power of two, 16 at least");
  if (B <= 0 || B > PLAN_MAX_REQUESTS || table_width <= 0 || num_pages <= 0 || tokens < 0)
    return host::fail(TYBOK_ERR_ARG, "page_plan: bad shape (1 to 8192 requests, table and pool not empty)");
  if (static_cast<long long>(num_pages) << shift > 0x7fffffffll) return host::fail(TYBOK_ERR_ARG, "page_plan: slots must fit 31 bits");
  const int same = (key_lens == key_lens_out) + (block_table == block_table_out) + (free_pages == free_pages_out) + (free_count == free_count_out);
  if (same != 0 && same != 4) return host::fail(TYBOK_ERR_ARG, "page_plan: the state is updated in place as a whole or not at all");
  if (int rc = host::require_sm100()) return rc;
  PlanParams p{};
  p.lens = key_lens; p.fresh = new_lens; p.finished = static_cast<const uint8_t*>(finished);
  p.table = block_table; p.stack = free_pages; p.count = free_count;
  p.lens_out = key_lens_out; p.table_out = block_table_out; p.stack_out = free_pages_out; p.count_out = free_count_out;
  p.cu = cu_tokens; p.pos = pos; p.slots = slots; p.missing = missing;
  p.B = B; p.W = table_width; p.P = num_pages; p.T = tokens; p.page_shift = shift; p.in_place = same == 4;
  p.pdl = host::pdl_enabled() ? 1 : 0;
  // entries to copy and write; each CTA pays the whole scan, so one has a few thousand of them at least
  const long long work = tokens + (p.in_place ? 0ll : num_pages + static_cast<long long>(B) * table_width);
  const int most = p.in_place ? 8 : host::sm_count();
  const int ctas = static_cast<int>(std::min<long long>(most, std::max<long long>(1, work / 4096)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.in_place && ctas > 1 ? 8 : ctas);
  cfg.blockDim = dim3(B <= 256 && work <= 4096 ? 256 : 1024);
  cfg.dynamicSmemBytes = sizeof(int) * (4 * static_cast<size_t>(B) + 3);
  cfg.stream = static_cast<cudaStream_t>(stream);
  static host::DeviceCache ready;
  const int set = host::per_device(ready, [] {
    return cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(sizeof(int) * (4 * PLAN_MAX_REQUESTS + 3))) == cudaSuccess ? 1 : 0;
  });
  if (!set) return host::fail_cuda("page_plan: shared memory");
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (p.pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.in_place) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = cfg.gridDim.x;
    attr[na].val.clusterDim.y = 1;
    attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  if (cudaLaunchKernelEx(&cfg, page_plan_kernel, p) != cudaSuccess) return host::fail_cuda("launch page_plan_kernel");
  host::count_launch();
  return TYBOK_OK;
}

int tybok_head_norm_rope_store(const void* src, int64_t ld, const int* pos, const int* slots, const float* cos_table,
                               const float* sin_table, int max_pos, int rot, int paired, const float* norm_q, const float* norm_k,
                               float eps, void* q_out, void* k_pages, const int64_t* k_strides, void* v_pages,
                               const int64_t* v_strides, int tokens, int H, int G, int D, int num_pages, int page_size,
                               int* status_word, void* stream) {
  using namespace tb;
  if (!src || !pos || !slots || !cos_table || !sin_table || !q_out || !k_pages || !v_pages || !k_strides || !v_strides)
    return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: null pointer argument");
  const int shift = page_shift_of(page_size);
  if (shift < 0) return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: the page size must be a power of two, 16 at least");
  if (D != 128 && D != 256) return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: head_dim must be 128 or 256");
  if (tokens <= 0 || H <= 0 || G <= 0 || num_pages <= 0 || max_pos <= 0 || rot <= 0 || rot > D || rot % 16 != 0)
    return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: bad shape (rotated channels: a multiple of 16, at most head_dim)");
  if (static_cast<long long>(num_pages) << shift > 0x7fffffffll) return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: slots must fit 31 bits");
  uintptr_t bits = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_pages) |
                   reinterpret_cast<uintptr_t>(v_pages) | reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table) |
                   reinterpret_cast<uintptr_t>(norm_q) | reinterpret_cast<uintptr_t>(norm_k);
  int64_t strides = ld;
  for (int i = 0; i < 3; ++i) strides |= k_strides[i] | v_strides[i];
  if ((bits & 15) || (strides & 7))
    return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: tensors must be 16-byte aligned, strides multiples of 8 elements");
  if (int rc = host::require_sm100()) return rc;
  HeadNormParams p{};
  p.src = static_cast<const __nv_bfloat16*>(src); p.ld = ld; p.pos = pos; p.slots = slots; p.cos = cos_table; p.sin = sin_table;
  p.wq = norm_q; p.wk = norm_k; p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.kp = static_cast<__nv_bfloat16*>(k_pages); p.vp = static_cast<__nv_bfloat16*>(v_pages);
  p.k_page = k_strides[0]; p.k_head = k_strides[1]; p.k_row = k_strides[2];
  p.v_page = v_strides[0]; p.v_head = v_strides[1]; p.v_row = v_strides[2];
  p.T = tokens; p.H = H; p.G = G; p.rot = rot; p.max_pos = max_pos; p.page_shift = shift; p.num_slots = num_pages << shift;
  p.paired = paired; p.eps = eps; p.status = status_word;
  p.pdl = host::pdl_enabled() ? 1 : 0;
  const int heads = 32 / (D / 8) * HN_LOADS, chunks = (H + 2 * G + heads - 1) / heads;
  const long long ctas = (static_cast<long long>(tokens) * chunks * 32 + HN_THREADS - 1) / HN_THREADS;
  if (ctas > 0x7fffffffll) return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: too many tokens for one launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(HN_THREADS);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl;
  if (cudaLaunchKernelEx(&cfg, D == 256 ? head_norm_rope_store_kernel<256> : head_norm_rope_store_kernel<128>, p) != cudaSuccess)
    return host::fail_cuda("launch head_norm_rope_store_kernel");
  host::count_launch();
  return TYBOK_OK;
}
}

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
// Bound by latency: the launch, the lengths, the scan, one table entry, the stores.  In a graph: 48 requests with a token each 3.8 us, 7 prompts
// 2.95, 2048 requests with 45,000 tokens 6.0 (2.5 MB).
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

__device__ __forceinline__ int plan_pages(long long tokens, int shift) { return static_cast<int>((tokens + (1ll << shift) - 1) >> shift); }

template <class T>
__device__ __forceinline__ T plan_scan(T x) {  // inclusive sums over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) >= o) x += y;
  }
  return x;
}

__global__ void __launch_bounds__(1024) page_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  __shared__ int sum_back[32], sum_more[32];
  __shared__ long long sum_new[32];
  int* back = plan_smem;             // [B + 1] pages that came back before request b
  int* more = back + p.B + 1;        // [B + 1] pages taken before request b
  int* cu = more + p.B + 1;          // [B + 1] tokens before request b
  int* base = cu + p.B + 1;          // [B] length that the new tokens follow
  const int tid = threadIdx.x, n = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = n >> 5;
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  const int count = *p.count;
  // Sums of each thread's requests, then over the threads.  Pages fit 31 bits (a request has at most a row of the table, or is
  // refused); tokens are summed in 64, so that no length overflows them before it is refused.
  const int per = (p.B + n - 1) / n, b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  int sb = 0, sm = 0;
  long long sn = 0;
  bool bad = count < 0 || count > p.P;
  for (int b = b0; b < b1; ++b) {
    const int len = p.lens[b], add = p.fresh[b];
    const bool gone = p.finished && p.finished[b];
    const int held = plan_pages(max(len, 0), p.page_shift), after = gone ? 0 : max(len, 0), kept = gone ? 0 : held;
    const int need = plan_pages(static_cast<long long>(after) + max(add, 0), p.page_shift);
    const bool out = len < 0 || add < 0 || held > p.W || need > p.W || static_cast<long long>(after) + max(add, 0) > 0x7fffffffll;
    bad = bad || out;
    back[b] = out ? 0 : held - kept;
    more[b] = out ? 0 : need - kept;
    cu[b] = out ? 0 : add;
    base[b] = after;
    sb += back[b];
    sm += more[b];
    sn += cu[b];
  }
  const int xb = plan_scan(sb), xm = plan_scan(sm);
  const long long xn = plan_scan(sn);
  if (lane == 31) {
    sum_back[warp] = xb;
    sum_more[warp] = xm;
    sum_new[warp] = xn;
  }
  bad = __syncthreads_or(bad);
  // every warp sums the warps
  const int wb = plan_scan(lane < warps ? sum_back[lane] : 0), wm = plan_scan(lane < warps ? sum_more[lane] : 0);
  const long long wn = plan_scan(lane < warps ? sum_new[lane] : 0ll);
  const int R = __shfl_sync(0xffffffffu, wb, 31), N = __shfl_sync(0xffffffffu, wm, 31);
  const long long tokens = __shfl_sync(0xffffffffu, wn, 31);
  const int before = max(warp - 1, 0);
  int ob = __shfl_sync(0xffffffffu, wb, before), om = __shfl_sync(0xffffffffu, wm, before);
  long long on = __shfl_sync(0xffffffffu, wn, before);
  if (warp == 0) ob = om = 0, on = 0;
  const bool refused = bad || tokens > p.T || R > p.P - count;
  const int missing = refused ? -1 : static_cast<int>(max(0ll, static_cast<long long>(N) - count - R));
  const bool ok = missing == 0;
  ob += xb - sb;
  om += xm - sm;
  on += xn - sn;
  for (int b = b0; b < b1; ++b) {
    const int vb = back[b], vm = more[b], vn = cu[b];
    back[b] = ob;
    more[b] = om;
    cu[b] = static_cast<int>(on);
    ob += vb;
    om += vm;
    on += vn;
  }
  if (tid == 0) {
    back[p.B] = R;
    more[p.B] = N;
    cu[p.B] = static_cast<int>(tokens);
  }
  __syncthreads();

  const int g0 = blockIdx.x * n + tid, gn = gridDim.x * n;
  const int nback = ok ? R : 0, nmore = ok ? N : 0;
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
    for (int b = g0 >> 5; b < p.B; b += gn >> 5) {  // a warp per row; the entries that are new come below
      const unsigned keep = ok ? plan_pages(base[b], p.page_shift) : p.W, to = keep + (ok ? more[b + 1] - more[b] : 0), width = p.W;
      const int* src = p.table + static_cast<long long>(b) * p.W;
      int* dst = p.table_out + static_cast<long long>(b) * p.W;
#pragma unroll 4
      for (unsigned j = lane; j < width; j += 32)
        if (j < keep || j >= to) dst[j] = src[j];
    }
  }
  auto taken = [&](int x) {  // the x-th page that is taken
    const int i = count + nback - 1 - x;
    if (p.in_place) return __ldcg(p.stack_out + i);
    return i < count ? p.stack[i] : back_page(i - count);
  };
  // The rest begins with other CTAs than the copies: each part is a chain of its own (48 requests 3.8 us against 5.1, 2048 requests 6.0 against 8.8).
  const int half = gridDim.x >> 1, g1 = (blockIdx.x < half ? blockIdx.x + gridDim.x - half : blockIdx.x - half) * n + tid;
  const int g2 = (gridDim.x - 1 - blockIdx.x) * n + tid;
  for (int x = g1; x < nmore; x += gn) {
    const int b = plan_find(more, p.B, x);
    p.table_out[static_cast<long long>(b) * p.W + plan_pages(base[b], p.page_shift) + x - more[b]] = taken(x);
  }
  const int page = 1 << p.page_shift, real = ok ? cu[p.B] : 0;
  for (unsigned i = g2; i < static_cast<unsigned>(p.T); i += gn) {  // (in 31 bits the last stride could go round and below zero)
    const int t = static_cast<int>(i);
    int at = 0, slot = -1;
    if (t < real) {
      const int b = plan_find(cu, p.B, t);
      at = base[b] + (t - cu[b]);
      const int j = at >> p.page_shift, keep = plan_pages(base[b], p.page_shift);
      const int number = j < keep ? p.table[static_cast<long long>(b) * p.W + j] : taken(more[b] + j - keep);
      slot = number * page + (at & (page - 1));
    }
    p.pos[t] = at;
    p.slots[t] = slot;
  }
  for (int b = g0; b <= p.B; b += gn) p.cu[b] = ok ? cu[b] : 0;
  for (int b = g0; b < p.B; b += gn) {
    if (ok) p.lens_out[b] = base[b] + (cu[b + 1] - cu[b]);
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
// D / 8 lanes hold a head, eight channels each, and a warp takes HN_LOADS such loads of one token at once: two where there are few tokens and
// latency counts, six where memory is to be kept busy (32 + 16 heads of 128, 300 tokens 2.97 against 4.40 us, 16384 tokens 98 against
// 73 us; equal near 1000).  Where all channels turn
// (HALVES), a lane holds four of the first half and their partners of the second; neighbours (PAIRED) lie in one lane anyway;
// with fewer channels turned in halves (SOME) the partners come by shuffle.  The weights are multiplied into the token's
// cosines and sines, which all of its heads share: a channel costs three multiplications and additions and the norm's two.
// Bound by memory: every byte is read once and written once (16384 tokens, 405 MB: 5.53 TB/s, 86 % of a plain copy; 33 tokens 2.1 us).
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
  int T, H, G, rot, max_pos, page_shift, num_slots, chunks;
  float eps;
  int* status;
  int pdl;
};
constexpr int HN_THREADS = 128;
enum HnForm { HN_HALVES, HN_PAIRED, HN_SOME };

// Pairs of channels as packed fp32 (one instruction for two).
__device__ __forceinline__ uint64_t hn_pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 hn_two(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t hn_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t hn_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t hn_swap(uint64_t v) {
  const float2 f = hn_two(v);
  return hn_pair(f.y, f.x);
}
__device__ __forceinline__ void hn_unpack(const uint4& v, uint64_t (&x)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = hn_pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
}

// A lane's eight channels: two runs of four, the second `gap` channels behind the first (4: side by side).
template <int GAP>
__device__ __forceinline__ uint4 hn_load(const __nv_bfloat16* src) {
  if (GAP == 4) return *reinterpret_cast<const uint4*>(src);
  const uint2 a = *reinterpret_cast<const uint2*>(src), b = *reinterpret_cast<const uint2*>(src + GAP);
  return make_uint4(a.x, a.y, b.x, b.y);
}
template <int GAP>
__device__ __forceinline__ void hn_store(__nv_bfloat16* dst, const uint4& v) {
  if (GAP == 4) {
    *reinterpret_cast<uint4*>(dst) = v;
  } else {
    *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(dst + GAP) = make_uint2(v.z, v.w);
  }
}
__device__ __forceinline__ void hn_floats(const float* src, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(src);
  x[0] = v.x;
  x[1] = v.y;
  x[2] = v.z;
  x[3] = v.w;
}

template <int D, HnForm FORM, int HN_LOADS>
__global__ void __launch_bounds__(HN_THREADS, 8) head_norm_rope_store_kernel(const HeadNormParams p) {
  constexpr int TEAM = D / 8, PER_LOAD = 32 / TEAM, HEADS = PER_LOAD * HN_LOADS;  // heads of a warp
  constexpr int GAP = FORM == HN_HALVES ? D / 2 : 4;
  const int lane = threadIdx.x & 31, l = lane % TEAM, sub = lane / TEAM;
  const int c0 = FORM == HN_HALVES ? 4 * l : 8 * l;  // first channel
  const int all = p.H + 2 * p.G;
  const unsigned w = (blockIdx.x * HN_THREADS + threadIdx.x) >> 5;  // (threads fit 32 bits; in another form it costs head_dim 128 a tenth: registers)
  const int t = static_cast<int>(w / p.chunks), h0 = static_cast<int>(w - static_cast<unsigned>(t) * p.chunks) * HEADS + sub;
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  if (t >= p.T) return;
  const int pos = p.pos[t], slot = p.slots[t];
  const __nv_bfloat16* row = p.src + t * p.ld + c0 + static_cast<long long>(h0) * D;
  uint4 raw[HN_LOADS];
#pragma unroll
  for (int i = 0; i < HN_LOADS; ++i) raw[i] = h0 + i * PER_LOAD < all ? hn_load<GAP>(row + i * PER_LOAD * D) : uint4{};
  const bool pos_ok = pos >= 0 && pos < p.max_pos, stored = slot >= 0 && slot < p.num_slots && pos_ok;
  if (lane == 0 && (!pos_ok || slot >= p.num_slots) && p.status) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
  const int half = p.rot >> 1;
  const bool turned = FORM == HN_HALVES || c0 < p.rot, first = c0 < half;
  const int away = FORM != HN_SOME || !turned ? 0 : first ? (half >> 3) : -(half >> 3);  // lanes to the partner
  const long long page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
  // Of channel e and its partner x'[e] = x[e] wc[e] + x[partner] ws[e]: the token's angles with the weights of the kind of head that the
  // lane is at in them.
  uint64_t wc[4], ws[4];
  auto coefficients = [&](const float* weight) {
    float a[8], b[8], cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = b[e] = cs[e] = 1.f, sn[e] = 0.f;
    if (weight) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v[4];
        hn_floats(weight + c0 + GAP * j, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * j + e] = v[e];
        if (FORM == HN_SOME) {
          hn_floats(weight + c0 + 4 * j + away * 8, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) b[4 * j + e] = v[e];
        }
      }
    }
    if (turned && pos_ok) {
      const long long at = static_cast<long long>(pos) * half;
      float c[4], s[4];
#pragma unroll
      for (int j = 0; j < (FORM == HN_SOME ? 2 : 1); ++j) {
        const long long i0 = at + (FORM == HN_SOME ? (first ? c0 : c0 - half) + 4 * j : FORM == HN_HALVES ? c0 : c0 >> 1);
        hn_floats(p.cos + i0, c);
        hn_floats(p.sin + i0, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (FORM == HN_SOME && (e >> 2) != j) continue;
          const int i = FORM == HN_PAIRED ? e >> 1 : e & 3;
          const bool minus = FORM == HN_SOME ? first : FORM == HN_HALVES ? e < 4 : !(e & 1);
          cs[e] = c[i];
          sn[e] = minus ? -s[i] : s[i];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float m[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int e = 2 * j + k;
        m[k] = (FORM == HN_HALVES ? a[e ^ 4] : FORM == HN_PAIRED ? a[e ^ 1] : b[e]) * sn[e];
      }
      wc[j] = hn_pair(a[2 * j] * cs[2 * j], a[2 * j + 1] * cs[2 * j + 1]);
      ws[j] = hn_pair(m[0], m[1]);
    }
  };
  int kind = -1;
#pragma unroll
  for (int i = 0; i < HN_LOADS; ++i) {
    const int h = h0 + i * PER_LOAD, now = h < p.H ? 0 : h < p.H + p.G ? 1 : 2;
    const float* weight = now == 0 ? p.wq : p.wk;
    if (now < 2 && now != kind) {
      kind = now;
      coefficients(weight);
    }
    if (__any_sync(0xffffffffu, now < 2)) {
      uint64_t x[4], mate[4];
      hn_unpack(raw[i], x);
      if (FORM == HN_SOME) {
        uint4 other;
        other.x = __shfl_sync(0xffffffffu, raw[i].x, lane + away);
        other.y = __shfl_sync(0xffffffffu, raw[i].y, lane + away);
        other.z = __shfl_sync(0xffffffffu, raw[i].z, lane + away);
        other.w = __shfl_sync(0xffffffffu, raw[i].w, lane + away);
        hn_unpack(other, mate);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) mate[j] = FORM == HN_HALVES ? x[j ^ 2] : hn_swap(x[j]);
      }
      float r = 1.f;
      if (p.wq || p.wk) {
        uint64_t two = hn_mul(x[0], x[0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) two = hn_fma(x[j], x[j], two);
        float ss = hn_two(two).x + hn_two(two).y;
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (weight) r = rsqrtf(ss * (1.f / D) + p.eps);
      }
      uint32_t packed[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint64_t z = hn_mul(x[j], wc[j]);
        if (FORM != HN_SOME || turned) z = hn_fma(mate[j], ws[j], z);
        const float2 f = hn_two(hn_mul(z, hn_pair(r, r)));
        const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
        packed[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
      const uint4 y = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      if (now == 0) hn_store<GAP>(p.q_out + (static_cast<long long>(t) * p.H + h) * D + c0, pos_ok ? y : uint4{});
      else if (now == 1 && stored) hn_store<GAP>(p.kp + page * p.k_page + (h - p.H) * p.k_head + off * p.k_row + c0, y);
    }
    if (now == 2 && h < all && stored) hn_store<GAP>(p.vp + page * p.v_page + (h - p.H - p.G) * p.v_head + off * p.v_row + c0, raw[i]);
  }
}

// Whether rows of `d` elements at these strides share none: each stride, from the smallest up, passes over all that lies inside it.
static bool rows_apart(const int64_t* strides, const int (&extents)[3], int d) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return strides[a] < strides[b]; });
  __int128 inside = d;
  for (const int i : order) {
    if (extents[i] <= 1) continue;
    if (strides[i] < inside) return false;
    inside += static_cast<__int128>(strides[i]) * (extents[i] - 1);
  }
  return true;
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
  if (static_cast<long long>(num_pages) << shift > 0x7fffffffll || static_cast<long long>(B) * table_width > 0x7fffffffll)
    return host::fail(TYBOK_ERR_ARG, "page_plan: slots and table entries must fit 31 bits");
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
  // Two threads for an entry to copy or write: every CTA pays the whole scan, but side by side, and the chains of the parts fall to different ones (7
  // prompts 2.95 us, 4.0 with two entries a thread; more than a CTA per SM costs 2048 requests 2.4 us).  In place, where one cluster meets, two entries a thread.
  const long long work = tokens + (p.in_place ? 0ll : num_pages + static_cast<long long>(B) * table_width);
  const int threads = B <= 256 ? 256 : B <= 1024 ? 512 : 1024, most = p.in_place ? 8 : host::sm_count();
  const int ctas = static_cast<int>(std::min<long long>(most, std::max<long long>(1, p.in_place ? work / (2 * threads) : 2 * work / threads)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.in_place && ctas > 1 ? 8 : ctas);
  cfg.blockDim = dim3(threads);
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
  const int extents[3] = {num_pages, G, page_size};
  for (int i = 0; i < 3; ++i)
    if (extents[i] > 1 && (k_strides[i] <= 0 || v_strides[i] <= 0)) return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: strides of the pools must be positive");
  uintptr_t bits = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_pages) |
                   reinterpret_cast<uintptr_t>(v_pages) | reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table) |
                   reinterpret_cast<uintptr_t>(norm_q) | reinterpret_cast<uintptr_t>(norm_k);
  int64_t strides = ld;
  for (int i = 0; i < 3; ++i) strides |= k_strides[i] | v_strides[i];
  if ((bits & 15) || (strides & 7))
    return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: tensors must be 16-byte aligned, strides multiples of 8 elements");
  if (!rows_apart(k_strides, extents, D) || !rows_apart(v_strides, extents, D) || k_pages == v_pages)
    return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: rows of the pools must not overlap");
  if (int rc = host::require_sm100()) return rc;
  HeadNormParams p{};
  p.src = static_cast<const __nv_bfloat16*>(src); p.ld = ld; p.pos = pos; p.slots = slots; p.cos = cos_table; p.sin = sin_table;
  p.wq = norm_q; p.wk = norm_k; p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.kp = static_cast<__nv_bfloat16*>(k_pages); p.vp = static_cast<__nv_bfloat16*>(v_pages);
  p.k_page = k_strides[0]; p.k_head = k_strides[1]; p.k_row = k_strides[2];
  p.v_page = v_strides[0]; p.v_head = v_strides[1]; p.v_row = v_strides[2];
  p.T = tokens; p.H = H; p.G = G; p.rot = rot; p.max_pos = max_pos; p.page_shift = shift; p.num_slots = num_pages << shift;
  p.eps = eps; p.status = status_word;
  p.pdl = host::pdl_enabled() ? 1 : 0;
  const int per_load = 32 / (D / 8), all = H + 2 * G;
  const bool few = static_cast<long long>(tokens) * all < 32768ll * per_load;
  p.chunks = (all + per_load * (few ? 2 : 6) - 1) / (per_load * (few ? 2 : 6));
  const long long ctas = (static_cast<long long>(tokens) * p.chunks * 32 + HN_THREADS - 1) / HN_THREADS;
  if (ctas > 0xffffffffll / HN_THREADS) return host::fail(TYBOK_ERR_ARG, "head_norm_rope_store: too many tokens for one launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(HN_THREADS);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl;
  using Kernel = void(const HeadNormParams);
  static Kernel* const kernels[2][3][2] = {
      {{head_norm_rope_store_kernel<128, HN_HALVES, 2>, head_norm_rope_store_kernel<128, HN_HALVES, 6>},
       {head_norm_rope_store_kernel<128, HN_PAIRED, 2>, head_norm_rope_store_kernel<128, HN_PAIRED, 6>},
       {head_norm_rope_store_kernel<128, HN_SOME, 2>, head_norm_rope_store_kernel<128, HN_SOME, 6>}},
      {{head_norm_rope_store_kernel<256, HN_HALVES, 2>, head_norm_rope_store_kernel<256, HN_HALVES, 6>},
       {head_norm_rope_store_kernel<256, HN_PAIRED, 2>, head_norm_rope_store_kernel<256, HN_PAIRED, 6>},
       {head_norm_rope_store_kernel<256, HN_SOME, 2>, head_norm_rope_store_kernel<256, HN_SOME, 6>}}};
  Kernel* kernel = kernels[D == 256][paired ? HN_PAIRED : rot == D ? HN_HALVES : HN_SOME][few ? 0 : 1];
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess)
    return host::fail_cuda("launch head_norm_rope_store_kernel");
  host::count_launch();
  return TYBOK_OK;
}
}

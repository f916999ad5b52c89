// Attention of new tokens over the paged cache of keys and values (layout: see paged.cu).
//
// Request b brings the n = cu[b+1] - cu[b] last of its key_lens[b] keys as queries; query i sees the keys j <= key_lens[b] - n + i
// (causal) or all of them.  Lengths are on the device, so the host sizes nothing by them: a persistent grid shares out the key
// blocks of all (request, key head, row tile) in one line, as evenly as blocks go.  A CTA's share may begin and end
// inside a tile; then it leaves (maximum, sum, unnormalised output) of its part behind, and a second kernel joins the parts in
// their order.  Queries of the same key head are rows of the same product (row = token * H / G + head).
//
// Algorithmic bytes: Q and O once, K and V of a request's keys once per row tile (L2 serves the tiles after the first).
// Flops: 4 * D * H per visible (query, key) pair.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/tybok_b200.h"
#include "host_util.h"
#include "ptx.cuh"
#include "split3.cuh"

namespace tb {

constexpr int PA_MAX_REQUESTS = 2048;

struct PagedAttnParams {
  const __nv_bfloat16* q;
  long long ldq;
  const __nv_bfloat16* kp;
  const __nv_bfloat16* vp;
  long long k_page, k_head, k_row, v_page, v_head, v_row;  // strides in elements
  const int* table;  // [B][ld_table]
  long long ld_table;
  const int* cu;
  const int* lens;
  __nv_bfloat16* out;
  uint8_t* out_planes;
  long long ld_out;  // H * D
  float plane_scale;
  int T, B, H, G, ratio, P, W, page_shift, causal;
  float scale_log2e;
  uint8_t* ws;
  int* status;
  int pdl;
};

// What a CTA's share needs to know of one request, out of range values brought back into range.
struct PaRequest {
  int start, n, len;
};
__device__ __forceinline__ PaRequest pa_request(const PagedAttnParams& p, int b) {
  PaRequest r;
  const int lo = p.cu[b], hi = p.cu[b + 1];
  r.start = max(0, min(lo, p.T));
  r.n = max(0, min(hi, p.T) - r.start);
  r.len = static_cast<int>(min(static_cast<long long>(max(0, p.lens[b])), static_cast<long long>(p.W) << p.page_shift));
  return r;
}
__device__ __forceinline__ bool pa_in_range(const PagedAttnParams& p, int b) {
  const int lo = p.cu[b], hi = p.cu[b + 1], len = p.lens[b];
  return lo >= 0 && lo <= hi && hi <= p.T && len >= 0 && len <= (static_cast<long long>(p.W) << p.page_shift);
}
// Keys that the rows before `row_end` of a request see: those of the last of them.
__device__ __forceinline__ int pa_seen(const PagedAttnParams& p, const PaRequest& r, int row_end) {
  if (!p.causal) return r.len;
  const int token = (row_end - 1) / p.ratio;
  return max(0, r.len - r.n + token + 1);
}
// Key blocks of a row tile; a tile that sees no key is one block of work all the same (its output is zero).
template <int ROWS, int BK>
__device__ __forceinline__ int pa_blocks(const PagedAttnParams& p, const PaRequest& r, int tile) {
  const int seen = pa_seen(p, r, min(r.n * p.ratio, (tile + 1) * ROWS));
  return max(1, (seen + BK - 1) / BK);
}

// ws: int4 per CTA (request, key head, tile, parts of the tile that this CTA begins and others go on with; parts = 0: none), then
// two partial tiles per CTA: [0] ends a tile begun by another CTA, [1] begins one that others go on with.
template <int ROWS, int D>
__host__ __device__ constexpr size_t pa_part_bytes() { return static_cast<size_t>(ROWS) * (D + 2) * 4; }
__host__ __device__ constexpr size_t pa_header_bytes(int ctas) { return (static_cast<size_t>(ctas) * 16 + 255) & ~size_t(255); }

// ------------------------------------------------------------------------------------------------ sixteen-row form
// Few rows per key head (single tokens): 16 rows of mma.m16n8k16, four warps that share the keys of a block and nothing else: each
// streams its own keys through its own ring and keeps its own maxima, sums and output in registers; they meet at the end of a tile.
constexpr int PR_ROWS = 16, PR_WARPS = 4, PR_THREADS = 128, PR_STAGES = 3;
__host__ __device__ constexpr int pr_sub(int d) { return d == 256 ? 16 : 32; }   // keys per warp and block: 16 KB of K and V
__host__ __device__ constexpr int pr_block(int d) { return PR_WARPS * pr_sub(d); }
constexpr int PR_STAGE_BYTES = 16384;
constexpr int PR_SMEM = PR_WARPS * PR_STAGES * PR_STAGE_BYTES;

__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight finished channels of an output row: bf16, and the three planes of the bf16 values.
__device__ __forceinline__ void pa_store8(const PagedAttnParams& p, long long at, const float (&o)[8]) {
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = pack_bf16(o[2 * j], o[2 * j + 1]);
  if (p.out) *reinterpret_cast<uint4*>(p.out + at) = make_uint4(b[0], b[1], b[2], b[3]);
  if (p.out_planes) {
    uint32_t w[3][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = bf16_round(o[4 * j + e]) * p.plane_scale;
      split3_quad(x, w[0][j], w[1][j], w[2][j]);
    }
    const long long plane = static_cast<long long>(p.T) * p.ld_out;
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(p.out_planes + k * plane + at) = make_uint2(w[k][0], w[k][1]);
  }
}

// Linear numbers of the key blocks: prefix[b] of them lie before request b.  By all threads of the CTA.
template <int ROWS, int BK, int NT>
__device__ void pa_schedule(const PagedAttnParams& p, long long* prefix) {
  __shared__ long long warp_sum[NT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long carry = 0;
  for (int base = 0; base < p.B; base += NT) {
    const int b = base + tid;
    PaRequest r{0, 0, 0};
    if (b < p.B) {
      r = pa_request(p, b);
      if (blockIdx.x == 0 && p.status && !pa_in_range(p, b)) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
    }
    const int tiles = (r.n * p.ratio + ROWS - 1) / ROWS;
    long long cost = 0;
    const bool many = p.causal && tiles > 4;  // their sums by the whole warp
    if (!many) {
      if (!p.causal) cost = static_cast<long long>(tiles) * max(1, (r.len + BK - 1) / BK);
      else
        for (int t = 0; t < tiles; ++t) cost += pa_blocks<ROWS, BK>(p, r, t);
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
      const int src = __ffs(left) - 1;
      const PaRequest o{0, __shfl_sync(0xffffffffu, r.n, src), __shfl_sync(0xffffffffu, r.len, src)};
      const int ot = __shfl_sync(0xffffffffu, tiles, src);
      long long sum = 0;
      for (int t = lane; t < ot; t += 32) sum += pa_blocks<ROWS, BK>(p, o, t);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == src) cost = sum;
    }
    cost *= p.G;
    long long x = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    long long before = carry, total = carry;
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      total += warp_sum[w];
    }
    if (b < p.B) prefix[b + 1] = before + x;
    carry = total;
    __syncthreads();
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
}

// A place in the line of key blocks: block `blk` of `nblk` of row tile `tile` of key head `g` of request `b`.
struct PaPlace {
  int b, g, tile, blk, nblk, tiles;
  PaRequest r;
};
// The tile that block x lies in.  By whole warps.
template <int ROWS, int BK>
__device__ PaPlace pa_locate(const PagedAttnParams& p, const long long* prefix, long long x) {
  PaPlace at;
  int lo = 0, hi = p.B;  // the last b with prefix[b] <= x (requests without queries have no blocks)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x) lo = mid;
    else hi = mid;
  }
  at.b = lo;
  at.r = pa_request(p, lo);
  const long long per_head = (prefix[lo + 1] - prefix[lo]) / p.G;
  long long rest = x - prefix[lo];
  at.g = static_cast<int>(rest / per_head);
  rest -= at.g * per_head;
  at.tiles = (at.r.n * p.ratio + ROWS - 1) / ROWS;
  if (!p.causal) {
    at.nblk = max(1, (at.r.len + BK - 1) / BK);
    at.tile = static_cast<int>(rest / at.nblk);
    at.blk = static_cast<int>(rest - static_cast<long long>(at.tile) * at.nblk);
    return at;
  }
  const int lane = threadIdx.x & 31;
  for (int t0 = 0;; t0 += 32) {  // 32 tiles at a time
    const int n = t0 + lane < at.tiles ? pa_blocks<ROWS, BK>(p, at.r, t0 + lane) : 0;
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, sum > rest);
    if (past || t0 + 32 >= at.tiles) {
      const int i = past ? __ffs(past) - 1 : 31;
      at.tile = t0 + i;
      at.nblk = __shfl_sync(0xffffffffu, n, i);
      at.blk = static_cast<int>(rest - (__shfl_sync(0xffffffffu, sum, i) - at.nblk));
      return at;
    }
    rest -= __shfl_sync(0xffffffffu, sum, 31);
  }
}
// The tile after this one (the caller knows that there is one).
template <int ROWS, int BK>
__device__ __forceinline__ void pa_next(const PagedAttnParams& p, PaPlace& at) {
  if (++at.tile == at.tiles) {
    at.tile = 0;
    if (++at.g == p.G) {
      at.g = 0;
      do {
        ++at.b;
        at.r = pa_request(p, at.b);
      } while (at.r.n == 0 && at.b + 1 < p.B);
      at.tiles = (at.r.n * p.ratio + ROWS - 1) / ROWS;
    }
  }
  at.blk = 0;
  at.nblk = pa_blocks<ROWS, BK>(p, at.r, at.tile);
}

// Output rows that belong to no request are zero.
template <int D>
__device__ __forceinline__ void pa_zero_rows(const PagedAttnParams& p, int nt) {
  const int first = max(0, min(p.cu[0], p.T)), last = max(first, min(p.cu[p.B], p.T));
  const long long per = p.ld_out / 8, rows = p.T - last + first, n = rows * per;
  const float zero[8] = {};
  for (long long i = static_cast<long long>(blockIdx.x) * nt + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * nt) {
    const long long row = i / per, c = i - row * per;
    pa_store8(p, (row < first ? row : row - first + last) * p.ld_out + c * 8, zero);
  }
}

template <int D>
__global__ void __launch_bounds__(PR_THREADS, 1) paged_rows_kernel(const PagedAttnParams p) {
  extern __shared__ __align__(128) uint8_t pr_smem[];
  __shared__ float s_m[PR_WARPS][PR_ROWS], s_l[PR_WARPS][PR_ROWS];
  constexpr int SUB = pr_sub(D), BK = pr_block(D), ROW_BYTES = D * 2, CHUNKS = D / 8, KS = D / 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long* prefix = reinterpret_cast<long long*>(pr_smem + PR_SMEM);
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  pa_zero_rows<D>(p, PR_THREADS);
  pa_schedule<PR_ROWS, BK, PR_THREADS>(p, prefix);
  const long long total = prefix[p.B], per = (total + gridDim.x - 1) / gridDim.x;
  const long long x1 = min(total, (blockIdx.x + 1) * per);
  long long x = min(total, blockIdx.x * per);
  int4 header = make_int4(0, 0, 0, 0);
  const uint32_t ring = smem_u32(pr_smem) + warp * (PR_STAGES * PR_STAGE_BYTES);
  PaPlace at{};
  if (x < x1) at = pa_locate<PR_ROWS, BK>(p, prefix, x);
  for (; x < x1;) {
    const int end = static_cast<int>(min(static_cast<long long>(at.nblk), at.blk + (x1 - x)));
    const int rows = at.r.n * p.ratio;
    // this thread's two rows of the tile: queries as operand fragments, keys they see
    uint32_t qf[KS][4];
    int limit[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = at.tile * PR_ROWS + h * 8 + (lane >> 2), token = row / p.ratio;
      const bool live = row < rows;
      limit[h] = !live ? 0 : p.causal ? max(0, at.r.len - at.r.n + token + 1) : at.r.len;
      const __nv_bfloat16* src = p.q + (at.r.start + token) * p.ldq + static_cast<long long>(at.g * p.ratio + row - token * p.ratio) * D + (lane & 3) * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[ks][h] = live ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
        qf[ks][h + 2] = live ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
      }
    }
    const int seen = pa_seen(p, at.r, min(rows, (at.tile + 1) * PR_ROWS));                    // by any row
    const int seen_all = p.causal ? max(0, at.r.len - at.r.n + at.tile * PR_ROWS / p.ratio + 1) : at.r.len;  // by every row
    auto fetch = [&](int j) {  // this warp's keys of block j
      const uint32_t slot = ring + (j % PR_STAGES) * PR_STAGE_BYTES;
      const int key0 = j * BK + warp * SUB;
#pragma unroll 1
      for (int k0 = 0; k0 < SUB; k0 += 16) {
        const int key = key0 + k0;
        int page = -1;
        if (key < seen) {
          page = p.table[at.b * p.ld_table + (key >> p.page_shift)];
          if (page < 0 || page >= p.P) {
            if (p.status && lane == 0) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
            page = -1;
          }
        }
        const long long off = key & ((1 << p.page_shift) - 1), pg = max(page, 0);
        const __nv_bfloat16* ks = p.kp + pg * p.k_page + at.g * p.k_head + off * p.k_row;
        const __nv_bfloat16* vs = p.vp + pg * p.v_page + at.g * p.v_head + off * p.v_row;
#pragma unroll
        for (int i = 0; i < 16 * CHUNKS / 32; ++i) {
          const int r = (i * 32 + lane) / CHUNKS, c = (i * 32 + lane) % CHUNKS;
          const int bytes = page >= 0 && key + r < seen ? 16 : 0;  // the others are zero
          const uint32_t dst = slot + (k0 + r) * ROW_BYTES + ((c ^ (r & 7)) << 4);
          const long long rr = bytes ? r : 0;
          cp_async16(dst, ks + rr * p.k_row + c * 8, bytes);
          cp_async16(dst + SUB * ROW_BYTES, vs + rr * p.v_row + c * 8, bytes);
        }
      }
    };
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PR_STAGES - 1; ++i) {
      if (at.blk + i < end) fetch(at.blk + i);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
#pragma unroll 1
    for (int j = at.blk; j < end; ++j) {
      if (j + PR_STAGES - 1 < end) fetch(j + PR_STAGES - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group %0;" ::"n"(PR_STAGES - 1) : "memory");
      __syncwarp();
      const int key0 = j * BK + warp * SUB;
      const uint32_t ka = ring + (j % PR_STAGES) * PR_STAGE_BYTES, va = ka + SUB * ROW_BYTES;
      if (key0 < seen) {
        float sc[SUB / 8][4];
#pragma unroll
        for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int u = 0; u < SUB / 16; ++u) {
            const int r = u * 16 + ((lane >> 4) << 3) + (lane & 7), c = ks * 2 + ((lane >> 3) & 1);
            uint32_t kf[4];
            ldsm4(ka + r * ROW_BYTES + ((c ^ (r & 7)) << 4), kf);
            mma_bf16(sc[2 * u], qf[ks], kf[0], kf[1]);
            mma_bf16(sc[2 * u + 1], qf[ks], kf[2], kf[3]);
          }
        const bool whole = key0 + SUB <= seen_all;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + i * 8 + (lane & 3) * 2 + (e & 1);
            float v = sc[i][e] * p.scale_log2e;
            if (!whole && key >= limit[e >> 1]) v = -INFINITY;
            sc[i][e] = v;
            mx[e >> 1] = fmaxf(mx[e >> 1], v);
          }
        float f[2], ref[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
          const float top = fmaxf(m[h], mx[h]);
          ref[h] = top == -INFINITY ? 0.f : top;
          f[h] = pa_exp2(m[h] - ref[h]);  // 0 for a first block
          m[h] = top;
          l[h] *= f[h];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] *= f[e >> 1];
        }
#pragma unroll
        for (int i = 0; i < SUB / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[i][e] = pa_exp2(sc[i][e] - ref[e >> 1]);
            l[e >> 1] += sc[i][e];
          }
#pragma unroll
        for (int u = 0; u < SUB / 16; ++u) {
          const uint32_t pf[4] = {pack_bf16(sc[2 * u][0], sc[2 * u][1]), pack_bf16(sc[2 * u][2], sc[2 * u][3]),
                                  pack_bf16(sc[2 * u + 1][0], sc[2 * u + 1][1]), pack_bf16(sc[2 * u + 1][2], sc[2 * u + 1][3])};
#pragma unroll
          for (int ds = 0; ds < KS; ++ds) {
            const int r = u * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), c = ds * 2 + (lane >> 4);
            uint32_t vf[4];
            ldsm4t(va + r * ROW_BYTES + ((c ^ (r & 7)) << 4), vf);
            mma_bf16(o[2 * ds], pf, vf[0], vf[1]);
            mma_bf16(o[2 * ds + 1], pf, vf[2], vf[3]);
          }
        }
      }
      __syncwarp();
    }
    // the four warps' parts meet
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    float* mine = reinterpret_cast<float*>(pr_smem + warp * (PR_STAGES * PR_STAGE_BYTES));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int row = h * 8 + (lane >> 2);
      if ((lane & 3) == 0) {
        s_m[warp][row] = m[h];
        s_l[warp][row] = l[h];
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(mine + row * D + ((i * 8 + (lane & 3) * 2) ^ ((row & 3) << 3))) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
    __syncthreads();
    const bool whole_tile = at.blk == 0 && end == at.nblk;
    const int part = at.blk > 0 ? 0 : 1;
    float* po = reinterpret_cast<float*>(p.ws + pa_header_bytes(gridDim.x) + (2ll * blockIdx.x + part) * pa_part_bytes<PR_ROWS, D>());
#pragma unroll 1
    for (int i = tid; i < PR_ROWS * D / 8; i += PR_THREADS) {
      const int row = i / (D / 8), c = (i % (D / 8)) * 8;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < PR_WARPS; ++w) top = fmaxf(top, s_m[w][row]);
      float sum = 0.f, v[8] = {};
#pragma unroll
      for (int w = 0; w < PR_WARPS; ++w) {
        const float f = pa_exp2(s_m[w][row] - (top == -INFINITY ? 0.f : top));
        sum += f * s_l[w][row];
        const float4* src = reinterpret_cast<const float4*>(pr_smem + w * (PR_STAGES * PR_STAGE_BYTES)) + (row * D + (c ^ ((row & 3) << 3))) / 4;
        const float4 a = src[0], b = src[1];
        v[0] += f * a.x; v[1] += f * a.y; v[2] += f * a.z; v[3] += f * a.w;
        v[4] += f * b.x; v[5] += f * b.y; v[6] += f * b.z; v[7] += f * b.w;
      }
      const int grow = at.tile * PR_ROWS + row;
      if (grow >= rows) continue;
      if (whole_tile) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inv;
        const int token = grow / p.ratio;
        pa_store8(p, (at.r.start + token) * p.ld_out + static_cast<long long>(at.g * p.ratio + grow - token * p.ratio) * D + c, v);
      } else {
        float4* dst = reinterpret_cast<float4*>(po + row * D + c);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        if (c == 0) {
          po[PR_ROWS * D + row] = top;
          po[PR_ROWS * D + PR_ROWS + row] = sum;
        }
      }
    }
    if (!whole_tile && at.blk == 0) header = make_int4(at.b, at.g, at.tile, static_cast<int>((x + at.nblk - 1) / per) - static_cast<int>(blockIdx.x) + 1);
    x += end - at.blk;
    __syncthreads();  // the ring is free again
    if (x < x1) pa_next<PR_ROWS, BK>(p, at);
  }
  if (tid == 0) reinterpret_cast<int4*>(p.ws)[blockIdx.x] = header;
}

// Joins the parts of the tile that CTA blockIdx.x of the kernel before began: four rows per CTA, a warp each.
template <int ROWS, int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttnParams p, int ctas) {
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  const int4 h = reinterpret_cast<const int4*>(p.ws)[blockIdx.x];
  if (h.w == 0) return;
  const int lane = threadIdx.x & 31, row = blockIdx.y * 4 + (threadIdx.x >> 5);
  const PaRequest r = pa_request(p, h.x);
  const int grow = h.z * ROWS + row;
  if (grow >= r.n * p.ratio) return;
  const uint8_t* parts = p.ws + pa_header_bytes(ctas);
  auto part = [&](int i) {  // the i-th part of the tile
    return reinterpret_cast<const float*>(parts + (2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * pa_part_bytes<ROWS, D>());
  };
  float top = -INFINITY;
  for (int i = lane; i < h.w; i += 32) top = fmaxf(top, part(i)[ROWS * D + row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;
  constexpr int N = D / 32;
  float sum = 0.f, v[N] = {};
  for (int i = 0; i < h.w; ++i) {
    const float* src = part(i);
    const float f = pa_exp2(src[ROWS * D + row] - top);
    sum += f * src[ROWS * D + ROWS + row];
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 a = *reinterpret_cast<const float4*>(src + row * D + lane * N + e);
      v[e] += f * a.x; v[e + 1] += f * a.y; v[e + 2] += f * a.z; v[e + 3] += f * a.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int token = grow / p.ratio;
  const long long at = (r.start + token) * p.ld_out + static_cast<long long>(h.y * p.ratio + grow - token * p.ratio) * D;
  float o[8];  // eight channels by one lane: its own, or (four channels per lane) its own and its neighbour's
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = v[e] * inv;
  if (N == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[4 + e] = __shfl_down_sync(0xffffffffu, o[e], 1);
    if (!(lane & 1)) pa_store8(p, at + lane * 4, o);
  } else {
    pa_store8(p, at + lane * 8, o);
  }
}

template <int D>
static int paged_launch_rows(const PagedAttnParams& p, int ctas, cudaStream_t stream) {
  const size_t smem = PR_SMEM + 8 * (static_cast<size_t>(p.B) + 1);
  static host::DeviceCache ready;
  const int set = host::per_device(ready, [] {
    return cudaFuncSetAttribute(paged_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PR_SMEM + 8 * (PA_MAX_REQUESTS + 1)) == cudaSuccess ? 1 : 0;
  });
  if (!set) return host::fail_cuda("paged_attention: shared memory");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(PR_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl;
  if (cudaLaunchKernelEx(&cfg, paged_rows_kernel<D>, p) != cudaSuccess) return host::fail_cuda("launch paged_rows_kernel");
  host::count_launch();
  cfg.gridDim = dim3(ctas, PR_ROWS / 4);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, paged_join_kernel<PR_ROWS, D>, p, ctas) != cudaSuccess) return host::fail_cuda("launch paged_join_kernel");
  host::count_launch();
  return TYBOK_OK;
}

template <int D>
static size_t paged_ws(int ctas) { return pa_header_bytes(ctas) + 2 * static_cast<size_t>(ctas) * pa_part_bytes<PR_ROWS, D>(); }

}  // namespace tb

extern "C" {

size_t tybok_paged_attention_workspace_bytes(int H, int G, int D, int max_tokens) {
  using namespace tb;
  if (H <= 0 || G <= 0 || max_tokens <= 0 || (D != 128 && D != 256)) return 0;
  const int ctas = host::sm_count();
  return D == 256 ? paged_ws<256>(ctas) : paged_ws<128>(ctas);
}

int tybok_paged_attention(const void* q, int64_t ldq, const void* k_pages, const int64_t* k_strides, const void* v_pages,
                          const int64_t* v_strides, const int* block_table, int64_t ld_table, const int* cu_tokens,
                          const int* key_lens, void* out, void* out_planes, int out_shift, int tokens, int B, int H, int G, int D,
                          int num_pages, int page_size, int table_width, int max_tokens, int causal, float scale, void* workspace,
                          size_t workspace_bytes, int* status_word, void* stream) {
  using namespace tb;
  if (!q || !k_pages || !v_pages || !k_strides || !v_strides || !block_table || !cu_tokens || !key_lens || (!out && !out_planes))
    return host::fail(TYBOK_ERR_ARG, "paged_attention: null pointer argument");
  if (D != 128 && D != 256) return host::fail(TYBOK_ERR_ARG, "paged_attention: head_dim must be 128 or 256");
  if (page_size < 16 || (page_size & (page_size - 1))) return host::fail(TYBOK_ERR_ARG, "paged_attention: the page size must be a power of two, 16 at least");
  if (tokens <= 0 || B <= 0 || B > PA_MAX_REQUESTS || H <= 0 || G <= 0 || H % G != 0 || num_pages <= 0 || table_width <= 0 || max_tokens <= 0)
    return host::fail(TYBOK_ERR_ARG, "paged_attention: bad shape (1 to 2048 requests, H % G == 0, pool and table not empty)");
  if (static_cast<long long>(tokens) * (H / G) > 0x7fffffffll) return host::fail(TYBOK_ERR_ARG, "paged_attention: query rows must fit 31 bits");
  const uintptr_t bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                         reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_planes);
  int64_t strides = ldq;
  for (int i = 0; i < 3; ++i) strides |= k_strides[i] | v_strides[i];
  if ((bits & 15) || (strides & 7))
    return host::fail(TYBOK_ERR_ARG, "paged_attention: tensors must be 16-byte aligned, strides multiples of 8 elements");
  if (out_shift < -60 || out_shift > 60) return host::fail(TYBOK_ERR_ARG, "paged_attention: exponent shift out of range");
  const size_t need = tybok_paged_attention_workspace_bytes(H, G, D, max_tokens);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return host::fail(TYBOK_ERR_WORKSPACE, "paged_attention: workspace must hold tybok_paged_attention_workspace_bytes(), 16-byte aligned");
  if (int rc = host::require_sm100()) return rc;
  PagedAttnParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq;
  p.kp = static_cast<const __nv_bfloat16*>(k_pages); p.vp = static_cast<const __nv_bfloat16*>(v_pages);
  p.k_page = k_strides[0]; p.k_head = k_strides[1]; p.k_row = k_strides[2];
  p.v_page = v_strides[0]; p.v_head = v_strides[1]; p.v_row = v_strides[2];
  p.table = block_table; p.ld_table = ld_table; p.cu = cu_tokens; p.lens = key_lens;
  p.out = static_cast<__nv_bfloat16*>(out); p.out_planes = static_cast<uint8_t*>(out_planes);
  p.ld_out = static_cast<long long>(H) * D; p.plane_scale = ldexpf(1.0f, out_shift);
  p.T = tokens; p.B = B; p.H = H; p.G = G; p.ratio = H / G; p.P = num_pages; p.W = table_width; p.causal = causal;
  for (p.page_shift = 4; (1 << p.page_shift) != page_size;) ++p.page_shift;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.ws = static_cast<uint8_t*>(workspace); p.status = status_word;
  p.pdl = host::pdl_enabled() ? 1 : 0;
  const int ctas = host::sm_count();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return D == 256 ? paged_launch_rows<256>(p, ctas, st) : paged_launch_rows<128>(p, ctas, st);
}
}

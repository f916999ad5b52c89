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
#include <limits>

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
  int tile_rows;     // query rows (token, head of the group) of a tile, at most those of the form
  int join_blocks;   // what leaving a tile to two CTAs costs, in key blocks
  float scale_log2e;     // softmax scale * log2(e), with its sign
  float abs_scale_log2e; // its magnitude, above zero, and the bit of the scores' instruction that negates Q instead
  uint32_t negate_q;
  long long wait_limit;  // SM clocks the softmax warps wait for their scores (kWaitLimitCycles in production)
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
template <int BK>
__device__ __forceinline__ int pa_blocks(const PagedAttnParams& p, const PaRequest& r, int tile) {
  const int seen = pa_seen(p, r, min(r.n * p.ratio, (tile + 1) * p.tile_rows));
  return max(1, (seen + BK - 1) / BK);
}
__device__ __forceinline__ int pa_tiles(const PagedAttnParams& p, int n) { return (n * p.ratio + p.tile_rows - 1) / p.tile_rows; }

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
// Returns the number of row tiles (of every key head).
template <int BK, int NT>
__device__ long long pa_schedule(const PagedAttnParams& p, long long* prefix) {
  __shared__ long long warp_sum[NT / 32], warp_tiles[NT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long carry = 0, all_tiles = 0;
  for (int base = 0; base < p.B; base += NT) {
    const int b = base + tid;
    PaRequest r{0, 0, 0};
    if (b < p.B) {
      r = pa_request(p, b);
      if (blockIdx.x == 0 && p.status && !pa_in_range(p, b)) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
    }
    const int tiles = pa_tiles(p, r.n);
    long long cost = 0;
    const bool many = p.causal && tiles > 4;  // their sums by the whole warp
    if (!many) {
      if (!p.causal) cost = static_cast<long long>(tiles) * max(1, (r.len + BK - 1) / BK);
      else
        for (int t = 0; t < tiles; ++t) cost += pa_blocks<BK>(p, r, t);
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
      const int src = __ffs(left) - 1;
      const PaRequest o{0, __shfl_sync(0xffffffffu, r.n, src), __shfl_sync(0xffffffffu, r.len, src)};
      const int ot = __shfl_sync(0xffffffffu, tiles, src);
      long long sum = 0;
      for (int t = lane; t < ot; t += 32) sum += pa_blocks<BK>(p, o, t);
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
    const int lane_tiles = __reduce_add_sync(0xffffffffu, tiles);
    if (lane == 31) {
      warp_sum[warp] = x;
      warp_tiles[warp] = lane_tiles;
    }
    __syncthreads();
    long long before = carry, total = carry;
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      total += warp_sum[w];
      all_tiles += warp_tiles[w];
    }
    if (b < p.B) prefix[b + 1] = before + x;
    carry = total;
    __syncthreads();
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
  return all_tiles * p.G;
}

// A place in the line of key blocks: block `blk` of `nblk` of row tile `tile` of key head `g` of request `b`.
struct PaPlace {
  int b, g, tile, blk, nblk, tiles;
  PaRequest r;
};
// The tile that block x lies in.  By whole warps.
template <int BK>
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
  at.tiles = pa_tiles(p, at.r.n);
  if (!p.causal) {
    at.nblk = max(1, (at.r.len + BK - 1) / BK);
    at.tile = static_cast<int>(rest / at.nblk);
    at.blk = static_cast<int>(rest - static_cast<long long>(at.tile) * at.nblk);
    return at;
  }
  const int lane = threadIdx.x & 31;
  for (int t0 = 0;; t0 += 32) {  // 32 tiles at a time
    const int n = t0 + lane < at.tiles ? pa_blocks<BK>(p, at.r, t0 + lane) : 0;
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
template <int BK>
__device__ __forceinline__ void pa_next(const PagedAttnParams& p, PaPlace& at) {
  if (++at.tile == at.tiles) {
    at.tile = 0;
    if (++at.g == p.G) {
      at.g = 0;
      do {
        ++at.b;
        at.r = pa_request(p, at.b);
      } while (at.r.n == 0 && at.b + 1 < p.B);
      at.tiles = pa_tiles(p, at.r.n);
    }
  }
  at.blk = 0;
  at.nblk = pa_blocks<BK>(p, at.r, at.tile);
}

// A CTA's share [x0, x1) of the line, the same for everyone who asks: equal numbers of blocks, borders moved to the edge of a tile
// that lies near.  With `whole` every border moves to the nearest edge, so no tile has two CTAs: where the rounds of whole tiles
// take no longer than an even share and the joining of its parts.
struct PaShare {
  long long per, x0, x1;
  bool whole;
};
__device__ __forceinline__ int pa_snap(const PaShare& sh, int blk, int nblk, int join_blocks) {
  const bool up = 2 * blk > nblk;
  const int away = up ? nblk - blk : blk;
  return sh.whole || away * 4ll <= min(sh.per, 4ll * join_blocks) - 4 ? (up ? nblk : 0) : blk;
}
template <int BK>
__device__ PaShare pa_share(const PagedAttnParams& p, const long long* prefix, long long tiles, PaPlace& first) {
  PaShare sh;
  const long long total = prefix[p.B], ctas = gridDim.x;
  sh.per = (total + ctas - 1) / ctas;
  sh.whole = (tiles + ctas - 1) / ctas * total <= (sh.per + p.join_blocks) * tiles;  // rounds * average length
  auto border = [&](long long c, PaPlace& at) {
    const long long x = c * sh.per;
    if (x >= total) return total;
    at = pa_locate<BK>(p, prefix, x);
    const int blk = pa_snap(sh, at.blk, at.nblk, p.join_blocks);
    const long long y = x - at.blk + blk;
    at.blk = blk;
    return y;
  };
  PaPlace next{};
  sh.x0 = border(blockIdx.x, first);
  sh.x1 = border(blockIdx.x + 1ll, next);
  if (sh.x0 < sh.x1 && first.blk == first.nblk) pa_next<BK>(p, first);
  return sh;
}
// How many CTAs the tile has that begins at x in this CTA's share and goes on behind it.
__device__ __forceinline__ int pa_parts(const PagedAttnParams& p, const PaShare& sh, long long x, int nblk) {
  const long long last = (x + nblk - 1) / sh.per;
  const int blk = static_cast<int>(last * sh.per - x);
  const bool gone = last > static_cast<long long>(blockIdx.x) && blk > 0 && pa_snap(sh, blk, nblk, p.join_blocks) == nblk;  // its border moved behind the tile
  return static_cast<int>(last - blockIdx.x) + (gone ? 0 : 1);
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
  const long long tiles = pa_schedule<BK, PR_THREADS>(p, prefix);
  PaPlace at{};
  const PaShare share = pa_share<BK>(p, prefix, tiles, at);
  const long long x1 = share.x1;
  long long x = share.x0;
  int4 header = make_int4(0, 0, 0, 0);
  const uint32_t ring = smem_u32(pr_smem) + warp * (PR_STAGES * PR_STAGE_BYTES);
  while (x < x1) {
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
    if (!whole_tile && at.blk == 0) header = make_int4(at.b, at.g, at.tile, pa_parts(p, share, x, at.nblk));
    x += end - at.blk;
    __syncthreads();  // the ring is free again
    if (x < x1) pa_next<BK>(p, at);
  }
  if (tid == 0) reinterpret_cast<int4*>(p.ws)[blockIdx.x] = header;
}

// ------------------------------------------------------------------------------------------------ tile forms
// Many rows per key head: 128-row tiles on the fifth-generation tensor cores.  Four control warps (keys, values, queries by TMA,
// one that issues the products) and two groups of four softmax warps with one query row per thread and tensor-memory lane.  The
// warp that fetches the queries walks the CTA's share and tells the others, a few tiles ahead; rings and barriers run on from
// tile to tile, so the next tile's queries, keys and first scores are on their way while this one's output is written.
//   scores   S = Q K^T into tensor memory, P = 2^(S c - m) in bf16 over it (m: a reference that moves only when a block's
//            maximum exceeds it by more than 2^8, then the row of O is rescaled), O += P V with P read from tensor memory.
//   head_dim 128 (paged_pair_kernel): two tiles of 128 rows share every key block of 128, a group each; the tiles take turns, one's
//            products run under the other's exponentials.
//   head_dim 256 (paged_wide_kernel): O of one tile takes half of the tensor memory; key blocks of 64 go round four score buffers and
//            the groups take every other block, so that a block's softmax has the time of two blocks' products.
// A page is one box of the tensor map and 64 channels (or a block's rows of a larger page); lanes of the copying warp issue one
// box each.  Page numbers out of range read as zero through the map's bounds.
// Values behind a request's last key are zeroed in shared memory before their product (their weights are zero, but what lies
// there may be anything).
constexpr int PT_THREADS = 384;
constexpr int PT_REGS_CONTROL = 72, PT_REGS_SOFTMAX = 216;  // launched with 168 each: 72 + 2 * 216 = 3 * 168
constexpr int PT_SMEM = 65536 + 4 * 32768 + 1024;           // queries, two key and two value blocks
constexpr float PT_RESCALE = 8.0f;
#define PA_MASKED 0xff800000u  // -infinity

__host__ __device__ constexpr int pt_bk(int d) { return d == 128 ? 128 : 64; }
__host__ __device__ constexpr int pt_rows(int d) { return d == 128 ? 256 : 128; }  // of a work item

// MN-major shared-memory operand with the 128-byte swizzle: 64-element runs along N, 8 K-rows per 1024-byte group; [16,30) leading
// byte offset >> 4 = distance between 64-wide N chunks, [32,46) stride byte offset >> 4 = distance between 8-row K groups.
__device__ __forceinline__ uint64_t pt_desc_mn(uint32_t smem_addr, uint32_t chunk_bytes) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | static_cast<uint64_t>(chunk_bytes >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
         static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
__device__ __forceinline__ float pt_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t pt_pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void pt_unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// What the CTA does with (a piece of) a tile.
struct __align__(16) PtPiece {
  int rows;         // query rows of the tile; 0 = the share is through
  int b, g;         // request and key head
  int blk, end;     // key blocks
  int len;          // keys of the request
  int seen, step;   // keys that the tile's first token sees, and how many more each later one does
  int token;        // first token of the tile, a row of q
  int part;         // 0 = the whole tile: the output; else 1 + which of the CTA's two partial tiles
  int pad[2];
};
constexpr int PT_PIECES = 4;

struct __align__(16) PtBars {
  PtPiece piece[PT_PIECES];
  uint64_t piece_full[PT_PIECES], piece_read[PT_PIECES];
  uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[4];     // pair: per tile; wide: per score buffer
  uint64_t p_full[2][4];  // pair: per tile and 32 keys; wide: [0] per score buffer
  uint64_t done[4];       // pair: per tile, its last product has landed; wide: per score buffer, the block's product has
  uint64_t o_free;        // wide: the output of a tile has been read
  uint64_t pub[2][4];     // wide: per group and warp: the reference maximum after this block; at the end of a tile, its sums
  uint64_t fin[2][4];
  uint64_t mma_done;
  uint32_t tmem_base;
  volatile int abort;
  float m_ref[2][128];                       // wide: per group and row
  float end_m[2][2][128], end_l[2][2][128];  // wide: per parity of the tile, group and row
};

// Piece n, read by a whole warp; false when there is none or the CTA has given up.
struct PtReader {
  uint32_t n = 0;
  bool ok = true;
  __device__ __forceinline__ bool next(PtBars& bars, PtPiece& at) {
    const uint32_t s = n % PT_PIECES;
    ok = __all_sync(0xffffffffu, wait_or_abort(&bars.piece_full[s], (n / PT_PIECES) & 1, &bars.abort));
    if (!ok) return false;
    const int4* src = reinterpret_cast<const int4*>(&bars.piece[s]);
    int4* dst = reinterpret_cast<int4*>(&at);
#pragma unroll
    for (int i = 0; i < 3; ++i) dst[i] = src[i];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bars.piece_read[s]);
    ++n;
    return at.rows > 0;
  }
};

// The walk over the CTA's share, and its queries: `tiles` of `rows` rows each (128 / ratio * ratio) per piece.  Leaves the header for the
// joining kernel behind.
template <int D>
__device__ __forceinline__ void pt_lead(const PagedAttnParams& p, const long long* prefix, long long tiles, const CUtensorMap* map, uint8_t* sq, PtBars& bars) {
  constexpr int NCH = D / 64, CH = 16384;
  const int lane = threadIdx.x & 31, half = 128 / p.ratio * p.ratio, tokens = 128 / p.ratio;
  PaPlace at{};
  const PaShare share = pa_share<pt_bk(D)>(p, prefix, tiles, at);
  int4 header = make_int4(0, 0, 0, 0);
  uint32_t n = 0, queries = 0;
  bool ok = true;
  long long x = share.x0;
  while (true) {
    const uint32_t s = n % PT_PIECES;
    if (n >= PT_PIECES) ok = __all_sync(0xffffffffu, wait_or_abort(&bars.piece_read[s], (n / PT_PIECES - 1) & 1, &bars.abort));
    if (!ok) break;
    const bool any = x < share.x1;
    PtPiece w{};
    if (any) {
      const int first = at.tile * p.tile_rows / p.ratio;
      w.rows = min(p.tile_rows, at.r.n * p.ratio - at.tile * p.tile_rows);
      w.b = at.b;
      w.g = at.g;
      w.blk = at.blk;
      w.end = static_cast<int>(min(static_cast<long long>(at.nblk), at.blk + (share.x1 - x)));
      w.len = at.r.len;
      w.seen = p.causal ? at.r.len - at.r.n + first + 1 : at.r.len;
      w.step = p.causal;
      w.token = at.r.start + first;
      w.part = w.blk == 0 && w.end == at.nblk ? 0 : w.blk > 0 ? 1 : 2;
      if (w.part == 2) header = make_int4(at.b, at.g, at.tile, pa_parts(p, share, x, at.nblk));
    }
    if (lane == 0) {
      bars.piece[s] = w;
      mbar_arrive(&bars.piece_full[s]);
    }
    __syncwarp();
    ++n;
    if (!any) break;
    if (queries > 0) ok = __all_sync(0xffffffffu, wait_or_abort(&bars.q_empty, (queries - 1) & 1, &bars.abort));
    if (!ok) break;
    const int nt = w.rows > half ? 2 : 1;
    if (lane == 0) {
      mbar_arrive_expect_tx(&bars.q_full, nt * NCH * half * 128);
      for (int i = 0; i < NCH * nt; ++i) tma_load_4d(sq + i * CH, map, &bars.q_full, (i % NCH) * 64, 0, w.g, w.token + (i / NCH) * tokens);
    }
    __syncwarp();
    ++queries;
    x += w.end - w.blk;
    if (x < share.x1) pa_next<pt_bk(D)>(p, at);
  }
  if (queries > 0) mbar_wait(&bars.q_full, (queries - 1) & 1);
  if (lane == 0) reinterpret_cast<int4*>(p.ws)[blockIdx.x] = header;
}

// Keys or values of the share: one block after the other into a ring of two.  A block's boxes: lane = piece of the block * chunks +
// chunk of 64 channels.  Stays until its last copies have landed.
template <int D>
__device__ __forceinline__ void pt_stream(const PagedAttnParams& p, const CUtensorMap* map, uint8_t* ring, uint64_t* full, uint64_t* empty, PtBars& bars) {
  constexpr int BK = pt_bk(D), NCH = D / 64, BYTES = BK * D * 2;
  const int lane = threadIdx.x & 31, rows = min(BK, 1 << p.page_shift), chunk = lane % NCH, row = lane / NCH * rows;
  // This lane's page of block j: -1 where nothing is to be copied, P (out of the map's bounds: zeros) for a bad number.
  auto page_of = [&](const PtPiece& at, int j) {
    const int key = j * BK + row;
    if (row >= BK || key >= at.len) return -1;
    int n = p.table[at.b * p.ld_table + (key >> p.page_shift)];
    if (n < 0 || n >= p.P) {
      if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
      n = p.P;
    }
    return n;
  };
  uint32_t i = 0;
  bool ok = true;
  PtReader reader;
  PtPiece at{};
  while (ok && reader.next(bars, at)) {
    int page = page_of(at, at.blk);
#pragma unroll 1
    for (int j = at.blk; j < at.end; ++j, ++i) {
      const int now = page, s = i & 1;
      if (j + 1 < at.end) page = page_of(at, j + 1);
      if (i >= 2 && !__all_sync(0xffffffffu, wait_or_abort(&empty[s], ((i >> 1) & 1) ^ 1, &bars.abort))) {
        ok = false;
        break;
      }
      const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, now >= 0));
      if (lane == 0) mbar_arrive_expect_tx(&full[s], boxes * rows * 128);
      __syncwarp();
      if (now >= 0)
        tma_load_4d(ring + s * BYTES + chunk * (BK * 128) + row * 128, map, &full[s], chunk * 64, (j * BK + row) & ((1 << p.page_shift) - 1), at.g, now);
    }
  }
  __syncwarp();
  for (uint32_t k = i < 2 ? 0 : i - 2; k < i; ++k) mbar_wait(&full[k & 1], (k >> 1) & 1);
}

// Zero the values of block j that lie behind the request's last key.  By a whole warp, after the block has landed.
template <int D>
__device__ __forceinline__ void pt_clear_tail(uint8_t* block, int len, int j) {
  constexpr int BK = pt_bk(D);
  const int first = max(0, len - j * BK);
  if (first >= BK) return;
  const int n = (BK - first) * 8;
#pragma unroll 1
  for (int c = 0; c < D / 64; ++c)
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < n; i += 32) *reinterpret_cast<uint4*>(block + c * (BK * 128) + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  __syncwarp();
}

// 32 finished or partial channels of a row.
__device__ __forceinline__ void pt_store32(const PagedAttnParams& p, float* part, long long at, const uint32_t (&o)[32], float inv) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[8 * k + e]) * inv;
    if (part) {
      float4* dst = reinterpret_cast<float4*>(part + 8 * k);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      pa_store8(p, at + 8 * k, v);
    }
  }
}

// Masks, maximum, exponentials and the bf16 weights of N words of 32 scores of one row; `seen` keys of them count.
template <int N>
__device__ __forceinline__ float pt_row_max(uint32_t (&v)[N][32], int seen) {
  float mx[4] = {-1e30f, -1e30f, -1e30f, -1e30f};
#pragma unroll
  for (int w = 0; w < N; ++w) {
    if (seen < 32 * N) {
      const int left = seen - 32 * w;
      const uint32_t bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!((bits >> e) & 1u)) v[w][e] = PA_MASKED;
    }
#pragma unroll
    for (int e = 0; e < 32; e += 2) mx[w & 3] = pt_max3(mx[w & 3], __uint_as_float(v[w][e]), __uint_as_float(v[w][e + 1]));
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
__device__ __forceinline__ void pt_weights(const uint32_t (&v)[32], uint64_t c2, uint64_t nm, uint64_t& sum, uint32_t (&pk)[16]) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    float x0, x1;
    pt_unpair(pt_fma2(pt_pair(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), c2, nm), x0, x1);
    const float p0 = pa_exp2(x0), p1 = pa_exp2(x1);
    sum = pt_add2(sum, pt_pair(p0, p1));
    pk[e >> 1] = pack_bf16(p0, p1);
  }
}
__device__ __forceinline__ void pt_rescale(uint32_t t_o, int words, float f) {
#pragma unroll 1
  for (int c = 0; c < words; ++c) {
    uint32_t o[32];
    tmem_ld32(t_o + c * 32, o);
    tc_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
    tmem_st32(t_o + c * 32, o);
  }
  tc_wait_st();
}

// Set-up that both tile forms share: barriers, tensor memory, the line of key blocks.
template <int D>
__device__ __forceinline__ long long pt_begin(const PagedAttnParams& p, PtBars& bars, long long* prefix) {
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < PT_PIECES; ++i) {
      mbar_init(&bars.piece_full[i], 1);
      mbar_init(&bars.piece_read[i], 11);  // eight softmax warps, keys, values, products
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.done[i], 1);
    }
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      for (int w = 0; w < 4; ++w) {
        mbar_init(&bars.p_full[i][w], 4);
        mbar_init(&bars.pub[i][w], 1);
        mbar_init(&bars.fin[i][w], 1);
      }
    }
    mbar_init(&bars.o_free, 8);
    mbar_init(&bars.mma_done, 1);
    bars.abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars.tmem_base, 512);
    tmem_relinquish();
  }
  if (p.pdl) {
    if (tid == 0) pdl_launch_dependents();
    pdl_wait();
  }
  pa_zero_rows<D>(p, PT_THREADS);
  const long long tiles = pa_schedule<pt_bk(D), PT_THREADS>(p, prefix);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return tiles;
}

__global__ void __launch_bounds__(PT_THREADS, 1)
paged_pair_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const PagedAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ PtBars bars;
  constexpr int D = 128, BK = 128, KV = 32768, CH = 16384;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = smem + 65536, *sv = sk + 2 * KV;
  long long* prefix = reinterpret_cast<long long*>(smem + PT_SMEM - 1024);
  const long long tiles = pt_begin<D>(p, bars, prefix);
  const uint32_t tmem = bars.tmem_base;  // S / P of tile t at 128 t, O of tile t at 256 + 128 t
  const int half = p.tile_rows >> 1;     // rows of a tile

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_CONTROL));
    if (warp == 0) {
      pt_stream<D>(p, &tm_k, sk, bars.k_full, bars.k_empty, bars);
    } else if (warp == 2) {
      pt_stream<D>(p, &tm_v, sv, bars.v_full, bars.v_empty, bars);
    } else if (warp == 3) {
      pt_lead<D>(p, prefix, tiles, &tm_q, sq, bars);
    } else {
      const bool leader = elect_one();
      const uint32_t idesc_s = idesc_bf16_f32(128, BK) | p.negate_q, idesc_o = idesc_bf16_f32(128, D) | (1u << 16);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, wait_or_abort(bar, parity, &bars.abort));
        return ok;
      };
      uint32_t i = 0, i_second = 0;  // blocks so far, and those with a second tile
      PtReader reader;
      PtPiece at{};
      auto piece = [&] {
        const int nt = at.rows > half ? 2 : 1, end = at.end;
        const uint32_t n = reader.n - 1;
        auto issue_s = [&](int t, uint32_t block) {
          const uint64_t qd = smem_desc_sw128(smem_u32(sq + t * 32768)), kd = smem_desc_sw128(smem_u32(sk + (block & 1) * KV));
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t o = (ks >> 2) * (CH >> 4) + (ks & 3) * 2;
            if (leader) umma_ss_bf16(tmem + t * 128, qd + o, kd + o, idesc_s, ks > 0 ? 1u : 0u);
          }
          if (leader) tc_commit(&bars.s_full[t]);
        };
        if (!wait(&bars.q_full, n & 1) || !wait(&bars.k_full[i & 1], (i >> 1) & 1)) return false;
        tc_fence_after();
        for (int t = 0; t < nt; ++t) issue_s(t, i);
        if (leader) {
          tc_commit(&bars.k_empty[i & 1]);
          if (at.blk + 1 == end) tc_commit(&bars.q_empty);
        }
        __syncwarp();
#pragma unroll 1
        for (int j = at.blk; j < end; ++j, ++i) {
          const int s = i & 1;
          const bool more = j + 1 < end;
          if (!wait(&bars.v_full[s], (i >> 1) & 1)) return false;
          pt_clear_tail<D>(sv + s * KV, at.len, j);
          if (more && !wait(&bars.k_full[s ^ 1], ((i + 1) >> 1) & 1)) return false;
          const uint64_t v_desc = pt_desc_mn(smem_u32(sv + s * KV), CH);
          for (int t = 0; t < nt; ++t) {
            const uint32_t par = (t ? i_second : i) & 1;
#pragma unroll
            for (int part = 0; part < 4; ++part) {  // each 32 keys' product starts under the next ones' exponentials
              if (!wait(&bars.p_full[t][part], par)) return false;
              tc_fence_after();
#pragma unroll
              for (int ks = 2 * part; ks < 2 * part + 2; ++ks)
                if (leader) umma_ts_bf16(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, v_desc + ks * (2048 >> 4), idesc_o, j > at.blk || ks ? 1u : 0u);
            }
            if (more) issue_s(t, i + 1);
            else if (leader) tc_commit(&bars.done[t]);
          }
          if (leader) {
            tc_commit(&bars.v_empty[s]);
            if (more) tc_commit(&bars.k_empty[s ^ 1]);
            if (j + 2 == end) tc_commit(&bars.q_empty);
          }
          __syncwarp();
          if (nt == 2) ++i_second;
        }
        return true;
      };
      while (reader.next(bars, at) && piece()) {
      }
      ok = ok && reader.ok;
      // nothing of this CTA's tensor work may be in flight when it gives up its tensor memory
      if (leader) tc_commit(&bars.mma_done);
      __syncwarp();
      if (!ok && lane == 0) {
        bars.abort = 1;
        if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_MMA);
      }
      mbar_wait(&bars.mma_done, 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    const int t = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t t_s = tmem + t * 128 + lane_addr, t_o = tmem + 256 + t * 128 + lane_addr;
    const uint64_t c2 = pt_pair(p.abs_scale_log2e, p.abs_scale_log2e);
    const int local = t * half + row, ahead = local / p.ratio;  // row of the piece; its token's number in it
    uint32_t n = 0, i = 0;  // tiles and blocks of this group
    bool ok = true;
    PtReader reader;
    PtPiece at{};
    while (ok && reader.next(bars, at)) {
      const int nvalid = min(half, at.rows - t * half);
      if (nvalid <= 0) continue;
      const bool live = q * 32 < nvalid, mine = row < nvalid;
      const int limit = at.seen + ahead * at.step;  // keys this row sees
      float m_ref = -1e30f, l = 0.f;
#pragma unroll 1
      for (int j = at.blk; j < at.end; ++j, ++i) {
        ok = __all_sync(0xffffffffu, wait_or_abort(&bars.s_full[t], i & 1, &bars.abort, p.wait_limit));
        if (!ok) break;
        if (live) {
          tc_fence_after();
          uint32_t v[4][32];
#pragma unroll
          for (int w = 0; w < 4; ++w) tmem_ld32(t_s + w * 32, v[w]);
          tc_wait_ld();
          const float m_blk = pt_row_max<4>(v, limit - j * BK) * p.abs_scale_log2e;
          const bool grow = m_blk > m_ref + PT_RESCALE;
          if (__any_sync(0xffffffffu, grow)) {
            if (j > at.blk) {  // the scores of this block came after the last one's product
              const float f = grow ? pa_exp2(m_ref - m_blk) : 1.0f;
              pt_rescale(t_o, 4, f);
              l *= f;
            }
            if (grow) m_ref = m_blk;
          }
          const uint64_t nm = pt_pair(-m_ref, -m_ref);
          uint64_t sum[2] = {pt_pair(0.f, 0.f), pt_pair(0.f, 0.f)};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t pk[16];
            pt_weights(v[w], c2, nm, sum[w & 1], pk);
            tmem_st16(t_s + w * 16, pk);
            tc_wait_st();
            if (w < 3) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars.p_full[t][w]);
            }
          }
          float a0, a1;
          pt_unpair(pt_add2(sum[0], sum[1]), a0, a1);
          l += a0 + a1;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (!live)
            for (int w = 0; w < 3; ++w) mbar_arrive(&bars.p_full[t][w]);
          mbar_arrive(&bars.p_full[t][3]);
        }
      }
      ok = ok && __all_sync(0xffffffffu, wait_or_abort(&bars.done[t], n & 1, &bars.abort));
      ++n;
      if (ok && live) {
        tc_fence_after();
        const float inv = at.part ? 1.f : l == 0.f ? 0.f : 1.f / l;
        float* part = !at.part ? nullptr
                               : reinterpret_cast<float*>(p.ws + pa_header_bytes(gridDim.x) + (2ll * blockIdx.x + at.part - 1) * pa_part_bytes<pt_rows(D), D>());
        const long long to = static_cast<long long>(at.token + ahead) * p.ld_out + static_cast<long long>(at.g * p.ratio + local - ahead * p.ratio) * D;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tc_wait_ld();
          if (mine) pt_store32(p, part ? part + local * D + c * 32 : nullptr, to + c * 32, o, inv);
        }
        if (part && mine) {
          part[pt_rows(D) * D + local] = m_ref;
          part[pt_rows(D) * D + pt_rows(D) + local] = l;
        }
        tc_fence_before();
      }
    }
    ok = ok && reader.ok;
    if (!ok && lane == 0) {
      bars.abort = 1;
      if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_EPILOGUE);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

__global__ void __launch_bounds__(PT_THREADS, 1)
paged_wide_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const PagedAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ PtBars bars;
  constexpr int D = 256, BK = 64, KV = 32768, QCH = 16384, CH = 8192, AHEAD = 3;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = smem + 65536, *sv = sk + 2 * KV;
  long long* prefix = reinterpret_cast<long long*>(smem + PT_SMEM - 1024);
  const long long tiles = pt_begin<D>(p, bars, prefix);
  const uint32_t tmem = bars.tmem_base;  // score buffers of 64 columns at 0, 64, 128, 192, O at 256

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_CONTROL));
    if (warp == 0) {
      pt_stream<D>(p, &tm_k, sk, bars.k_full, bars.k_empty, bars);
    } else if (warp == 2) {
      pt_stream<D>(p, &tm_v, sv, bars.v_full, bars.v_empty, bars);
    } else if (warp == 3) {
      pt_lead<D>(p, prefix, tiles, &tm_q, sq, bars);
    } else {
      const bool leader = elect_one();
      const uint32_t idesc_s = idesc_bf16_f32(128, BK) | p.negate_q, idesc_o = idesc_bf16_f32(128, D) | (1u << 16);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, wait_or_abort(bar, parity, &bars.abort));
        return ok;
      };
      const uint64_t qd = smem_desc_sw128(smem_u32(sq));
      uint32_t i = 0;  // blocks so far
      PtReader reader;
      PtPiece at{};
      while (ok && reader.next(bars, at)) {
        const uint32_t n = reader.n - 1;
        auto issue_s = [&](uint32_t block) {
          if (!wait(&bars.k_full[block & 1], (block >> 1) & 1)) return;
          tc_fence_after();
          const uint64_t kd = smem_desc_sw128(smem_u32(sk + (block & 1) * KV));
#pragma unroll
          for (int ks = 0; ks < 16; ++ks) {
            const uint32_t qo = (ks >> 2) * (QCH >> 4) + (ks & 3) * 2, ko = (ks >> 2) * (CH >> 4) + (ks & 3) * 2;
            if (leader) umma_ss_bf16(tmem + (block & 3) * 64, qd + qo, kd + ko, idesc_s, ks > 0 ? 1u : 0u);
          }
          if (leader) {
            tc_commit(&bars.k_empty[block & 1]);
            tc_commit(&bars.s_full[block & 3]);
          }
          __syncwarp();
        };
        const int nb = at.end - at.blk;
        if (!wait(&bars.q_full, n & 1)) break;
#pragma unroll 1
        for (int j = -AHEAD; j < nb && ok; ++j) {
          if (j >= 0) {
            const uint32_t block = i + j;
            const int s = block & 1;
            if (j == 0 && n > 0 && !wait(&bars.o_free, (n - 1) & 1)) break;  // the last tile's output has been read
            if (!wait(&bars.v_full[s], (block >> 1) & 1)) break;
            pt_clear_tail<D>(sv + s * KV, at.len, at.blk + j);
            if (!wait(&bars.p_full[0][block & 3], (block >> 2) & 1)) break;
            tc_fence_after();
            const uint64_t v_desc = pt_desc_mn(smem_u32(sv + s * KV), CH);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              if (leader) umma_ts_bf16(tmem + 256, tmem + (block & 3) * 64 + ks * 8, v_desc + ks * (2048 >> 4), idesc_o, j > 0 || ks ? 1u : 0u);
            if (leader) {
              tc_commit(&bars.v_empty[s]);
              tc_commit(&bars.done[block & 3]);
            }
            __syncwarp();
          }
          if (j + AHEAD < nb) {
            issue_s(i + j + AHEAD);
            if (ok && j + AHEAD == nb - 1) {
              if (leader) tc_commit(&bars.q_empty);
              __syncwarp();
            }
          }
        }
        i += nb;
      }
      ok = ok && reader.ok;
      if (leader) tc_commit(&bars.mma_done);
      __syncwarp();
      if (!ok && lane == 0) {
        bars.abort = 1;
        if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_MMA);
      }
      mbar_wait(&bars.mma_done, 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    const int grp = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t t_o = tmem + 256 + lane_addr;
    const uint64_t c2 = pt_pair(p.abs_scale_log2e, p.abs_scale_log2e);
    const int ahead = row / p.ratio;  // number of the row's token in the tile
    uint32_t i = 0;                   // blocks so far (of both groups)
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, wait_or_abort(bar, parity, &bars.abort));
      return ok;
    };
    PtReader reader;
    PtPiece at{};
    auto piece = [&] {
      const uint32_t n = reader.n - 1;
      const bool live = q * 32 < at.rows, mine = row < at.rows;
      const int limit = at.seen + ahead * at.step;
      float m_own = -1e30f, l = 0.f;  // the reference that l is relative to
#pragma unroll 1
      for (int j = at.blk; j < at.end; ++j, ++i) {
        if ((i & 1) != static_cast<uint32_t>(grp)) continue;
        const uint32_t buf = i & 3;
        if (!__all_sync(0xffffffffu, wait_or_abort(&bars.s_full[buf], (i >> 2) & 1, &bars.abort, p.wait_limit))) return ok = false;
        uint32_t v[2][32];
        float m_blk = 0.f;
        const uint32_t t_s = tmem + buf * 64 + lane_addr;
        if (live) {
          tc_fence_after();
#pragma unroll
          for (int w = 0; w < 2; ++w) tmem_ld32(t_s + w * 32, v[w]);
          tc_wait_ld();
          m_blk = pt_row_max<2>(v, limit - j * BK) * p.abs_scale_log2e;
        }
        // the reference after the block before, which the other group has
        float m_ref = -1e30f;
        if (j > at.blk) {
          if (!wait(&bars.pub[grp ^ 1][q], ((i - 1) >> 1) & 1)) return false;
          m_ref = bars.m_ref[grp ^ 1][row];
        }
        const bool grow = live && m_blk > m_ref + PT_RESCALE;
        const float m_new = grow ? m_blk : m_ref;
        bars.m_ref[grp][row] = m_new;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.pub[grp][q]);
        if (live) {
          if (__any_sync(0xffffffffu, grow) && j > at.blk) {
            // The product before must have landed.  (This block's scores came after that of block i - 3, so the barrier's phase
            // before has passed, and its next waits for this block's weights.)
            if (!wait(&bars.done[(i - 1) & 3], ((i - 1) >> 2) & 1)) return false;
            tc_fence_after();
            pt_rescale(t_o, 8, grow ? pa_exp2(m_ref - m_blk) : 1.0f);
          }
          l *= pa_exp2(m_own - m_new);
          m_own = m_new;
          const uint64_t nm = pt_pair(-m_new, -m_new);
          uint64_t sum[2] = {pt_pair(0.f, 0.f), pt_pair(0.f, 0.f)};
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t pk[16];
            pt_weights(v[w], c2, nm, sum[w], pk);
            tmem_st16(t_s + w * 16, pk);
          }
          float a0, a1;
          pt_unpair(pt_add2(sum[0], sum[1]), a0, a1);
          l += a0 + a1;
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[0][buf]);
      }
      // both groups' sums, relative to the later reference
      bars.end_m[n & 1][grp][row] = m_own;
      bars.end_l[n & 1][grp][row] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.fin[grp][q]);
      if (!wait(&bars.fin[grp ^ 1][q], n & 1)) return false;
      const float m_other = bars.end_m[n & 1][grp ^ 1][row], m_end = fmaxf(m_own, m_other);
      l = l * pa_exp2(m_own - m_end) + bars.end_l[n & 1][grp ^ 1][row] * pa_exp2(m_other - m_end);
      if (!wait(&bars.done[(i - 1) & 3], ((i - 1) >> 2) & 1)) return false;
      if (live) {
        tc_fence_after();
        const float inv = at.part ? 1.f : l == 0.f ? 0.f : 1.f / l;
        float* part = !at.part ? nullptr
                               : reinterpret_cast<float*>(p.ws + pa_header_bytes(gridDim.x) + (2ll * blockIdx.x + at.part - 1) * pa_part_bytes<pt_rows(D), D>());
        const long long to = static_cast<long long>(at.token + ahead) * p.ld_out + static_cast<long long>(at.g * p.ratio + row - ahead * p.ratio) * D;
#pragma unroll 1
        for (int c = 4 * grp; c < 4 * grp + 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tc_wait_ld();
          if (mine) pt_store32(p, part ? part + row * D + c * 32 : nullptr, to + c * 32, o, inv);
        }
        if (part && mine && grp == 0) {
          part[pt_rows(D) * D + row] = m_end;
          part[pt_rows(D) * D + pt_rows(D) + row] = l;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.o_free);
      return true;
    };
    while (reader.next(bars, at) && piece()) {
    }
    ok = ok && reader.ok;
    if (!ok && lane == 0) {
      bars.abort = 1;
      if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_EPILOGUE);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the tile that CTA blockIdx.x of the kernel before began; a warp per row.
template <int ROWS, int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttnParams p, int ctas) {
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  const int4 h = reinterpret_cast<const int4*>(p.ws)[blockIdx.x];
  if (h.w == 0) return;
  const PaRequest r = pa_request(p, h.x);
  const uint8_t* parts = p.ws + pa_header_bytes(ctas);
  auto part = [&](int i) {  // the i-th part of the tile
    return reinterpret_cast<const float*>(parts + (2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * pa_part_bytes<ROWS, D>());
  };
  const int lane = threadIdx.x & 31, rows = min(p.tile_rows, r.n * p.ratio - h.z * p.tile_rows);
  for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < rows; row += gridDim.y * 4) {
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
    const int grow = h.z * p.tile_rows + row, token = grow / p.ratio;
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
}

// ------------------------------------------------------------------------------------------------ host
// Which form: the rows of a key head that the largest request is known to bring.
static bool pa_tile_form(int ratio, int max_tokens) { return ratio <= 128 && static_cast<long long>(ratio) * max_tokens > PR_ROWS; }
static int pa_form_rows(int D, bool tiles) { return tiles ? pt_rows(D) : PR_ROWS; }

static size_t pa_workspace(int D, bool tiles, int ctas) {
  return pa_header_bytes(ctas) + 2 * static_cast<size_t>(ctas) * pa_form_rows(D, tiles) * (D + 2) * 4;
}

using PaRowsKernel = void(const PagedAttnParams);
using PaTileKernel = void(const CUtensorMap, const CUtensorMap, const CUtensorMap, const PagedAttnParams);
using PaJoinKernel = void(const PagedAttnParams, int);

static int pa_set_attributes() {
  static host::DeviceCache ready;
  const int set = host::per_device(ready, [] {
    const auto smem = [](auto* kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess; };
    const int rows = PR_SMEM + 8 * (PA_MAX_REQUESTS + 1);
    const int tiles = PT_SMEM + 8 * (PA_MAX_REQUESTS + 1);
    return smem(paged_rows_kernel<128>, rows) && smem(paged_rows_kernel<256>, rows) && smem(paged_pair_kernel, tiles) && smem(paged_wide_kernel, tiles);
  });
  return set ? TYBOK_OK : host::fail_cuda("paged_attention: shared memory");
}

// Tensor map of a pool [P][G][page][D]: boxes of 64 channels and one page's rows (or a block's).
static int pa_pool_map(CUtensorMap* map, const void* base, const int64_t* strides, int P, int G, int page, int D) {
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(page), static_cast<uint64_t>(G), static_cast<uint64_t>(P)};
  const uint64_t pitch[3] = {static_cast<uint64_t>(strides[2]) * 2, static_cast<uint64_t>(strides[1]) * 2, static_cast<uint64_t>(strides[0]) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(std::min(page, pt_bk(D))), 1, 1};
  return host::tensor_map_4d(map, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, pitch, box);
}

}  // namespace tb

extern "C" {

size_t tybok_paged_attention_workspace_bytes(int H, int G, int D, int max_tokens) {
  using namespace tb;
  if (H <= 0 || G <= 0 || max_tokens <= 0 || (D != 128 && D != 256)) return 0;
  return pa_workspace(D, pa_tile_form(H / G, max_tokens), host::sm_count());
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
  // the tile forms want a scale above zero (at zero: one that no score brings above 2^-22)
  p.abs_scale_log2e = fabsf(p.scale_log2e);
  if (p.abs_scale_log2e == 0.f) p.abs_scale_log2e = std::numeric_limits<float>::denorm_min();
  p.negate_q = scale < 0.f ? 1u << 13 : 0u;
  p.wait_limit = host::epilogue_wait_limit() > 0 ? host::epilogue_wait_limit() : kWaitLimitCycles;
  p.ws = static_cast<uint8_t*>(workspace); p.status = status_word;
  p.pdl = host::pdl_enabled() ? 1 : 0;
  const bool tiles = pa_tile_form(p.ratio, max_tokens);
  p.tile_rows = !tiles ? PR_ROWS : 128 / p.ratio * p.ratio * (D == 128 ? 2 : 1);
  p.join_blocks = tiles ? (D == 128 ? 3 : 6) : 4;
  CUtensorMap tm_q, tm_k, tm_v;
  if (tiles) {
    const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.ratio), static_cast<uint64_t>(G), static_cast<uint64_t>(tokens)};
    const uint64_t pitch[3] = {static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(p.ratio) * D * 2, static_cast<uint64_t>(ldq) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(p.ratio), 1, static_cast<uint32_t>(128 / p.ratio)};
    if (int rc = host::tensor_map_4d(&tm_q, q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, pitch, box)) return rc;
    if (int rc = pa_pool_map(&tm_k, k_pages, k_strides, num_pages, G, page_size, D)) return rc;
    if (int rc = pa_pool_map(&tm_v, v_pages, v_strides, num_pages, G, page_size, D)) return rc;
  }
  if (int rc = pa_set_attributes()) return rc;
  const int ctas = host::sm_count();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(tiles ? PT_THREADS : PR_THREADS);
  cfg.dynamicSmemBytes = (tiles ? PT_SMEM : PR_SMEM) + 8 * (static_cast<size_t>(B) + 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl;
  cudaError_t e;
  if (tiles) {
    PaTileKernel* kernel = D == 256 ? paged_wide_kernel : paged_pair_kernel;
    e = cudaLaunchKernelEx(&cfg, kernel, tm_q, tm_k, tm_v, p);
  } else {
    PaRowsKernel* kernel = D == 256 ? paged_rows_kernel<256> : paged_rows_kernel<128>;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
  }
  if (e != cudaSuccess) return host::fail_cuda("launch paged_attention");
  host::count_launch();
  cfg.gridDim = dim3(ctas, tiles ? 8 : PR_ROWS / 4);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  PaJoinKernel* join = tiles ? (D == 256 ? paged_join_kernel<pt_rows(256), 256> : paged_join_kernel<pt_rows(128), 128>)
                             : (D == 256 ? paged_join_kernel<PR_ROWS, 256> : paged_join_kernel<PR_ROWS, 128>);
  if (cudaLaunchKernelEx(&cfg, join, p, ctas) != cudaSuccess) return host::fail_cuda("launch paged_join_kernel");
  host::count_launch();
  return TYBOK_OK;
}
}

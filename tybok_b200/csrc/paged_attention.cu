// Attention of new tokens over the paged cache of keys and values (layout: see paged.cu).
//
// Request b brings the n = cu[b+1] - cu[b] last of its key_lens[b] keys as queries; query i sees the keys j <= key_lens[b] - n + i
// (causal) or all of them.  Lengths are on the device, so the host sizes nothing by them: a persistent grid shares out the key
// blocks of all (request, key head, row tile) in one line, as evenly as blocks go.  A CTA's share may begin and end
// inside a tile; then it leaves (maximum, sum, unnormalised output) of its part behind, and a second kernel joins the parts in
// their order.  Queries of the same key head are rows of the same product (row = token * H / G + head).
//
// Where the tiles are few and the caches short, a cluster of CTAs takes each tile instead and joins its parts over distributed
// shared memory: no second kernel, no trip through global memory (3 requests of 10 keys, 8 heads of 256: 6.5 us against 8.6; 8 requests of
// 50 tokens over up to 970 keys: 14.7 against 21.8).
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
  uint32_t ratio_mul;
  int ratio_shift;
  int tile_rows;     // query rows (token, head of the group) of a tile, at most those of the form
  int tile_tokens;   // tokens of a tile where it holds whole ones, else 0
  int wide_out;      // the outputs are 32-byte aligned
  int join_blocks;   // what leaving a tile to two CTAs costs, in key blocks
  int tile_blocks;   // what beginning and ending a tile costs, in key blocks
  int cluster;       // > 0: one row tile per cluster of that many CTAs, which share its key blocks and join their parts themselves
  float scale_log2e;     // softmax scale * log2(e), with its sign
  float abs_scale_log2e; // its magnitude, above zero, and the bit of the scores' instruction that negates Q instead
  uint32_t negate_q;
  long long wait_limit;  // SM clocks the softmax warps wait for their scores (kWaitLimitCycles in production)
  uint8_t* ws;
  int* status;
  int pdl;
};

// n / ratio for 0 <= n < 2^31, by a product with ratio_mul = ceil(2^(31 + bits) / ratio), bits = ceil(log2(ratio)): exact for 31 bits, and no
// division (150 clocks and more) on the way to the first keys.
__device__ __forceinline__ int pa_token(const PagedAttnParams& p, int row) {
  return p.ratio == 1 ? row : static_cast<int>(__umulhi(static_cast<uint32_t>(row), p.ratio_mul) >> p.ratio_shift);
}

// What a CTA's share needs to know of one request, out of range values brought back into range.
struct PaRequest {
  int start, n, len;
};
__device__ __forceinline__ PaRequest pa_request(const PagedAttnParams& p, int b) {
  PaRequest r;
  const int lo = p.cu[b], hi = p.cu[b + 1];
  r.start = max(0, min(lo, p.T));
  r.n = max(r.start, min(hi, p.T)) - r.start;  // (cut before the difference, which could go round for a bound near -2^31)
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
  return max(0, r.len - r.n + (row_end > 0 ? pa_token(p, row_end - 1) : -1) + 1);
}
// Key blocks of a row tile; a tile that sees no key is one block of work all the same (its output is zero).
template <int BK>
__device__ __forceinline__ int pa_blocks(const PagedAttnParams& p, const PaRequest& r, int tile) {
  // (tiles of whole tokens need no division: a tile form's, or of one row per token)
  const int seen = p.tile_tokens ? (p.causal ? r.len - r.n + min(r.n, (tile + 1) * p.tile_tokens) : r.len)
                                 : pa_seen(p, r, min(r.n * p.ratio, (tile + 1) * p.tile_rows));
  return max(1, (seen + BK - 1) / BK);
}
__device__ __forceinline__ int pa_tiles(const PagedAttnParams& p, int n) {
  if (n * p.ratio <= p.tile_rows) return n > 0;
  return (n * p.ratio + p.tile_rows - 1) / p.tile_rows;
}

// ws: per CTA what the joining kernel is to know of the tile that it begins and others go on with, then two partial tiles per CTA: [0] ends
// a tile begun by another CTA, [1] begins one that others go on with.
struct __align__(16) PaHeader {
  int parts;        // CTAs that have a part of the tile; 0 = there is none to join
  int rows, first;  // rows of the tile, and the first one's number among the request's
  int start, g;     // first token of the request, key head
  int pad[3];
};
template <int ROWS, int D>
__host__ __device__ constexpr size_t pa_part_bytes() { return static_cast<size_t>(ROWS) * (D + 2) * 4; }
__host__ __device__ constexpr size_t pa_header_bytes(int ctas) { return (static_cast<size_t>(ctas) * sizeof(PaHeader) + 255) & ~size_t(255); }

// ------------------------------------------------------------------------------------------------ sixteen-row form
// Few rows per key head (single tokens): 16 rows of mma.m16n8k16, four warps that share the keys of a block and nothing else: each
// streams its own keys through its own ring and keeps its own maxima, sums and output in registers; they meet at the end of a tile.
constexpr int PR_ROWS = 16, PR_WARPS = 4, PR_THREADS = 128, PR_STAGES = 3;
constexpr int PR_SUB = 16;                                                            // keys per warp and block
constexpr int PR_BLOCK = PR_WARPS * PR_SUB;
__host__ __device__ constexpr int pr_stage(int d) { return 2 * PR_SUB * d * 2; }      // a warp's keys and values of a block
__host__ __device__ constexpr int pr_ring(int d) { return PR_WARPS * PR_STAGES * pr_stage(d); }
__host__ __device__ constexpr int pr_smem(int d) { return pr_ring(d) + PR_ROWS * (d + 2) * 4; }  // and what a cluster's CTAs send
// CTAs per SM.  At head_dim 128 one's copies go on while the other joins its warps' parts or begins a tile; at 256 the ring that keeps
// memory busy fills the SM.
__host__ __device__ constexpr int pr_ctas(int d) { return d == 128 ? 2 : 1; }

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

// The line: the key blocks of all (request, key head, row tile), numbered in that order; where the shares are long enough for it to count,
// each tile's are led by `extra` places that stand for its beginning and end.  Whole warps ask, each for itself:
// request 32 k + lane at a time, and the sums of such groups stay in the lanes.
struct PaGroup {      // 32 requests
  PaRequest r;        // this lane's
  int tiles;
  uint32_t cost, sum; // places of one of its key heads; places of all of them up to this lane's request
};
struct PaLine {
  uint32_t places, tiles;
  int extra;
  bool whole;                             // no tile is to have two CTAs
  uint32_t sums[PA_MAX_REQUESTS / 1024];  // places of group 32 i + lane
  PaGroup last;
};
__device__ __forceinline__ uint32_t pa_scan(uint32_t x) {  // inclusive sums over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) >= o) x += y;
  }
  return x;
}
// Blocks of one key head of this lane's request.
template <int BK>
__device__ __forceinline__ uint32_t pa_cost(const PagedAttnParams& p, const PaRequest& r, int tiles) {
  uint32_t cost = 0;
  if (p.cluster) return tiles;  // (a line of tiles)
  if (!p.causal) return static_cast<uint32_t>(tiles) * max(1, (r.len + BK - 1) / BK);
  const bool many = tiles > 8;  // their sums by the whole warp
  if (!many)
    for (int t = 0; t < tiles; ++t) cost += pa_blocks<BK>(p, r, t);
  for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
    const int src = __ffs(left) - 1, lane = threadIdx.x & 31;
    const PaRequest o{0, __shfl_sync(0xffffffffu, r.n, src), __shfl_sync(0xffffffffu, r.len, src)};
    const int n = __shfl_sync(0xffffffffu, tiles, src);
    uint32_t sum = 0;
    for (int t = lane; t < n; t += 32) sum += pa_blocks<BK>(p, o, t);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == src) cost = sum;
  }
  return cost;
}
template <int BK>
__device__ __forceinline__ PaGroup pa_group(const PagedAttnParams& p, int k, int extra) {
  const int b = 32 * k + (threadIdx.x & 31);
  PaGroup g;
  g.r = {0, 0, 0};
  if (b < p.B) g.r = pa_request(p, b);
  g.tiles = pa_tiles(p, g.r.n);
  g.cost = pa_cost<BK>(p, g.r, g.tiles) + g.tiles * extra;
  g.sum = pa_scan(g.cost * p.G);
  return g;
}
template <int BK>
__device__ __forceinline__ PaLine pa_line(const PagedAttnParams& p) {
  const int lane = threadIdx.x & 31;
  PaLine line{};
  int longest = 0;  // tile, in blocks
  uint32_t tiles[PA_MAX_REQUESTS / 1024] = {}, all_tiles = 0;  // up to this lane's request in the last group
#pragma unroll 1
  for (int k = 0; 32 * k < p.B; ++k) {
    line.last = pa_group<BK>(p, k, 0);
    all_tiles = pa_scan(static_cast<uint32_t>(line.last.tiles) * p.G);
    if (!p.cluster && line.last.tiles > 0) longest = max(longest, pa_blocks<BK>(p, line.last.r, line.last.tiles - 1));
    const uint32_t sum = __shfl_sync(0xffffffffu, line.last.sum, 31), count = __shfl_sync(0xffffffffu, all_tiles, 31);
#pragma unroll
    for (int i = 0; i < PA_MAX_REQUESTS / 1024; ++i)
      if (k == 32 * i + lane) line.sums[i] = sum, tiles[i] = count;
    line.places += sum;
    line.tiles += count;
  }
  if (p.cluster) return line;
  const uint32_t ctas = gridDim.x;
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (line.places >= p.tile_blocks * ctas) line.extra = p.tile_blocks;
  const uint32_t per = (line.places + line.tiles * line.extra + ctas - 1) / ctas;
  line.whole = static_cast<float>((line.tiles + ctas - 1) / ctas) * (longest + line.extra) <= static_cast<float>(per + line.extra + p.join_blocks);
  if (line.whole) line.extra = 0;  // about equal tiles
  line.places += line.tiles * line.extra;
#pragma unroll
  for (int i = 0; i < PA_MAX_REQUESTS / 1024; ++i) line.sums[i] += tiles[i] * line.extra;
  line.last.cost += line.last.tiles * line.extra;
  line.last.sum += all_tiles * line.extra;
  return line;
}

// A place in the line: place `blk` of `nblk` of row tile `tile` of key head `g` of request `b`.
struct PaPlace {
  int b, g, tile, blk, nblk, tiles;
  PaRequest r;
};
// Where place x < line.places lies.
template <int BK>
__device__ __forceinline__ PaPlace pa_locate(const PagedAttnParams& p, const PaLine& line, uint32_t x) {
  const int lane = threadIdx.x & 31;
  int k = 0;
  PaGroup g = line.last;
  if (p.B > 32) {
    uint32_t before = 0;
#pragma unroll 1
    for (int i = 0; i < PA_MAX_REQUESTS / 1024; ++i) {
      const uint32_t sum = pa_scan(line.sums[i]) + before, past = __ballot_sync(0xffffffffu, sum <= x);
      k += __popc(past);
      before = __shfl_sync(0xffffffffu, sum, 31);
      if (past != 0xffffffffu) {
        const int at = __popc(past);
        x -= __shfl_sync(0xffffffffu, sum, at) - __shfl_sync(0xffffffffu, line.sums[i], at);
        break;
      }
    }
    g = pa_group<BK>(p, k, line.extra);
  }
  const int src = __popc(__ballot_sync(0xffffffffu, g.sum <= x));
  const uint32_t per_head = __shfl_sync(0xffffffffu, g.cost, src);
  x -= __shfl_sync(0xffffffffu, g.sum, src) - per_head * p.G;
  PaPlace at{};
  at.b = min(32 * k + src, p.B - 1);  // (only tokens counted many times over could lead beyond the line)
  at.r = {__shfl_sync(0xffffffffu, g.r.start, src), __shfl_sync(0xffffffffu, g.r.n, src), __shfl_sync(0xffffffffu, g.r.len, src)};
  at.tiles = __shfl_sync(0xffffffffu, g.tiles, src);
  at.g = p.G == 1 ? 0 : static_cast<int>(min(x / max(per_head, 1u), p.G - 1u));
  x -= at.g * per_head;
  if (p.cluster) {
    at.tile = static_cast<int>(x);
    at.blk = 0;
    at.nblk = pa_blocks<BK>(p, at.r, at.tile);
    return at;
  }
  if (!p.causal) {
    at.nblk = max(1, (at.r.len + BK - 1) / BK) + line.extra;
    at.tile = static_cast<int>(x / at.nblk);
    at.blk = static_cast<int>(x) - at.tile * at.nblk;
    return at;
  }
#pragma unroll 1
  for (at.tile = 0; at.tile < at.tiles; at.tile += 32) {  // 32 tiles at a time
    const uint32_t n = at.tile + lane < at.tiles ? pa_blocks<BK>(p, at.r, at.tile + lane) + line.extra : 0, to = pa_scan(n);
    const uint32_t past = __ballot_sync(0xffffffffu, to <= x);
    if (past != 0xffffffffu) {
      const int i = __popc(past);
      at.tile += i;
      at.nblk = __shfl_sync(0xffffffffu, n, i);
      at.blk = static_cast<int>(x - (__shfl_sync(0xffffffffu, to, i) - at.nblk));
      return at;
    }
    x -= __shfl_sync(0xffffffffu, to, 31);
  }
  return at;  // (not reached: x lies in the line)
}
// The tile after this one (the caller knows that there is one).
template <int BK>
__device__ __forceinline__ void pa_next(const PagedAttnParams& p, PaPlace& at, int extra) {
  if (++at.tile == at.tiles) {
    at.tile = 0;
    if (++at.g == p.G) {
      at.g = 0;
      do {
        at.b = min(at.b + 1, p.B - 1);
        at.r = pa_request(p, at.b);
      } while (at.r.n == 0 && at.b + 1 < p.B);
      at.tiles = pa_tiles(p, at.r.n);
    }
  }
  at.blk = 0;
  at.nblk = pa_blocks<BK>(p, at.r, at.tile) + extra;
}

// A CTA's share [x0, x1) of the line: equal numbers of places, borders moved to the edge of a tile that lies near (and from a tile's
// leading places to its beginning).  With `whole` every border moves to the nearest edge: where the rounds of the longest tile take
// no longer than an even share, the second beginning that it brings and the joining of its parts.
struct PaShare {
  uint32_t per, x0, x1;
  int extra;
  bool whole;
};
__device__ __forceinline__ int pa_snap(const PaShare& sh, int blk, int nblk, int join_blocks) {
  const bool up = 2 * blk > nblk;
  const int away = up ? nblk - blk : blk;
  if (sh.whole || 4 * away <= static_cast<int>(min(sh.per, 4u * join_blocks)) - 4) return up ? nblk : 0;
  return blk <= sh.extra ? 0 : blk;
}
// Where share `number` begins, and the place there.
template <int BK>
__device__ __forceinline__ uint32_t pa_border(const PagedAttnParams& p, const PaLine& line, const PaShare& sh, unsigned number, PaPlace& next) {
  const unsigned long long x = static_cast<unsigned long long>(number) * sh.per;
  if (x >= line.places) return line.places;
  next = pa_locate<BK>(p, line, static_cast<uint32_t>(x));
  const int blk = pa_snap(sh, next.blk, next.nblk, p.join_blocks);
  const uint32_t border = static_cast<uint32_t>(x) - next.blk + blk;
  next.blk = blk;
  return border;
}
template <int BK>
__device__ PaShare pa_share(const PagedAttnParams& p, PaPlace& first) {
  const PaLine line = pa_line<BK>(p);
  PaShare sh;
  sh.extra = line.extra;
  sh.whole = line.whole;
  if (p.cluster) {  // tile number blockIdx.x / cluster; `per` blocks of it to each CTA
    sh.per = sh.x0 = sh.x1 = 0;
    const uint32_t x = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
    if (x >= line.tiles) return sh;
    first = pa_locate<BK>(p, line, x);
    sh.per = (first.nblk + p.cluster - 1) / p.cluster;
    first.blk = min(static_cast<uint32_t>(first.nblk), rank * sh.per);
    sh.x1 = min(static_cast<uint32_t>(first.nblk) - first.blk, sh.per);
    return sh;
  }
  sh.per = (line.places + gridDim.x - 1) / gridDim.x;
#pragma unroll 1
  for (int i = 1; i >= 0; --i) {
    const uint32_t border = pa_border<BK>(p, line, sh, blockIdx.x + i, first);
    if (i) sh.x1 = border;
    else sh.x0 = border;
  }
  if (sh.x0 < sh.x1 && first.blk == first.nblk) pa_next<BK>(p, first, sh.extra);
  return sh;
}
__device__ __forceinline__ void pa_send4(uint32_t to, float4 v) {  // to another CTA of the cluster
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void pa_send(const void* local, int rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dsmem_addr(smem_u32(local), rank)), "f"(v) : "memory");
}

// How many CTAs the tile has that begins at x in this CTA's share and goes on behind it.
__device__ __forceinline__ int pa_parts(const PagedAttnParams& p, const PaShare& sh, uint32_t x, int nblk) {
  const uint32_t last = (x + nblk - 1) / sh.per;
  const int blk = static_cast<int>(last * sh.per - x);
  const bool gone = last > blockIdx.x && blk > 0 && pa_snap(sh, blk, nblk, p.join_blocks) == nblk;  // its border moved behind the tile
  return static_cast<int>(last - blockIdx.x) + (gone ? 0 : 1);
}
// Lengths that reach beyond what they index: the status word says so (the kernels cut them).
__device__ __forceinline__ void pa_check(const PagedAttnParams& p, int t, int nt) {
  if (blockIdx.x != 0 || !p.status) return;
  for (int b = t; b < p.B; b += nt)
    if (!pa_in_range(p, b)) atomicCAS(p.status, 0, TYBOK_DEV_BAD_INDEX);
}

// Output rows that belong to no request are zero.
template <int D>
__device__ __forceinline__ void pa_zero_rows(const PagedAttnParams& p, int t, int nt) {
  const int first = max(0, min(p.cu[0], p.T)), last = max(first, min(p.cu[p.B], p.T));
  const long long per = p.ld_out / 8, rows = p.T - last + first, n = rows * per;
  const float zero[8] = {};
  for (long long i = static_cast<long long>(blockIdx.x) * nt + t; i < n; i += static_cast<long long>(gridDim.x) * nt) {
    const long long row = i / per, c = i - row * per;
    pa_store8(p, (row < first ? row : row - first + last) * p.ld_out + c * 8, zero);
  }
}

template <int D>
__global__ void __launch_bounds__(PR_THREADS, pr_ctas(D)) paged_rows_kernel(const PagedAttnParams p) {
  extern __shared__ __align__(128) uint8_t pr_shared[];
  __shared__ float s_m[PR_WARPS][PR_ROWS], s_l[PR_WARPS][PR_ROWS];
  constexpr int SUB = PR_SUB, BK = PR_BLOCK, STAGE = pr_stage(D), ROW_BYTES = D * 2, CHUNKS = D / 8, KS = D / 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.cluster) cluster_arrive_relaxed();  // this CTA is there: its shared memory may be written
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  PaPlace at{};
  const PaShare share = pa_share<BK>(p, at);
  const uint32_t x1 = share.x1;
  uint32_t x = share.x0;
  PaHeader header{};
  // cluster: [CTA][row of this CTA's share][D], then the references and the sums, as the CTAs send them
  float* parts = reinterpret_cast<float*>(pr_shared + pr_ring(D));
  const int each = p.cluster ? PR_ROWS / p.cluster : PR_ROWS, each_bits = __ffs(each) - 1, rank = p.cluster ? static_cast<int>(cluster_ctarank()) : 0;
  bool tidied = false;
  auto tidy = [&] {  // under the first keys' way
    pa_check(p, tid, PR_THREADS);
    pa_zero_rows<D>(p, tid, PR_THREADS);
    tidied = true;
  };
  const uint32_t ring = smem_u32(pr_shared) + warp * (PR_STAGES * STAGE);
  while (x < x1) {
    const int end = static_cast<int>(min(static_cast<uint32_t>(at.nblk), at.blk + (x1 - x)));
    const int rows = at.r.n * p.ratio;
    const int seen = pa_seen(p, at.r, min(rows, (at.tile + 1) * PR_ROWS));                    // by any row
    const int seen_all = p.causal ? max(0, at.r.len - at.r.n + pa_token(p, at.tile * PR_ROWS) + 1) : at.r.len;  // by every row
    uint32_t in = 0, out = 0;  // ring slots
    auto fetch = [&](int j) {  // this warp's keys of block j
      const uint32_t slot = ring + in * STAGE;
      in = in + 1 == PR_STAGES ? 0 : in + 1;
      const int key = j * BK + warp * SUB;  // sixteen keys lie in one page
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
      for (int i = 0; i < SUB * CHUNKS / 32; ++i) {
        const int r = (i * 32 + lane) / CHUNKS, c = (i * 32 + lane) % CHUNKS;
        const int bytes = page >= 0 && key + r < seen ? 16 : 0;  // the others are zero
        const uint32_t dst = slot + r * ROW_BYTES + ((c ^ (r & 7)) << 4);
        const long long rr = bytes ? r : 0;
        cp_async16(dst, ks + rr * p.k_row + c * 8, bytes);
        cp_async16(dst + SUB * ROW_BYTES, vs + rr * p.v_row + c * 8, bytes);
      }
    };
    uint32_t qf[KS][4];
    int limit[2];
    // this thread's two rows of the tile: queries as operand fragments, keys they see
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = at.tile * PR_ROWS + h * 8 + (lane >> 2), token = pa_token(p, row);
      const bool live = row < rows;
      limit[h] = !live ? 0 : p.causal ? max(0, at.r.len - at.r.n + token + 1) : at.r.len;
      const __nv_bfloat16* src = p.q + (at.r.start + token) * p.ldq + static_cast<long long>(at.g * p.ratio + row - token * p.ratio) * D + (lane & 3) * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[ks][h] = live ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
        qf[ks][h + 2] = live ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
    for (int j = at.blk - (PR_STAGES - 1); j < end; ++j) {  // (the code that fetches once)
      if (j + PR_STAGES - 1 < end) fetch(j + PR_STAGES - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (j < at.blk) continue;
      if (j == at.blk && !tidied) tidy();
      asm volatile("cp.async.wait_group %0;" ::"n"(PR_STAGES - 1) : "memory");
      __syncwarp();
      const int key0 = j * BK + warp * SUB;
      const uint32_t ka = ring + out * STAGE, va = ka + SUB * ROW_BYTES;
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
      out = out + 1 == PR_STAGES ? 0 : out + 1;
      __syncwarp();
    }
    // the four warps' parts meet
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    float* mine = reinterpret_cast<float*>(pr_shared + warp * (PR_STAGES * STAGE));
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
    if (p.cluster) cluster_wait_acquire();  // the others are there
    float* po = reinterpret_cast<float*>(p.ws + pa_header_bytes(gridDim.x) + (2ll * blockIdx.x + part) * pa_part_bytes<PR_ROWS, D>());
#pragma unroll
    for (int i = tid; i < PR_ROWS * D / 8; i += PR_THREADS) {
      const int row = i / (D / 8), c = (i % (D / 8)) * 8;
      float f[PR_WARPS], top = -INFINITY, sum = 0.f, v[8] = {};
#pragma unroll
      for (int w = 0; w < PR_WARPS; ++w) top = fmaxf(top, s_m[w][row]);
#pragma unroll
      for (int w = 0; w < PR_WARPS; ++w) {
        f[w] = pa_exp2(s_m[w][row] - (top == -INFINITY ? 0.f : top));
        sum += f[w] * s_l[w][row];
        const float4* src = reinterpret_cast<const float4*>(pr_shared + w * (PR_STAGES * STAGE)) + (row * D + (c ^ ((row & 3) << 3))) / 4;
        const float4 a = src[0], b = src[1];
        v[0] += f[w] * a.x; v[1] += f[w] * a.y; v[2] += f[w] * a.z; v[3] += f[w] * a.w;
        v[4] += f[w] * b.x; v[5] += f[w] * b.y; v[6] += f[w] * b.z; v[7] += f[w] * b.w;
      }
      const int grow = at.tile * PR_ROWS + row;
      if (grow >= rows) continue;
      if (whole_tile) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inv;
        const int token = pa_token(p, grow);
        pa_store8(p, (at.r.start + token) * p.ld_out + static_cast<long long>(at.g * p.ratio + grow - token * p.ratio) * D + c, v);
      } else if (p.cluster) {
        const int owner = row >> each_bits, at_owner = rank * each + (row & (each - 1));
        const uint32_t to = dsmem_addr(smem_u32(parts + at_owner * D + c), owner);
        pa_send4(to, make_float4(v[0], v[1], v[2], v[3]));
        pa_send4(to + 16, make_float4(v[4], v[5], v[6], v[7]));
        if (c == 0) {
          pa_send(parts + PR_ROWS * D + at_owner, owner, top);
          pa_send(parts + PR_ROWS * D + PR_ROWS + at_owner, owner, sum);
        }
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
    if (p.cluster) break;
    if (!whole_tile && at.blk == 0) header = {pa_parts(p, share, x, at.nblk), min(PR_ROWS, rows - at.tile * PR_ROWS), at.tile * PR_ROWS, at.r.start, at.g};
    x += end - at.blk;
    __syncthreads();  // the ring is free again
    if (x < x1) pa_next<BK>(p, at, 0);
  }
  if (!tidied) tidy();
  if (!p.cluster) {
    if (tid == 0) reinterpret_cast<PaHeader*>(p.ws)[blockIdx.x] = header;
    return;
  }
  const bool alone = share.per > 0 && share.per >= static_cast<uint32_t>(at.nblk);  // one CTA of the cluster has had all of the tile
  if (x == x1) {  // a CTA without blocks has nothing to add
    cluster_wait_acquire();
    if (share.per > 0 && !alone && tid < PR_ROWS) pa_send(parts + PR_ROWS * D + rank * each + (tid & (each - 1)), tid >> each_bits, -INFINITY);
  }
  if (alone) return;
  __syncwarp();
  cluster_sync_all();  // every part has arrived
  if (share.per == 0) return;  // no tile for the whole cluster
  const int rows = at.r.n * p.ratio;
  for (int i = tid; i < each * D / 8; i += PR_THREADS) {
    const int mine = i / (D / 8), c = (i % (D / 8)) * 8, row = rank * each + mine, grow = at.tile * PR_ROWS + row;
    if (grow >= rows) continue;
    float m[8], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = k < p.cluster ? parts[PR_ROWS * D + k * each + mine] : -INFINITY;
      top = fmaxf(top, m[k]);
    }
    float sum = 0.f, v[8] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (m[k] == -INFINITY) continue;
      const float f = pa_exp2(m[k] - top);
      sum += f * parts[PR_ROWS * D + PR_ROWS + k * each + mine];
      const float4* src = reinterpret_cast<const float4*>(parts + (k * each + mine) * D + c);
      const float4 a = src[0], b = src[1];
      v[0] += f * a.x; v[1] += f * a.y; v[2] += f * a.z; v[3] += f * a.w;
      v[4] += f * b.x; v[5] += f * b.y; v[6] += f * b.z; v[7] += f * b.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inv;
    const int token = pa_token(p, grow);
    pa_store8(p, (at.r.start + token) * p.ld_out + static_cast<long long>(at.g * p.ratio + grow - token * p.ratio) * D + c, v);
  }
}

// ------------------------------------------------------------------------------------------------ tile forms
// Many rows per key head: 128-row tiles on the fifth-generation tensor cores.  Four control warps (keys, products, values, and the
// CTA's share with the queries) and two groups of four softmax warps with one query row per thread and tensor-memory
// lane.  The warp that walks the CTA's share tells the others, a few tiles ahead; rings and barriers run on from tile to tile, so
// the next tile's queries, keys and first scores are on their way while this one's output is written.
//   S = Q K^T into tensor memory, P = 2^(S c - m) in bf16 over it (m: a reference that moves only when a block's maximum exceeds
//   it by more than 2^8, then the row of O is rescaled), O += P V with P read from tensor memory.
//   head_dim 128 (paged_pair_kernel): two tiles of 128 rows share every block of 128 keys, a group of softmax warps each; queries in
//            shared memory.  Tensor memory: S / P and O of both tiles, 128 columns each; a tile's S(j+1) follows its PV(j).
//            One warp issues the products of both, so the tiles take turns: one's products run under the other's exponentials
//            (a warp for each fell into step with the other: 562 to 600 us against 530 on 2 requests of 2048 tokens over
//            8250 keys; blocks of 64 keys with scores in two buffers 597).  Bound by the exponentials (2048 of the special-function unit's
//            clocks a block), the products (2048) and the hand-overs between them: 3450 clocks a block.
//   head_dim 256 (paged_wide_kernel): O of one tile takes half of the tensor memory.  The groups take every other block of 64 keys, with a
//            score buffer each: PV(j), S(j+2).  The queries are in tensor memory too: as a shared-memory operand their 64 KB
//            would be read again for every 64 keys, and with the keys, the values and what the copies write, shared
//            memory (128 bytes a clock) would set the pace (1790 clocks a block, and 1570 so, of which 1024 are products).
// Measured on a B200: 32 heads on 8 key heads of 128, 2 requests of 2048 new tokens over 8250 keys each, causal, 425 us once and
// 470 to 490 back to back under the power cap, 1.0 to 1.1 PF/s; 16 + 16 heads of 128, 19 requests from one token to 700 over up to 5000
// keys 56 us; 8 heads on 1 of 256: 8 requests of 50 tokens over up to 970 keys 14.7 us, 5 of 402 to 627 tokens over themselves 30.5.
// A page is one box of the tensor map and 64 channels (or a block's rows of a larger page); lanes of the copying warp issue one
// box each.  Page numbers out of range read as zero through the map's bounds.
// Values behind a request's last key are zeroed in shared memory before their product (their weights are zero, but what lies
// there may be anything).
constexpr int PT_THREADS = 384;
constexpr int PT_REGS_CONTROL = 72, PT_REGS_SOFTMAX = 216;  // launched with 168 each: 72 + 2 * 216 = 3 * 168
constexpr int PT_SMEM = 196608 + 1024;  // queries, two key and two value blocks
constexpr float PT_RESCALE = 8.0f;
#define PA_MASKED 0xff800000u  // -infinity
// Where a row's reference starts, and its least value: finite, so that a masked score's distance from it is -infinity and not NaN, and
// below every finite score.
constexpr float PT_LOWEST = -3.402823466e38f;

__host__ __device__ constexpr int pt_rows(int d) { return d == 128 ? 256 : 128; }  // of a work item
__host__ __device__ constexpr int pt_bk(int d) { return d == 128 ? 128 : 64; }     // keys of a block (32 KB)

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

// 4-D tiled load (crd0 innermost).
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int crd0, int crd1, int crd2, int crd3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(crd0), "r"(crd1), "r"(crd2), "r"(crd3)
      : "memory");
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
constexpr int PT_PIECES = 4;  // (the barriers below come in fours)

struct __align__(16) PtBars {
  PtPiece piece[PT_PIECES];
  uint64_t piece_full[PT_PIECES], piece_read[PT_PIECES];
  uint64_t q_full, q_empty;      // the queries of a tile have landed in shared memory; may be overwritten there
  uint64_t q_in, q_used;         // wide: they are in tensor memory; may be overwritten there
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2];            // pair: per tile; wide: per score buffer
  uint64_t p_full[2][4];         // the same, and 32 of the block's keys
  uint64_t done[2];              // pair: per tile, its last product has landed; wide: [block % 2], the block's product has
  uint64_t o_free;        // wide: the output of a tile has been read
  uint64_t pub[2][4];     // wide: per group and warp: the reference maximum after this block
  uint64_t fin[2][2][4];  // the same, per parity of the tile: its sums at the tile's end
  uint64_t mma_done;
  uint32_t tmem_base;
  volatile int abort;
  float m_ref[2][128];                       // wide: per group and row
  float end_m[2][2][128], end_l[2][2][128];  // wide: per parity of the tile, group and row
  PtPiece item;                              // cluster: the tile (rows = 0: none), and this CTA's part of its statistics
  float part_m[256], part_l[256];
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

// Several barriers in the time of one: a wait is a round trip of a hundred clocks even where the phase has passed, and lanes can ask for
// different ones.
struct PtWait {
  uint64_t* bar;
  uint32_t parity;
};
__device__ __forceinline__ bool pt_wait(const PtWait& a, const PtWait& b, const PtWait& c, volatile int* abort_flag) {
  const int which = threadIdx.x & 3;
  return __all_sync(0xffffffffu, wait_or_abort(which == 0 ? a.bar : which == 1 ? b.bar : c.bar, which == 0 ? a.parity : which == 1 ? b.parity : c.parity, abort_flag));
}

// How many of a block's weights (32 keys at a time) after the first have been handed over, in their order.
template <int N>
__device__ __forceinline__ int pt_handed(uint64_t* handed, uint32_t parity) {
  const int lane = threadIdx.x & 31;
  return __ffs(~__ballot_sync(0xffffffffu, lane < N - 1 && mbar_test_wait(&handed[1 + min(lane, N - 2)], parity))) - 1;
}

// What an issuing warp is about to need: a block's weights, 32 keys at a time (parts), its values, and the keys of the scores after it.  A wait
// is a round trip of a hundred clocks even where the phase has passed, and the tensor core runs dry meanwhile (it holds a
// few instructions).  So lanes ask for different barriers at once, and for a turn while the one before is still being issued.
struct PtTurn {
  uint64_t *parts, *values, *keys;
  uint32_t part_parity, value_parity, key_parity;
  bool more;  // the keys count
  // The barrier that this lane asks for.
  template <int N>
  __device__ __forceinline__ bool lane_done(int lane) const {
    uint64_t* bar = lane < N ? parts + lane : lane == N ? values : keys;
    const uint32_t parity = lane < N ? part_parity : lane == N ? value_parity : key_parity;
    return lane > N + 1 || (lane == N + 1 && !more) || mbar_test_wait(bar, parity & 1);
  }
  // Parts that need no wait: none unless the values and keys are there.
  template <int N>
  __device__ __forceinline__ int ready() const {
    const uint32_t done = __ballot_sync(0xffffffffu, lane_done<N>(threadIdx.x & 31));
    return ((done >> N) & 3u) == 3u ? __ffs(~(done & ((1u << N) - 1u))) - 1 : 0;
  }
  // Until the values, the keys and one part are there; 0 when the CTA has given up.
  template <int N>
  __device__ __forceinline__ int wait(volatile int* abort_flag) const {
    int n = ready<N>();
    const long long t0 = clock64();
    while (n == 0) {
      if (*abort_flag || clock64() - t0 > kWaitLimitCycles) break;
      n = ready<N>();
    }
    return __shfl_sync(0xffffffffu, n, 0);
  }
};

// Products whose descriptors differ in the low word only (start address, leading offset): the high word (stride 1024 bytes, version,
// 128-byte swizzle) is a constant.
constexpr uint32_t PT_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t pt_desc_lo(uint32_t smem_addr, uint32_t chunk_bytes) { return (smem_addr & 0x3FFFF) >> 4 | chunk_bytes >> 4 << 16; }
// By the lane with `leader` set; predicated, so that the warp's control flow stays uniform.
__device__ __forceinline__ void pt_mma_ss(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(PT_DESC_HI), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(PT_DESC_HI), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void pt_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}

// The same value in every lane, known to the compiler as such (a reduction ends in a uniform register).  The operands of the tensor-core
// instructions are uniform registers: from values that only happen to agree, each instruction pays for moving its own.
__device__ __forceinline__ int pt_uniform(int x) { return static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<uint32_t>(x))); }

// The walk over the CTA's share, and its queries: one or two tiles of whole tokens per piece.  Leaves the header for the joining kernel
// behind.
template <int D>
__device__ __forceinline__ void pt_lead(const PagedAttnParams& p, PaPlace at, const PaShare& share, const CUtensorMap* map, uint8_t* sq, PtBars& bars) {
  constexpr int NCH = D / 64, CH = 16384, TILES = pt_rows(D) / 128;
  const int lane = threadIdx.x & 31, tokens = p.tile_tokens / TILES, half = tokens * p.ratio;
  PaHeader header{};
  if (p.cluster && lane == 0) {
    PtPiece w{};
    if (share.per > 0) {
      w.rows = min(p.tile_rows, at.r.n * p.ratio - at.tile * p.tile_rows);
      w.g = at.g;
      w.token = at.r.start + at.tile * p.tile_tokens;
    }
    bars.item = w;
  }
  uint32_t n = 0, queries = 0;
  bool ok = true;
  uint32_t x = share.x0;
  while (true) {
    const uint32_t s = n % PT_PIECES;
    if (n >= PT_PIECES) ok = __all_sync(0xffffffffu, wait_or_abort(&bars.piece_read[s], (n / PT_PIECES - 1) & 1, &bars.abort));
    if (!ok) break;
    const bool any = x < share.x1;
    int end = 0;
    PtPiece w{};
    if (any) {
      const int first = at.tile * p.tile_tokens;
      w.rows = min(p.tile_rows, at.r.n * p.ratio - at.tile * p.tile_rows);
      w.b = at.b;
      w.g = at.g;
      end = static_cast<int>(min(static_cast<uint32_t>(at.nblk), at.blk + (share.x1 - x)));
      w.blk = max(0, at.blk - share.extra);
      w.end = end - share.extra;
      w.len = at.r.len;
      w.seen = p.causal ? at.r.len - at.r.n + first + 1 : at.r.len;
      w.step = p.causal;
      w.token = at.r.start + first;
      w.part = p.cluster ? 1 : at.blk == 0 && end == at.nblk ? 0 : at.blk > 0 ? 1 : 2;
      if (w.part == 2) header = {pa_parts(p, share, x, at.nblk), w.rows, at.tile * p.tile_rows, at.r.start, at.g};
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
    x += end - at.blk;
    if (x < share.x1) pa_next<pt_bk(D)>(p, at, share.extra);
  }
  if (queries > 0) mbar_wait(&bars.q_full, (queries - 1) & 1);
  if (lane == 0 && !p.cluster) reinterpret_cast<PaHeader*>(p.ws)[blockIdx.x] = header;
}

// Keys or values of the share: one block after the other into a ring of two.  A block's boxes: lane = piece of the block * chunks + chunk of
// 64 channels.  Stays until its last copies have landed.
struct PtRing {
  const CUtensorMap* map;
  uint8_t* at;
  uint64_t *full, *empty;
};
template <int D>
__device__ __forceinline__ void pt_stream(const PagedAttnParams& p, const PtRing& ring, PtBars& bars) {
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
  uint32_t blocks = 0, i = 0;  // blocks requested; blocks begun
  bool ok = true;
  PtReader reader;
  PtPiece at{};
  while (ok && reader.next(bars, at)) {
    int page = page_of(at, at.blk);
#pragma unroll 1
    for (int j = at.blk; j < at.end && ok; ++j, ++i) {
      const int now = page, s = i & 1, off = (j * BK + row) & ((1 << p.page_shift) - 1);
      if (j + 1 < at.end) page = page_of(at, j + 1);
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, now >= 0)) * rows * 128, par = ((i >> 1) & 1) ^ 1;
      if (i >= 2) ok = __all_sync(0xffffffffu, wait_or_abort(&ring.empty[s], par, &bars.abort));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&ring.full[s], bytes);
      __syncwarp();
      if (now >= 0) tma_load_4d(ring.at + s * BYTES + chunk * (BK * 128) + row * 128, ring.map, &ring.full[s], chunk * 64, off, at.g, now);
      blocks = i + 1;
    }
  }
  __syncwarp();
  for (uint32_t k = blocks < 2 ? 0 : blocks - 2; k < blocks; ++k) mbar_wait(&ring.full[k & 1], (k >> 1) & 1);
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
#pragma unroll(D == 256 ? 4 : 1)
    for (int i = threadIdx.x & 31; i < n; i += 32) *reinterpret_cast<uint4*>(block + c * (BK * 128) + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  __syncwarp();
}

// 32 bytes of registers (r[first] ..) to global memory: one 256-bit store, or two of 128 bits where the caller's tensor is
// only 16-byte aligned.
template <int N>
__device__ __forceinline__ void pt_store_32b(void* dst, const uint32_t (&r)[N], int first, int wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(r[first]), "r"(r[first + 1]), "r"(r[first + 2]),
                 "r"(r[first + 3]), "r"(r[first + 4]), "r"(r[first + 5]), "r"(r[first + 6]), "r"(r[first + 7])
                 : "memory");
  } else {
    uint4* d = static_cast<uint4*>(dst);
    d[0] = make_uint4(r[first], r[first + 1], r[first + 2], r[first + 3]);
    d[1] = make_uint4(r[first + 4], r[first + 5], r[first + 6], r[first + 7]);
  }
}
// 32 channels of a finished row, `at` elements into the output: whole 32-byte sectors straight from a thread's registers.
__device__ __forceinline__ void pt_store32(const PagedAttnParams& p, long long at, const uint32_t (&o)[32], float inv) {
  uint32_t ob[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) ob[e] = pack_bf16(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
  if (p.out) {
    pt_store_32b(p.out + at, ob, 0, p.wide_out);
    pt_store_32b(p.out + at + 16, ob, 8, p.wide_out);
  }
  if (p.out_planes) {
    uint32_t w[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x[4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ob[2 * e + k]));
        x[2 * k] = f.x * p.plane_scale;
        x[2 * k + 1] = f.y * p.plane_scale;
      }
      split3_quad(x, w[0][e], w[1][e], w[2][e]);
    }
    const long long plane = static_cast<long long>(p.T) * p.ld_out;
#pragma unroll
    for (int k = 0; k < 3; ++k) pt_store_32b(p.out_planes + k * plane + at, w[k], 0, p.wide_out);
  }
}
// A partial tile in the workspace: four channels of 128 rows side by side, so that a warp's rows are one run: float4 number
// [column / 4][row].
__device__ __forceinline__ void pt_part32(float4* part, int column, int row, const uint32_t (&o)[32]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    part[(column / 4 + e) * 128 + row] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
}

// Masks, maximum, exponentials and the bf16 weights of 32 scores of one row, of which the first `left` keys count.
template <int N>
__device__ __forceinline__ void pt_row_max(uint32_t (&v)[32], int left, float (&mx)[N]) {
  if (left < 32) {
    const uint32_t bits = left <= 0 ? 0u : (1u << left) - 1u;
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (!((bits >> e) & 1u)) v[e] = PA_MASKED;
  }
#pragma unroll
  for (int e = 0; e < 32; e += 2) mx[(e >> 1) % N] = pt_max3(mx[(e >> 1) % N], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
}
// Ties 32 registers to this point of the program: their load has been waited for.
__device__ __forceinline__ void pt_landed(uint32_t (&v)[32]) {
  asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
               "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
               "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]));
  asm volatile("" : "+r"(v[30]), "+r"(v[31]));
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

// Set-up that both tile forms share: barriers, tensor memory, and (warp 3) the CTA's share.
template <int D>
__device__ __forceinline__ PaShare pt_begin(const PagedAttnParams& p, PtBars& bars, const CUtensorMap* q, const CUtensorMap* k, const CUtensorMap* v, PaPlace& first) {
  const int tid = threadIdx.x, warp = tid >> 5;
  PaShare share{};
  if (warp == 3) {
    if (p.pdl) pdl_wait();
    share = pa_share<pt_bk(D)>(p, first);
  }
  if (tid == 0) {
    tma_prefetch_desc(q);
    tma_prefetch_desc(k);
    tma_prefetch_desc(v);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars.piece_full[i], 1);
      mbar_init(&bars.piece_read[i], 11);  // eight softmax warps, keys, values, products
      for (int w = 0; w < 2; ++w) {
        mbar_init(&bars.p_full[w][i], 4);
        mbar_init(&bars.pub[w][i], 1);
        mbar_init(&bars.fin[0][w][i], 1);
        mbar_init(&bars.fin[1][w][i], 1);
      }
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.done[i], 1);
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, D == 128 ? 1 : 8);  // wide: eight warps take them to tensor memory
    mbar_init(&bars.q_in, 8);
    mbar_init(&bars.q_used, 1);
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
    if (warp != 3) pdl_wait();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return share;
}

// What a softmax warp does with N * 32 scores of a row that are in tensor memory at t_s: the block's maximum ...
template <int N>
__device__ __forceinline__ float pt_scores(uint32_t t_s, uint32_t (&v)[N][32], int seen, float scale) {
  tc_fence_after();
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  tmem_ld32(t_s, v[0]);
#pragma unroll
  for (int w = 0; w < N; ++w) {  // 32 scores' maximum under the load of the next ones
    tc_wait_ld();
    pt_landed(v[w]);
    if (w + 1 < N) tmem_ld32(t_s + (w + 1) * 32, v[w + 1 < N ? w + 1 : 0]);
    pt_row_max<4>(v[w], seen - 32 * w, mx);
  }
  return fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale, PT_LOWEST);
}
// ... and the weights relative to m over them, handed over 32 keys at a time (the last ones by the caller); returns their sum.
template <int N>
__device__ __forceinline__ float pt_probabilities(uint32_t t_s, const uint32_t (&v)[N][32], float m, uint64_t c2, uint64_t* handed) {
  const uint64_t nm = pt_pair(-m, -m);
  uint64_t sum[2] = {pt_pair(0.f, 0.f), pt_pair(0.f, 0.f)};
#pragma unroll
  for (int w = 0; w < N; ++w) {
    uint32_t pk[16];
    pt_weights(v[w], c2, nm, sum[w & 1], pk);
    tmem_st16(t_s + w * 16, pk);
    tc_wait_st();
    if (w < N - 1) {
      tc_fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&handed[w]);
    }
  }
  float a0, a1;
  pt_unpair(pt_add2(sum[0], sum[1]), a0, a1);
  return a0 + a1;
}
// Hands over the last weights of a block; all of them in a warp without query rows.
template <int N>
__device__ __forceinline__ void pt_hand_over(bool live, uint64_t* handed) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if (!live)
      for (int w = 0; w < N - 1; ++w) mbar_arrive(&handed[w]);
    mbar_arrive(&handed[N - 1]);
  }
}

// The CTAs of a cluster join their parts of a tile. Each owns a share of the rows; once all have left their rings, the softmax warps send
// every row's part, from tensor memory, to its owner: [part][column / 4][row of the share], over the ring. With everything here the owner
// adds the parts up in their order, a thread per row and 32 columns. (All threads of the cluster meet before and after the sending.)
__device__ __forceinline__ void pt_meet() {
  __syncwarp();
  cluster_arrive_release();
  cluster_wait_acquire();
}
// chunks [c0, c1) of 32 columns of tile t's `row`; m = -INFINITY: no part of it here
template <int D>
__device__ __forceinline__ void pt_send(const PagedAttnParams& p, PtBars& bars, float4* parts, uint32_t t_o, int t, int row, int c0, int c1, bool live, bool mine, float m, float l) {
  const int each = pt_rows(D) / p.cluster, at = t * 128 + row, owner = at >> (__ffs(each) - 1), here = at & (each - 1), rank = cluster_ctarank();
  if (c0 == 0) {
    pa_send(&bars.part_m[rank * each + here], owner, mine ? m : -INFINITY);
    pa_send(&bars.part_l[rank * each + here], owner, l);
  }
  if (!live) return;
  const uint32_t to = dsmem_addr(smem_u32(parts + rank * (D / 4) * each + here), owner), step = each * 16;
  tc_fence_after();
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    uint32_t o[32];
    tmem_ld32(t_o + c * 32, o);
    tc_wait_ld();
    if (mine)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pa_send4(to + (c * 8 + e) * step, make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3])));
  }
}
template <int D>
__device__ __forceinline__ void pt_join(const PagedAttnParams& p, const PtBars& bars, const float4* parts) {
  if (bars.item.rows == 0) return;
  const int each = pt_rows(D) / p.cluster, rank = cluster_ctarank(), half = p.tile_rows / (pt_rows(D) / 128);
  for (int i = threadIdx.x - 128; i < each * (D / 32); i += 256) {
    const int here = i & (each - 1), at = rank * each + here, c = i >> (__ffs(each) - 1), local = (at >> 7) * half + (at & 127);
    if ((at & 127) >= half || local >= bars.item.rows) continue;
    float m[8], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = k < p.cluster ? bars.part_m[k * each + here] : -INFINITY;
      top = fmaxf(top, m[k]);
    }
    uint32_t o[32] = {};
#pragma unroll 1
    for (int k = 0; k < p.cluster; ++k) {
      const float mk = bars.part_m[k * each + here];
      if (mk == -INFINITY) continue;
      const float f = pa_exp2(mk - top);
      sum += f * bars.part_l[k * each + here];
      const float4* src = parts + (k * (D / 4) + c * 8) * each + here;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float4 a = src[e * each];
        o[4 * e] = __float_as_uint(__uint_as_float(o[4 * e]) + f * a.x);
        o[4 * e + 1] = __float_as_uint(__uint_as_float(o[4 * e + 1]) + f * a.y);
        o[4 * e + 2] = __float_as_uint(__uint_as_float(o[4 * e + 2]) + f * a.z);
        o[4 * e + 3] = __float_as_uint(__uint_as_float(o[4 * e + 3]) + f * a.w);
      }
    }
    const int ahead = pa_token(p, local);
    pt_store32(p, static_cast<long long>(bars.item.token + ahead) * p.ld_out + static_cast<long long>(bars.item.g * p.ratio + local - ahead * p.ratio) * D + c * 32, o,
               sum == 0.f ? 0.f : 1.f / sum);
  }
}

__global__ void __launch_bounds__(PT_THREADS, 1)
paged_pair_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const PagedAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ PtBars bars;
  constexpr int D = 128, BK = pt_bk(D), KV = 32768, CH = 16384;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = smem + 65536, *sv = sk + 2 * KV;
  PaPlace first{};
  const PaShare share = pt_begin<D>(p, bars, &tm_q, &tm_k, &tm_v, first);
  constexpr uint32_t tmem = 0;           // all 512 columns are this CTA's: S / P of tile t at 128 t, O of tile t at 256 + 128 t
  const int half = p.tile_rows >> 1;     // rows of a tile

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_CONTROL));
    if (warp == 3) {
      pt_lead<D>(p, first, share, &tm_q, sq, bars);
    } else if (warp != 1) {
      const bool k = warp == 0;
      pt_stream<D>(p, {k ? &tm_k : &tm_v, k ? sk : sv, k ? bars.k_full : bars.v_full, k ? bars.k_empty : bars.v_empty}, bars);
    } else {
      const uint32_t leader = elect_one();
      const uint32_t idesc_s = idesc_bf16_f32(128, BK) | p.negate_q, idesc_o = idesc_bf16_f32(128, D) | (1u << 16);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, wait_or_abort(bar, parity, &bars.abort));
        return ok;
      };
      uint32_t i = 0, i_second = 0;  // blocks so far, and those with a second tile
      PtReader reader;
      PtPiece at{};
      while (ok && reader.next(bars, at)) {
        const int nt = pt_uniform(at.rows > half ? 2 : 1), nb = pt_uniform(at.end - at.blk), blk = pt_uniform(at.blk), len = pt_uniform(at.len);
        if (!wait(&bars.q_full, (reader.n - 1) & 1)) break;
#pragma unroll 1
        for (int j = -1; j < nb && ok; ++j) {
          const bool more = j + 1 < nb;
          const uint32_t vb = i + j, kb = i + j + 1;  // blocks of this product and of the scores after it
          const uint32_t v_desc = pt_desc_lo(smem_u32(sv + (vb & 1) * KV), CH), k_desc = pt_desc_lo(smem_u32(sk + (kb & 1) * KV), 16);
          const PtWait keys{&bars.k_full[kb & 1], (kb >> 1) & 1}, values{&bars.v_full[vb & 1], (vb >> 1) & 1};
#pragma unroll 1
          for (int t = 0; t < nt && ok; ++t) {
            if (j < 0) {
              ok = t > 0 || wait(keys.bar, keys.parity);
              tc_fence_after();
            } else {
              const PtWait weights{&bars.p_full[t][0], ((t ? i_second : i) + j) & 1};
              ok = t ? wait(weights.bar, weights.parity) : pt_wait(values, weights, more ? keys : values, &bars.abort);
              if (!ok) break;
              tc_fence_after();
              if (t == 0) pt_clear_tail<D>(sv + (vb & 1) * KV, len, blk + j);
              int ready = 0;  // parts after the first that need no wait
#pragma unroll
              for (int part = 0; part < 4; ++part) {  // each 32 keys' product starts under the next ones' exponentials
                if (part == 1) ready = pt_handed<4>(bars.p_full[t], weights.parity);
                if (part > ready && !wait(&bars.p_full[t][part], weights.parity)) break;
                if (part) tc_fence_after();
#pragma unroll
                for (int ks = 2 * part; ks < 2 * part + 2; ++ks)
                  pt_mma_ts(leader, tmem + 256 + t * 128, tmem + t * 128 + ks * 8, v_desc + ks * (2048 >> 4), idesc_o, j > 0 || ks ? 1u : 0u);
              }
            }
            if (!ok) break;
            if (more) {
              const uint32_t q_desc = pt_desc_lo(smem_u32(sq + t * 32768), 16);
#pragma unroll
              for (int ks = 0; ks < 8; ++ks) {
                const uint32_t o = (ks >> 2) * (CH >> 4) + (ks & 3) * 2;
                pt_mma_ss(leader, tmem + t * 128, q_desc + o, k_desc + o, idesc_s, ks > 0 ? 1u : 0u);
              }
              pt_commit(leader, &bars.s_full[t]);
            } else {
              pt_commit(leader, &bars.done[t]);
            }
          }
          if (!ok) break;
          if (more) pt_commit(leader, &bars.k_empty[kb & 1]);
          if (j + 2 == nb) pt_commit(leader, &bars.q_empty);  // the last scores have been issued
          if (j >= 0) pt_commit(leader, &bars.v_empty[vb & 1]);
        }
        i += nb;
        if (nt == 2) i_second += nb;
      }
      ok = ok && reader.ok;
      // nothing of this CTA's tensor work may be in flight when it gives up its tensor memory
      pt_commit(leader, &bars.mma_done);
      if (!ok && lane == 0) {
        bars.abort = 1;
        if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_MMA);
      }
      mbar_wait(&bars.mma_done, 0);
    }
    if (p.cluster) {
      pt_meet();
      pt_meet();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    const int t = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t t_s = tmem + t * 128 + lane_addr, t_o = tmem + 256 + t * 128 + lane_addr;
    const uint64_t c2 = pt_pair(p.abs_scale_log2e, p.abs_scale_log2e);
    const int local = t * half + row, ahead = pa_token(p, local);  // row of the piece; its token's number in it
    pa_check(p, tid - 128, 256);
    pa_zero_rows<D>(p, tid - 128, 256);
    uint32_t n = 0, i = 0;  // tiles and blocks of this group
    bool ok = true;
    float part_m = -INFINITY, part_l = 0.f;  // cluster: of this row
    PtReader reader;
    PtPiece at{};
    while (ok && reader.next(bars, at)) {
      const int nvalid = min(half, at.rows - t * half);
      if (nvalid <= 0) continue;
      const bool live = q * 32 < nvalid, mine = row < nvalid;
      const int limit = at.seen + ahead * at.step;  // keys this row sees
      float m_ref = PT_LOWEST, l = 0.f;
#pragma unroll 1
      for (int j = at.blk; j < at.end; ++j, ++i) {
        ok = __all_sync(0xffffffffu, wait_or_abort(&bars.s_full[t], i & 1, &bars.abort, p.wait_limit));
        if (!ok) break;
        if (live) {
          uint32_t v[4][32];
          const float m_blk = pt_scores<4>(t_s, v, limit - j * BK, p.abs_scale_log2e);
          const bool grow = m_blk > m_ref + PT_RESCALE;
          if (__any_sync(0xffffffffu, grow)) {
            if (j > at.blk) {  // the scores of this block came after the last one's product
              const float f = grow ? pa_exp2(m_ref - m_blk) : 1.0f;
              pt_rescale(t_o, 4, f);
              l *= f;
            }
            if (grow) m_ref = m_blk;
          }
          l += pt_probabilities<4>(t_s, v, m_ref, c2, bars.p_full[t]);
        }
        pt_hand_over<4>(live, bars.p_full[t]);
      }
      ok = ok && __all_sync(0xffffffffu, wait_or_abort(&bars.done[t], n & 1, &bars.abort));
      ++n;
      if (p.cluster) {
        if (ok) part_m = m_ref, part_l = l;
        break;  // the only piece
      }
      if (ok && live) {
        tc_fence_after();
        const float inv = at.part ? 1.f : l == 0.f ? 0.f : 1.f / l;
        // [tile][column / 4][row], then the references and sums of both tiles
        float4* part = reinterpret_cast<float4*>(p.ws + pa_header_bytes(gridDim.x) + (2ll * blockIdx.x + at.part - 1) * pa_part_bytes<pt_rows(D), D>());
        const long long to = static_cast<long long>(at.token + ahead) * p.ld_out + static_cast<long long>(at.g * p.ratio + local - ahead * p.ratio) * D;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tc_wait_ld();
          if (at.part) pt_part32(part + t * (D / 4) * 128, c * 32, row, o);
          else if (mine) pt_store32(p, to + c * 32, o, inv);
        }
        if (at.part) {
          float* stat = reinterpret_cast<float*>(part + pt_rows(D) * D / 4);
          stat[t * 128 + row] = m_ref;
          stat[pt_rows(D) + t * 128 + row] = l;
        }
        tc_fence_before();
      }
    }
    ok = ok && reader.ok;
    if (!ok && lane == 0) {
      if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_EPILOGUE);
      bars.abort = 1;
    }
    if (p.cluster) {
      const int valid = at.rows - t * half;  // (no piece: no rows)
      pt_meet();
      pt_send<D>(p, bars, reinterpret_cast<float4*>(sk), t_o, t, row, 0, 4, q * 32 < valid && __any_sync(0xffffffffu, part_m > -INFINITY), row < valid, part_m, part_l);
      pt_meet();
      pt_join<D>(p, bars, reinterpret_cast<const float4*>(sk));
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
  constexpr int D = 256, BK = pt_bk(D), KV = 32768, QCH = 16384, CH = BK * 128;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = smem + 65536, *sv = sk + 2 * KV;
  PaPlace first{};
  const PaShare share = pt_begin<D>(p, bars, &tm_q, &tm_k, &tm_v, first);
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: two score buffers of 64 columns, queries from 128 (two channels a column), O from 256

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_CONTROL));
    if (warp == 3) {
      pt_lead<D>(p, first, share, &tm_q, sq, bars);
    } else if (warp != 1) {
      const bool k = warp == 0;
      // a key block's place is free when its scores are there, a value block's when its product is: no barriers of their own
      pt_stream<D>(p, {k ? &tm_k : &tm_v, k ? sk : sv, k ? bars.k_full : bars.v_full, k ? bars.s_full : bars.done}, bars);
    } else {
      const uint32_t leader = elect_one();
      const uint32_t idesc_s = idesc_bf16_f32(128, BK) | p.negate_q, idesc_o = idesc_bf16_f32(128, D) | (1u << 16);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, wait_or_abort(bar, parity, &bars.abort));
        return ok;
      };
      uint32_t i = 0;  // blocks so far
      PtReader reader;
      PtPiece at{};
      while (ok && reader.next(bars, at)) {
        const uint32_t n = reader.n - 1;
        const int nb = pt_uniform(at.end - at.blk), blk = pt_uniform(at.blk), len = pt_uniform(at.len);
        if (!wait(&bars.q_in, n & 1)) break;
        auto turn = [&](int j) {  // product of block j of the piece, then scores of block j + 2
          const uint32_t vb = i + j, s = vb & 1;
          return PtTurn{bars.p_full[s], &bars.v_full[s], &bars.k_full[s], vb >> 1, vb >> 1, (vb + 2) >> 1, j + 2 < nb};
        };
        int parts = 0;  // of this turn's weights, known to be there
#pragma unroll 1
        for (int j = -2; j < nb; ++j) {
          const bool more = j + 2 < nb;
          const uint32_t vb = i + j, kb = vb + 2, s = vb & 1;  // blocks of this product and of the scores after it, their buffer
          if (j == 0 && n > 0 && !wait(&bars.o_free, (n - 1) & 1)) break;  // the last tile's output has been read
          if (j >= 0) {
            if (parts == 0) parts = turn(j).wait<2>(&bars.abort);
            ok = parts > 0;
          } else if (more) {
            wait(&bars.k_full[s], (kb >> 1) & 1);
          }
          if (!ok) break;
          tc_fence_after();
          if (j >= 0) {
            pt_clear_tail<D>(sv + s * KV, len, blk + j);
            const uint32_t v_desc = pt_desc_lo(smem_u32(sv + s * KV), CH);
#pragma unroll
            for (int part = 0; part < 2; ++part) {  // the first 32 keys' product starts under the others' exponentials
              if (part >= parts) {
                if (!wait(&bars.p_full[s][1], (vb >> 1) & 1)) break;
                tc_fence_after();
              }
#pragma unroll
              for (int ks = 2 * part; ks < 2 * part + 2; ++ks)
                pt_mma_ts(leader, tmem + 256, tmem + s * 64 + ks * 8, v_desc + ks * (2048 >> 4), idesc_o, j > 0 || ks ? 1u : 0u);
            }
            if (!ok) break;
          }
          parts = j + 1 >= 0 && j + 1 < nb ? turn(j + 1).ready<2>() : 0;
          if (more) {
            const uint32_t k_desc = pt_desc_lo(smem_u32(sk + s * KV), 16);
#pragma unroll
            for (int ks = 0; ks < 16; ++ks) {
              const uint32_t o = (ks >> 2) * (CH >> 4) + (ks & 3) * 2;
              pt_mma_ts(leader, tmem + s * 64, tmem + 128 + ks * 8, k_desc + o, idesc_s, ks > 0 ? 1u : 0u);
            }
            pt_commit(leader, &bars.s_full[s]);
            if (j + 3 == nb) pt_commit(leader, &bars.q_used);  // the last scores have been issued
          }
          if (j >= 0) pt_commit(leader, &bars.done[s]);
        }
        i += nb;
      }
      ok = ok && reader.ok;
      pt_commit(leader, &bars.mma_done);
      if (!ok && lane == 0) {
        bars.abort = 1;
        if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_MMA);
      }
      mbar_wait(&bars.mma_done, 0);
    }
    if (p.cluster) {
      pt_meet();
      pt_meet();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    const int grp = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t t_o = tmem + 256 + lane_addr, t_s = tmem + grp * 64 + lane_addr;
    const uint64_t c2 = pt_pair(p.abs_scale_log2e, p.abs_scale_log2e);
    const int ahead = pa_token(p, row);  // number of the row's token in the tile
    uint32_t i = 0;                   // blocks so far (of both groups)
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, wait_or_abort(bar, parity, &bars.abort));
      return ok;
    };
    // this thread's half of its query row (two chunks of 64 channels) of tile n, from shared to tensor memory
    auto queries = [&](uint32_t n) {
      if (!wait(&bars.q_full, n & 1) || (n > 0 && !wait(&bars.q_used, (n - 1) & 1))) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        const uint8_t* src = sq + (2 * grp + c) * QCH + row * 128;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + ((e ^ (row & 7)) << 4));
          v[4 * e] = x.x;
          v[4 * e + 1] = x.y;
          v[4 * e + 2] = x.z;
          v[4 * e + 3] = x.w;
        }
        tmem_st32(tmem + 128 + (2 * grp + c) * 32 + lane_addr, v);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars.q_in);
        mbar_arrive(&bars.q_empty);
      }
      return true;
    };
    PtReader reader;
    PtPiece at{}, next{};
    float part_m = -INFINITY, part_l = 0.f;  // cluster: of this row
    bool any = reader.next(bars, at) && queries(0);
    pa_check(p, tid - 128, 256);
    pa_zero_rows<D>(p, tid - 128, 256);
#pragma unroll 1
    for (uint32_t n = 0; any; ++n) {
      const bool live = q * 32 < at.rows, mine = row < at.rows;
      const int limit = at.seen + ahead * at.step;
      float m_own = PT_LOWEST, l = 0.f;  // the reference that l is relative to
#pragma unroll 1
      for (int j = at.blk; j < at.end; ++j, ++i) {
        if ((i & 1) != static_cast<uint32_t>(grp)) continue;
        // The scores, and the product of this group's block before (half of the lanes each, in the time of one wait).  That product's next
        // phase needs this block's weights, so nothing of it is missed here, and what this group has seen the other one knows by `pub`
        // and `fin`: both can wait for either's last product below.  (The scores alone say that it has been done, not that its
        // arrival is there: that is a commit of its own, and a wait for the phase after it would have passed at once.)
        const bool product = (lane & 1) && i >= 2;
        ok = __all_sync(0xffffffffu, wait_or_abort(product ? &bars.done[grp] : &bars.s_full[grp], product ? ((i >> 1) - 1) & 1 : (i >> 1) & 1, &bars.abort, p.wait_limit));
        if (!ok) break;
        uint32_t v[2][32];
        float m_blk = 0.f;
        if (live) m_blk = pt_scores<2>(t_s, v, limit - j * BK, p.abs_scale_log2e);
        // the reference after the block before, which the other group has
        float m_ref = PT_LOWEST;
        if (j > at.blk) {
          if (!wait(&bars.pub[grp ^ 1][q], ((i - 1) >> 1) & 1)) break;
          m_ref = bars.m_ref[grp ^ 1][row];
        }
        const bool grow = live && m_blk > m_ref + PT_RESCALE;
        const float m_new = grow ? m_blk : m_ref;
        bars.m_ref[grp][row] = m_new;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.pub[grp][q]);
        if (live) {
          if (__any_sync(0xffffffffu, grow) && j > at.blk) {
            // The product before must have landed.  (The barrier's phase before has passed: the other group saw it before `pub`; its next waits
            // for this block's weights.)
            if (!wait(&bars.done[(i - 1) & 1], ((i - 1) >> 1) & 1)) break;
            tc_fence_after();
            pt_rescale(t_o, 8, grow ? pa_exp2(m_ref - m_blk) : 1.0f);
          }
          l = l * pa_exp2(m_own - m_new) + pt_probabilities<2>(t_s, v, m_new, c2, bars.p_full[grp]);
          m_own = m_new;
        }
        pt_hand_over<2>(live, bars.p_full[grp]);
      }
      if (!ok) break;
      // Both groups' sums, relative to the later reference.  (With one barrier for all tiles a short next tile, whose blocks may all be the
      // other group's, could be through before this one has asked.  The tile after that needs this group's sums of the next one.)
      bars.end_m[n & 1][grp][row] = m_own;
      bars.end_l[n & 1][grp][row] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.fin[n & 1][grp][q]);
      any = reader.next(bars, next);
      if (!reader.ok || (any && !queries(n + 1))) break;  // the next scores may begin
      if (!wait(&bars.fin[n & 1][grp ^ 1][q], (n >> 1) & 1)) break;
      const float m_other = bars.end_m[n & 1][grp ^ 1][row], m_end = fmaxf(m_own, m_other);
      l = l * pa_exp2(m_own - m_end) + bars.end_l[n & 1][grp ^ 1][row] * pa_exp2(m_other - m_end);
      if (!wait(&bars.done[(i - 1) & 1], ((i - 1) >> 1) & 1)) break;
      if (p.cluster) {
        part_m = m_end, part_l = l;
        break;  // the only piece
      }
      if (live) {
        tc_fence_after();
        const float inv = at.part ? 1.f : l == 0.f ? 0.f : 1.f / l;
        float4* part = reinterpret_cast<float4*>(p.ws + pa_header_bytes(gridDim.x) + (2ll * blockIdx.x + at.part - 1) * pa_part_bytes<pt_rows(D), D>());
        const long long to = static_cast<long long>(at.token + ahead) * p.ld_out + static_cast<long long>(at.g * p.ratio + row - ahead * p.ratio) * D;
#pragma unroll 1
        for (int c = 4 * grp; c < 4 * grp + 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tc_wait_ld();
          if (at.part) pt_part32(part, c * 32, row, o);
          else if (mine) pt_store32(p, to + c * 32, o, inv);
        }
        if (at.part && grp == 0) {
          float* stat = reinterpret_cast<float*>(part + pt_rows(D) * D / 4);
          stat[row] = m_end;
          stat[pt_rows(D) + row] = l;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.o_free);
      at = next;
    }
    ok = ok && reader.ok;
    if (!ok && lane == 0) {
      if (p.status) atomicCAS(p.status, 0, TYBOK_DEV_TIMEOUT_EPILOGUE);
      bars.abort = 1;
    }
    if (p.cluster) {
      pt_meet();
      pt_send<D>(p, bars, reinterpret_cast<float4*>(sk), t_o, 0, row, 4 * grp, 4 * grp + 4, q * 32 < at.rows && __any_sync(0xffffffffu, part_m > -INFINITY), row < at.rows, part_m, part_l);
      pt_meet();
      pt_join<D>(p, bars, reinterpret_cast<const float4*>(sk));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the tile that CTA blockIdx.x of a tile form began: a thread per row and 32 columns.
template <int D>
__global__ void __launch_bounds__(128) paged_join_tile_kernel(const PagedAttnParams p, int ctas) {
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  const PaHeader h = reinterpret_cast<const PaHeader*>(p.ws)[blockIdx.x];
  if (h.parts == 0) return;
  constexpr int ROWS = pt_rows(D), COLS = D / 32;  // grid.y = 32 columns of 128 rows
  const int t = blockIdx.y / COLS, c = blockIdx.y % COLS, row = threadIdx.x, half = p.tile_rows / (pt_rows(D) / 128), local = t * half + row;
  if (row >= half || local >= h.rows) return;
  const uint8_t* parts = p.ws + pa_header_bytes(ctas);
  auto part = [&](int i) {  // the i-th part of the tile
    return reinterpret_cast<const float4*>(parts + (2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * pa_part_bytes<ROWS, D>());
  };
  auto stat = [&](int i) { return reinterpret_cast<const float*>(part(i) + ROWS * D / 4) + t * 128 + row; };
  float top = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < h.parts; ++i) top = fmaxf(top, *stat(i));
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f;
  uint32_t o[32] = {};
#pragma unroll 2
  for (int i = 0; i < h.parts; ++i) {
    const float4* src = part(i) + (t * (D / 4) + c * 8) * 128 + row;
    float4 a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = src[e * 128];
    const float f = pa_exp2(*stat(i) - top);
    sum += f * stat(i)[ROWS];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[4 * e] = __float_as_uint(__uint_as_float(o[4 * e]) + f * a[e].x);
      o[4 * e + 1] = __float_as_uint(__uint_as_float(o[4 * e + 1]) + f * a[e].y);
      o[4 * e + 2] = __float_as_uint(__uint_as_float(o[4 * e + 2]) + f * a[e].z);
      o[4 * e + 3] = __float_as_uint(__uint_as_float(o[4 * e + 3]) + f * a[e].w);
    }
  }
  const int grow = h.first + local, token = pa_token(p, grow);
  pt_store32(p, static_cast<long long>(h.start + token) * p.ld_out + static_cast<long long>(h.g * p.ratio + grow - token * p.ratio) * D + c * 32, o, sum == 0.f ? 0.f : 1.f / sum);
}

// The same for the sixteen-row form; a warp per row.
template <int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttnParams p, int ctas) {
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait();
  }
  const PaHeader h = reinterpret_cast<const PaHeader*>(p.ws)[blockIdx.x];
  if (h.parts == 0) return;
  constexpr int ROWS = PR_ROWS;
  const uint8_t* parts = p.ws + pa_header_bytes(ctas);
  auto part = [&](int i) {  // the i-th part of the tile
    return reinterpret_cast<const float*>(parts + (2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * pa_part_bytes<ROWS, D>());
  };
  const int lane = threadIdx.x & 31;
  for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < h.rows; row += gridDim.y * 4) {
    float top = -INFINITY;
    for (int i = lane; i < h.parts; i += 32) top = fmaxf(top, part(i)[ROWS * D + row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.f;
    constexpr int N = D / 32;
    float sum = 0.f, v[N] = {};
#pragma unroll 4
    for (int i = 0; i < h.parts; ++i) {
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
    const int grow = h.first + row, token = pa_token(p, grow);
    const long long at = static_cast<long long>(h.start + token) * p.ld_out + static_cast<long long>(h.g * p.ratio + grow - token * p.ratio) * D;
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
// Whether clusters take the tiles: CTAs of a cluster per tile, or 0.  All tiles that these sizes allow must run at once, and even a full cache must
// take a cluster no longer than an even share of all tiles and the joining of its parts would take all CTAs.
template <class Kernel, int D>
static int pa_clusters(Kernel* kernel, int threads, int smem, int size) {  // of `size` CTAs that the device holds at once
  static host::DeviceCache cache[9];
  return host::per_device(cache[size], [&] {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 1;
    }
    return n;
  });
}
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
    return smem(paged_rows_kernel<128>, pr_smem(128)) && smem(paged_rows_kernel<256>, pr_smem(256)) && smem(paged_pair_kernel, PT_SMEM) && smem(paged_wide_kernel, PT_SMEM);
  });
  return set ? TYBOK_OK : host::fail_cuda("paged_attention: shared memory");
}

// Tensor map of a pool [P][G][page][D]: boxes of 64 channels and one page's rows (or a block's).
static int pa_pool_map(CUtensorMap* map, const void* base, const int64_t* strides, int P, int G, int page, int D) {
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(page), static_cast<uint64_t>(G), static_cast<uint64_t>(P)};
  auto bytes = [&](int i, int extent) { return static_cast<uint64_t>(extent > 1 ? strides[i] : D) * 2; };  // (of an extent of one it does not matter)
  const uint64_t pitch[3] = {bytes(2, page), bytes(1, G), bytes(0, P)};
  const uint32_t box[4] = {64, static_cast<uint32_t>(std::min(page, pt_bk(D))), 1, 1};
  return host::tensor_map_4d(map, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, pitch, box);
}

}  // namespace tb

extern "C" {

size_t tybok_paged_attention_workspace_bytes(int H, int G, int D, int max_tokens) {
  using namespace tb;
  if (H <= 0 || G <= 0 || max_tokens <= 0 || (D != 128 && D != 256)) return 0;
  const bool tiles = pa_tile_form(H / G, max_tokens);
  return pa_workspace(D, tiles, host::sm_count() * (tiles ? 1 : pr_ctas(D)));
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
  if (static_cast<long long>(table_width) * page_size > 0x7fffff00ll) return host::fail(TYBOK_ERR_ARG, "paged_attention: a request's keys must fit 31 bits");
  const int extents[3] = {num_pages, G, page_size};
  for (int i = 0; i < 3; ++i)
    if (extents[i] > 1 && (k_strides[i] <= 0 || v_strides[i] <= 0)) return host::fail(TYBOK_ERR_ARG, "paged_attention: strides of the pools must be positive");
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
  int ratio_bits = 1;
  while ((1ll << ratio_bits) < p.ratio) ++ratio_bits;
  p.ratio_mul = static_cast<uint32_t>(((1ull << (31 + ratio_bits)) + p.ratio - 1) / p.ratio);  // (not used for a ratio of one)
  p.ratio_shift = ratio_bits - 1;
  p.scale_log2e = scale * 1.4426950408889634f;
  // the tile forms want a scale above zero (at zero: one that no score brings above 2^-22)
  p.abs_scale_log2e = fabsf(p.scale_log2e);
  if (p.abs_scale_log2e == 0.f) p.abs_scale_log2e = std::numeric_limits<float>::denorm_min();
  p.negate_q = scale < 0.f ? 1u << 13 : 0u;
  p.wait_limit = host::epilogue_wait_limit() > 0 ? host::epilogue_wait_limit() : kWaitLimitCycles;
  p.ws = static_cast<uint8_t*>(workspace); p.status = status_word;
  p.pdl = host::pdl_enabled() ? 1 : 0;
  p.wide_out = ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_planes)) & 31) == 0;
  const bool tiles = pa_tile_form(p.ratio, max_tokens);
  p.tile_rows = !tiles ? PR_ROWS : 128 / p.ratio * p.ratio * (D == 128 ? 2 : 1);
  const double most_tiles = static_cast<double>(tokens) * p.ratio / p.tile_rows + B, most_blocks = static_cast<double>(table_width) * page_size / 64 + 8;
  if (most_tiles * G * most_blocks > 4e9) return host::fail(TYBOK_ERR_ARG, "paged_attention: more than 2^32 key blocks could fall to one call");
  p.tile_tokens = p.tile_rows % p.ratio == 0 ? p.tile_rows / p.ratio : 0;
  // Both sides measured.  Joining: head_dim 128, 19 requests from one token to 700, 2 blocks 55.7 us, 3 56.3, 4 57.2 and 8 prompts of 1024 tokens 81.4,
  // 79.8, 79.8; head_dim 256, five prompts of 402 to 627 tokens 7 blocks 31.7, 9 30.3, 12 30.3 and twelve of 300 to 968 57.9, 58.0, 60.4.  A tile's
  // edges: the 19 requests with 1 block 59.2, 2 56.3, 3 58.6; the twelve prompts with 4 60.3, 5 58.0, 7 59.5.
  p.join_blocks = tiles ? (D == 128 ? 3 : 9) : 4;
  p.tile_blocks = !tiles ? 0 : D == 128 ? 2 : 5;
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
  const int sms = host::sm_count(), threads = tiles ? PT_THREADS : PR_THREADS, smem = tiles ? PT_SMEM : pr_smem(D);
  PaTileKernel* tile_kernel = D == 256 ? paged_wide_kernel : paged_pair_kernel;
  PaRowsKernel* rows_kernel = D == 256 ? paged_rows_kernel<256> : paged_rows_kernel<128>;
  // Tiles at most (a request's last one may be partly empty), key blocks of a full cache.
  const double items = G * (B + std::floor(static_cast<double>(tokens) * p.ratio / p.tile_rows));
  const double blocks = static_cast<double>(table_width) * page_size / (tiles ? pt_bk(D) : PR_BLOCK);
  for (int size = 8; size >= 2 && !p.cluster; size /= 2) {
    if (items * size > sms || blocks * (1.0 / size - items / sms) > p.join_blocks) continue;
    const int room = tiles ? (D == 256 ? pa_clusters<PaTileKernel, 256>(tile_kernel, threads, smem, size) : pa_clusters<PaTileKernel, 128>(tile_kernel, threads, smem, size))
                           : (D == 256 ? pa_clusters<PaRowsKernel, 256>(rows_kernel, threads, smem, size) : pa_clusters<PaRowsKernel, 128>(rows_kernel, threads, smem, size));
    if (items <= room) p.cluster = size;
  }
  const int ctas = p.cluster ? static_cast<int>(items) * p.cluster : tiles ? sms : sms * pr_ctas(D);
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (p.pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = na;
  if (p.cluster) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = p.cluster;
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    cfg.numAttrs = na + 1;
  }
  const cudaError_t e = tiles ? cudaLaunchKernelEx(&cfg, tile_kernel, tm_q, tm_k, tm_v, p) : cudaLaunchKernelEx(&cfg, rows_kernel, p);
  if (e != cudaSuccess) return host::fail_cuda("launch paged_attention");
  host::count_launch();
  if (p.cluster) return TYBOK_OK;
  cfg.gridDim = dim3(ctas, tiles ? 8 : PR_ROWS / 4);  // tile forms: 128 rows x 32 columns each
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  PaJoinKernel* join = tiles ? (D == 256 ? paged_join_tile_kernel<256> : paged_join_tile_kernel<128>)
                             : (D == 256 ? paged_join_kernel<256> : paged_join_kernel<128>);
  if (cudaLaunchKernelEx(&cfg, join, p, ctas) != cudaSuccess) return host::fail_cuda("launch paged_join_kernel");
  host::count_launch();
  return TYBOK_OK;
}
}

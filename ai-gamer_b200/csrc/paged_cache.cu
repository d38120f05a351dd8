// paged_cache.cu -- copies of a cache's pages, and attention of one new token of each sequence over its pages.
#include <cooperative_groups.h>
#include <float.h>
#include <string.h>

#include <new>
#include <type_traits>
#include <vector>

#include "long_context.h"

namespace cg = cooperative_groups;

namespace {

// ---------------------------------------------------------------------------------------------
// Page copies.  The pairs travel as kernel parameters: nothing to upload, nothing that a later call could overwrite while
// an earlier one (or a captured graph) still reads it.  Bound by memory: 1021 pages of 128 KB in 43 us, 6.2 TB/s.
constexpr int kFewPairs = 32, kManyPairs = 2000;  // per launch: a fork's few parameters are not carried in 16 KB
constexpr int kCopyThreads = 256, kCopyUnroll = 4;

struct CopyShape {
  uint4 *k, *v;
  long long page, place, head;  // strides in 16-byte units
  int run, heads;               // consecutive 16-byte units of a run; runs: places x heads (1 x 1 where a page is one run)
  int units, blocks;            // of a page, and blocks that copy it
};
template <int N>
struct CopyParams : CopyShape {
  int32_t src[N], dst[N];
};

template <int N>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams<N> p) {
  griddep_launch_dependents();
  griddep_wait();
  const int pair = blockIdx.x / p.blocks;
  const int first = (blockIdx.x - pair * p.blocks) * kCopyThreads * kCopyUnroll + threadIdx.x;
  uint4* const base = blockIdx.y ? p.v : p.k;
  const uint4* const src = base + p.src[pair] * p.page;
  uint4* const dst = base + p.dst[pair] * p.page;
  uint4 got[kCopyUnroll];
  long long at[kCopyUnroll];
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    const int u = first + i * kCopyThreads;
    const int run = u / p.run, place = run / p.heads;
    at[i] = place * p.place + (run - place * p.heads) * p.head + (u - run * p.run);
    if (u < p.units) got[i] = __ldcs(src + at[i]);
  }
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i)
    if (first + i * kCopyThreads < p.units) dst[at[i]] = got[i];
}

template <int N>
int launch_copies(aig_ctx* ctx, const CopyShape& shape, const int32_t* src, const int32_t* dst, int pairs) {
  CopyParams<N> p;
  static_cast<CopyShape&>(p) = shape;
  for (int done = 0; done < pairs; done += N) {
    const int n = pairs - done < N ? pairs - done : N;
    memcpy(p.src, src + done, n * sizeof(int32_t));
    memcpy(p.dst, dst + done, n * sizeof(int32_t));
    if ((long long)n * p.blocks > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "kv copy pages: too much for one call");
    AIG_CUDA_OK(ctx, launch_pdl(ctx, copy_pages_kernel<N>, dim3((unsigned)(n * p.blocks), 2), dim3(kCopyThreads), 0, p));
  }
  return AIG_OK;
}

// ---------------------------------------------------------------------------------------------
// Attention of one new token.  For each (sequence, cached head) the visible positions are split over the CTAs of a cluster
// and over their warps; a warp takes tiles of 16 or 32 positions through a ring of shared memory filled by cp.async.  Products
// are mma.sync with the positions as rows and the group's query heads as the 8 columns, S^T = K Q^T and O^T = V^T P^T: K and
// V come from shared memory as they lie there, P turns from result to operand by movmatrix, and eight query heads cost no more
// than one.  (The kernel is bound by reading the cache, then by issuing instructions: with the heads as 16 rows
// it took 430 instructions for 16 positions of 64, and 33 us where it takes 24, 128 sequences of up to 516 visible.)
// Softmax with a running maximum and sum in fp32; the weights enter the second product as a sum of two 16-bit values each, so
// that their rounding does not add to the result's.  Warps are joined in shared memory, CTAs over the cluster's distributed
// shared memory, in a fixed order: one launch, no scratch in global memory, nothing that two calls or captured
// graphs could share.
constexpr int kMaxCluster = 16;

struct AttendParams {
  const uint8_t *k, *v, *q;
  uint8_t* out;
  long long page, place, head;                 // cache strides in bytes
  long long q_seq, q_head, out_seq, out_head;  // in bytes
  const int32_t *table, *lengths;
  int table_width, num_pages;
  Divisor page_size;
  int kv_heads, group, row_blocks;             // query heads per cached one, in blocks of 8 or 16
  int splits;
  int window, sinks;
  float scale_log2;                            // scale * log2(e)
  int* gerr;
};

// W warps.  Where there are more sequences and heads than the device holds CTAs, small CTAs of two warps, seven to an SM, hide one
// another's beginnings and ends; few long sequences need the reads of four warps per CTA (128 sequences, 8 heads of 64: 22.9 us
// with two, 25.5 with four; 8 sequences of up to 65536, 8 heads of 128: 214 with two, 177 to 192 with four).
template <int D, int HT, int W>
struct AttendShape {
  static constexpr int kTile = 16;                                  // positions (32 need more shared memory: fewer CTAs, 26 us)
  static constexpr int kRows = 8 * HT;                              // query heads per CTA
  static constexpr int kStages = 3;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTileBytes = kTile * kRowBytes;              // of keys, and of values: 2 KB or 4 KB
  static constexpr int kRing = W * kStages * 2 * kTileBytes;        // 24 to 96 KB
  static constexpr int kPitch = D + 4;                              // of a row of sums: lanes' stores fall into different banks
  static constexpr int kJoin = W * kRows * (kPitch + 2) * 4;        // the warps' sums take the ring's place
  static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
  static constexpr int kCtasPerSm = W == 2 ? (D == 64 ? (HT == 1 ? 7 : 5) : 4) : (D == 64 ? (HT == 1 ? 4 : 3) : 2);
};

template <class T, int D, int HT, int W>
__global__ void __launch_bounds__(W * 32, AttendShape<D, HT, W>::kCtasPerSm) paged_attention_kernel(const __grid_constant__ AttendParams p) {
  using S = AttendShape<D, HT, W>;
  constexpr int kChunks = D / 8;                // 16-byte pieces of a row
  constexpr int kLoads = S::kTile * kChunks / 32;
  constexpr int kTile = S::kTile, kRows = S::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_scale[kMaxCluster][kRows];
  cg::cluster_group cluster = cg::this_cluster();
  griddep_launch_dependents();
  griddep_wait();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits;
  int item = blockIdx.x / p.splits;
  const int row_block = item % p.row_blocks;
  item /= p.row_blocks;
  const int b = item / p.kv_heads, kvh = item - b * p.kv_heads;
  const int rows = min(p.group - row_block * kRows, kRows);
  const int q_head0 = kvh * p.group + row_block * kRows;

  // visible positions: `front` of them from 0 on, the others from `back` on
  int len = p.lengths[b];
  const long long most = (long long)p.table_width * p.page_size.by;
  if (len > most) {
    if (threadIdx.x == 0) note_error(p.gerr, kErrBadPlace);
    len = (int)most;
  }
  int front = 0, back = 0, visible = max(len, 0);
  if (p.window > 0 && len > p.window) {
    back = len - p.window;
    front = min(p.sinks, back);
    visible = front + p.window;
  }
  // this CTA's share, in whole tiles; its warps take the tiles in turn
  const int tiles = (int)(((unsigned)visible + kTile - 1) / kTile);
  const int share = (tiles + p.splits - 1) / p.splits;
  const int tile_end = min((split + 1) * share, tiles);
  const int tile0 = split * share + warp;

  // ---- queries as the B operand: columns are query heads
  uint32_t qb[HT][D / 16][2];
  {
    const int c = (lane & 3) * 2;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int r = ht * 8 + (lane >> 2);
      const uint8_t* q = p.q + b * p.q_seq + (q_head0 + r) * p.q_head + c * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) qb[ht][ks][e] = r < rows ? *reinterpret_cast<const uint32_t*>(q + (ks * 16 + e * 8) * 2) : 0u;
    }
  }

  const uint32_t ring = smem_u32(smem) + warp * S::kStages * 2 * S::kTileBytes;
  const uint8_t* const kbase = p.k + kvh * p.head + (lane % kChunks) * 16;
  const uint8_t* const vbase = p.v + kvh * p.head + (lane % kChunks) * 16;
  const int32_t* const pages = p.table + (long long)b * p.table_width;

  // Row `lane` of a tile: its page (-1: none) and its place there, looked up one tile before it is loaded so that the table's
  // latency is not in the way.
  int row_page = -1, row_place = 0;
  auto look_up = [&](int tile) {
    const int i = tile * kTile + (lane & (kTile - 1));
    row_page = -1;
    if (tile < tile_end && i < visible) {
      const int t = i < front ? i : back + (i - front);
      const int slot = p.page_size.divide(t);
      row_place = t - slot * (int)p.page_size.by;
      row_page = pages[slot];
      if ((unsigned)row_page >= (unsigned)p.num_pages) {
        note_error(p.gerr, kErrBadPage);
        row_page = -1;
      }
    }
  };
  // (returns which of the tile's positions take part, as bits)
  auto load = [&](int tile, int stage) {
    uint32_t there = 0;
    if (tile < tile_end) {
      const long long mine = row_page < 0 ? -1 : row_page * p.page + row_place * p.place;
      there = __ballot_sync(0xffffffffu, row_page >= 0);
      const uint32_t kd = ring + stage * 2 * S::kTileBytes, vd = kd + S::kTileBytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = i * (32 / kChunks) + lane / kChunks, c = lane % kChunks;
        long long at = __shfl_sync(0xffffffffu, mine, r);
        const uint32_t to = r * S::kRowBytes + ((c ^ (r & 7)) << 4);  // pieces of 8 rows fall into different banks
        const int bytes = at < 0 ? 0 : 16;
        at = at < 0 ? 0 : at;
        cp_async16(kd + to, kbase + at, bytes);
        cp_async16(vd + to, vbase + at, bytes);
      }
    }
    cp_async_commit();  // (an empty group where there is no tile: groups are counted)
    return there;
  };

  // sums O^T: rows d, columns heads 2 (lane % 4) and the next; maxima and sums of these two heads
  float o[HT][D / 16][4], top[HT][2], sum[HT][2];
#pragma unroll
  for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[ht][n][e] = 0.f;
    top[ht][0] = top[ht][1] = -INFINITY;
    sum[ht][0] = sum[ht][1] = 0.f;
  }

  look_up(tile0);
  uint32_t there[S::kStages];  // of the tiles on their way, the next to be taken first
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) {
    there[s] = load(tile0 + s * W, s);
    look_up(tile0 + (s + 1) * W);
  }
  int stage = 0;
  for (int tile = tile0; tile < tile_end; tile += W, stage = stage + 1 == S::kStages ? 0 : stage + 1) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();
    {
      const int next = tile + (S::kStages - 1) * W;
      there[S::kStages - 1] = load(next, stage == 0 ? S::kStages - 1 : stage - 1);
      look_up(next + W);
    }
    const uint32_t shown = there[0];
#pragma unroll
    for (int s = 0; s + 1 < S::kStages; ++s) there[s] = there[s + 1];
    if (shown == 0) continue;  // none of them has a page
    const uint32_t kd = ring + stage * 2 * S::kTileBytes, vd = kd + S::kTileBytes;
    // ---- scores: 16 positions a block
    float sc[HT][kTile / 16][4];
#pragma unroll
    for (int kb = 0; kb < kTile / 16; ++kb) {
#pragma unroll
      for (int ht = 0; ht < HT; ++ht)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[ht][kb][e] = 0.f;
      const int r = kb * 16 + (lane & 15), c0 = lane >> 4;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t ka[4];
        ldmatrix4(kd + r * S::kRowBytes + (((ks * 2 + c0) ^ (r & 7)) << 4), ka);
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) mma16816<T>(sc[ht][kb], ka, qb[ht][ks][0], qb[ht][ks][1]);
      }
    }
    if (shown != 0xffffffffu) {  // behind the last position, or without a page
      static_assert(kTile <= 32, "a bit for each position");
#pragma unroll
      for (int kb = 0; kb < kTile / 16; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int ht = 0; ht < HT; ++ht)
            if (!(shown >> (kb * 16 + (lane >> 2) + (e >> 1) * 8) & 1)) sc[ht][kb][e] = -INFINITY;
    }
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      float mx[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = sc[ht][0][h];
#pragma unroll
        for (int kb = 0; kb < kTile / 16; ++kb) m = fmaxf(fmaxf(m, sc[ht][kb][h]), sc[ht][kb][h + 2]);
        // (scores of minus infinity are held against a finite value, which gives them the weight 0; top = -inf says that there was no
        // position at all)
        mx[h] = fmaxf(m * p.scale_log2, -FLT_MAX);
      }
#pragma unroll
      for (int s = 4; s < 32; s <<= 1)
#pragma unroll
        for (int h = 0; h < 2; ++h) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], s));
      if (__any_sync(0xffffffffu, mx[0] > top[ht][0] || mx[1] > top[ht][1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float m = fmaxf(mx[h], top[ht][h]);
          const float f = ex2(top[ht][h] - m);  // (a tile has a visible position, so m is above -inf)
          top[ht][h] = m;
          sum[ht][h] *= f;
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            o[ht][n][h] *= f;
            o[ht][n][h + 2] *= f;
          }
        }
      }
    }
#pragma unroll
    for (int kb = 0; kb < kTile / 16; ++kb) {
      uint32_t hi[HT][2], lo[HT][2];
#pragma unroll
      for (int ht = 0; ht < HT; ++ht)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = ex2(fmaf(sc[ht][kb][2 * e], p.scale_log2, -top[ht][0])), y = ex2(fmaf(sc[ht][kb][2 * e + 1], p.scale_log2, -top[ht][1]));
          sum[ht][0] += x;
          sum[ht][1] += y;
          split2<T>(x, y, hi[ht][e], lo[ht][e]);
          hi[ht][e] = movmatrix_trans(hi[ht][e]);
          lo[ht][e] = movmatrix_trans(lo[ht][e]);
        }
      // matrices of 8 positions x 8 elements, turned: elements are rows
      const int r = kb * 16 + (lane & 7) + ((lane >> 4) << 3), c0 = (lane >> 3) & 1;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t va[4];
        ldmatrix4_trans(vd + r * S::kRowBytes + (((n * 2 + c0) ^ (r & 7)) << 4), va);
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
          mma16816<T>(o[ht][n], va, hi[ht][0], hi[ht][1]);
          mma16816<T>(o[ht][n], va, lo[ht][0], lo[ht][1]);
        }
      }
    }
    __syncwarp();  // the stage is free for the load after next
  }
  cp_async_wait<0>();
#pragma unroll
  for (int ht = 0; ht < HT; ++ht)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) sum[ht][h] += __shfl_xor_sync(0xffffffffu, sum[ht][h], s);

  // ---- join the warps: [warp][row][D] weighted sums, then [warp][row] maxima and sums, in the ring's place
  __syncthreads();
  constexpr int kPitch = S::kPitch;
  float* const acc = reinterpret_cast<float*>(smem);
  float* const tops = acc + W * kRows * kPitch;
  float* const sums = tops + W * kRows;
#pragma unroll
  for (int ht = 0; ht < HT; ++ht)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = ht * 8 + (lane & 3) * 2 + h;
      if (r < rows) {
        float* const to = acc + (warp * kRows + r) * kPitch + (lane >> 2);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          to[n * 16] = o[ht][n][h];
          to[n * 16 + 8] = o[ht][n][h + 2];
        }
      }
      if (lane < 4) {
        tops[warp * kRows + r] = top[ht][h];
        sums[warp * kRows + r] = sum[ht][h];
      }
    }
  __syncthreads();
  // each warp's factor, and the CTA's maximum and sum in the first warp's place
  if (threadIdx.x < kRows) {
    const int r = threadIdx.x;
    float m = tops[r], f[W], total = 0.f;
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, tops[w * kRows + r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = tops[w * kRows + r];
      f[w] = mw == -INFINITY ? 0.f : ex2(mw - m);  // a warp without a position has the weight 0
      total += f[w] * sums[w * kRows + r];
    }
#pragma unroll
    for (int w = 0; w < W; ++w) s_scale[w][r] = f[w];
    tops[r] = m;
    sums[r] = total;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += W * 32) {
    const int r = i / D, at = r * kPitch + (i - r * D);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v = fmaf(s_scale[w][r], acc[w * kRows * kPitch + at], v);
    acc[at] = v;
  }
  // ---- join the CTAs: each takes a share of the outputs
  if (p.splits > 1) cluster.sync();
  else __syncthreads();
  if (threadIdx.x < kRows) {
    const int r = threadIdx.x;
    float m = -INFINITY, total = 0.f;
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, *cluster.map_shared_rank(tops + r, s));
    for (int s = 0; s < p.splits; ++s) {
      const float ms = *cluster.map_shared_rank(tops + r, s);
      const float f = ms == -INFINITY ? 0.f : ex2(ms - m);
      s_scale[s][r] = f;
      total += f * *cluster.map_shared_rank(sums + r, s);
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / total;  // nothing visible: zeros (every score minus infinity: 0 / 0)
    for (int s = 0; s < p.splits; ++s) s_scale[s][r] *= inv;
  }
  __syncthreads();
  const int pairs = rows * (D / 2);
  for (int i = split * W * 32 + threadIdx.x; i < pairs; i += p.splits * W * 32) {
    const int r = i / (D / 2), c = (i - r * (D / 2)) * 2;
    float2 v = make_float2(0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
      const float2 x = *reinterpret_cast<const float2*>(cluster.map_shared_rank(acc + r * kPitch + c, s));
      const float f = s_scale[s][r];
      v.x = fmaf(f, x.x, v.x);
      v.y = fmaf(f, x.y, v.y);
    }
    uint8_t* out = p.out + b * p.out_seq + (q_head0 + r) * p.out_head;
    *reinterpret_cast<uint32_t*>(out + c * 2) = pack2<T>(v.x, v.y);
  }
  if (p.splits > 1) cluster.sync();  // nobody leaves while its shared memory is read
}

template <class T, int D, int HT, int W>
int launch_attend(aig_ctx* ctx, AttendParams& p, int items, long long max_visible) {
  using S = AttendShape<D, HT, W>;
  // Splits: enough CTAs for every SM four times, each with a tile per warp at least.  Clusters of 16 leave SMs idle that
  // a group of 16 does not fit on (8 sequences of up to 65536: 179 to 191 us with 8, 192 to 200 with 16, five runs of each): only where
  // 8 would leave more (one sequence of 65536, 8 heads of 128: 104 with 8, 71 with 16).
  const int most = items * 8 < ctx->sm_count ? kMaxCluster : 8;
  p.splits = 1;
  while (p.splits < most && items * p.splits < 4 * ctx->sm_count && max_visible > (long long)p.splits * W * S::kTile) p.splits *= 2;
  auto kernel = paged_attention_kernel<T, D, HT, W>;
  AIG_CUDA_OK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
  if (p.splits > 8) AIG_CUDA_OK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)items * p.splits);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1] = pdl_attribute(ctx);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  AIG_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, kernel, p));
  return AIG_OK;
}
template <class T, int D, int HT>
int launch_attend(aig_ctx* ctx, AttendParams& p, int batch, long long max_visible) {
  p.row_blocks = ceil_div(p.group, 8 * HT);
  const long long items = (long long)batch * p.kv_heads * p.row_blocks;
  if (items * kMaxCluster > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "paged attention: too many sequences and heads for one call");
  return items >= 4 * ctx->sm_count ? launch_attend<T, D, HT, 2>(ctx, p, (int)items, max_visible) : launch_attend<T, D, HT, 4>(ctx, p, (int)items, max_visible);
}
template <class T, int D>
int launch_attend(aig_ctx* ctx, AttendParams& p, int batch, long long max_visible) {
  return p.group <= 8 ? launch_attend<T, D, 1>(ctx, p, batch, max_visible) : launch_attend<T, D, 2>(ctx, p, batch, max_visible);
}

}  // namespace

extern "C" {

int aig_kv_copy_pages(aig_ctx* ctx, const aig_kv_cache* cache, const int32_t* src, const int32_t* dst, int pairs) {
  if (!ctx) return AIG_ERR_INVALID;
  DeviceGuard g(ctx->device);
  const int rc = check_cache(ctx, cache, "kv copy pages");
  if (rc != AIG_OK) return rc;
  AIG_REQUIRE(ctx, pairs >= 0 && (pairs == 0 || (src && dst)), "kv copy pages: null list or negative number");
  for (int i = 0; i < pairs; ++i)
    AIG_REQUIRE(ctx, src[i] >= 0 && src[i] < cache->num_pages && dst[i] >= 0 && dst[i] < cache->num_pages,
                "kv copy pages: pair %d (%d -> %d) names no page of the pool", i, src[i], dst[i]);
  const char* const twice = "kv copy pages: pair %d (%d -> %d): a page is a destination twice, or a source and a destination";
  if (pairs <= kFewPairs) {  // (a fork's copy does not pay for a large pool)
    for (int i = 0; i < pairs; ++i)
      for (int j = 0; j < pairs; ++j) AIG_REQUIRE(ctx, dst[i] != src[j] && (i == j || dst[i] != dst[j]), twice, i, src[i], dst[i]);
  } else {
    try {
      std::vector<uint8_t> role(cache->num_pages, 0);  // 1: a source, 2: a destination
      for (int i = 0; i < pairs; ++i) {
        AIG_REQUIRE(ctx, role[dst[i]] == 0 && !(role[src[i]] & 2) && src[i] != dst[i], twice, i, src[i], dst[i]);
        role[src[i]] |= 1;
        role[dst[i]] |= 2;
      }
    } catch (const std::bad_alloc&) {
      return aig_fail(ctx, AIG_ERR_CUDA, "kv copy pages: out of host memory");
    }
  }
  CopyShape p;
  p.k = (uint4*)cache->k;
  p.v = (uint4*)cache->v;
  p.page = cache->page_stride / 8;
  p.place = cache->token_stride / 8;
  p.head = cache->head_stride / 8;
  const long long units = (long long)cache->page_size * cache->kv_heads * (cache->head_dim / 8);
  if (units > (1ll << 30)) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "kv copy pages: pages above 16 GB");
  p.units = (int)units;
  const int row = cache->head_dim / 8;
  const bool places_outside = (cache->kv_heads == 1 || p.head == row) && (cache->page_size == 1 || p.place == (long long)row * cache->kv_heads);
  const bool heads_outside = (cache->page_size == 1 || p.place == row) && (cache->kv_heads == 1 || p.head == (long long)row * cache->page_size);
  p.run = places_outside || heads_outside ? p.units : row;
  p.heads = places_outside || heads_outside ? 1 : cache->kv_heads;
  p.blocks = (int)ceil_div_ll(units, kCopyThreads * kCopyUnroll);
  return pairs <= kFewPairs ? launch_copies<kFewPairs>(ctx, p, src, dst, pairs) : launch_copies<kManyPairs>(ctx, p, src, dst, pairs);
}

int aig_paged_attention(aig_ctx* ctx, const aig_kv_cache* cache, const aig_heads* q, const aig_heads* out, const int32_t* table, int table_width,
                        const int32_t* lengths, int batch, int max_length, float scale, int window, int sinks) {
  if (!ctx) return AIG_ERR_INVALID;
  DeviceGuard g(ctx->device);
  const int rc = check_cache(ctx, cache, "paged attention");
  if (rc != AIG_OK) return rc;
  if (cache->head_dim != 64 && cache->head_dim != 128)
    return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "paged attention: head dimension must be 64 or 128 (got %d)", cache->head_dim);
  AIG_REQUIRE(ctx, batch >= 0 && table_width > 0 && max_length >= 0 && sinks >= 0, "paged attention: bad extents");
  AIG_REQUIRE(ctx, scale > 0.f && scale - scale == 0.f, "paged attention: the scale has to be positive and finite");
  if (batch == 0) return AIG_OK;
  AIG_REQUIRE(ctx, heads_sane(q) && heads_sane(out) && table && lengths && aligned_to(table, 4) && aligned_to(lengths, 4),
              "paged attention: null tensor, negative stride, or integers off a 4-byte boundary");
  AIG_REQUIRE(ctx, heads_vectorised(*q) && heads_vectorised(*out), "paged attention: q and out on 16-byte boundaries, strides multiples of 8");
  AIG_REQUIRE(ctx, q->heads == out->heads && q->heads % cache->kv_heads == 0, "paged attention: %d query heads, %d in the output, %d cached", q->heads,
              out->heads, cache->kv_heads);
  AttendParams p{};
  p.k = (const uint8_t*)cache->k;
  p.v = (const uint8_t*)cache->v;
  p.q = (const uint8_t*)q->data;
  p.out = (uint8_t*)out->data;
  p.page = cache->page_stride * 2;
  p.place = cache->token_stride * 2;
  p.head = cache->head_stride * 2;
  p.q_seq = q->token_stride * 2;
  p.q_head = q->head_stride * 2;
  p.out_seq = out->token_stride * 2;
  p.out_head = out->head_stride * 2;
  p.table = table;
  p.lengths = lengths;
  p.table_width = table_width;
  p.page_size = Divisor::of(cache->page_size);
  p.num_pages = cache->num_pages;
  p.kv_heads = cache->kv_heads;
  p.group = q->heads / cache->kv_heads;
  p.window = window;
  p.sinks = sinks;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.gerr = ctx->d_err;
  long long visible = max_length;
  if (window > 0 && visible > (long long)window + sinks) visible = (long long)window + sinks;
  if (cache->dtype == AIG_F16)
    return cache->head_dim == 64 ? launch_attend<__half, 64>(ctx, p, batch, visible) : launch_attend<__half, 128>(ctx, p, batch, visible);
  return cache->head_dim == 64 ? launch_attend<__nv_bfloat16, 64>(ctx, p, batch, visible) : launch_attend<__nv_bfloat16, 128>(ctx, p, batch, visible);
}

}  // extern "C"

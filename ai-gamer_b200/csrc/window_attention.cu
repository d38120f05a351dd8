// window_attention.cu -- causal attention over whole sequences with a sliding window and first tokens that stay visible
// (sinks), and its gradients.
//
//   S = scale * Q K^T,  P = softmax(S) over the keys j <= p that are within `window` of p or below `sinks`,  O = P V
//   dV = P^T dO,  dP = dO V^T,  D = rowsum(dO o O),  dS = scale * P o (dP - D),  dQ = dS K,  dK = dS^T Q
//
// Forward: tiles of 128 queries x 128 keys on tcgen05.  A CTA has one or two tiles of queries, each with 128 threads that
// own a row of scores; one warp fetches tiles by TMA, one issues the products.  Scores and outputs stay in TMEM; the
// weights go back to TMEM as 16-bit values over the scores and are the second product's A operand from there, V its B
// operand as it lies in memory (MN-major).  Tiles that the window, the sinks and the causal order leave empty are not
// visited; only tiles that they cut are masked.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "long_context.h"

namespace {

constexpr int kTile = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct View {
  uint8_t* data;
  long long batch, token, head;  // strides in elements
};

struct WinParams {
  View q, k, v, o, dout, dq, dk, dv;
  float *lse, *delta;
  const int32_t* lengths;
  int batch, q_len, kv_len, heads, kv_heads;
  int window, sinks;
  float scale;
  int blocks;  // of query rows per head
  int first_block, split;  // of a launch of the dK and dV kernel: its first block of keys, log2 of CTAs per block
  bool leads, after;        // it overlaps the launch behind it, before it
  int* gerr;
};

// ---- PTX that the other kernels have no use for
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* desc, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(desc)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// tcgen05.mma and commit by the lane whose `issue` is set.  The predicate is inside: the whole warp runs the code around it
// with the same values, so that descriptors are advanced in uniform registers.  (In a branch that one lane takes, every
// operand is moved from a vector register: four products and two commits took 365 clocks to issue.)  Descriptors are given by
// their low words; the high word is the same for all tiles here.
constexpr uint32_t kDescHi = umma_desc_hi(128);
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t issue, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 l, %6, 0;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(accumulate), "r"(issue)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t issue, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 l, %6, 0;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(accumulate), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t issue, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %1, 0;\n\t"
      "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// two operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 pair_of(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
// bits 0 .. n-1
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
constexpr uint32_t kMinusInf = 0xff800000u;
// The roles' shares of a block's registers (by all warps of a group of four)
template <int R>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
// A bounded wait whose answer all lanes of the warp share
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* gerr, int code) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, gerr, code));
}
template <class T>
__host__ __device__ constexpr uint32_t idesc_for(int m, int n, bool b_mn_major) {
  return umma_idesc_f16(m, n) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7 | 1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u);
}

// A tile of R rows of D elements as D/64 blocks of [R rows][64 elements], 128-byte swizzled
template <int D, int R>
constexpr uint32_t kTileBytes = R * D * 2;
// by boxes of B rows
template <int D, int R, int B>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int row, int b) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int r = 0; r < R; r += B) tma_load_4d(dst + (c * R + r) * 128, map, bar, c * 64, head, row + r, b);
}
// Low descriptor words of a tile as a K-major operand, K step `ks` of 16 elements of its rows (128-byte swizzled, groups of
// eight rows 1024 bytes apart) ...
template <int R>
__device__ __forceinline__ uint32_t desc_k(uint32_t tile, int ks) { return umma_desc_lo(tile) + (((ks >> 2) * R * 128 + (ks & 3) * 32) >> 4); }
// ... and with its rows as the K dimension, K step of 16 rows (64 elements of N per row, the next 64 a block further on)
template <int R>
__device__ __forceinline__ uint32_t desc_rows(uint32_t tile, int ks) { return ((tile & 0x3FFFFu) >> 4 | (uint32_t)(R * 128 / 16) << 16) + ks * (16 * 128 / 16); }
// Rows from `from` on become zeros (a product with the weight 0 would keep a NaN); by one warp, before the product reads them
template <int D, int R>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int from, int lane) {
  const int pieces = (R - from) * 8;
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    for (int i = lane; i < pieces; i += 32) *reinterpret_cast<uint4*>(tile + c * R * 128 + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// N values of a row in TMEM, times f, to memory (every lane takes part in the reads)
template <class T, int N>
__device__ __forceinline__ void store_row(uint32_t taddr, T* out, float f, bool there) {
#pragma unroll
  for (int c0 = 0; c0 < N; c0 += 32) {
    uint32_t v[32];
    tmem_ld_32x32(taddr + c0, v);
    tmem_ld_wait();
    if (there) {
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        uint4 x;
        x.x = pack2<T>(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f);
        x.y = pack2<T>(__uint_as_float(v[e + 2]) * f, __uint_as_float(v[e + 3]) * f);
        x.z = pack2<T>(__uint_as_float(v[e + 4]) * f, __uint_as_float(v[e + 5]) * f);
        x.w = pack2<T>(__uint_as_float(v[e + 6]) * f, __uint_as_float(v[e + 7]) * f);
        *reinterpret_cast<uint4*>(out + c0 + e) = x;
      }
    }
  }
}

// N sums of a row in TMEM, times f
template <int N>
__device__ __forceinline__ void scale_row(uint32_t taddr, float f) {
#pragma unroll 1
  for (int c0 = 0; c0 < N; c0 += 16) {
    uint32_t v[16];
    tmem_ld_32x16(taddr + c0, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
    tmem_st_32x16(taddr + c0, v);
  }
}

// Tiles of R keys that queries at positions first .. last visit: [0, sink_end) and [begin, end)
struct KeyTiles {
  int sink_end, begin, end;
  __device__ __forceinline__ bool has(int t) const { return t < sink_end || (t >= begin && t < end); }
};
template <int R>
__device__ __forceinline__ KeyTiles key_tiles(int first, int last, int window, int sinks) {
  KeyTiles k;
  k.begin = window > 0 ? max(0, first - window + 1) / R : 0;
  k.end = last < first ? k.begin : last / R + 1;
  k.sink_end = window > 0 && last >= first ? min((sinks + R - 1) / R, k.begin) : 0;
  return k;
}

// ---- CTAs of a cluster that share a sum: each keeps its part in its shared memory, rows of N floats, 16-byte pieces exchanged so that
// eight threads' own rows fall into different banks
template <int N>
__device__ __forceinline__ uint32_t kept_at(int r, int column) {
  return (uint32_t)(r * 4 * N + ((column / 4 ^ (r & 7)) << 4));
}
template <int N, int Columns>
__device__ __forceinline__ void keep_row(uint32_t taddr, uint32_t to, int r, int column, float f) {
#pragma unroll
  for (int c0 = 0; c0 < Columns; c0 += 32) {
    uint32_t v[32];
    tmem_ld_32x32(taddr + c0, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; e += 4)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + kept_at<N>(r, column + c0 + e)), "f"(__uint_as_float(v[e]) * f),
                   "f"(__uint_as_float(v[e + 1]) * f), "f"(__uint_as_float(v[e + 2]) * f), "f"(__uint_as_float(v[e + 3]) * f)
                   : "memory");
  }
}
__device__ __forceinline__ float2 peer_load2(uint32_t cluster_addr) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(cluster_addr) : "memory");
  return x;
}
__device__ __forceinline__ float4 peer_load(uint32_t cluster_addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(cluster_addr) : "memory");
  return x;
}

// first of n units of work of part r of 2^split
__device__ __forceinline__ int part_begin(int n, int split, int r) { return (n >> split) * r + min(r, n & ((1 << split) - 1)); }
// The parts' sums of a share of the 128 rows for each CTA, in a fixed order, eight reads under way per thread; `work`: units that were
// shared (a part may have had none).  store(row, column, four sums).
template <int N, int Threads, class Store>
__device__ __forceinline__ void join_rows(uint32_t base, int work, int split, int part, Store store) {
  const int parts = 1 << split, rows = kTile >> split, units = rows * (N / 4);  // of four columns
  for (int i = threadIdx.x; i < units; i += Threads << (3 - split)) {
    float4 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int n = k & (parts - 1), at = i + (k >> split) * Threads;
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at < units && part_begin(work, split, n + 1) > part_begin(work, split, n))
        x[k] = peer_load(mapa_shared(base + kept_at<N>(part * rows + at / (N / 4), at % (N / 4) * 4), (uint32_t)n));
    }
#pragma unroll
    for (int step = 1; step < 8; step *= 2)
#pragma unroll
      for (int k = 0; k < 8; k += 2 * step)
        if (step < parts) x[k] = make_float4(x[k].x + x[k + step].x, x[k].y + x[k + step].y, x[k].z + x[k + step].z, x[k].w + x[k + step].w);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int at = i + (k >> split) * Threads;
      if ((k & (parts - 1)) == 0 && at < units) store(part * rows + at / (N / 4), at % (N / 4) * 4, x[k]);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Forward
template <int D, int NT, bool Split>  // NT tiles of queries
struct FwdShape {
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kThreads = 128 + 128 * NT;
  static constexpr int kCtasPerSm = NT == 1 && D == 64 && !Split ? 2 : 1;
  // registers of the warps that fetch and issue, and of those that hold a row of scores: 128 x 64 + 256 x 216 of a block's 384 x 168,
  // 128 x 64 + 128 x 192 of its 256 x 128 (with 40 the issuing warp spills: 72 us where it takes 69); one CTA of one tile to an SM has enough
  static constexpr int kFewer = NT == 2 || kCtasPerSm == 2 ? 64 : 0, kMore = NT == 2 ? 216 : 192;
  static constexpr int kTmemCols = NT == 2 ? 512 : 256;  // scores 128 columns a tile, then outputs D columns a tile
  static constexpr uint32_t kQ = NT * kTileBytes<D, kTile>;
  static constexpr size_t kSmem = kQ + 2 * kStages * kTileBytes<D, kTile> + 256;
};
constexpr float kLazy = 8.f;  // a row's maximum may grow by 2^8 before its sums are rescaled: weights stay below 2^8

// Split: a tile of queries is a cluster's, each of whose CTAs has a part of the keys.
template <class T, int D, int NT, bool Split>
__global__ void __launch_bounds__((FwdShape<D, NT, Split>::kThreads), (FwdShape<D, NT, Split>::kCtasPerSm))
window_forward_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                      const __grid_constant__ WinParams p) {
  static_assert(!Split || NT == 1, "one tile of queries is shared");
  using S = FwdShape<D, NT, Split>;
  constexpr int NS = S::kStages;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t base = smem_u32(sm);
  if (base & 1023u) {  // (never seen; tiles could not be fetched)
    if (threadIdx.x == 0) note_error(p.gerr, 1100);
    return;
  }
  const uint32_t sQ = base, sK = sQ + S::kQ, sV = sK + NS * kTileBytes<D, kTile>;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + S::kQ + 2 * NS * kTileBytes<D, kTile>);
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, s_full = bar0 + 8, p_full = s_full + 8 * NT, o_full = p_full + 8 * NT, k_full = o_full + 8 * NT,
                 k_free = k_full + 8 * NS, v_full = k_free + 8 * NS, v_free = v_full + 8 * NS;
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + 1 + 3 * NT + 4 * NS);
  volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  float2* const s_stat = reinterpret_cast<float2*>(sm + kTile * D * 4);  // [128], behind a part's rows
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  // the blocks of the last queries, which see the most keys, come first
  const int split = Split ? p.split : 0, parts = 1 << split, part = blockIdx.x & (parts - 1);
  int item = blockIdx.x >> split;
  const int b = item % p.batch;
  item /= p.batch;
  const int h = item % p.heads, block = p.blocks - 1 - item / p.heads;
  const int kvh = h / (p.heads / p.kv_heads);
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.kv_len) : p.kv_len;
  const int off = p.kv_len - p.q_len;  // position of query row 0
  const int rows_end = min(p.q_len, len - off);
  KeyTiles kt[NT];
  int sink_end = 0, begin = 0x7fffffff, end = 0;
#pragma unroll
  for (int w = 0; w < NT; ++w) {
    const int r0 = (block * NT + w) * kTile;
    kt[w] = key_tiles<kTile>(off + r0, off + min(r0 + kTile, rows_end) - 1, p.window, p.sinks);
    if (kt[w].end > kt[w].begin) {
      sink_end = max(sink_end, kt[w].sink_end);
      begin = min(begin, kt[w].begin);
      end = max(end, kt[w].end);
    }
  }
  if (end == 0) return;  // no query row within the sequence
  begin = max(begin, sink_end);
  const int all_tiles = sink_end + end - begin;
  const int skipped = part_begin(all_tiles, split, part), tiles = part_begin(all_tiles, split, part + 1) - skipped;
  auto tile_at = [&](int it) { return (Split ? it + skipped : it) < sink_end ? (Split ? it + skipped : it) : begin + ((Split ? it + skipped : it) - sink_end); };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int w = 0; w < NT; ++w) {
      mbar_init(s_full + 8 * w, 1);
      mbar_init(p_full + 8 * w, 128);
      mbar_init(o_full + 8 * w, 1);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(k_full + 8 * s, 1);
      mbar_init(k_free + 8 * s, 1);
      mbar_init(v_full + 8 * s, 1);
      mbar_init(v_free + 8 * s, 1);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(s_tmem), S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const uint32_t tS = tmem, tO = tmem + 128 * NT;

  if (S::kFewer > 0 && warp < 4) fewer_registers<S::kFewer>();
  if (warp == 0) {
    if (lane == 0 && (!Split || tiles > 0)) {
      mbar_expect_tx(q_full, S::kQ);
#pragma unroll
      for (int w = 0; w < NT; ++w) load_tile<D, kTile, kTile>(sQ + w * kTileBytes<D, kTile>, &mapQ, q_full, h, (block * NT + w) * kTile, b);
      for (int it = 0; it < tiles; ++it) {
        const int s = it % NS, row = tile_at(it) * kTile;
        const uint32_t ph = (uint32_t)(it / NS + 1) & 1u;  // (the first round finds the stages free)
        if (it >= NS && !mbar_wait_bounded(k_free + 8 * s, ph, s_abort, p.gerr, 1101)) break;
        mbar_expect_tx(k_full + 8 * s, kTileBytes<D, kTile>);
        load_tile<D, kTile, kTile>(sK + s * kTileBytes<D, kTile>, &mapK, k_full + 8 * s, kvh, row, b);
        if (it >= NS && !mbar_wait_bounded(v_free + 8 * s, ph, s_abort, p.gerr, 1102)) break;
        mbar_expect_tx(v_full + 8 * s, kTileBytes<D, kTile>);
        load_tile<D, kTile, kTile>(sV + s * kTileBytes<D, kTile>, &mapV, v_full + 8 * s, kvh, row, b);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = idesc_for<T>(kTile, kTile, false), idesc_o = idesc_for<T>(kTile, D, true);
    const uint32_t leader = elect_one() ? 1u : 0u;
    int done[NT];  // tiles whose second product has been issued
#pragma unroll
    for (int w = 0; w < NT; ++w) done[w] = 0;
    auto scores = [&](int w, int it) {
      const uint32_t k = sK + (it % NS) * kTileBytes<D, kTile>;
      {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) mma_ss(leader, tS + 128 * w, desc_k<kTile>(sQ + w * kTileBytes<D, kTile>, ks), desc_k<kTile>(k, ks), idesc_s, ks != 0);
        commit(leader, s_full + 8 * w);
      }
    };
    bool ok = (!Split || tiles > 0) && warp_wait(q_full, 0, s_abort, p.gerr, 1103) && warp_wait(k_full, 0, s_abort, p.gerr, 1104);
    if (ok) {
      tc_fence_after();
#pragma unroll
      for (int w = 0; w < NT; ++w)
        if (kt[w].has(tile_at(0))) scores(w, 0);
      commit(leader, k_free);
      for (int it = 0; it < tiles && ok; ++it) {
        const int t = tile_at(it), s = it % NS, next = it + 1, ns = next % NS;
        if (next < tiles && !warp_wait(k_full + 8 * ns, (uint32_t)(next / NS) & 1u, s_abort, p.gerr, 1105)) break;
        if (!warp_wait(v_full + 8 * s, (uint32_t)(it / NS) & 1u, s_abort, p.gerr, 1106)) break;
        if (t * kTile + kTile > len) clear_rows<D, kTile>(sm + (sV - base) + s * kTileBytes<D, kTile>, len - t * kTile, lane);
#pragma unroll
        for (int w = 0; w < NT; ++w) {
          if (kt[w].has(t)) {
            if (!(ok = warp_wait(p_full + 8 * w, (uint32_t)done[w] & 1u, s_abort, p.gerr, 1107))) break;
            tc_fence_after();
            {
#pragma unroll
              for (int ks = 0; ks < kTile / 16; ++ks)
                mma_ts(leader, tO + D * w, tS + 128 * w + ks * 8, desc_rows<kTile>(sV + s * kTileBytes<D, kTile>, ks), idesc_o, done[w] != 0 || ks != 0);
            }
            ++done[w];
            if (Split ? next == tiles : t + 1 == kt[w].end) commit(leader, o_full + 8 * w);
          }
          if (next < tiles && kt[w].has(tile_at(next))) scores(w, next);
        }
        {
          commit(leader, v_free + 8 * s);
          if (next < tiles) commit(leader, k_free + 8 * ns);
        }
      }
    }
  } else if (warp >= 4) {
    if (S::kFewer > 0) more_registers<S::kMore>();
    const int w = (warp - 4) >> 2, q = warp & 3;
    const int row = (block * NT + w) * kTile + q * 32 + lane, pos = off + row;
    const int first = off + (block * NT + w) * kTile;  // position of the tile's first row
    KeyTiles mine = kt[0];
    if (NT == 2 && w == 1) mine = kt[NT - 1];
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t tSw = tS + 128 * w + lanes, tOw = tO + D * w + lanes;
    const float c = p.scale * kLog2e;
    float top = -INFINITY, sum = 0.f;  // top: in units of log2, what the weights are relative to
    int n = 0;
    bool ok = true;
    for (int it = 0; it < tiles; ++it) {
      const int t = tile_at(it);
      if (!mine.has(t)) continue;
      if (!(ok = warp_wait(s_full + 8 * w, (uint32_t)n & 1u, s_abort, p.gerr, 1108))) break;
      tc_fence_after();
      const int j0 = t * kTile;
      const bool cut = j0 + kTile - 1 > first || (p.window > 0 && j0 <= first + kTile - 1 - p.window && j0 + kTile > p.sinks);
      const int lo = p.window > 0 ? pos - p.window + 1 - j0 : -1, hi = pos - j0, sinks = p.sinks - j0;  // columns
      uint32_t v[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld_32x32(tSw + 32 * i, v[i]);
      tmem_ld_wait();
      if (cut) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t shown = bits_below(hi + 1 - 32 * i) & (~bits_below(lo - 32 * i) | bits_below(sinks - 32 * i));
#pragma unroll
          for (int e = 0; e < 32; ++e) v[i][e] = shown >> e & 1 ? v[i][e] : kMinusInf;
        }
      }
      float part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part[i] = __uint_as_float(v[i][0]);
#pragma unroll
        for (int e = 1; e < 31; e += 2) part[i] = fmaxf(fmaxf(part[i], __uint_as_float(v[i][e])), __uint_as_float(v[i][e + 1]));
        part[i] = fmaxf(part[i], __uint_as_float(v[i][31]));
      }
      const float m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * c;
      const bool grew = m > top + kLazy;  // (from -inf any finite value)
      if (__any_sync(0xffffffffu, grew)) {
        const float f = grew ? ex2(top - m) : 1.f;
        if (grew) {
          top = m;
          sum *= f;
        }
        if (n > 0) scale_row<D>(tOw, f);  // the products that went into the output have completed: the scores were issued behind them
      }
      const float ref = top == -INFINITY ? 0.f : top;  // a row that has seen no key yet
      float2 sums[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = fma2(pair_of(v[i][e], v[i][e + 1]), make_float2(c, c), make_float2(-ref, -ref));
          const float2 y = make_float2(ex2(x.x), ex2(x.y));
          sums[(e >> 1) & 3] = i == 0 && e < 8 ? y : add2(sums[(e >> 1) & 3], y);
          o[e / 2] = pack2<T>(y.x, y.y);
        }
        tmem_st_32x16(tSw + 16 * i, o);  // over scores that have been read
      }
      sums[0] = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
      sum += sums[0].x + sums[0].y;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full + 8 * w);
      ++n;
    }
    if (ok && n > 0 && warp_wait(o_full + 8 * w, 0, s_abort, p.gerr, 1109)) {
      tc_fence_after();
      if constexpr (Split) {  // (the tiles' places are free: every product is done)
        keep_row<D, D>(tOw, base, q * 32 + lane, 0, 1.f);
        s_stat[q * 32 + lane] = make_float2(top, sum);
      } else {
        const float inv = 1.f / sum;
        T* const out = reinterpret_cast<T*>(p.o.data) + b * p.o.batch + row * p.o.token + h * p.o.head;
        store_row<T, D>(tOw, out, inv, row < rows_end);
        if (row < rows_end) p.lse[((long long)b * p.heads + h) * p.q_len + row] = fmaf(top, kLn2, logf(sum));
      }
    }
  }

  if (*s_abort) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
  if constexpr (Split) {  // the parts' sums, in a fixed order: a share of the rows for each CTA, eight reads under way per thread
    cluster_sync_all();
    const int rows = kTile >> split, units = rows * (D / 4);  // of four columns
    for (int i = threadIdx.x; i < units; i += S::kThreads << (3 - split)) {
      float4 x[8];
      float2 stat[8];  // what the weights are relative to, their sum
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int n = k & (parts - 1), at = i + (k >> split) * S::kThreads, r = part * rows + at / (D / 4);
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        stat[k] = make_float2(-INFINITY, 0.f);
        if (at < units && part_begin(all_tiles, split, n + 1) > part_begin(all_tiles, split, n)) {  // (a part may have had no keys)
          x[k] = peer_load(mapa_shared(base + kept_at<D>(r, at % (D / 4) * 4), (uint32_t)n));
          stat[k] = peer_load2(mapa_shared(smem_u32(s_stat + r), (uint32_t)n));
        }
      }
#pragma unroll
      for (int step = 1; step < 8; step *= 2)
#pragma unroll
        for (int k = 0; k < 8; k += 2 * step)
          if (step < parts) {
            const float top = fmaxf(stat[k].x, stat[k + step].x), ref = top == -INFINITY ? 0.f : top;
            const float f = ex2(stat[k].x - ref), g = ex2(stat[k + step].x - ref);
            x[k] = make_float4(f * x[k].x + g * x[k + step].x, f * x[k].y + g * x[k + step].y, f * x[k].z + g * x[k + step].z, f * x[k].w + g * x[k + step].w);
            stat[k] = make_float2(top, f * stat[k].y + g * stat[k + step].y);
          }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = i + (k >> split) * S::kThreads, row = block * kTile + part * rows + at / (D / 4), c = at % (D / 4) * 4;
        if ((k & (parts - 1)) != 0 || at >= units || row >= rows_end) continue;
        const float inv = 1.f / stat[k].y;
        T* const to = reinterpret_cast<T*>(p.o.data) + b * p.o.batch + row * p.o.token + h * p.o.head + c;
        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(x[k].x * inv, x[k].y * inv), pack2<T>(x[k].z * inv, x[k].w * inv));
        if (c == 0) p.lse[((long long)b * p.heads + h) * p.q_len + row] = fmaf(stat[k].x, kLn2, logf(stat[k].y));
      }
    }
    cluster_sync_all();  // nobody leaves while its shared memory is read
  }
}

// ---------------------------------------------------------------------------------------------
// Forward, short sequences: 64 queries of a head per CTA of four warps, products by mma.sync.  A sequence of 64 is half a tile of
// the tcgen05 kernel, whose CTA owns an SM and spends its time on the way there and back; of these CTAs four or seven to an
// SM hide one another's (1024 heads of 64 x 64: 8.7 us against 31.5; four to an SM 10.8).  One or two tiles of keys, fetched at once.
constexpr int kShort = 64;

template <int D, int Tiles>
struct ShortShape {
  static constexpr uint32_t kTileB = kShort * D * 2;
  static constexpr size_t kSmem = (1 + 2 * Tiles) * kTileB;  // queries, keys and values
  static constexpr int kCtasPerSm = Tiles == 1 && D == 64 ? 7 : 4;
};

// 64 rows of D elements, 16-byte pieces of a row exchanged so that those of eight rows fall into different banks
template <int D>
__device__ __forceinline__ uint32_t short_at(int r, int c) {
  return (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4));
}
template <class T, int D>
__device__ __forceinline__ void short_load(uint32_t to, const View& v, int b, int h, int first, int end, int tid) {
  constexpr int kPieces = D / 8, kStep = 128 / kPieces;  // rows that the CTA's threads fetch at once
  const int r = tid / kPieces, c = tid % kPieces;
  const T* from = reinterpret_cast<const T*>(v.data) + b * v.batch + h * v.head + (first + r) * v.token + c * 8;
  const T* const some = reinterpret_cast<const T*>(v.data);  // (an address for copies of no bytes)
#pragma unroll
  for (int i = 0; i < kShort / kStep; ++i, from += kStep * v.token) {
    const bool there = first + r + i * kStep < end;
    cp_async16(to + short_at<D>(r + i * kStep, c), there ? from : some, there ? 16 : 0);
  }
}

template <class T, int D, int Tiles>
__global__ void __launch_bounds__(128, (ShortShape<D, Tiles>::kCtasPerSm)) window_short_kernel(const __grid_constant__ WinParams p) {
  using S = ShortShape<D, Tiles>;
  extern __shared__ __align__(1024) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int item = blockIdx.x;
  const int b = item % p.batch;
  item /= p.batch;
  const int h = item % p.heads, r0 = (p.blocks - 1 - item / p.heads) * kShort;
  const int kvh = h / (p.heads / p.kv_heads);
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.kv_len) : p.kv_len;
  const int off = p.kv_len - p.q_len;
  const int rows_end = min(p.q_len, len - off);
  if (r0 >= rows_end) return;
  const KeyTiles kt = key_tiles<kShort>(off + r0, off + min(r0 + kShort, rows_end) - 1, p.window, p.sinks);
  const int tiles = Tiles == 1 ? 1 : kt.sink_end + kt.end - kt.begin;
  auto first_key = [&](int u) { return Tiles == 1 ? 0 : (u < kt.sink_end ? u : kt.begin + (u - kt.sink_end)) * kShort; };
  const uint32_t sQ = smem_u32(sm);
  auto stage = [&](int u) { return sQ + S::kTileB * (1 + 2 * u); };  // keys, then values
  auto fetch = [&](int u) {
    if (u < tiles) {
      short_load<T, D>(stage(u), p.k, b, kvh, first_key(u), len, threadIdx.x);
      short_load<T, D>(stage(u) + S::kTileB, p.v, b, kvh, first_key(u), len, threadIdx.x);
    }
    cp_async_commit();
  };
  short_load<T, D>(sQ, p.q, b, h, r0, rows_end, threadIdx.x);
#pragma unroll
  for (int u = 0; u < Tiles; ++u) fetch(u);
  cp_async_wait<Tiles - 1>();
  __syncthreads();
  float o[D / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};  // of rows lane/4 and lane/4 + 8 of the warp's 16
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  const float c = p.scale * kLog2e;
  const int first = off + r0 + warp * 16;  // position of the warp's first row
  for (int u = 0; u < tiles; ++u) {
    if (u > 0) {
      cp_async_wait<0>();
      __syncthreads();
    }
    const uint32_t sK = stage(u), sV = sK + S::kTileB;
    const int j0 = first_key(u);
    const int keys = first + 16 - j0;  // of the tile, up to the warp's last row's own
    float sc[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][e] = (n & ~1) * 8 < keys ? 0.f : -INFINITY;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t qa[4];  // (read again for every tile: held, they would cost an SM some of its CTAs)
      ldmatrix4(sQ + short_at<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)), qa);
#pragma unroll
      for (int n = 0; n < 8; n += 2) {
        if (n * 8 >= keys) continue;
        uint32_t kb[4];
        ldmatrix4(sK + short_at<D>(n * 8 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), kb);
        mma16816<T>(sc[n], qa, kb[0], kb[1]);
        mma16816<T>(sc[n + 1], qa, kb[2], kb[3]);
      }
    }
    const bool cut = j0 + kShort - 1 > first || (p.window > 0 && j0 <= first + 15 - p.window && j0 + kShort > p.sinks);
    if (cut) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int pos = first + (lane >> 2) + 8 * x - j0, lo = p.window > 0 ? pos - p.window + 1 : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // 32 keys, this thread's from bit 0 on
          const uint32_t shown = (bits_below(pos + 1 - 32 * i) & (~bits_below(lo - 32 * i) | bits_below(p.sinks - j0 - 32 * i))) >> ((lane & 3) * 2);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (!(shown >> (8 * n) & 1)) sc[4 * i + n][2 * x] = -INFINITY;
            if (!(shown >> (8 * n + 1) & 1)) sc[4 * i + n][2 * x + 1] = -INFINITY;
          }
        }
      }
    }
    float ref[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float m = fmaxf(sc[0][2 * x], sc[0][2 * x + 1]);
#pragma unroll
      for (int n = 1; n < 8; ++n) m = fmaxf(fmaxf(m, sc[n][2 * x]), sc[n][2 * x + 1]);
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2)) * c, top[x]);
      if (u == 0) {
        top[x] = m;
      } else if (__any_sync(0xffffffffu, m > top[x])) {
        const float f = m > top[x] ? ex2(top[x] - m) : 1.f;
        top[x] = m;
        sum[x] *= f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * x] *= f;
          o[n][2 * x + 1] *= f;
        }
      }
      ref[x] = top[x] == -INFINITY ? 0.f : top[x];  // a row that has seen no key yet
    }
    uint32_t w[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // rows lane/4 and + 8 of 8 keys, then of the next 8
        const float x = ex2(fmaf(sc[2 * ks + (e >> 1)][2 * (e & 1)], c, -ref[e & 1])), y = ex2(fmaf(sc[2 * ks + (e >> 1)][2 * (e & 1) + 1], c, -ref[e & 1]));
        sum[e & 1] += x + y;
        w[ks][e] = pack2<T>(x, y);
      }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks * 16 >= keys) continue;
      const int r = ks * 16 + (lane & 15), c0 = lane >> 4;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t vb[4];
        ldmatrix4_trans(sV + short_at<D>(r, n * 2 + c0), vb);
        mma16816<T>(o[2 * n], w[ks], vb[0], vb[1]);
        mma16816<T>(o[2 * n + 1], w[ks], vb[2], vb[3]);
      }
    }
  }
  // ---- results through the warp's own rows of the queries' place, so that they leave in 16-byte pieces
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
    sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
    const float inv = 1.f / sum[x];
    const int r = warp * 16 + (lane >> 2) + 8 * x, row = r0 + r;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<uint32_t*>(sm + short_at<D>(r, n) + (lane & 3) * 4) = pack2<T>(o[n][2 * x] * inv, o[n][2 * x + 1] * inv);
    if ((lane & 3) == 0 && row < rows_end) p.lse[((long long)b * p.heads + h) * p.q_len + row] = fmaf(top[x], kLn2, logf(sum[x]));
  }
  __syncwarp();
  T* const out = reinterpret_cast<T*>(p.o.data) + b * p.o.batch + h * p.o.head;
#pragma unroll
  for (int i = 0; i < 16 * (D / 8) / 32; ++i) {
    const int r = warp * 16 + (i * 32 + lane) / (D / 8), piece = (i * 32 + lane) % (D / 8);
    if (r0 + r < rows_end) *reinterpret_cast<uint4*>(out + (r0 + r) * p.o.token + piece * 8) = *reinterpret_cast<const uint4*>(sm + short_at<D>(r, piece));
  }
}

// ---------------------------------------------------------------------------------------------
// Backward: one kernel for dQ (a tile of 128 queries stays, keys pass by), one for dK and dV (a tile of 128 keys stays, the
// queries of the group's heads pass by).  Each computes the weights again from lse: two more products than one kernel that
// adds dQ into memory with atomics would need, but every sum has a fixed order.  A thread owns a row of scores, 64 columns of it
// at a time.  Bound by the chain from products to exponentials to products: so two tiles are under way on an SM, in two groups of
// 128 threads of one CTA or in two CTAs.  (2 x 4099, 16 heads of 64: 208 us; one tile of 128 at a time for both groups 257; now 210.)
//
// fp16 has few small numbers: weights of a row over thousands of keys, and dS of small gradients, would be rounded to
// multiples of 2^-24.  So the weights are multiplied by 2^8, and dS by a power of two 2^k that follows the largest
// |dO| * |V| seen so far: typical ones lie around 1.  dS = P (dP - D), and D comes from the values of all keys that a query sees, other
// tiles' too (this one's may be zero): the power follows the queries' |D| as well.  Then 2^k |dP| < 2^14 (|dO| |V| times 2^3, 2^4
// for heads of 128, is held below 2^11, and a sum of 64 or 128 products is at most 2^3 times that) and 2^k |D| < 2^11: no dS passes fp16's
// largest value.  Where a tile asks for a smaller power the sums so far are scaled (rare: it keeps two bits in hand).
constexpr int kSub = 64;
template <class T>
constexpr int kWeightBits = std::is_same<T, __half>::value ? 8 : 0;
constexpr int kMostBits = 11, kAimBits = 9;  // of 2^k * |dO| * |V| * sqrt(D)

__device__ __forceinline__ float pow2(int k) { return __int_as_float((k + 127) << 23); }  // -126 .. 127

// Exponent e with x < 2^e (x finite and not negative, as bits; -126 at least)
__device__ __forceinline__ int exponent_of(uint32_t x) { return (int)(x >> 23) - 126; }
// ... with |x| < 2^e for this lane's values of rows [0, rows) of a tile in shared memory ...
template <int D, int R>
__device__ __forceinline__ int lane_exponent(const uint8_t* tile, int rows, int lane) {
  __half2 m[2] = {__half2half2(__ushort_as_half(0)), __half2half2(__ushort_as_half(0))};
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll 4
    for (int i = lane; i < rows * 8; i += 32) {
      const uint4 v = *reinterpret_cast<const uint4*>(tile + c * R * 128 + i * 16);
      const __half2* h = reinterpret_cast<const __half2*>(&v);
      m[0] = __hmax2(m[0], __hmax2(__habs2(h[0]), __habs2(h[1])));
      m[1] = __hmax2(m[1], __hmax2(__habs2(h[2]), __habs2(h[3])));
    }
  const __half2 both = __hmax2(m[0], m[1]);
  return min(exponent_of(__float_as_uint(fmaxf(__low2float(both), __high2float(both)))), 20);
}
// ... and for all of them, by one warp
template <int D, int R>
__device__ __forceinline__ int tile_exponent(const uint8_t* tile, int rows, int lane) {
  return __reduce_max_sync(0xffffffffu, lane_exponent<D, R>(tile, rows, lane));
}
// the power for a tile whose bound has the exponent e, given the one so far
__device__ __forceinline__ int next_power(int k, int e) {
  return e + k > kMostBits ? max(kAimBits - e, -100) : k;
}
constexpr int kFirstPower = 100;

// ---------------------------------------------------------------------------------------------
// Backward, sequences of one tile of 64 keys: a cached head of a sequence per CTA of four warps, products by mma.sync, all three
// gradients at once.  A warp has 16 queries for scores, weights, dS and dQ, then 16 keys for dV = P^T dO and dK = dS^T Q, whose
// operands come through shared memory; the heads of the group follow one another, 4 us each.  D = sum of P o dP, in fp32: every visible key is at
// hand.  Bound, like the forward, by the way there and back, which several CTAs to an SM hide.
template <int D>
struct ShortGradShape {
  static constexpr uint32_t kTileB = kShort * D * 2, kWeights = kShort * kShort * 2;
  static constexpr size_t kSmem = 4 * kTileB + 2 * kWeights + 64;  // keys, values, queries, gradients of outputs; weights, dS; largest |dS| of each warp
  static constexpr int kCtasPerSm = D == 64 ? 3 : 2;
};
// acc += A^T B over `rows` rows: 16 columns of A (64 wide) from `column` on, B of D columns
template <class T, int D>
__device__ __forceinline__ void short_product(float (&acc)[D / 8][4], uint32_t a, uint32_t b, int column, int rows, int lane) {
#pragma unroll
  for (int ks = 0; ks < kShort / 16; ++ks) {
    if (ks * 16 >= rows) break;
    uint32_t w[4];
    ldmatrix4_trans(a + short_at<kShort>(ks * 16 + (lane & 7) + ((lane >> 4) << 3), column / 8 + ((lane >> 3) & 1)), w);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      uint32_t vb[4];
      ldmatrix4_trans(b + short_at<D>(ks * 16 + (lane & 15), n * 2 + (lane >> 4)), vb);
      mma16816<T>(acc[2 * n], w, vb[0], vb[1]);
      mma16816<T>(acc[2 * n + 1], w, vb[2], vb[3]);
    }
  }
}
// 16 rows that a warp holds, times f, through its rows of `tile`, to memory in 16-byte pieces; rows before `end`
template <class T, int D>
__device__ __forceinline__ void short_store(const float (&acc)[D / 8][4], float f, uint8_t* tile, const View& v, int b, int h, int first, int end, int lane) {
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<uint32_t*>(tile + short_at<D>(first + (lane >> 2) + 8 * x, n) + (lane & 3) * 4) = pack2<T>(acc[n][2 * x] * f, acc[n][2 * x + 1] * f);
  __syncwarp();
  T* const out = reinterpret_cast<T*>(v.data) + b * v.batch + h * v.head;
#pragma unroll
  for (int i = 0; i < 16 * (D / 8) / 32; ++i) {
    const int r = first + (i * 32 + lane) / (D / 8), piece = (i * 32 + lane) % (D / 8);
    if (r < end) *reinterpret_cast<uint4*>(out + r * v.token + piece * 8) = *reinterpret_cast<const uint4*>(tile + short_at<D>(r, piece));
  }
}

template <class T, int D>
__global__ void __launch_bounds__(128, ShortGradShape<D>::kCtasPerSm) window_short_backward_kernel(const __grid_constant__ WinParams p) {
  using S = ShortGradShape<D>;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x % p.batch, kvh = blockIdx.x / p.batch, group = p.heads / p.kv_heads;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.kv_len) : p.kv_len;
  const int off = p.kv_len - p.q_len;
  const int rows_end = min(p.q_len, len - off);
  if (len == 0) return;
  uint8_t* const tQ = sm + 2 * S::kTileB;
  const uint32_t sK = smem_u32(sm), sV = sK + S::kTileB, sQ = sV + S::kTileB, sG = sQ + S::kTileB, sP = sG + S::kTileB, sD = sP + S::kWeights;
  uint8_t* const tP = sm + 4 * S::kTileB;
  float* const s_most = reinterpret_cast<float*>(tP + 2 * S::kWeights);  // [4]
  float dk[D / 8][4], dv[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;
  if (rows_end > 0) {
    short_load<T, D>(sK, p.k, b, kvh, 0, len, threadIdx.x);
    short_load<T, D>(sV, p.v, b, kvh, 0, len, threadIdx.x);
  }
  const float c = p.scale * kLog2e;
  const int first = off + warp * 16, keys = warp * 16 < rows_end ? min(first + 16, len) : 0;  // of the warp's rows: position, keys up to the last one's own
  int power = kFirstPower;  // of dS in the sums for dK
  for (int i = 0; i < group && rows_end > 0; ++i) {
    const int h = kvh * group + i;
    short_load<T, D>(sQ, p.q, b, h, 0, rows_end, threadIdx.x);
    short_load<T, D>(sG, p.dout, b, h, 0, rows_end, threadIdx.x);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    float sc[8][4], dp[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][e] = dp[n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t qa[4], ga[4];
      ldmatrix4(sQ + short_at<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)), qa);
      ldmatrix4(sG + short_at<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)), ga);
#pragma unroll
      for (int n = 0; n < 8; n += 2) {
        if (n * 8 >= keys) continue;
        uint32_t kb[4];
        ldmatrix4(sK + short_at<D>(n * 8 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), kb);
        mma16816<T>(sc[n], qa, kb[0], kb[1]);
        mma16816<T>(sc[n + 1], qa, kb[2], kb[3]);
        ldmatrix4(sV + short_at<D>(n * 8 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), kb);
        mma16816<T>(dp[n], ga, kb[0], kb[1]);
        mma16816<T>(dp[n + 1], ga, kb[2], kb[3]);
      }
    }
    float most = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = warp * 16 + (lane >> 2) + 8 * x, pos = off + row, lo = p.window > 0 ? pos - p.window + 1 : 0;
      const bool there = row < rows_end, single = pos == 0 || (p.window == 1 && p.sinks == 0);  // (one visible key: no gradient through its weight)
      const float lse2 = there ? p.lse[((long long)b * p.heads + h) * p.q_len + row] * kLog2e : 0.f;
      float own = 0.f;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 2 * x; e < 2 * x + 2; ++e) {
          const int j = n * 8 + (lane & 3) * 2 + (e & 1);
          const bool shown = there && j <= pos && (j >= lo || j < p.sinks);
          sc[n][e] = shown ? ex2(fmaf(sc[n][e], c, -lse2)) : 0.f;
          if (shown) own = fmaf(sc[n][e], dp[n][e], own);
        }
      own += __shfl_xor_sync(0xffffffffu, own, 1);
      own += __shfl_xor_sync(0xffffffffu, own, 2);
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 2 * x; e < 2 * x + 2; ++e) {
          dp[n][e] = single || sc[n][e] == 0.f ? 0.f : sc[n][e] * (dp[n][e] - own);
          most = fmaxf(most, fabsf(dp[n][e]));
        }
    }
    // powers of two of dS, as its largest value asks: this head's for dQ, the smallest so far for dK
    int k_dq = 0, k_dk = 0;
    if (kScaled) {
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));  // (not negative: as integers)
      if (lane == 0) s_most[warp] = most;
      __syncthreads();
      most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
      k_dq = max(min(13 + 127 - (int)(__float_as_uint(most) >> 23), kFirstPower), -kFirstPower);
      k_dk = min(power, k_dq);
      if (k_dk != power) {
        const float f = pow2(max(k_dk - power, -126));
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) dk[n][e] *= f;
        power = k_dk;
      }
    }
    const float f_dq = kScaled ? pow2(k_dq) : 1.f, f_dk = kScaled ? pow2(k_dk) : 1.f, f_p = pow2(kWeightBits<T>);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t at = short_at<kShort>(warp * 16 + (lane >> 2) + 8 * x, n) + (lane & 3) * 4;
        *reinterpret_cast<uint32_t*>(tP + at) = pack2<T>(sc[n][2 * x] * f_p, sc[n][2 * x + 1] * f_p);
        *reinterpret_cast<uint32_t*>(tP + S::kWeights + at) = pack2<T>(dp[n][2 * x] * f_dk, dp[n][2 * x + 1] * f_dk);
      }
    uint32_t w[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[ks][e] = pack2<T>(dp[2 * ks + (e >> 1)][2 * (e & 1)] * f_dq, dp[2 * ks + (e >> 1)][2 * (e & 1) + 1] * f_dq);
    float dq[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) dq[n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks * 16 >= keys) continue;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t kb[4];
        ldmatrix4_trans(sK + short_at<D>(ks * 16 + (lane & 15), n * 2 + (lane >> 4)), kb);
        mma16816<T>(dq[2 * n], w[ks], kb[0], kb[1]);
        mma16816<T>(dq[2 * n + 1], w[ks], kb[2], kb[3]);
      }
    }
    __syncthreads();
    if (warp * 16 < len) {
      short_product<T, D>(dv, sP, sG, warp * 16, rows_end, lane);
      short_product<T, D>(dk, sD, sQ, warp * 16, rows_end, lane);
    }
    __syncthreads();  // everyone is done with the head's tiles
    if (keys > 0) short_store<T, D>(dq, p.scale * (kScaled ? pow2(-k_dq) : 1.f), tQ, p.dq, b, h, warp * 16, rows_end, lane);
    if (i + 1 < group) __syncthreads();
  }
  __syncthreads();
  if (warp * 16 < len) {
    short_store<T, D>(dk, p.scale * (kScaled ? pow2(-power) : 1.f), sm, p.dk, b, kvh, warp * 16, len, lane);
    short_store<T, D>(dv, pow2(-kWeightBits<T>), sm + S::kTileB, p.dv, b, kvh, warp * 16, len, lane);
  }
}

// Shared memory is handed out to the last kilobytes at D = 128 (a tile has to be fetched two before it is needed): dynamic
// shared memory starts on a 1024-byte boundary, which the tiles' swizzling needs.
// A place in a ring of N stages, and the parity of its barriers' phases
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1u;
    }
  }
};

// G groups of 128 threads, each with a tile of 64 rows of its own in hand.  A CTA of two groups has an SM to itself.  Heads of 64
// leave room for two CTAs of one group, which hide each other's beginnings and ends too, but each is slower by itself: they are
// taken where no CTA has more than its half SM's share of all tiles.  2 x 4099 with a window of 1024, 16
// heads: dQ 92 us with one group, 109 with two; dK and dV, where two sinks make one CTA the longest by far, 190 and 116;
// 4096 without a window, 4 heads: 57 + 74 against 39 + 46.
//
// A block of keys that many queries see (all heads of its group; all of a sequence where it holds a sink) is one long walk, and few
// blocks leave SMs idle.  It is then shared by the CTAs of a cluster, a part of the queries each, joined through their shared memory
// in a fixed order.  Blocks that only sinks make long get a launch of their own, beside that of the other blocks.  dK and dV of one
// sequence, 8 query heads on one of 64: 4096 tokens 305 -> 77 us, with a window of 512 and 4 sinks 444 -> 68; 8 on 2 heads, 32768 tokens,
// window 1024, 4 sinks 1817 -> 254 (heads of 128 1947 -> 300); 2 x 1000, 4 on 2 heads 26 -> 15.  So are dQ's tiles of queries where they
// are no more than the SMs: 4096 tokens, one head of 64 38 -> 18, of 128 50 -> 23; 2048, 4 heads 23 -> 18, 30 -> 23.
template <int D, int G>
struct BwdShape {
  static constexpr int kCtasPerSm = G == 1 ? 2 : 1;
  static constexpr int kThreads = 128 + 128 * G;
  static constexpr int kTmemCols = 256 * G;
};
// dQ, heads of 128: both groups share tiles of 128 keys, half of the columns each.  A product of 128 x 128 takes 67 clocks, two of
// 128 x 64 100 (both operands come from shared memory), and the products are what heads of 128 wait for.
template <int D, int G>
struct DqShape : BwdShape<D, G> {
  static constexpr int kKeyRows = D == 128 ? 128 : kSub;              // of a tile
  static constexpr int kStreams = D == 128 ? 1 : G, kHalves = G / kStreams;
  static constexpr int kKeys = D == 128 ? 3 : G == 2 ? 8 : 5, kValues = D == 128 ? 2 : G == 2 ? 6 : 4;  // stages: keys are needed for longer
  static constexpr uint32_t kFixed = 2 * kTileBytes<D, kTile>, kStage = kTileBytes<D, kKeyRows>;
  static constexpr uint32_t kTiles = kFixed + (kKeys + kValues) * kStage;
  static constexpr size_t kSmem = kTiles + 2048 + 512;
  static_assert((11 + 3 * kKeys + kValues) * 8 + 2 * kKeys * 4 + 8 + 16 <= 512, "barriers, powers and flags behind the sums");
};
template <int D, int G>
struct DkvShape : BwdShape<D, G> {
  static constexpr int kStages = D == 128 ? 5 : G == 2 ? 7 : 4;
  static constexpr uint32_t kFixed = 2 * kTileBytes<D, kTile>, kStage = 2 * kTileBytes<D, kSub>;
  static constexpr uint32_t kTiles = kFixed + kStages * kStage;
  static constexpr size_t kSmem = kTiles + kStages * kSub * 8 + 384;
};

// Split: a tile of queries is a cluster's, each of whose CTAs has a part of the keys.
template <class T, int D, int G, bool Split>
__global__ void __launch_bounds__(DqShape<D, G>::kThreads, DqShape<D, G>::kCtasPerSm)
window_dq_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                 const __grid_constant__ CUtensorMap mapG, const __grid_constant__ WinParams p) {
  using S = DqShape<D, G>;
  constexpr int NK = S::kKeys, NV = S::kValues, KR = S::kKeyRows, ST = S::kStreams, H = S::kHalves;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t base = smem_u32(sm);
  if (base & 1023u) {  // (never seen; tiles could not be fetched)
    if (threadIdx.x == 0) note_error(p.gerr, 1100);
    return;
  }
  const uint32_t sQ = base, sG = sQ + kTileBytes<D, kTile>, sK = base + S::kFixed, sV = sK + NK * S::kStage;
  float* const s_sum = reinterpret_cast<float*>(sm + S::kTiles);  // [2][128]
  float* const s_own = s_sum + 256;                                // [2][128]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(s_own + 256);
  const uint32_t bar0 = smem_u32(bars);
  // of each stream of tiles: scores and dP are there, they have been read; of each of its two buffers: dS is there
  const uint32_t q_full = bar0, dq_full = bar0 + 8, sd_full = bar0 + 16, sd_free = sd_full + 16, ds_full = sd_free + 16, kv_full = ds_full + 32,
                 k_free = kv_full + 8 * NK, v_free = k_free + 8 * NK, st_full = v_free + 8 * NV, d_full = st_full + 8 * NK;
  int* const s_power = reinterpret_cast<int*>(bars + 11 + 3 * NK + NV);  // [NK]
  int* const s_step = s_power + NK;                                       // [NK]: its change against the tile before
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_step + NK);
  volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  uint32_t* const s_most = s_tmem + 2;  // [4]: each warp's largest |D|, as bits
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  const int split = Split ? p.split : 0, parts = 1 << split, part = blockIdx.x & (parts - 1);
  int item = blockIdx.x >> split;
  const int b = item % p.batch;
  item /= p.batch;
  const int h = item % p.heads, block = p.blocks - 1 - item / p.heads;
  const int kvh = h / (p.heads / p.kv_heads);
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.kv_len) : p.kv_len;
  const int off = p.kv_len - p.q_len, r0 = block * kTile;
  const int rows_end = min(p.q_len, len - off);
  if (r0 >= rows_end) return;
  const KeyTiles kt = key_tiles<KR>(off + r0, off + min(r0 + kTile, rows_end) - 1, p.window, p.sinks);
  // D = dO . O has the output's rounding in it, which is large against dP where a row sees a few keys.  Rows that see only the
  // first tile's keys take the sum of P o dP over them instead; with a window of few keys all rows do, in a pass of its own over
  // the tiles ahead of the one that adds up dQ.
  const int seen = kt.sink_end + kt.end - kt.begin;
  const int ahead = !Split && p.window > 0 && p.window + p.sinks <= kSub ? seen : 0;
  // (where rows see only the first tile's keys, there are few tiles: the first part has them all)
  const bool shared = Split && (kt.sink_end > 0 ? 0 : kt.begin) * KR + KR <= off + r0;
  const int skipped = shared ? part_begin(seen, split, part) : part == 0 ? 0 : seen, tiles = ahead + (shared ? part_begin(seen, split, part + 1) : seen) - skipped;
  auto first_key = [&](int u) {
    const int t = (u < ahead ? u : u - ahead) + (Split ? skipped : 0);
    return (t < kt.sink_end ? t : kt.begin + (t - kt.sink_end)) * KR;
  };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(dq_full, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(sd_full + 8 * i, 1);
      mbar_init(sd_free + 8 * i, 128 * H);
    }
    for (int i = 0; i < 2 * ST; ++i) mbar_init(ds_full + 8 * i, 128 * H);
    for (int s = 0; s < NK; ++s) {
      mbar_init(kv_full + 8 * s, 1);
      mbar_init(k_free + 8 * s, 1);
      mbar_init(st_full + 8 * s, 1);
    }
    mbar_init(d_full, 4);
    // the products are done with it, and so is the search for its largest value
    for (int s = 0; s < NV; ++s) mbar_init(v_free + 8 * s, kScaled ? 2 : 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(s_tmem), S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // of each stream: scores, dP; then each stream's two buffers for dS; then dQ
  const uint32_t tmem = *s_tmem, tdS = tmem + 2 * KR * ST, tdQ = tmem + 3 * KR * ST;
  if (S::kCtasPerSm == 2 && warp < 4) fewer_registers<64>();

  if (warp == 0) {
    if (lane == 0 && (!Split || tiles > 0)) {
      mbar_expect_tx(q_full, S::kFixed);
      load_tile<D, kTile, kSub>(sQ, &mapQ, q_full, h, r0, b);
      load_tile<D, kTile, kSub>(sG, &mapG, q_full, h, r0, b);
      Ring<NK> kr;
      Ring<NV> vr;
      for (int u = 0; u < tiles; ++u, kr.next(), vr.next()) {
        if (u >= NK && !mbar_wait_bounded(k_free + 8 * kr.s, kr.ph ^ 1u, s_abort, p.gerr, 1121)) break;
        mbar_expect_tx(kv_full + 8 * kr.s, 2 * S::kStage);
        load_tile<D, KR, kSub>(sK + kr.s * S::kStage, &mapK, kv_full + 8 * kr.s, kvh, first_key(u), b);
        if (u >= NV && !mbar_wait_bounded(v_free + 8 * vr.s, vr.ph ^ 1u, s_abort, p.gerr, 1133)) break;
        load_tile<D, KR, kSub>(sV + vr.s * S::kStage, &mapV, kv_full + 8 * kr.s, kvh, first_key(u), b);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = idesc_for<T>(kTile, KR, false), idesc_q = idesc_for<T>(kTile, D, true);
    const uint32_t leader = elect_one() ? 1u : 0u;
    Ring<NK> kr, kd;  // of the next scores, of the next product with dS
    Ring<NV> vr;
    auto scores = [&](int u) {
      const uint32_t k = sK + kr.s * S::kStage, v = sV + vr.s * S::kStage, t = tmem + 2 * KR * (u % ST);
      if (!warp_wait(kv_full + 8 * kr.s, kr.ph, s_abort, p.gerr, 1122)) return false;
      if (first_key(u) + KR > len) clear_rows<D, KR>(sm + (k - base), len - first_key(u), lane);
      tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) mma_ss(leader, t, desc_k<kTile>(sQ, ks), desc_k<KR>(k, ks), idesc_s, ks != 0);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) mma_ss(leader, t + KR, desc_k<kTile>(sG, ks), desc_k<KR>(v, ks), idesc_s, ks != 0);
      // (whoever finds the scores finds their power too: awaited by each thread that scales, dQ of 2 x 4099 took 95 us, not 92)
      if (kScaled && !warp_wait(st_full + 8 * kr.s, kr.ph, s_abort, p.gerr, 1129)) return false;
      commit(leader, sd_full + 8 * (u % ST));
      commit(leader, v_free + 8 * vr.s);
      kr.next();
      vr.next();
      return true;
    };
    auto add = [&](int x) {  // dQ += dS K
      if (x >= ahead) {
#pragma unroll
        for (int ks = 0; ks < KR / 16; ++ks)
          mma_ts(leader, tdQ, tdS + KR / 2 * (x % (2 * ST)) + ks * 8, desc_rows<KR>(sK + kd.s * S::kStage, ks), idesc_q, x != ahead || ks != 0);
      }
      commit(leader, k_free + 8 * kd.s);
      kd.next();
    };
    bool ok = (!Split || tiles > 0) && warp_wait(q_full, 0, s_abort, p.gerr, 1123);
    for (int u = 0; u < ST && u < tiles && ok; ++u) ok = scores(u);
    for (int u = 0; u + ST < tiles && ok; ++u) {
      // The stream's threads have read tile u: they have written dS of their tile before.  That product goes ahead of the next scores, so that
      // whoever finds these knows its buffer free.
      if (!(ok = warp_wait(sd_free + 8 * (u % ST), (uint32_t)(u / ST) & 1u, s_abort, p.gerr, 1124))) break;
      tc_fence_after();
      if (u >= ST) add(u - ST);
      ok = scores(u + ST);
    }
    for (int x = max(tiles - 2 * ST, 0); x < tiles && ok; ++x) {
      if (!(ok = warp_wait(ds_full + 8 * (x % (2 * ST)), (uint32_t)(x / (2 * ST)) & 1u, s_abort, p.gerr, 1125))) break;
      tc_fence_after();
      add(x);
    }
    if (ok) commit(leader, dq_full);
  } else if (warp == 2) {
    if (kScaled && (!Split || tiles > 0) && warp_wait(q_full, 0, s_abort, p.gerr, 1126)) {
      const int eg = tile_exponent<D, kTile>(sm + (sG - base), min(kTile, rows_end - r0), lane) + (D == 64 ? 3 : 4);
      int k = kFirstPower;
      Ring<NK> kr;
      Ring<NV> vr;
      for (int u = 0; u < tiles; ++u, kr.next(), vr.next()) {
        if (!warp_wait(kv_full + 8 * kr.s, kr.ph, s_abort, p.gerr, 1127)) break;
        int e = eg + tile_exponent<D, KR>(sm + (sV - base) + vr.s * S::kStage, min(KR, len - first_key(u)), lane);
        if (u == 0 && ahead == 0) {  // (with two passes the first, over all keys, meets what D is made of)
          if (!warp_wait(d_full, 0, s_abort, p.gerr, 1134)) break;
          e = max(e, exponent_of(max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]))));
        }
        const int k_new = next_power(k, e);
        __syncwarp();
        if (lane == 0) {
          s_power[kr.s] = k_new;
          s_step[kr.s] = u == 0 ? 0 : k_new - k;
          mbar_arrive(st_full + 8 * kr.s);
          mbar_arrive(v_free + 8 * vr.s);
        }
        k = k_new;
      }
    }
  } else if (warp >= 4) {
    if (S::kCtasPerSm == 2) more_registers<192>();
    const int w = (warp - 4) >> 2, q = warp & 3, in_tile = q * 32 + lane;
    const int stream = w % ST, half = H == 2 ? w : 0;
    const int row = r0 + in_tile, pos = off + row;
    const bool there = row < rows_end;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const float c = p.scale * kLog2e;
    const long long stat = ((long long)b * p.heads + h) * p.q_len + row;
    const float lse2 = there ? p.lse[stat] * kLog2e : INFINITY;  // (weights of 0)
    // a query that sees one key has the weight 1 whatever its score: no gradient through it
    const bool single = pos == 0 || (p.window == 1 && p.sinks == 0);
    const bool few = ahead == 0 && !shared && first_key(0) + KR > off + r0, mine_few = first_key(0) + KR > pos;
    constexpr int kShare = D / G;  // a row's dot product and its result are shared by the groups
    float delta = 0.f;
    if (there && ahead == 0) {
      const T* g = reinterpret_cast<const T*>(p.dout.data) + b * p.dout.batch + row * p.dout.token + h * p.dout.head + w * kShare;
      const T* o = reinterpret_cast<const T*>(p.o.data) + b * p.o.batch + row * p.o.token + h * p.o.head + w * kShare;
#pragma unroll
      for (int i = 0; i < kShare; i += 8) {
        const uint4 x = *reinterpret_cast<const uint4*>(g + i), y = *reinterpret_cast<const uint4*>(o + i);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = unpack2<T>(xs[e]), z = unpack2<T>(ys[e]);
          delta = fmaf(a.x, z.x, fmaf(a.y, z.y, delta));
        }
      }
    }
    auto join = [&] {  // the groups' parts of it
      if (G == 2) {
        s_sum[w * 128 + in_tile] = delta;
        named_bar_sync(2, 256);
        delta = s_sum[in_tile] + s_sum[128 + in_tile];
      }
    };
    bool joined = ahead == 0;
    if (joined) join();
    if (kScaled && w == 0) {
      const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(delta)));
      if (lane == 0) {
        s_most[q] = most;
        mbar_arrive(d_full);
      }
    }
    bool ok = true;
    Ring<NK> kr;
    if (stream == 1) kr.next();
    for (int u = stream, n = 0; u < tiles; u += ST, ++n) {
      const int s = kr.s, j0 = first_key(u);
      if (!joined && u >= ahead) {
        join();
        joined = true;
      }
      const uint32_t t = tmem + 2 * KR * stream + 64 * half + lanes;
      float r = 1.f;
      int step = 0;
      ok = warp_wait(sd_full + 8 * stream, (uint32_t)n & 1u, s_abort, p.gerr, 1128);
      if (kScaled) {
        r = pow2(s_power[s]);
        step = s_step[s];
      }
      if (!ok) {
        if (H == 2 && few && u == 0) named_bar_sync(2, 256);  // (the other half may be waiting below)
        break;
      }
      tc_fence_after();
      uint32_t sc[2][32], dp[2][32];
      tmem_ld_32x32(t, sc[0]);
      tmem_ld_32x32(t + 32, sc[1]);
      tmem_ld_32x32(t + KR, dp[0]);
      tmem_ld_32x32(t + KR + 32, dp[1]);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(sd_free + 8 * stream);
      if (single) r = 0.f;
      const bool cut = j0 + KR - 1 > off + r0 || (p.window > 0 && j0 <= off + r0 + kTile - 1 - p.window && j0 + KR > p.sinks);
      if (cut) {
        const int c0 = j0 + 64 * half, lo = p.window > 0 ? pos - p.window + 1 - c0 : -1, hi = pos - c0, sinks = p.sinks - c0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t shown = bits_below(hi + 1 - 32 * i) & (~bits_below(lo - 32 * i) | bits_below(sinks - 32 * i));
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            sc[i][e] = shown >> e & 1 ? sc[i][e] : kMinusInf;
            dp[i][e] = shown >> e & 1 ? dp[i][e] : 0u;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = fma2(pair_of(sc[i][e], sc[i][e + 1]), make_float2(c, c), make_float2(-lse2, -lse2));
          const float2 y = make_float2(ex2(x.x), ex2(x.y));
          sc[i][e] = __float_as_uint(y.x);
          sc[i][e + 1] = __float_as_uint(y.y);
        }
      if (u < ahead || (few && u == 0)) {
        float2 own = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 32; e += 2) own = fma2(pair_of(sc[i][e], sc[i][e + 1]), pair_of(dp[i][e], dp[i][e + 1]), own);
        float sum = own.x + own.y;
        if (u < ahead) {
          delta += sum;
        } else {
          if (H == 2) {
            s_own[w * 128 + in_tile] = sum;
            named_bar_sync(2, 256);
            sum = s_own[in_tile] + s_own[128 + in_tile];
          }
          if (mine_few) delta = sum;
        }
      }
      if (kScaled && step != 0 && u > ahead) {  // what has been summed so far, the other group's last tile included, follows
        if (!(ok = warp_wait(k_free + 8 * ((u - 1) % NK), (uint32_t)((u - 1) / NK) & 1u, s_abort, p.gerr, 1131))) break;
        tc_fence_after();
        scale_row<D / H>(tdQ + lanes + half * (D / H), pow2(max(step, -126)));
      }
      if (u >= ahead) {
        const float shift = -delta * r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t o[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = mul2(pair_of(sc[i][e], sc[i][e + 1]), fma2(pair_of(dp[i][e], dp[i][e + 1]), make_float2(r, r), make_float2(shift, shift)));
            o[e / 2] = pack2<T>(x.x, x.y);
          }
          tmem_st_32x16(tdS + KR / 2 * (u % (2 * ST)) + 32 * half + lanes + 16 * i, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(ds_full + 8 * (u % (2 * ST)));
      for (int i = 0; i < ST; ++i) kr.next();
    }
    if (!joined) join();
    if (ok && (!Split || tiles > 0) && warp_wait(dq_full, 0, s_abort, p.gerr, 1132)) {
      tc_fence_after();
      if (there && w == 0 && part == 0) p.delta[stat] = delta;
      float f = p.scale;
      if (kScaled) f *= pow2(-s_power[(tiles - 1) % NK]);
      if constexpr (Split) {  // (the tiles' places are free: every product is done)
        keep_row<D, kShare>(tdQ + lanes + w * kShare, base, in_tile, w * kShare, f);
      } else {
        T* const out = reinterpret_cast<T*>(p.dq.data) + b * p.dq.batch + row * p.dq.token + h * p.dq.head + w * kShare;
        store_row<T, kShare>(tdQ + lanes + w * kShare, out, f, there);
      }
    }
  }

  if (*s_abort) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
  if constexpr (Split) {
    cluster_sync_all();
    join_rows<D, S::kThreads>(base, shared ? seen : 1, split, part, [&](int r, int c, float4 x) {
      const int row = r0 + r;
      if (row < rows_end)
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.dq.data) + b * p.dq.batch + row * p.dq.token + h * p.dq.head + c) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    });
    cluster_sync_all();  // nobody leaves while its shared memory is read
  }
}

// Split: a block of keys is a cluster's, each of whose CTAs has a part of the queries.
template <class T, int D, int G, bool Split>
__global__ void __launch_bounds__(DkvShape<D, G>::kThreads, DkvShape<D, G>::kCtasPerSm)
window_dkv_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                  const __grid_constant__ CUtensorMap mapG, const __grid_constant__ WinParams p) {
  using S = DkvShape<D, G>;
  constexpr int NS = S::kStages;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t base = smem_u32(sm);
  // Where two launches overlap, the second ends after the first, so that what follows finds both complete: its last CTA waits.  (It
  // starts once every CTA of the first has, and reads nothing that the first writes.)
  if (p.leads) griddep_launch_dependents();
  auto leave = [&] {
    if (p.after && threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) griddep_wait();
  };
  if (base & 1023u) {  // (never seen; tiles could not be fetched)
    if (threadIdx.x == 0) note_error(p.gerr, 1100);
    return leave();
  }
  const uint32_t sK = base, sV = sK + kTileBytes<D, kTile>, ring = base + S::kFixed;  // a stage: queries, gradients of outputs
  float* const s_lse = reinterpret_cast<float*>(sm + S::kTiles);  // [NS][64]: -lse in log2, plus the weights' power
  float* const s_delta = s_lse + NS * kSub;                       // [NS][64]: -delta
  uint64_t* const bars = reinterpret_cast<uint64_t*>(s_delta + NS * kSub);
  const uint32_t bar0 = smem_u32(bars);
  // of each group: scores are there, weights are there, dP is there, dS is there
  const uint32_t kv_full = bar0, all_done = bar0 + 8, s_full = bar0 + 16, p_full = s_full + 16, dp_full = p_full + 16, ds_full = dp_full + 16,
                 q_full = ds_full + 16, q_free = q_full + 8 * NS, st_full = q_free + 8 * NS;
  int* const s_power = reinterpret_cast<int*>(bars + 10 + 3 * NS);  // [NS]
  int* const s_step = s_power + NS;                                 // [NS]
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_step + NS);
  volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  const int split = Split ? p.split : 0, parts = 1 << split, part = blockIdx.x & (parts - 1);
  int item = blockIdx.x >> split;
  const int b = item % p.batch;
  item /= p.batch;
  const int kvh = item % p.kv_heads, j0 = (p.first_block + item / p.kv_heads) * kTile;
  const int group = p.heads / p.kv_heads;
  const int len = p.lengths ? min(max(__ldcg(p.lengths + b), 0), p.kv_len) : p.kv_len;
  const int off = p.kv_len - p.q_len;
  const int rows_end = min(p.q_len, len - off);
  if (j0 >= len) return leave();
  // tiles of queries that see a key of this one: rows from the first key's position on, as far as the window of the last key
  // reaches, or all where a key is a sink
  const int j1 = min(j0 + kTile, len) - 1;
  const int row_first = max(0, j0 - off);
  const int row_last = p.window > 0 && j0 >= p.sinks ? min(rows_end - 1, j1 + p.window - 1 - off) : rows_end - 1;
  const int t_first = row_first / kSub, per_head = row_last < row_first ? 0 : row_last / kSub - t_first + 1;
  const int all_tiles = per_head * group;
  const int begin = part_begin(all_tiles, split, part), tiles = part_begin(all_tiles, split, part + 1) - begin;
  // the tiles one after the other: those of a head, then the next head's
  struct Walk {
    int t, h, per_head;
    __device__ __forceinline__ void next() {
      if (++t == per_head) {
        t = 0;
        ++h;
      }
    }
  };
  // (the same for all threads, which the compiler has to know: products are issued from uniform registers)
  const int skipped = !Split || per_head == 0 ? 0 : __shfl_sync(0xffffffffu, begin / per_head, 0);
  const Walk start{begin - skipped * per_head, kvh * group + skipped, per_head};
  auto first_row = [&](const Walk& at) { return (t_first + at.t) * kSub; };

  if (all_tiles == 0) {  // no query sees these keys
    for (int i = threadIdx.x; part == 0 && i < (j1 - j0 + 1) * (D / 8); i += S::kThreads) {
      const int j = j0 + i / (D / 8), c = i % (D / 8) * 8;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.dk.data) + b * p.dk.batch + j * p.dk.token + kvh * p.dk.head + c) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.dv.data) + b * p.dv.batch + j * p.dv.token + kvh * p.dv.head + c) = make_uint4(0, 0, 0, 0);
    }
    return leave();
  }

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(all_done, 1);
    for (int w = 0; w < G; ++w) {
      mbar_init(s_full + 8 * w, 1);
      mbar_init(p_full + 8 * w, 128);
      mbar_init(dp_full + 8 * w, 1);
      mbar_init(ds_full + 8 * w, 128);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(q_full + 8 * s, 1);
      mbar_init(q_free + 8 * s, 1);
      mbar_init(st_full + 8 * s, kScaled ? 2 : 1);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(s_tmem), S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // of each group: 64 columns of scores, then weights, 64 of dP, then dS; then dV and dK
  const uint32_t tmem = *s_tmem, tdV = tmem + 128 * G, tdK = tdV + D;
  if (S::kCtasPerSm == 2 && warp < 4) fewer_registers<64>();

  if (warp == 0) {
    if (lane == 0 && (!Split || tiles > 0)) {
      mbar_expect_tx(kv_full, S::kFixed);
      load_tile<D, kTile, kSub>(sK, &mapK, kv_full, kvh, j0, b);
      load_tile<D, kTile, kSub>(sV, &mapV, kv_full, kvh, j0, b);
      Ring<NS> ring_at;
      Walk at = start;
      for (int u = 0; u < tiles; ++u, ring_at.next(), at.next()) {
        const int s = ring_at.s;
        if (u >= NS && !mbar_wait_bounded(q_free + 8 * s, ring_at.ph ^ 1u, s_abort, p.gerr, 1141)) break;
        mbar_expect_tx(q_full + 8 * s, S::kStage);
        load_tile<D, kSub, kSub>(ring + s * S::kStage, &mapQ, q_full + 8 * s, at.h, first_row(at), b);
        load_tile<D, kSub, kSub>(ring + s * S::kStage + kTileBytes<D, kSub>, &mapG, q_full + 8 * s, at.h, first_row(at), b);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = idesc_for<T>(kTile, kSub, false), idesc_g = idesc_for<T>(kTile, D, true);
    const uint32_t leader = elect_one() ? 1u : 0u;
    Ring<NS> rs, rp, rv, rk;  // of the next scores, dP, product for dV, product for dK
    Walk at = start;
    auto scores = [&](int u) {
      const uint32_t q = ring + rs.s * S::kStage;
      if (!warp_wait(q_full + 8 * rs.s, rs.ph, s_abort, p.gerr, 1142)) return false;
      if (first_row(at) + kSub > rows_end) {  // rows behind the sequence's end are summed over too
        clear_rows<D, kSub>(sm + (q - base), rows_end - first_row(at), lane);
        clear_rows<D, kSub>(sm + (q - base) + kTileBytes<D, kSub>, rows_end - first_row(at), lane);
      }
      tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) mma_ss(leader, tmem + 128 * (u % G), desc_k<kTile>(sK, ks), desc_k<kSub>(q, ks), idesc_s, ks != 0);
      commit(leader, s_full + 8 * (u % G));
      rs.next();
      at.next();
      return true;
    };
    auto dps = [&](int u) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        mma_ss(leader, tmem + 128 * (u % G) + 64, desc_k<kTile>(sV, ks), desc_k<kSub>(ring + rp.s * S::kStage + kTileBytes<D, kSub>, ks), idesc_s, ks != 0);
      commit(leader, dp_full + 8 * (u % G));
      rp.next();
    };
    bool ok = (!Split || tiles > 0) && warp_wait(kv_full, 0, s_abort, p.gerr, 1143);
    for (int u = 0; u < G && u < tiles && ok; ++u) {
      ok = scores(u);
      if (ok) dps(u);
    }
    // a tile's weights, then the dS of the tile before (of the other group, where there are two)
    for (int u = 0; u < tiles + G - 1 && ok; ++u) {
      if (u < tiles) {
        if (!warp_wait(p_full + 8 * (u % G), (uint32_t)(u / G) & 1u, s_abort, p.gerr, 1144)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < kSub / 16; ++ks)
          mma_ts(leader, tdV, tmem + 128 * (u % G) + ks * 8, desc_rows<kSub>(ring + rv.s * S::kStage + kTileBytes<D, kSub>, ks), idesc_g, u != 0 || ks != 0);
        rv.next();
        if (u + G < tiles && !scores(u + G)) break;
      }
      const int x = u - (G - 1);
      if (x < 0) continue;
      if (!warp_wait(ds_full + 8 * (x % G), (uint32_t)(x / G) & 1u, s_abort, p.gerr, 1145)) break;
      tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < kSub / 16; ++ks)
        mma_ts(leader, tdK, tmem + 128 * (x % G) + 64 + ks * 8, desc_rows<kSub>(ring + rk.s * S::kStage, ks), idesc_g, x != 0 || ks != 0);
      commit(leader, q_free + 8 * rk.s);
      rk.next();
      if (x + 1 == tiles) commit(leader, all_done);
      if (x + G < tiles) dps(x + G);
    }
  } else if (warp == 2) {
    // statistics of the queries, the next tile's on their way while the stage is awaited
    auto fetch = [&](int u, const Walk& at, float2 (&x)[2]) {
      const int row = first_row(at);
      const long long stat = ((long long)b * p.heads + at.h) * p.q_len + row;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = lane + 32 * i;
        const bool there = u < tiles && row + r < rows_end;
        x[i].x = there ? __ldcg(p.lse + stat + r) : INFINITY;  // (a weight of 0)
        x[i].y = there ? __ldcg(p.delta + stat + r) : 0.f;
      }
    };
    float2 x[2];
    Ring<NS> ring_at;
    Walk at = start;
    fetch(0, at, x);
    for (int u = 0; u < tiles; ++u, ring_at.next()) {
      const int s = ring_at.s;
      if (u >= NS && !warp_wait(q_free + 8 * s, ring_at.ph ^ 1u, s_abort, p.gerr, 1147)) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s_lse[s * kSub + lane + 32 * i] = fmaf(x[i].x, -kLog2e, (float)kWeightBits<T>);
        s_delta[s * kSub + lane + 32 * i] = -x[i].y;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(st_full + 8 * s);
      at.next();
      fetch(u + 1, at, x);
    }
  } else if (warp == 3) {
    // the power for dS, as this block's values and the queries' D ask; D of the next tile on its way while the stage is awaited
    Walk at = start;
    float d0, d1;
    auto fetch = [&] {  // of this lane's two queries (the last one's again where there are none)
      const float* const delta = p.delta + ((long long)b * p.heads + at.h) * p.q_len;
      const int row = first_row(at) + lane;
      d0 = __ldcg(delta + min(row, rows_end - 1));
      d1 = __ldcg(delta + min(row + 32, rows_end - 1));
    };
    if (kScaled && (!Split || tiles > 0)) {
      fetch();
      if (warp_wait(kv_full, 0, s_abort, p.gerr, 1146)) {
        const int ev = tile_exponent<D, kTile>(sm + (sV - base), min(kTile, len - j0), lane) + (D == 64 ? 3 : 4);
        int k = kFirstPower;
        Ring<NS> ring_at;
        for (int u = 0; u < tiles; ++u, ring_at.next()) {
          const int s = ring_at.s;
          if (!warp_wait(q_full + 8 * s, ring_at.ph, s_abort, p.gerr, 1148)) break;
          const int eg = lane_exponent<D, kSub>(sm + S::kFixed + s * S::kStage + kTileBytes<D, kSub>, min(kSub, rows_end - first_row(at)), lane);
          const int k_new = next_power(k, __reduce_max_sync(0xffffffffu, max(ev + eg, exponent_of(__float_as_uint(fmaxf(fabsf(d0), fabsf(d1)))))));
          if (lane == 0) {
            s_power[s] = k_new;
            s_step[s] = u == 0 ? 0 : k_new - k;
            mbar_arrive(st_full + 8 * s);
          }
          k = k_new;
          at.next();
          if (u + 1 < tiles) fetch();
        }
      }
    }
  } else {
    if (S::kCtasPerSm == 2) more_registers<192>();
    const int w = (warp - 4) >> 2, q = warp & 3, in_tile = q * 32 + lane;
    const int key = j0 + in_tile;
    const uint32_t lanes = (uint32_t)(q * 32) << 16, t = tmem + 128 * w + lanes;
    const float c = p.scale * kLog2e;
    const bool sink = key < p.sinks, no_ds = p.window == 1 && p.sinks == 0;
    bool ok = true;
    Ring<NS> ring_at;
    Walk at = start;
    if (w == 1) {
      ring_at.next();
      at.next();
    }
    for (int u = w, n = 0; u < tiles; u += G, ++n) {
      const int s = ring_at.s, first = off + first_row(at);  // position of the tile's first query
      const float4 *lse2 = reinterpret_cast<const float4*>(s_lse + s * kSub), *delta = reinterpret_cast<const float4*>(s_delta + s * kSub);
      const bool cut = j0 + kTile - 1 > first || (p.window > 0 && j0 <= first + kSub - 1 - p.window && j0 + kTile > p.sinks);
      // columns whose queries see this thread's key: from `from` on, and before `to` unless it is a sink
      const int from = key - first, to = p.window > 0 && !sink ? from + p.window : 0x7fffffff;
      if (!(ok = warp_wait(st_full + 8 * s, ring_at.ph, s_abort, p.gerr, 1149))) break;
      if (!(ok = warp_wait(s_full + 8 * w, (uint32_t)n & 1u, s_abort, p.gerr, 1150))) break;
      tc_fence_after();
      uint32_t wt[2][32];
      tmem_ld_32x32(t, wt[0]);
      tmem_ld_32x32(t + 32, wt[1]);
      tmem_ld_wait();
      if (cut) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t shown = ~bits_below(from - 32 * i) & bits_below(to - 32 * i);
#pragma unroll
          for (int e = 0; e < 32; ++e) wt[i][e] = shown >> e & 1 ? wt[i][e] : kMinusInf;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 l = lse2[8 * i + e / 4];
          const float2 x = fma2(pair_of(wt[i][e], wt[i][e + 1]), make_float2(c, c), make_float2(l.x, l.y));
          const float2 y = fma2(pair_of(wt[i][e + 2], wt[i][e + 3]), make_float2(c, c), make_float2(l.z, l.w));
          const float4 z = make_float4(ex2(x.x), ex2(x.y), ex2(y.x), ex2(y.y));
          wt[i][e] = __float_as_uint(z.x);
          wt[i][e + 1] = __float_as_uint(z.y);
          wt[i][e + 2] = __float_as_uint(z.z);
          wt[i][e + 3] = __float_as_uint(z.w);
          o[e / 2] = pack2<T>(z.x, z.y);
          o[e / 2 + 1] = pack2<T>(z.z, z.w);
        }
        tmem_st_32x16(t + 16 * i, o);  // over scores that have been read
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full + 8 * w);
      float r = no_ds ? 0.f : 1.f;
      if (!(ok = warp_wait(dp_full + 8 * w, (uint32_t)n & 1u, s_abort, p.gerr, 1151))) break;
      tc_fence_after();
      if (kScaled) {
        const int step = s_step[s];
        if (step != 0) {  // what has been summed so far, the other group's last tile included, follows
          if (!(ok = warp_wait(q_free + 8 * ((u - 1) % NS), (uint32_t)((u - 1) / NS) & 1u, s_abort, p.gerr, 1152))) break;
          tc_fence_after();
          scale_row<D>(tdK + lanes, pow2(max(step, -126)));
        }
        r *= pow2(s_power[s] - kWeightBits<T>);
      }
      uint32_t d[2][32];
      tmem_ld_32x32(t + 64, d[0]);
      tmem_ld_32x32(t + 96, d[1]);
      tmem_ld_wait();
      if (cut) {
        // hidden values may be of rows that are not there; the query at position 0 sees one key: no gradient through it
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int alone = -first - 32 * i;
          const uint32_t shown = ~bits_below(from - 32 * i) & bits_below(to - 32 * i) & ~(bits_below(alone + 1) & ~bits_below(alone));
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            d[i][e] = shown >> e & 1 ? d[i][e] : 0u;
            wt[i][e] = shown >> e & 1 ? wt[i][e] : 0u;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 l = delta[8 * i + e / 4];
          const float2 x = mul2(mul2(pair_of(wt[i][e], wt[i][e + 1]), make_float2(r, r)), add2(pair_of(d[i][e], d[i][e + 1]), make_float2(l.x, l.y)));
          const float2 y = mul2(mul2(pair_of(wt[i][e + 2], wt[i][e + 3]), make_float2(r, r)), add2(pair_of(d[i][e + 2], d[i][e + 3]), make_float2(l.z, l.w)));
          o[e / 2] = pack2<T>(x.x, x.y);
          o[e / 2 + 1] = pack2<T>(y.x, y.y);
        }
        tmem_st_32x16(t + 64 + 16 * i, o);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(ds_full + 8 * w);
      for (int i = 0; i < G; ++i) {
        ring_at.next();
        at.next();
      }
    }
    if (ok && (!Split || tiles > 0) && warp_wait(all_done, 0, s_abort, p.gerr, 1153)) {
      tc_fence_after();
      float f = p.scale;
      if (kScaled) f *= pow2(-s_power[(tiles - 1) % NS]);
      constexpr int kShare = D / G;
      if constexpr (!Split) {
        T* const dk = reinterpret_cast<T*>(p.dk.data) + b * p.dk.batch + key * p.dk.token + kvh * p.dk.head + w * kShare;
        T* const dv = reinterpret_cast<T*>(p.dv.data) + b * p.dv.batch + key * p.dv.token + kvh * p.dv.head + w * kShare;
        store_row<T, kShare>(tdV + lanes + w * kShare, dv, pow2(-kWeightBits<T>), key < len);
        store_row<T, kShare>(tdK + lanes + w * kShare, dk, f, key < len);
      } else {  // (the tiles' places are free: every product is done)
        keep_row<2 * D, kShare>(tdV + lanes + w * kShare, base, in_tile, w * kShare, pow2(-kWeightBits<T>));
        keep_row<2 * D, kShare>(tdK + lanes + w * kShare, base, in_tile, D + w * kShare, f);
      }
    }
  }

  if (*s_abort) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
  if constexpr (Split) {
    cluster_sync_all();
    join_rows<2 * D, S::kThreads>(base, all_tiles, split, part, [&](int r, int c, float4 x) {  // columns of dV, then of dK
      const int j = j0 + r;
      if (j >= len) return;
      T* const to = c < D ? reinterpret_cast<T*>(p.dv.data) + b * p.dv.batch + j * p.dv.token + kvh * p.dv.head + c
                          : reinterpret_cast<T*>(p.dk.data) + b * p.dk.batch + j * p.dk.token + kvh * p.dk.head + c - D;
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    });
    cluster_sync_all();  // nobody leaves while its shared memory is read
  }
  leave();
}

// (a stride of 0 over a dimension above 1 is refused: TMA has none)
bool tensor_ok(const aig_seq_heads* t, int batch, int tokens, int heads) {
  return t && t->data && (t->batch_stride > 0 || batch == 1) && (t->token_stride > 0 || tokens == 1) && (t->head_stride > 0 || heads == 1) && aligned_to(t->data, 16) && t->batch_stride >= 0 && t->token_stride >= 0 && t->head_stride >= 0 && t->batch_stride % 8 == 0 &&
         t->token_stride % 8 == 0 && t->head_stride % 8 == 0;
}
View view_of(const aig_seq_heads* t) { return View{(uint8_t*)t->data, t->batch_stride, t->token_stride, t->head_stride}; }

int check_desc(aig_ctx* ctx, const aig_window_desc* d, const char* who) {
  AIG_REQUIRE(ctx, d && dtype_known(d->dtype), "%s: null description or unknown element type", who);
  AIG_REQUIRE(ctx, d->batch >= 0 && d->q_len >= 0 && d->kv_len >= d->q_len && d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0 && d->sinks >= 0,
              "%s: bad extents (q_len at most kv_len, heads a multiple of kv_heads)", who);
  AIG_REQUIRE(ctx, d->scale > 0.f && d->scale - d->scale == 0.f, "%s: the scale has to be positive and finite", who);
  if (d->head_dim != 64 && d->head_dim != 128)
    return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "%s: head dimension must be 64 or 128 (got %d)", who, d->head_dim);
  if (d->kv_len > 1 << 30) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "%s: more than 2^30 keys", who);
  return AIG_OK;
}
WinParams params_of(const aig_window_desc* d) {
  WinParams p{};
  p.batch = d->batch;
  p.q_len = d->q_len;
  p.kv_len = d->kv_len;
  p.heads = d->heads;
  p.kv_heads = d->kv_heads;
  p.window = d->window > 0 && d->window < d->kv_len ? d->window : 0;  // (one that hides nothing is none)
  p.sinks = d->sinks < d->kv_len ? d->sinks : d->kv_len;
  p.scale = d->scale;
  return p;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeTiledFn>(f) : nullptr;
  }();
  return fn;
}

// A tensor [batch][tokens][heads][D] in boxes of B tokens x 64 elements of one head; tokens behind the last read as zeros.
template <class T, int D, int B>
int encode(aig_ctx* ctx, CUtensorMap* m, const View& v, int batch, int tokens, int heads) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return aig_fail(ctx, AIG_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
  // (the stride of a dimension of one has no meaning, but has to be a possible one)
  const cuuint64_t strides[3] = {(cuuint64_t)(heads > 1 ? v.head : D) * 2, (cuuint64_t)(tokens > 1 ? v.token : D) * 2, (cuuint64_t)(batch > 1 ? v.batch : D) * 2};
  const cuuint32_t box[4] = {64, 1, B, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, v.data, dims, strides,
                         box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return aig_fail(ctx, AIG_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)r);
  return AIG_OK;
}

cudaLaunchAttribute cluster_attribute(int ctas) {
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeClusterDimension;
  a.val.clusterDim.x = ctas;
  a.val.clusterDim.y = a.val.clusterDim.z = 1;
  return a;
}
// CTAs of a cluster that share a long walk over tiles: `blocks` of them, the longest of `most` tiles, `all` together, one CTA to an SM.
// A card of 148 SMs holds 74 clusters of two, 33 of four, 15 of eight; a CTA's beginning and end cost as much as `alone` tiles, with the
// join as `joined`.
int cluster_size(double sms, double blocks, double most, double all, double alone, double joined) {
  int size = 1;
  double least = 1e300;
  for (int n = 1; n <= 8; n *= 2) {
    const double waves = std::ceil(blocks / (sms * (n == 1 ? 1. : n == 2 ? 0.5 : n == 4 ? 0.223 : 0.102)));
    const double t = std::max(most, all / blocks * waves) / n + (n == 1 ? alone : joined) * waves;
    if (t < least) least = t, size = n;
  }
  return size;
}

template <class T, int D, int NT, bool Split>
int launch_forward(aig_ctx* ctx, WinParams& p, int parts, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv) {
  using S = FwdShape<D, NT, Split>;
  static_assert(!Split || kTile * (D + 2) * 4 <= S::kSmem - 256, "a part's sums take the tiles' place");
  p.blocks = ceil_div(p.q_len, kTile * NT);
  p.split = parts == 8 ? 3 : parts >> 1;
  const long long grid = (long long)p.blocks * p.heads * p.batch * parts;
  if (grid > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "window attention: too many rows for one call");
  AIG_CUDA_OK(ctx, cudaFuncSetAttribute(window_forward_kernel<T, D, NT, Split>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  if (Split) attr[cfg.numAttrs++] = cluster_attribute(parts);
  AIG_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, window_forward_kernel<T, D, NT, Split>, mq, mk, mv, (const WinParams&)p));
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
}

template <class T, int D, int Tiles>
int launch_short(aig_ctx* ctx, WinParams& p) {
  using S = ShortShape<D, Tiles>;
  p.blocks = ceil_div(p.q_len, kShort);
  const long long grid = (long long)p.blocks * p.heads * p.batch;
  if (grid > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "window attention: too many rows for one call");
  if (S::kSmem > (48u << 10)) AIG_CUDA_OK(ctx, cudaFuncSetAttribute(window_short_kernel<T, D, Tiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  window_short_kernel<T, D, Tiles><<<(unsigned)grid, 128, S::kSmem, ctx->stream>>>(p);
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
}

template <class T, int D>
int forward(aig_ctx* ctx, WinParams& p) {
  p.gerr = ctx->d_err;
  // 128 keys of 64 or 64 of 128: at twice that the two kernels are level (1024 heads: 64 x 64 x 64 8.7 us against 31.5, 128 x 128 x 64
  // 22 against 34, 256 x 256 x 64 in 512 heads 31 against 27; 64 x 64 x 128 17 against 36, 128 x 128 x 128 50 against 46)
  if (p.kv_len <= kShort) return launch_short<T, D, 1>(ctx, p);
  if constexpr (D == 64) {
    if (p.kv_len <= 2 * kShort) return launch_short<T, D, 2>(ctx, p);
  }
  CUtensorMap mq, mk, mv;
  int rc = encode<T, D, kTile>(ctx, &mq, p.q, p.batch, p.q_len, p.heads);
  if (rc == AIG_OK) rc = encode<T, D, kTile>(ctx, &mk, p.k, p.batch, p.kv_len, p.kv_heads);
  if (rc == AIG_OK) rc = encode<T, D, kTile>(ctx, &mv, p.v, p.batch, p.kv_len, p.kv_heads);
  if (rc != AIG_OK) return rc;
  // Where every tile of queries finds an SM of its own, or more, clusters share tiles that see many keys: 64 rows over 8192 keys, 8 heads
  // of 128 on 2, 101 -> 21 us; 4096 rows of one head of 64 44 -> 16; 512 rows over 8192, 8 heads of 64 84 -> 27.
  const double n = (double)ceil_div(p.q_len, kTile) * p.heads * p.batch, reach = p.window > 0 ? std::min(p.window + p.sinks + 2. * kTile, (double)p.kv_len) : p.kv_len;
  if (n <= ctx->sm_count) {
    const int parts = cluster_size(ctx->sm_count, n, reach / kTile, std::min(reach, p.kv_len - 0.5 * p.q_len) / kTile * n, 6, 9);
    return parts == 1 ? launch_forward<T, D, 1, false>(ctx, p, 1, mq, mk, mv) : launch_forward<T, D, 1, true>(ctx, p, parts, mq, mk, mv);
  }
  // Heads of 64 leave room for two CTAs with a tile of queries each on an SM, which hide each other's beginnings and ends (2 x 4099,
  // 16 heads: 69 us; one CTA with two tiles 77); heads of 128 for one, whose two tiles share the keys they fetch (4096 without a window, 4
  // heads, a tile for each SM: 59 us against 54; 8 heads with a window of 256, twice as many: 14 against 20).
  if (D == 64 || p.q_len <= kTile) return launch_forward<T, D, 1, false>(ctx, p, 1, mq, mk, mv);
  if constexpr (D == 128) return launch_forward<T, D, 2, false>(ctx, p, 1, mq, mk, mv);
}
template <class T, int D, int G, bool Split>
int launch_dq(aig_ctx* ctx, WinParams p, int parts, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mg) {
  using S = DqShape<D, G>;
  static_assert(kTile * D * 4 <= S::kTiles, "a part's sums take the tiles' place");
  p.split = parts == 8 ? 3 : parts >> 1;
  AIG_CUDA_OK(ctx, cudaFuncSetAttribute(window_dq_kernel<T, D, G, Split>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.blocks * p.heads * p.batch * parts);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  if (Split) attr[cfg.numAttrs++] = cluster_attribute(parts);
  AIG_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, window_dq_kernel<T, D, G, Split>, mq, mk, mv, mg, (const WinParams&)p));
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
}
// dK and dV of `blocks` blocks of 128 keys from the first on, each in `parts` CTAs of a cluster; `leads`, `after`: beside the launch behind it,
// before it
template <class T, int D, int G, bool Split>
int launch_dkv(aig_ctx* ctx, WinParams p, int first, int blocks, int parts, bool leads, bool after, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
               const CUtensorMap& mg) {
  using S = DkvShape<D, G>;
  static_assert(kTile * 2 * D * 4 <= S::kTiles, "a part's sums take the tiles' place");
  p.first_block = first;
  p.leads = leads;
  p.after = after;
  p.split = parts == 8 ? 3 : parts >> 1;
  const long long grid = (long long)blocks * p.kv_heads * p.batch * parts;
  if (grid > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "window attention backward: too many rows for one call");
  AIG_CUDA_OK(ctx, cudaFuncSetAttribute(window_dkv_kernel<T, D, G, Split>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (Split) attr[cfg.numAttrs++] = cluster_attribute(parts);
  if (after) attr[cfg.numAttrs++] = pdl_attribute(ctx);
  AIG_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, window_dkv_kernel<T, D, G, Split>, mq, mk, mv, mg, (const WinParams&)p));
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
}

template <class T, int D>
int launch_short_backward(aig_ctx* ctx, const WinParams& p) {
  using S = ShortGradShape<D>;
  const long long grid = (long long)p.kv_heads * p.batch;
  if (grid > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "window attention backward: too many rows for one call");
  AIG_CUDA_OK(ctx, cudaFuncSetAttribute(window_short_backward_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  window_short_backward_kernel<T, D><<<(unsigned)grid, 128, S::kSmem, ctx->stream>>>(p);
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
}

template <class T, int D>
int backward(aig_ctx* ctx, WinParams& p) {
  p.gerr = ctx->d_err;
  // Sequences of one tile, unless a few CTAs would take the heads of large groups one after the other (1024 heads of 64 x 64 x 64 23 us, the
  // two kernels 47; of 64 x 64 x 128 45 and 115; 64 x 64 x 64, 16 heads on 2: of 128 sequences 46 and 61, of one 37 and 17).
  if (p.kv_len <= kShort && (p.heads <= 2 * p.kv_heads || (long long)p.kv_heads * p.batch >= ctx->sm_count)) return launch_short_backward<T, D>(ctx, p);
  CUtensorMap mq{}, mk, mv, mg{};
  int rc = encode<T, D, kSub>(ctx, &mk, p.k, p.batch, p.kv_len, p.kv_heads);
  if (rc == AIG_OK) rc = encode<T, D, kSub>(ctx, &mv, p.v, p.batch, p.kv_len, p.kv_heads);
  if (rc == AIG_OK) rc = encode<T, D, kSub>(ctx, &mq, p.q, p.batch, p.q_len, p.heads);
  if (rc == AIG_OK) rc = encode<T, D, kSub>(ctx, &mg, p.dout, p.batch, p.q_len, p.heads);
  if (rc != AIG_OK) return rc;
  p.blocks = ceil_div(p.q_len, kTile);
  const int blocks_kv = ceil_div(p.kv_len, kTile);
  const long long grid = (long long)p.blocks * p.heads * p.batch, grid_kv = (long long)blocks_kv * p.kv_heads * p.batch;
  if (grid > 0x7fffffffll || grid_kv > 0x7fffffffll) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "window attention backward: too many rows for one call");
  // tiles of 64 that pass by: of all CTAs together, of the longest
  const double sms = ctx->sm_count, reach = p.window > 0 ? (double)p.window + kTile : p.kv_len;
  const double all = std::min(reach, p.kv_len - 0.5 * p.q_len) * p.blocks * p.batch * p.heads / kSub;
  const double most_dq = p.window > 0 ? std::min(reach + p.sinks, (double)p.kv_len) : p.kv_len;
  const bool two = D == 64 && most_dq / kSub * 2 * sms <= all, again = p.window > 0 && p.window + p.sinks <= kSub;  // (again: two passes over the keys, few)
  constexpr int kr = DqShape<D, 2>::kKeyRows;
  const int parts = two || again || grid > ctx->sm_count ? 1 : cluster_size(sms, (double)grid, most_dq / kr, all * kSub / kr, 512. / kr, 900. / kr);
  if (parts > 1) rc = launch_dq<T, D, 2, true>(ctx, p, parts, mq, mk, mv, mg);
  else if (D == 64 && two) rc = launch_dq<T, D, D == 64 ? 1 : 2, false>(ctx, p, 1, mq, mk, mv, mg);
  else rc = launch_dq<T, D, 2, false>(ctx, p, 1, mq, mk, mv, mg);
  if (rc != AIG_OK) return rc;
  const double group = (double)(p.heads / p.kv_heads) / kSub, heads = (double)p.kv_heads * p.batch;  // tiles per query that sees a block
  auto keys = [&](int first, int blocks, bool leads, bool after, double most, double all) {  // most: tiles of the longest block
    if (blocks == 0) return (int)AIG_OK;
    if constexpr (D == 64) {
      if (most * 2 * sms <= all) return launch_dkv<T, D, 1, false>(ctx, p, first, blocks, 1, leads, after, mq, mk, mv, mg);
    }
    const int parts = cluster_size(sms, blocks * heads, most, all, 3, 7);
    return parts == 1 ? launch_dkv<T, D, 2, false>(ctx, p, first, blocks, 1, leads, after, mq, mk, mv, mg)
                      : launch_dkv<T, D, 2, true>(ctx, p, first, blocks, parts, leads, after, mq, mk, mv, mg);
  };
  // one launch where the longest block holds nothing up, else two
  const int sinks = p.window > 0 && reach < p.q_len ? std::min((int)(((long long)p.sinks + kTile - 1) / kTile), blocks_kv) : 0;  // blocks that every query sees
  const double most = std::min(reach, (double)p.q_len) * group, of_sinks = p.q_len * group * sinks * heads;
  if (sinks == 0 || p.q_len * group * sms <= 1.25 * (all + of_sinks)) return keys(0, blocks_kv, false, false, sinks ? p.q_len * group : most, all + of_sinks);
  rc = keys(0, sinks, sinks < blocks_kv, false, p.q_len * group, of_sinks);
  return rc != AIG_OK ? rc : keys(sinks, blocks_kv - sinks, false, true, most, all);
}

}  // namespace

extern "C" {

int aig_window_attention_forward(aig_ctx* ctx, const aig_window_desc* d, const aig_seq_heads* q, const aig_seq_heads* k, const aig_seq_heads* v,
                                 const aig_seq_heads* out, float* lse, const int32_t* lengths) {
  if (!ctx) return AIG_ERR_INVALID;
  DeviceGuard g(ctx->device);
  const int rc = check_desc(ctx, d, "window attention");
  if (rc != AIG_OK) return rc;
  if (d->batch == 0 || d->q_len == 0) return AIG_OK;
  const int b = d->batch, tq = d->q_len, tk = d->kv_len, h = d->heads, hk = d->kv_heads;
  AIG_REQUIRE(ctx, tensor_ok(q, b, tq, h) && tensor_ok(k, b, tk, hk) && tensor_ok(v, b, tk, hk) && tensor_ok(out, b, tq, h) && lse && aligned_to(lse, 4) &&
                       aligned_to(lengths, 4),
              "window attention: null tensor, data off a 16-byte boundary, or strides that are not positive multiples of 8");
  WinParams p = params_of(d);
  p.q = view_of(q);
  p.k = view_of(k);
  p.v = view_of(v);
  p.o = view_of(out);
  p.lse = lse;
  p.lengths = lengths;
  if (d->dtype == AIG_F16) return d->head_dim == 64 ? forward<__half, 64>(ctx, p) : forward<__half, 128>(ctx, p);
  return d->head_dim == 64 ? forward<__nv_bfloat16, 64>(ctx, p) : forward<__nv_bfloat16, 128>(ctx, p);
}

int aig_window_attention_backward(aig_ctx* ctx, const aig_window_desc* d, const aig_seq_heads* q, const aig_seq_heads* k, const aig_seq_heads* v,
                                  const aig_seq_heads* out, const float* lse, const aig_seq_heads* dout, const aig_seq_heads* dq,
                                  const aig_seq_heads* dk, const aig_seq_heads* dv, float* delta, const int32_t* lengths) {
  if (!ctx) return AIG_ERR_INVALID;
  DeviceGuard g(ctx->device);
  const int rc = check_desc(ctx, d, "window attention backward");
  if (rc != AIG_OK) return rc;
  if (d->batch == 0 || d->kv_len == 0) return AIG_OK;
  const int b = d->batch, tq = d->q_len, tk = d->kv_len, h = d->heads, hk = d->kv_heads;
  AIG_REQUIRE(ctx, tq > 0, "window attention backward: no queries");
  AIG_REQUIRE(ctx, tensor_ok(q, b, tq, h) && tensor_ok(k, b, tk, hk) && tensor_ok(v, b, tk, hk) && tensor_ok(out, b, tq, h) && tensor_ok(dout, b, tq, h) &&
                       tensor_ok(dq, b, tq, h) && tensor_ok(dk, b, tk, hk) && tensor_ok(dv, b, tk, hk) && lse && delta && aligned_to(lse, 4) && aligned_to(delta, 4) &&
                       aligned_to(lengths, 4),
              "window attention backward: null tensor, data off a 16-byte boundary, or strides that are not positive multiples of 8");
  WinParams p = params_of(d);
  p.q = view_of(q);
  p.k = view_of(k);
  p.v = view_of(v);
  p.o = view_of(out);
  p.dout = view_of(dout);
  p.dq = view_of(dq);
  p.dk = view_of(dk);
  p.dv = view_of(dv);
  p.lse = const_cast<float*>(lse);
  p.delta = delta;
  p.lengths = lengths;
  if (d->dtype == AIG_F16) return d->head_dim == 64 ? backward<__half, 64>(ctx, p) : backward<__half, 128>(ctx, p);
  return d->head_dim == 64 ? backward<__nv_bfloat16, 64>(ctx, p) : backward<__nv_bfloat16, 128>(ctx, p);
}

}  // extern "C"

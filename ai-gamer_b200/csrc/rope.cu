// rope.cu -- rotary positions of queries and keys, alone or on the way into a paged key/value cache.
//
// A pair (a, b) of a head at position p becomes m * (a cos - b sin, b cos + a sin) with the angle p * f[j]; the transpose
// has the sine's sign turned.  A frequency is kept as a 64-bit fraction of a turn: p * f modulo 2^64 is the angle modulo a
// turn, exact but for f's own last bit (position 2^31: 2^-33 of a turn), where a product in fp32 loses the angle from a few
// thousand positions on and one in fp64 costs the SM's few fp64 units.  Its top 32 bits, as a signed fraction, go to the
// special-function unit's sine and cosine, whose error within half a turn either way (2^-21) lies below the fp16 results' 2^-12.
//
// Bound by memory: every value is read once and written once.  A thread turns the same pairs of several heads, so that
// sines are computed once for them; a pair's halves arrive as the widest vectors that the layout allows.
#include <cmath>
#include <new>
#include <vector>

#include "long_context.h"

struct aig_rope_plan {
  aig_ctx* ctx = nullptr;
  aig_rope_desc desc{};
  uint64_t* turns = nullptr;  // [rot_dim / 2] fractions of a turn per position, in 2^-64
};

namespace {

constexpr int kThreads = 128;

struct Side {
  const uint8_t* in;
  uint8_t* out;
  long long in_token, in_head, out_token, out_head;  // strides in elements
};

struct RopeParams {
  Side part[3];            // queries, keys, values
  int end[3];              // heads up to and with each part, counted over the parts
  int turned_heads;        // heads below it are turned, the others copied
  int rot_items, half;     // an item of a head: rot_items that turn V pairs, then those that copy 2 V values; half = rot_dim / 2
  Divisor groups;          // items of a head
  Divisor chunks;          // a token's heads in chunks of HP that one thread takes
  uint32_t items;
  const int32_t* positions;
  const uint64_t* turns;
  float magnitude, sign;
  // keys and values into pages (page.by > 0)
  const int32_t *seqs, *table;
  int batch, table_width, num_pages;
  Divisor page;
  long long page_stride, place_stride;
  int* gerr;
};

template <int V>
struct Vec;
template <>
struct Vec<1> { using type = uint16_t; };
template <>
struct Vec<2> { using type = uint32_t; };
template <>
struct Vec<4> { using type = uint2; };
template <>
struct Vec<8> { using type = uint4; };

template <class T, int V>
struct Row {
  T v[V];
  __device__ __forceinline__ void load(const T* p) { *reinterpret_cast<typename Vec<V>::type*>(v) = *reinterpret_cast<const typename Vec<V>::type*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename Vec<V>::type*>(p) = *reinterpret_cast<const typename Vec<V>::type*>(v); }
};

// One item: V pairs (or 2 V values to copy) of HP heads of a token.  All of them are read before the first is written: the
// reads of several heads are under way together (an output may be its input, so the compiler cannot move reads ahead itself).
template <class T, int V, int HP, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  if (item >= p.items) return;
  const uint32_t row = p.groups.divide(item);
  const int g = item - row * p.groups.by;
  const uint32_t token = p.chunks.divide(row);
  const int first = (row - token * p.chunks.by) * HP;
  const int position = p.positions[token];
  long long place = 0;   // where the token's keys and values go
  int heads = p.end[2];  // without a place for them only queries are turned
  if (p.page.by > 0) {
    if (position < 0) return;
    const int seq = p.seqs ? p.seqs[token] : (int)token;
    const int slot = p.page.divide(position);
    int page = -1;
    if (seq < 0 || seq >= p.batch || slot >= p.table_width) {
      note_error(p.gerr, kErrBadPlace);
    } else {
      page = p.table[(long long)seq * p.table_width + slot];
      if (page < 0 || page >= p.num_pages) {
        note_error(p.gerr, kErrBadPage);
        page = -1;
      }
    }
    if (page < 0) heads = p.end[0];
    place = page * p.page_stride + (long long)(position - slot * (int)p.page.by) * p.place_stride;
  }
  const bool turn = g < p.rot_items;
  // elements of the item's two vectors within a head
  const int a0 = turn ? (INTERLEAVED ? 2 * V * g : V * g) : 2 * p.half + 2 * V * (g - p.rot_items);
  const int b0 = turn && !INTERLEAVED ? a0 + p.half : a0 + V;
  Row<T, V> a[HP], b[HP];
  T* out[HP];
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    const int h = first + i;
    if (h < heads) {
      const int w = h < p.end[0] ? 0 : h < p.end[1] ? 1 : 2;
      const Side& s = p.part[w];
      const int head = w == 0 ? h : h - p.end[w - 1];
      const T* in = reinterpret_cast<const T*>(s.in) + token * s.in_token + head * s.in_head;
      out[i] = reinterpret_cast<T*>(s.out) + (w > 0 && p.page.by > 0 ? place : token * s.out_token) + head * s.out_head;
      a[i].load(in + a0);
      b[i].load(in + b0);
    }
  }
  float cs[V], sn[V];
  if (turn) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint64_t angle = (uint64_t)(int64_t)position * p.turns[V * g + e];
      const float rad = (float)(int32_t)(angle >> 32) * 1.4629180792671596e-9f;  // 2 pi / 2^32
      float s, c;
      __sincosf(rad, &s, &c);
      cs[e] = c * p.magnitude;
      sn[e] = s * p.magnitude * p.sign;
    }
  }
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    const int h = first + i;
    if (h >= heads) break;
    if (turn && h < p.turned_heads) {
      if (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < V; ++e) {  // pairs lie side by side: the first half of them in a, the second in b
          T* x = 2 * e < V ? &a[i].v[2 * e % V] : &b[i].v[2 * e % V];
          T* y = 2 * e + 1 < V ? &a[i].v[(2 * e + 1) % V] : &b[i].v[(2 * e + 1) % V];
          const float u = to_f32(*x), v = to_f32(*y);
          *x = from_f32<T>(u * cs[e] - v * sn[e]);
          *y = from_f32<T>(v * cs[e] + u * sn[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float u = to_f32(a[i].v[e]), v = to_f32(b[i].v[e]);
          a[i].v[e] = from_f32<T>(u * cs[e] - v * sn[e]);
          b[i].v[e] = from_f32<T>(v * cs[e] + u * sn[e]);
        }
      }
    }
    a[i].store(out[i] + a0);
    b[i].store(out[i] + b0);
  }
}

template <class T, int HP>
void (*pick_kernel(int v, bool interleaved))(const RopeParams) {
  switch (v) {
    case 8: return interleaved ? rope_kernel<T, 8, HP, true> : rope_kernel<T, 8, HP, false>;
    case 4: return interleaved ? rope_kernel<T, 4, HP, true> : rope_kernel<T, 4, HP, false>;
    case 2: return interleaved ? rope_kernel<T, 2, HP, true> : rope_kernel<T, 2, HP, false>;
    default: return interleaved ? rope_kernel<T, 1, HP, true> : rope_kernel<T, 1, HP, false>;
  }
}
template <class T>
void (*pick_kernel(int v, int hp, bool interleaved))(const RopeParams) {
  return hp == 4 ? pick_kernel<T, 4>(v, interleaved) : pick_kernel<T, 1>(v, interleaved);
}

// The widest vectors that head_dim, rot_dim and all tensors' addresses and strides are multiples of.
int vector_width(int head_dim, int rot, const RopeParams& p) {
  long long all = (head_dim / 2) | (rot / 2);
  for (const Side& s : p.part)
    if (s.in) all |= (long long)((uintptr_t)s.in / 2) | (long long)((uintptr_t)s.out / 2) | s.in_token | s.in_head | s.out_token | s.out_head;
  if (p.page.by > 0) all |= p.page_stride | p.place_stride;
  return all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
}

int launch(aig_ctx* ctx, int dtype, int head_dim, int rot, bool interleaved, long long tokens, RopeParams& p) {
  const int v = vector_width(head_dim, rot, p);
  p.half = rot / 2;
  p.rot_items = rot / 2 / v;
  const int groups = head_dim / 2 / v, heads = p.end[2];
  // Heads per thread: sines are shared by more of them and more reads are under way, but few tokens need every head as a
  // thread of its own to fill the device.
  const int hp = (double)tokens * groups * heads >= 4.0 * 1024 * ctx->sm_count ? 4 : 1;
  const long long per_token = (long long)ceil_div(heads, hp) * groups;
  if (tokens * (double)per_token > 2147483647.0 - kThreads)
    return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "rotary positions: too many values for one call");
  p.groups = Divisor::of(groups);
  p.chunks = Divisor::of(ceil_div(heads, hp));
  p.items = (uint32_t)(tokens * per_token);
  p.gerr = ctx->d_err;
  void (*kernel)(const RopeParams) = dtype == AIG_F16 ? pick_kernel<__half>(v, hp, interleaved) : pick_kernel<__nv_bfloat16>(v, hp, interleaved);
  AIG_CUDA_OK(ctx, launch_pdl(ctx, kernel, dim3((p.items + kThreads - 1) / kThreads), dim3(kThreads), 0, p));
  return AIG_OK;
}

Side side_of(const aig_heads* in, const aig_heads* out) {
  return Side{(const uint8_t*)in->data, (uint8_t*)out->data, in->token_stride, in->head_stride, out->token_stride, out->head_stride};
}

int check_pair(aig_ctx* ctx, const aig_heads* in, const aig_heads* out, const char* who) {
  AIG_REQUIRE(ctx, heads_sane(in) && heads_sane(out), "%s: null tensor, negative stride or data off a 2-byte boundary", who);
  AIG_REQUIRE(ctx, in->heads == out->heads, "%s: input and output have different numbers of heads (%d, %d)", who, in->heads, out->heads);
  return AIG_OK;
}

bool desc_ok(const aig_rope_desc* d) {
  if (!d || d->head_dim <= 0 || d->head_dim % 2 || d->head_dim > 1024 || d->rot_dim <= 0 || d->rot_dim % 2 || d->rot_dim > d->head_dim) return false;
  if (!(d->base > 1.f) || !std::isfinite(d->base) || !std::isfinite(d->magnitude)) return false;
  if (d->scaling < AIG_ROPE_PLAIN || d->scaling > AIG_ROPE_TURNS) return false;
  if (d->scaling != AIG_ROPE_PLAIN && (!(d->factor >= 1.f) || !std::isfinite(d->factor))) return false;
  if (d->scaling >= AIG_ROPE_RAMP && (d->original_len <= 0 || !(d->low > 0.f) || !(d->high > d->low) || !std::isfinite(d->high))) return false;
  return true;
}

int turn_tensors(aig_rope_plan* pl, int dtype, const int32_t* positions, long long tokens, const aig_heads* q, const aig_heads* q_out,
                 const aig_heads* k, const aig_heads* k_out, float sign, const char* who) {
  if (!pl) return AIG_ERR_INVALID;
  aig_ctx* ctx = pl->ctx;
  DeviceGuard g(ctx->device);
  AIG_REQUIRE(ctx, dtype_known(dtype), "%s: unknown element type %d", who, dtype);
  AIG_REQUIRE(ctx, tokens >= 0, "%s: negative number of tokens", who);
  if (tokens == 0) return AIG_OK;
  int rc = check_pair(ctx, q, q_out, who);
  if (rc != AIG_OK) return rc;
  AIG_REQUIRE(ctx, (k == nullptr) == (k_out == nullptr), "%s: k and k_out come together", who);
  if (k && (rc = check_pair(ctx, k, k_out, who)) != AIG_OK) return rc;
  AIG_REQUIRE(ctx, positions && aligned_to(positions, 4), "%s: null positions, or off a 4-byte boundary", who);
  RopeParams p{};
  p.part[0] = side_of(q, q_out);
  p.end[0] = p.end[1] = p.end[2] = q->heads;
  if (k) {
    p.part[1] = side_of(k, k_out);
    p.end[1] = p.end[2] = q->heads + k->heads;
  }
  p.turned_heads = p.end[2];
  p.positions = positions;
  p.turns = pl->turns;
  p.magnitude = pl->desc.magnitude;
  p.sign = sign;
  return launch(ctx, dtype, pl->desc.head_dim, pl->desc.rot_dim, pl->desc.interleaved != 0, tokens, p);
}

}  // namespace

extern "C" {

int aig_rope_frequencies(const aig_rope_desc* d, double* out, int n) {
  if (!desc_ok(d) || !out || n != d->rot_dim / 2) return AIG_ERR_INVALID;
  const double two_pi = 6.283185307179586476925286766559, rot = d->rot_dim, base = d->base, len = d->original_len;
  double ramp_from = 0, ramp_to = 0;
  if (d->scaling == AIG_ROPE_RAMP) {
    auto pair_with = [&](double turns) { return rot * std::log(len / (two_pi * turns)) / (2.0 * std::log(base)); };
    ramp_from = std::fmax(std::floor(pair_with(d->high)), 0.0);
    ramp_to = std::fmin(std::ceil(pair_with(d->low)), rot - 1.0);
  }
  for (int j = 0; j < n; ++j) {
    double f = std::pow(base, -2.0 * j / rot);
    double share = 0.0;  // of the frequency that the longer context asks for
    if (d->scaling == AIG_ROPE_LINEAR) share = 1.0;
    if (d->scaling == AIG_ROPE_RAMP) share = std::fmin(1.0, std::fmax(0.0, (j - ramp_from) / std::fmax(ramp_to - ramp_from, 0.001)));
    if (d->scaling == AIG_ROPE_TURNS) share = 1.0 - std::fmin(1.0, std::fmax(0.0, (len * f / two_pi - d->low) / ((double)d->high - d->low)));
    out[j] = share == 0.0 ? f : f * (1.0 - share) + f / d->factor * share;
  }
  return AIG_OK;
}

int aig_rope_plan_create(aig_ctx* ctx, const aig_rope_desc* desc, aig_rope_plan** out) {
  if (!ctx || !out) return AIG_ERR_INVALID;
  *out = nullptr;
  DeviceGuard g(ctx->device);
  AIG_REQUIRE(ctx, desc_ok(desc), "rope plan: head_dim even and at most 1024, rot_dim even and at most head_dim, base above 1, factor at least 1, "
                                  "original_len and 0 < low < high with scalings that use them, everything finite");
  try {
    const int n = desc->rot_dim / 2;
    std::vector<double> f(n);
    std::vector<uint64_t> turns(n);
    aig_rope_frequencies(desc, f.data(), n);
    // f is at most 1 radian, so f / 2 pi * 2^64 fits; long double keeps all 64 bits
    for (int j = 0; j < n; ++j) turns[j] = (uint64_t)((long double)f[j] / 6.283185307179586476925286766559005768L * 18446744073709551616.0L + 0.5L);
    aig_rope_plan* pl = new aig_rope_plan();
    pl->ctx = ctx;
    pl->desc = *desc;
    if (cudaMalloc(&pl->turns, n * sizeof(uint64_t)) != cudaSuccess ||
        cudaMemcpyAsync(pl->turns, turns.data(), n * sizeof(uint64_t), cudaMemcpyHostToDevice, ctx->stream) != cudaSuccess ||
        cudaStreamSynchronize(ctx->stream) != cudaSuccess) {
      aig_rope_plan_destroy(pl);
      return aig_fail(ctx, AIG_ERR_CUDA, "rope plan: device allocation or copy failed");
    }
    *out = pl;
    return AIG_OK;
  } catch (const std::bad_alloc&) {
    return aig_fail(ctx, AIG_ERR_CUDA, "rope plan: out of host memory");
  }
}

int aig_rope_plan_destroy(aig_rope_plan* pl) {
  if (!pl) return AIG_OK;
  DeviceGuard g(pl->ctx->device);
  cudaStreamSynchronize(pl->ctx->stream);
  cudaFree(pl->turns);
  delete pl;
  return AIG_OK;
}

int aig_rope_forward(aig_rope_plan* pl, int dtype, const int32_t* positions, long long tokens, const aig_heads* q, const aig_heads* q_out,
                     const aig_heads* k, const aig_heads* k_out) {
  return turn_tensors(pl, dtype, positions, tokens, q, q_out, k, k_out, 1.f, "rope forward");
}

int aig_rope_backward(aig_rope_plan* pl, int dtype, const int32_t* positions, long long tokens, const aig_heads* dq, const aig_heads* dq_out,
                      const aig_heads* dk, const aig_heads* dk_out) {
  return turn_tensors(pl, dtype, positions, tokens, dq, dq_out, dk, dk_out, -1.f, "rope backward");
}

int aig_kv_append(aig_ctx* ctx, const aig_kv_cache* cache, aig_rope_plan* rope, const aig_heads* k, const aig_heads* v, const aig_heads* q,
                  const aig_heads* q_out, const int32_t* seqs, const int32_t* positions, long long tokens, const int32_t* table, int batch,
                  int table_width) {
  if (!ctx) return AIG_ERR_INVALID;
  DeviceGuard g(ctx->device);
  int rc = check_cache(ctx, cache, "kv append");
  if (rc != AIG_OK) return rc;
  AIG_REQUIRE(ctx, tokens >= 0 && batch >= 0 && table_width >= 0, "kv append: bad extents");
  if (tokens == 0) return AIG_OK;
  AIG_REQUIRE(ctx, heads_sane(k) && heads_sane(v), "kv append: null tensor, negative stride or data off a 2-byte boundary");
  AIG_REQUIRE(ctx, k->heads == cache->kv_heads && v->heads == cache->kv_heads, "kv append: %d and %d heads for a cache of %d", k->heads, v->heads,
              cache->kv_heads);
  AIG_REQUIRE(ctx, (q == nullptr) == (q_out == nullptr), "kv append: q and q_out come together");
  if (q && (rc = check_pair(ctx, q, q_out, "kv append")) != AIG_OK) return rc;
  AIG_REQUIRE(ctx, seqs || tokens <= batch, "kv append: %lld tokens without sequence numbers for a batch of %d", tokens, batch);
  AIG_REQUIRE(ctx, !rope || (rope->ctx->device == ctx->device && rope->desc.head_dim == cache->head_dim),
              "kv append: the rope plan is for another device or head dimension");
  AIG_REQUIRE(ctx, positions && table && aligned_to(positions, 4) && aligned_to(table, 4) && aligned_to(seqs, 4),
              "kv append: null positions or table, or integers off a 4-byte boundary");
  RopeParams p{};
  if (q) p.part[0] = side_of(q, q_out);
  p.end[0] = q ? q->heads : 0;
  p.part[1] = Side{(const uint8_t*)k->data, (uint8_t*)cache->k, k->token_stride, k->head_stride, 0, cache->head_stride};
  p.part[2] = Side{(const uint8_t*)v->data, (uint8_t*)cache->v, v->token_stride, v->head_stride, 0, cache->head_stride};
  p.end[1] = p.end[0] + cache->kv_heads;
  p.end[2] = p.end[1] + cache->kv_heads;
  p.turned_heads = rope ? p.end[1] : 0;
  p.positions = positions;
  p.turns = rope ? rope->turns : nullptr;
  p.magnitude = rope ? rope->desc.magnitude : 1.f;
  p.sign = 1.f;
  p.seqs = seqs;
  p.table = table;
  p.batch = batch;
  p.table_width = table_width;
  p.page = Divisor::of(cache->page_size);
  p.num_pages = cache->num_pages;
  p.page_stride = cache->page_stride;
  p.place_stride = cache->token_stride;
  return launch(ctx, cache->dtype, cache->head_dim, rope ? rope->desc.rot_dim : 0, rope && rope->desc.interleaved, tokens, p);
}

}  // extern "C"

// window_attention.cu -- causal attention over whole sequences with a sliding window and first tokens that stay visible
// (sinks), and its gradients.
//
//   S = scale * Q K^T,  P = softmax(S) over the keys j <= p that are within `window` of p or below `sinks`,  O = P V
//   dV = P^T dO,  dP = dO V^T,  D = rowsum(dO o O),  dS = scale * P o (dP - D),  dQ = dS K,  dK = dS^T Q
//
// A row per warp, a value of the head per lane and register; softmax with a running maximum and sum in fp32.
#include "long_context.h"

namespace {

constexpr int kWarps = 4;

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
};

template <class T>
__device__ __forceinline__ T* row_of(const View& v, int b, int t, int h) {
  return reinterpret_cast<T*>(v.data) + b * v.batch + t * v.token + h * v.head;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ int length_of(const WinParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.kv_len) : p.kv_len;
}
template <class T, int N>
__device__ __forceinline__ void load_row(float (&x)[N], const T* p, int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f32(p[i * 32 + lane]);
}
template <int N>
__device__ __forceinline__ float dot(const float (&a)[N], const float (&b)[N]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(a[i], b[i], s);
  return warp_sum(s);
}

// keys of a query at position pos: [0, front) and [back, pos]
__device__ __forceinline__ void keys_of(const WinParams& p, int pos, int& front, int& back) {
  back = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  front = min(p.sinks, back);
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) forward_rows_kernel(const __grid_constant__ WinParams p) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31, i = blockIdx.x * kWarps + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  const int pos = i + p.kv_len - p.q_len;
  if (i >= p.q_len || pos >= length_of(p, b)) return;
  const int kvh = h / (p.heads / p.kv_heads);
  float q[N], o[N] = {}, x[N];
  load_row<T>(q, row_of<T>(p.q, b, i, h), lane);
  float top = -INFINITY, sum = 0.f;
  int front, back;
  keys_of(p, pos, front, back);
  for (int j = front > 0 ? 0 : back; j <= pos; j = j + 1 == front ? back : j + 1) {
    load_row<T>(x, row_of<T>(p.k, b, j, kvh), lane);
    const float s = dot(q, x) * p.scale, m = fmaxf(top, s), f = expf(top - m), w = expf(s - m);
    load_row<T>(x, row_of<T>(p.v, b, j, kvh), lane);
    sum = sum * f + w;
    top = m;
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = fmaf(o[n], f, w * x[n]);
  }
  T* out = row_of<T>(p.o, b, i, h);
#pragma unroll
  for (int n = 0; n < N; ++n) out[n * 32 + lane] = from_f32<T>(o[n] / sum);
  if (lane == 0) p.lse[((long long)b * p.heads + h) * p.q_len + i] = top + logf(sum);
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) backward_q_kernel(const __grid_constant__ WinParams p) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31, i = blockIdx.x * kWarps + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  const int pos = i + p.kv_len - p.q_len;
  if (i >= p.q_len || pos >= length_of(p, b)) return;
  const int kvh = h / (p.heads / p.kv_heads);
  float q[N], g[N], x[N], dq[N] = {};
  load_row<T>(q, row_of<T>(p.q, b, i, h), lane);
  load_row<T>(g, row_of<T>(p.dout, b, i, h), lane);
  load_row<T>(x, row_of<T>(p.o, b, i, h), lane);
  const float delta = dot(g, x);
  const long long stat = ((long long)b * p.heads + h) * p.q_len + i;
  const float lse = p.lse[stat];
  if (lane == 0) p.delta[stat] = delta;
  int front, back;
  keys_of(p, pos, front, back);
  for (int j = front > 0 ? 0 : back; j <= pos; j = j + 1 == front ? back : j + 1) {
    load_row<T>(x, row_of<T>(p.v, b, j, kvh), lane);
    const float dp = dot(g, x);
    load_row<T>(x, row_of<T>(p.k, b, j, kvh), lane);
    const float ds = expf(dot(q, x) * p.scale - lse) * (dp - delta) * p.scale;
#pragma unroll
    for (int n = 0; n < N; ++n) dq[n] = fmaf(ds, x[n], dq[n]);
  }
  T* out = row_of<T>(p.dq, b, i, h);
#pragma unroll
  for (int n = 0; n < N; ++n) out[n * 32 + lane] = from_f32<T>(dq[n]);
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) backward_kv_kernel(const __grid_constant__ WinParams p) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31, j = blockIdx.x * kWarps + (threadIdx.x >> 5), kvh = blockIdx.y, b = blockIdx.z;
  const int len = length_of(p, b), first = p.kv_len - p.q_len, group = p.heads / p.kv_heads;
  if (j >= len) return;
  float k[N], v[N], x[N], g[N], dk[N] = {}, dv[N] = {};
  load_row<T>(k, row_of<T>(p.k, b, j, kvh), lane);
  load_row<T>(v, row_of<T>(p.v, b, j, kvh), lane);
  // queries that see key j: positions j .. last
  const int last = p.window > 0 && j >= p.sinks ? (int)min((long long)len - 1, (long long)j + p.window - 1) : len - 1;
  for (int h = kvh * group; h < (kvh + 1) * group; ++h)
    for (int pos = max(j, first); pos <= last; ++pos) {
      const int i = pos - first;
      const long long stat = ((long long)b * p.heads + h) * p.q_len + i;
      load_row<T>(x, row_of<T>(p.q, b, i, h), lane);
      load_row<T>(g, row_of<T>(p.dout, b, i, h), lane);
      const float w = expf(dot(k, x) * p.scale - p.lse[stat]);
      const float ds = w * (dot(v, g) - p.delta[stat]) * p.scale;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        dk[n] = fmaf(ds, x[n], dk[n]);
        dv[n] = fmaf(w, g[n], dv[n]);
      }
    }
  T *out_k = row_of<T>(p.dk, b, j, kvh), *out_v = row_of<T>(p.dv, b, j, kvh);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    out_k[n * 32 + lane] = from_f32<T>(dk[n]);
    out_v[n * 32 + lane] = from_f32<T>(dv[n]);
  }
}

bool tensor_ok(const aig_seq_heads* t) {
  return t && t->data && aligned_to(t->data, 16) && t->batch_stride >= 0 && t->token_stride >= 0 && t->head_stride >= 0 && t->batch_stride % 8 == 0 &&
         t->token_stride % 8 == 0 && t->head_stride % 8 == 0;
}
View view_of(const aig_seq_heads* t) { return View{(uint8_t*)t->data, t->batch_stride, t->token_stride, t->head_stride}; }

int check_desc(aig_ctx* ctx, const aig_window_desc* d, const char* who) {
  AIG_REQUIRE(ctx, d && dtype_known(d->dtype), "%s: null description or unknown element type", who);
  AIG_REQUIRE(ctx, d->batch >= 0 && d->q_len >= 0 && d->kv_len >= d->q_len && d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0 && d->sinks >= 0,
              "%s: bad extents (q_len at most kv_len, heads a multiple of kv_heads)", who);
  AIG_REQUIRE(ctx, d->scale == d->scale && d->scale - d->scale == 0.f, "%s: the scale is not finite", who);
  if (d->head_dim != 64 && d->head_dim != 128)
    return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "%s: head dimension must be 64 or 128 (got %d)", who, d->head_dim);
  if (d->batch > 65535 || d->heads > 65535) return aig_fail(ctx, AIG_ERR_UNSUPPORTED, "%s: more than 65535 sequences or heads", who);
  return AIG_OK;
}
WinParams params_of(const aig_window_desc* d) {
  WinParams p{};
  p.batch = d->batch;
  p.q_len = d->q_len;
  p.kv_len = d->kv_len;
  p.heads = d->heads;
  p.kv_heads = d->kv_heads;
  p.window = d->window;
  p.sinks = d->sinks;
  p.scale = d->scale;
  return p;
}

template <class T, int D>
int forward(aig_ctx* ctx, const WinParams& p) {
  forward_rows_kernel<T, D><<<dim3(ceil_div(p.q_len, kWarps), p.heads, p.batch), kWarps * 32, 0, ctx->stream>>>(p);
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
}
template <class T, int D>
int backward(aig_ctx* ctx, const WinParams& p) {
  backward_q_kernel<T, D><<<dim3(ceil_div(p.q_len, kWarps), p.heads, p.batch), kWarps * 32, 0, ctx->stream>>>(p);
  AIG_LAUNCH_OK(ctx);
  backward_kv_kernel<T, D><<<dim3(ceil_div(p.kv_len, kWarps), p.kv_heads, p.batch), kWarps * 32, 0, ctx->stream>>>(p);
  AIG_LAUNCH_OK(ctx);
  return AIG_OK;
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
  AIG_REQUIRE(ctx, tensor_ok(q) && tensor_ok(k) && tensor_ok(v) && tensor_ok(out) && lse,
              "window attention: null tensor, data off a 16-byte boundary, or strides that are negative or no multiples of 8");
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
  AIG_REQUIRE(ctx, tensor_ok(q) && tensor_ok(k) && tensor_ok(v) && tensor_ok(out) && tensor_ok(dout) && tensor_ok(dq) && tensor_ok(dk) && tensor_ok(dv) &&
                       lse && delta,
              "window attention backward: null tensor, data off a 16-byte boundary, or strides that are negative or no multiples of 8");
  AIG_REQUIRE(ctx, d->q_len > 0, "window attention backward: no queries");
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

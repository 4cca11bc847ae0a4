// KV write with the rotation of queries and keys on the way: what a layer otherwise does with a rotation
// of q and k in place and reshape_and_cache behind it, in one launch that reads every tensor once.
//
// A pair (a, b) of a head's dimensions becomes (a cos - b sin, b cos + a sin), with the cosine and the sine of
// the token's position from a table [position][cos of rot / 2 pairs, sin of rot / 2 pairs].  Pairs are
// (d, d + rot / 2), or neighbours (2 d, 2 d + 1); dimensions from rot on stay as they are.  The arithmetic is
// fp32 and what comes out is rounded once, to the query's type or to the cache's code of k / k_scale: keys are
// NOT rounded to the query's type before they are quantised, as a separate rotation would.
#include <algorithm>
#include <type_traits>

#include "kv_quant.cuh"

namespace b200pa {

struct RotaryParams {
  void* query_out;
  const void* query;
  const void* key;
  const void* value;
  void* key_cache;
  void* value_cache;
  const int64_t* positions;
  const int64_t* slots;
  const void* table;
  const float* k_scale;
  const float* v_scale;
  int64_t query_out_stride;  // elements between two tokens
  int64_t query_stride;
  int64_t key_stride;
  int64_t value_stride;
  int64_t block_stride;  // flash layout: elements of the cache
  int64_t page_stride;
  int64_t head_stride;
  int64_t max_position;  // rows of the table
  int num_tokens;
  int num_heads;
  int num_kv_heads;
  int head_size;
  int rot;
  int block_size;
  int x;            // x-layout: elements per chunk of K; 0: flash layout
  bool neighbours;  // pairs are neighbours
  bool table_f32;   // else the table has the query's type
};

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fffffff); }

// Every type, size, stride and alignment: a CTA to a token, a thread to a pair.
template <typename in_t, typename cache_t, int KV>
__global__ void __launch_bounds__(256) rotary_write_plain_kernel(const RotaryParams p) {
  grid_dependency_wait();
  const int64_t tok = blockIdx.x;
  const int D = p.head_size, HK = p.num_kv_heads, half = p.rot / 2;
  const int64_t pos = p.positions[tok], slot = p.slots[tok];
  const bool known = pos >= 0 && pos < p.max_position;
  const int64_t blk = slot >= 0 ? slot / p.block_size : 0;
  const int off = int(slot >= 0 ? slot - blk * p.block_size : 0);
  auto entry = [&](int i) -> float {
    if (!known) return nan_f32();
    const int64_t at = pos * p.rot + i;
    return p.table_f32 ? static_cast<const float*>(p.table)[at] : to_f32(static_cast<const in_t*>(p.table)[at]);
  };
  auto store = [](float v, float scale) -> cache_t {
    if constexpr (KV == kKvAuto) return from_f32<cache_t>(v);
    else return f32_to_fp8<KV == kKvE5M2>(__fdiv_rn(v, scale));
  };
  auto flash_at = [&](int h, int d) { return blk * p.block_stride + off * p.page_stride + h * p.head_stride + d; };
  const float k_scale = KV == kKvAuto ? 1.f : *p.k_scale, v_scale = KV == kKvAuto ? 1.f : *p.v_scale;
  cache_t* kc = static_cast<cache_t*>(p.key_cache);
  cache_t* vc = static_cast<cache_t*>(p.value_cache);
  const int units = half + D - p.rot;  // pairs, then what is not rotated
  for (int i = threadIdx.x; i < (p.num_heads + HK) * units; i += blockDim.x) {
    const int head = i / units, u = i % units;
    const bool is_key = head >= p.num_heads;
    if (is_key && slot < 0) continue;
    const int h = is_key ? head - p.num_heads : head;
    const in_t* src = is_key ? static_cast<const in_t*>(p.key) + tok * p.key_stride + int64_t(h) * D
                             : static_cast<const in_t*>(p.query) + tok * p.query_stride + int64_t(h) * D;
    auto put = [&](int d, float v) {
      if (!is_key) static_cast<in_t*>(p.query_out)[tok * p.query_out_stride + int64_t(h) * D + d] = from_f32<in_t>(v);
      else if (p.x == 0) kc[flash_at(h, d)] = store(v, k_scale);
      else kc[(((blk * HK + h) * (D / p.x) + d / p.x) * p.block_size + off) * p.x + d % p.x] = store(v, k_scale);
    };
    if (u < half) {
      const int da = p.neighbours ? 2 * u : u, db = p.neighbours ? 2 * u + 1 : u + half;
      const float a = to_f32(src[da]), b = to_f32(src[db]), c = entry(u), s = entry(half + u);
      put(da, fmaf(a, c, -(b * s)));
      put(db, fmaf(b, c, a * s));
    } else {
      const int d = p.rot + u - half;
      put(d, to_f32(src[d]));
    }
  }
  if (slot < 0) return;
  const in_t* v = static_cast<const in_t*>(p.value) + tok * p.value_stride;
  for (int i = threadIdx.x; i < HK * D; i += blockDim.x) {
    const int h = i / D, d = i % D;
    vc[p.x == 0 ? flash_at(h, d) : ((blk * HK + h) * D + d) * p.block_size + off] = store(to_f32(v[i]), v_scale);
  }
}

template <typename in_t, typename cache_t, int KV>
static int launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  const cudaError_t e = launch_dependent(rotary_write_plain_kernel<in_t, cache_t, KV>, dim3(p.num_tokens), dim3(256), 0, stream, p);
  count_launch();
  if (e != cudaSuccess) {
    set_error("rotary KV write kernel launch failed: %s", cudaGetErrorString(e));
    return B200PA_ECUDA;
  }
  return B200PA_OK;
}

template <typename in_t>
static int dispatch_rotary(const RotaryParams& p, int kv_dtype, cudaStream_t s) {
  switch (kv_dtype) {
    case B200PA_KV_AUTO: return launch_rotary<in_t, in_t, kKvAuto>(p, s);
    case B200PA_KV_FP8_E4M3: return launch_rotary<in_t, uint8_t, kKvE4M3>(p, s);
    case B200PA_KV_FP8_E5M2: return launch_rotary<in_t, uint8_t, kKvE5M2>(p, s);
  }
  set_error("Unsupported data type of kv cache: %d", kv_dtype);
  return B200PA_EUNSUPPORTED;
}

static int rotary_entry(const b200pa_rotary_args* r, const b200pa_cache_args* a, void* stream, bool flash) {
  B200PA_CHECK_ARG(r != nullptr && a != nullptr, "args is NULL");
  B200PA_CHECK_ARG(a->num_tokens >= 0 && a->num_heads > 0 && a->head_size > 0 && a->block_size > 0 && r->num_heads > 0,
                   "bad sizes: num_tokens=%d num_heads=%d num_kv_heads=%d head_size=%d block_size=%d", a->num_tokens,
                   r->num_heads, a->num_heads, a->head_size, a->block_size);
  B200PA_CHECK_ARG(int64_t(r->num_heads + int64_t(a->num_heads)) * a->head_size <= INT32_MAX, "too many heads: %d and %d of %d",
                   r->num_heads, a->num_heads, a->head_size);
  B200PA_CHECK_ARG(r->rot_dim > 0 && r->rot_dim % 2 == 0 && r->rot_dim <= a->head_size,
                   "rot_dim %d has to be even and at most the head size %d", r->rot_dim, a->head_size);
  B200PA_CHECK_ARG(r->max_position > 0, "the rotation table is empty");
  if (a->in_dtype != B200PA_F32 && a->in_dtype != B200PA_F16 && a->in_dtype != B200PA_BF16) {
    set_error("Unsupported input type of kv cache: %d", a->in_dtype);
    return B200PA_EUNSUPPORTED;
  }
  if (a->kv_dtype != B200PA_KV_AUTO && a->kv_dtype != B200PA_KV_FP8_E4M3 && a->kv_dtype != B200PA_KV_FP8_E5M2) {
    set_error("Unsupported data type of kv cache: %d", a->kv_dtype);
    return B200PA_EUNSUPPORTED;
  }
  B200PA_CHECK_ARG(r->table_dtype == B200PA_F32 || r->table_dtype == a->in_dtype,
                   "the rotation table has to be float32 or of the query's type");
  if (!flash)
    B200PA_CHECK_ARG(a->x > 0 && a->head_size % a->x == 0, "head_size %d is not a multiple of x=%d",
                     a->head_size, a->x);
  if (a->num_tokens == 0) return B200PA_OK;
  B200PA_CHECK_ARG(r->query_out && r->query && r->positions && r->cos_sin && a->key && a->value && a->key_cache &&
                       a->value_cache && a->slot_mapping,
                   "null tensor pointer");
  B200PA_CHECK_ARG(a->kv_dtype == B200PA_KV_AUTO || (a->k_scale && a->v_scale), "fp8 kv cache needs k_scale and v_scale");
  RotaryParams p{};
  p.query_out = r->query_out;
  p.query = r->query;
  p.key = a->key;
  p.value = a->value;
  p.key_cache = a->key_cache;
  p.value_cache = a->value_cache;
  p.positions = r->positions;
  p.slots = a->slot_mapping;
  p.table = r->cos_sin;
  p.k_scale = a->k_scale;
  p.v_scale = a->v_scale;
  p.query_out_stride = r->query_out_stride;
  p.query_stride = r->query_stride;
  p.key_stride = a->key_stride;
  p.value_stride = a->value_stride;
  p.block_stride = a->block_stride;
  p.page_stride = a->page_stride;
  p.head_stride = a->head_stride;
  p.max_position = r->max_position;
  p.num_tokens = a->num_tokens;
  p.num_heads = r->num_heads;
  p.num_kv_heads = a->num_heads;
  p.head_size = a->head_size;
  p.rot = r->rot_dim;
  p.block_size = a->block_size;
  p.x = flash ? 0 : a->x;
  p.neighbours = r->neighbours != 0;
  p.table_f32 = r->table_dtype == B200PA_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->in_dtype) {
    case B200PA_F32: return dispatch_rotary<float>(p, a->kv_dtype, s);
    case B200PA_F16: return dispatch_rotary<__half>(p, a->kv_dtype, s);
    default: return dispatch_rotary<__nv_bfloat16>(p, a->kv_dtype, s);
  }
}

}  // namespace b200pa

extern "C" int b200pa_rotary_reshape_and_cache(const b200pa_rotary_args* rotary, const b200pa_cache_args* args, void* stream) {
  return b200pa::rotary_entry(rotary, args, stream, false);
}

extern "C" int b200pa_rotary_reshape_and_cache_flash(const b200pa_rotary_args* rotary, const b200pa_cache_args* args,
                                                     void* stream) {
  return b200pa::rotary_entry(rotary, args, stream, true);
}

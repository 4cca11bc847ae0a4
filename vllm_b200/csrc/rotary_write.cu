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

#include "decode_common.cuh"
#include "kv_quant.cuh"
#include "kv_write_windows.h"
#include "launch_state.cuh"

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

// Every type, size, stride and alignment: a CTA to a token, a thread to a pair.  8192 tokens of 32 / 8 heads of 96, 24
// dimensions rotated, bf16, 148 us (HBM alone 23), 32 / 32 heads of 80, 20 rotated, 278 (38), fp32 heads of 128 156 (62).
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

// How a launch of the kernel below is divided.
struct RotaryPlan {
  int units;                       // of a head: pairs of 16-byte chunks that are rotated together, then chunks
  int tokens, lanes;               // tokens of a block; heads that its threads work on at once (Q, K, flash V)
  int q_heads, q_parts, q_blocks;  // heads of a block, parts that they make, blocks
  int k_heads, k_parts, k_blocks;  // ... of K; in the flash layout V as well
  int v_heads, v_parts, v_blocks;  // V of the x-layout: tiles of 16 tokens
  int v_dims;                      // head dimensions of a warp's item there
  bool few;                        // less than a wave of blocks
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPitch = 64 * 2 + 16;  // bytes between two token rows of a transposed tile

template <typename in_t>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<in_t, __nv_bfloat16>) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}
template <typename in_t>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  constexpr bool kBf = std::is_same_v<in_t, __nv_bfloat16>;
  return make_uint4(pack2<kBf>(f[0], f[1]), pack2<kBf>(f[2], f[3]), pack2<kBf>(f[4], f[5]), pack2<kBf>(f[6], f[7]));
}

// 16-bit tensors, everything in chunks of 8 elements.  What bounds it: HBM for prefill steps, of whose bytes the
// queries are most; a chain of trips to memory (position -> table, slot -> store) for decode steps.  Blocks of one
// launch do different things:
//   * Q, K and V of the flash layout: a thread owns one unit of a head (the two chunks that a rotation of halves
//     combines, or one chunk) of one token, loads its cosines and sines once and walks over heads, four chunks at a time;
//   * V of the x-layout is a transpose: a warp takes 16 tokens x up to 64 dimensions of a head through shared
//     memory (ldmatrix.trans gives a lane four tokens of a dimension).  Tiles are moved onto 16-slot boundaries of
//     the cache as in the other KV write kernels (kv_write_windows.h).
// Measured on B200: 8192 tokens of 32 / 8 heads of 128, bf16, 42 us (4.9 TB/s of the 206 MB that it has to move); 16384
// of 64 / 8 heads to fp8, chunks that start anywhere, 122 (5.3 TB/s; 139 with 24 warps to an SM and eight chunks a
// thread, 24 and six 129, 16 and sixteen 141, 32 and eight 152); flash layout, neighbours, a quarter rotated, to e5m2,
// 47 (5.3).  32 warps leave 64 registers, of which all twelve instantiations spill: 20 to 88 bytes a thread stored, up
// to 116 loaded.  24 warps with eight chunks store 0 to 56 and are slower, 32 with eight up to 224.  With the next heads'
// chunks on their way under the ones in work: 47 -> 57.  What is left is latency (a warp loads, waits, turns and
// stores) and, for a step of 8192 tokens, 2560 unequal blocks on 592 places: 4.3 waves.
template <typename in_t, int KV, bool kHalves>
__global__ void __launch_bounds__(kRotaryThreads, 4) rotary_write_kernel(const RotaryParams p, const RotaryPlan plan) {
  using cache_t = std::conditional_t<KV == kKvAuto, in_t, uint8_t>;
  constexpr int E = sizeof(cache_t), HU = kHalves ? 2 : 4;
  __shared__ __align__(16) unsigned char s_tile[kRotaryThreads / 32][16 * kRotaryPitch];
  const int tid = threadIdx.x;
  const int D = p.head_size, HK = p.num_kv_heads, B = p.block_size, N = p.num_tokens;
  if (plan.few) grid_dependency();  // (with more blocks the next grid's would take the places of this one's)
  else grid_dependency_wait();

  int b = blockIdx.x;
  if (b < plan.v_blocks) {
    // ================================================= V of the x-layout
    const int lane = tid & 31, warp = tid >> 5;
    const int tile = b / plan.v_parts, h0 = (b - tile * plan.v_parts) * plan.v_heads, h1 = min(HK, h0 + plan.v_heads);
    const int t0 = tile * 16;
    auto slot_at = [&](int tok) -> int64_t { return tok >= 0 && tok < N ? __ldg(p.slots + tok) : int64_t(-1); };
    const int64_t now = slot_at(t0 + lane);
    int d = 0, before = 0, after = 0;
    if (B % 16 == 0) {
      const int64_t back = lane < 3 ? slot_at(t0 - 16 + (lane == 0 ? 0 : lane == 1 ? 8 : 15)) : int64_t(-1);
      auto from = [&](int64_t v, int l) { return __shfl_sync(0xffffffffu, v, l); };
      d = tile_shift(from(now, 0), from(now, 8), from(now, 15));
      before = tile_shift(from(back, 0), from(back, 1), from(back, 2));
      after = tile_shift(from(now, 16), from(now, 24), from(now, 31));
    }
    const ScaledDiv div(KV == kKvAuto ? 1.f : *p.v_scale);
    const int DG = plan.v_dims, groups = (D + DG - 1) / DG, items = (h1 - h0) * groups;
    unsigned char* mine = s_tile[warp];
    auto window = [&](const TileWindow& w, int64_t slot) {  // slot: of row `lane` (lanes 0 .. 15)
      if (w.lo >= w.hi) return;
      const int64_t own = lane >= w.lo && lane < w.hi ? slot : int64_t(-1);
      const int j = lane & 3;
      int64_t at[4];  // element of (head 0, this lane's dimension 0) of tokens 4 j .. 4 j + 3
      bool have[4], quad = B % 4 == 0;
      int64_t first = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t s = __shfl_sync(0xffffffffu, own, 4 * j + k);
        if (k == 0) first = s;
        have[k] = s >= 0;
        quad = quad && have[k] && s == first + k;
        const int64_t blk = have[k] ? s / B : 0;
        at[k] = blk * HK * int64_t(D) * B + (have[k] ? int(s - blk * B) : 0) + int64_t(lane >> 2) * B;
      }
      quad = quad && (first & 3) == 0;
      uint4 in[4];
      auto load = [&](int item) {
        const int h = h0 + item / groups, d0 = item % groups * DG;
        const in_t* src = static_cast<const in_t*>(p.value) + int64_t(h) * D + d0 + (lane & 7) * 8;
        const bool col = (lane & 7) * 8 < min(DG, D - d0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * i + (lane >> 3);
          if (col && r >= w.lo && r < w.hi) in[i] = *reinterpret_cast<const uint4*>(src + int64_t(w.tok + r) * p.value_stride);
        }
      };
      if (warp < items) load(warp);
      for (int item = warp; item < items; item += kRotaryThreads / 32) {
        const int h = h0 + item / groups, d0 = item % groups * DG;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(mine + (4 * i + (lane >> 3)) * kRotaryPitch + (lane & 7) * 16) = in[i];
        __syncwarp();
        if (item + kRotaryThreads / 32 < items) load(item + kRotaryThreads / 32);
        const int mr = lane & 7, mi = lane >> 3, mtok = (mr >> 1) * 4 + (mr & 1) + (mi & 1) * 2;
        const uint32_t row = smem_u32(mine) + mtok * kRotaryPitch + (mi >> 1) * 16;
        const int n16 = min(DG, D - d0) / 16;
        for (int i16 = 0; i16 < n16; ++i16) {
          uint32_t r[4];  // (tokens 4j, 4j+1), (4j+2, 4j+3) of row d; the same of row d + 8
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                       : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                       : "r"(row + i16 * 32));
          const int64_t to = (int64_t(h) * D + d0 + i16 * 16) * B;
          cache_t* base = static_cast<cache_t*>(p.value_cache) + to;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t w2[2] = {r[2 * i], r[2 * i + 1]};
            if constexpr (KV != kKvAuto) {
              uint32_t o[1];
              convert_words<in_t, KV, 2>(w2, o, div);
              w2[0] = o[0];
            }
            if (quad) {
              cache_t* dst = base + at[0] + 8 * i * B;
              if constexpr (E == 1) *reinterpret_cast<uint32_t*>(dst) = w2[0];
              else *reinterpret_cast<uint2*>(dst) = make_uint2(w2[0], w2[1]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (!have[k]) continue;
                cache_t* dst = base + at[k] + 8 * i * B;
                if constexpr (E == 1) *reinterpret_cast<unsigned char*>(dst) = static_cast<unsigned char>(w2[0] >> (8 * k));
                else *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(w2[k >> 1] >> (16 * (k & 1)));
              }
            }
          }
        }
        __syncwarp();
      }
    };
    const TileWindow own = tile_window(t0, N, d, after), front = tile_front_window(t0, d, before);
    window(own, __shfl_sync(0xffffffffu, now, (lane + d) & 31));
    window(front, __shfl_sync(0xffffffffu, now, (lane + d) & 15));
    return;
  }
  b -= plan.v_blocks;

  // ================================================= rows: K (and flash V), then Q
  const int unit = tid % plan.units, row = tid / plan.units;
  const int tl = row % plan.tokens, hl = row / plan.tokens;
  if (hl >= plan.lanes) return;
  const int rot_units = p.rot / (kHalves ? 16 : 8);
  const bool turned = unit < rot_units;
  // dimensions of the unit's chunks
  const int d0 = kHalves && turned ? unit * 8 : p.rot + (unit - rot_units) * 8;
  const int d1 = d0 + p.rot / 2;  // (halves only)
  const bool is_q = b >= plan.k_blocks;
  const bool is_v = !is_q && p.x == 0 && b >= plan.k_blocks / 2;  // (flash: as many blocks of V as of K)
  if (is_q) b -= plan.k_blocks;
  else if (is_v) b -= plan.k_blocks / 2;
  const int parts = is_q ? plan.q_parts : plan.k_parts, per = is_q ? plan.q_heads : plan.k_heads;
  const int tile = b / parts;
  const int h_end = min(is_q ? p.num_heads : HK, (b - tile * parts + 1) * per);
  const int tok = tile * plan.tokens + tl;
  int h = (b - tile * parts) * per + hl;
  if (tok >= N || h >= h_end) return;
  const in_t* src = is_q ? static_cast<const in_t*>(p.query) + int64_t(tok) * p.query_stride
                         : is_v ? static_cast<const in_t*>(p.value) + int64_t(tok) * p.value_stride
                                : static_cast<const in_t*>(p.key) + int64_t(tok) * p.key_stride;
  const bool rotate = turned && !is_v;
  const bool two = kHalves && turned;
  uint4 in[HU][2];
  auto load = [&](int i, int head) {
    const in_t* s = src + int64_t(head) * D;
    in[i][0] = *reinterpret_cast<const uint4*>(s + d0);
    if (two) in[i][1] = *reinterpret_cast<const uint4*>(s + d1);
  };
#pragma unroll
  for (int i = 0; i < HU; ++i)
    if (h + i * plan.lanes < h_end) load(i, h + i * plan.lanes);
  constexpr int NP = kHalves ? 8 : 4;  // pairs of a unit
  float cosine[NP], sine[NP];
  if (rotate) {
    const int64_t pos = p.positions[tok];
    if (pos < 0 || pos >= p.max_position) {
#pragma unroll
      for (int i = 0; i < NP; ++i) cosine[i] = sine[i] = nan_f32();
    } else if (p.table_f32) {
      const float* t = static_cast<const float*>(p.table) + pos * p.rot + unit * NP;
#pragma unroll
      for (int i = 0; i < NP; i += 4) {
        *reinterpret_cast<float4*>(cosine + i) = __ldg(reinterpret_cast<const float4*>(t + i));
        *reinterpret_cast<float4*>(sine + i) = __ldg(reinterpret_cast<const float4*>(t + p.rot / 2 + i));
      }
    } else {
      const in_t* t = static_cast<const in_t*>(p.table) + pos * p.rot + unit * NP;
      float c8[8], s8[8];
      if constexpr (kHalves) {
        unpack8<in_t>(__ldg(reinterpret_cast<const uint4*>(t)), c8);
        unpack8<in_t>(__ldg(reinterpret_cast<const uint4*>(t + p.rot / 2)), s8);
      } else {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(t)), s = __ldg(reinterpret_cast<const uint2*>(t + p.rot / 2));
        unpack8<in_t>(make_uint4(c.x, c.y, 0, 0), c8);
        unpack8<in_t>(make_uint4(s.x, s.y, 0, 0), s8);
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        cosine[i] = c8[i];
        sine[i] = s8[i];
      }
    }
  }
  // where the chunks go: element of head 0, elements between heads
  int64_t to0, to1, step;
  if (is_q) {
    to0 = int64_t(tok) * p.query_out_stride + d0;
    to1 = to0 + p.rot / 2;
    step = D;
  } else {
    const int64_t slot = __ldg(p.slots + tok);
    if (slot < 0) return;
    const int64_t blk = slot / B;
    const int off = int(slot - blk * B);
    if (p.x == 0) {
      to0 = blk * p.block_stride + off * p.page_stride + d0;
      to1 = to0 + p.rot / 2;
      step = p.head_stride;
    } else {
      constexpr int X = 16 / E;
      const int64_t base = blk * HK * int64_t(D) * B + off * X;
      to0 = base + d0 / X * X * B + d0 % X;
      to1 = base + d1 / X * X * B + d1 % X;
      step = int64_t(D) * B;
    }
  }
  const ScaledDiv div(KV == kKvAuto || is_q ? 1.f : is_v ? *p.v_scale : *p.k_scale);
  auto put = [&](const float (&f)[8], int64_t at) {
    if (is_q) {
      *reinterpret_cast<uint4*>(static_cast<in_t*>(p.query_out) + at) = pack8<in_t>(f);
    } else {
      cache_t* c = static_cast<cache_t*>(is_v ? p.value_cache : p.key_cache) + at;
      if constexpr (KV == kKvAuto) {
        *reinterpret_cast<uint4*>(c) = pack8<in_t>(f);
      } else {
        __align__(8) uint8_t o[8];
        convert_n<float, uint8_t, KV, 8>(f, o, div);
        *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(o);
      }
    }
  };
  for (; h < h_end; h += HU * plan.lanes) {
    const int next = h + HU * plan.lanes;
#pragma unroll
    for (int i = 0; i < HU; ++i) {
      const int hi = h + i * plan.lanes;
      if (hi >= h_end) break;
      float a[8], bb[8];
      unpack8<in_t>(in[i][0], a);
      if (two) unpack8<in_t>(in[i][1], bb);
      if (rotate) {
        if constexpr (kHalves) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float x = a[k], y = bb[k];
            a[k] = fmaf(x, cosine[k], -(y * sine[k]));
            bb[k] = fmaf(y, cosine[k], x * sine[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = a[2 * k], y = a[2 * k + 1];
            a[2 * k] = fmaf(x, cosine[k], -(y * sine[k]));
            a[2 * k + 1] = fmaf(y, cosine[k], x * sine[k]);
          }
        }
      }
      put(a, to0 + hi * step);
      if (two) put(bb, to1 + hi * step);
    }
    if (next >= h_end) break;
#pragma unroll
    for (int i = 0; i < HU; ++i)
      if (next + i * plan.lanes < h_end) load(i, next + i * plan.lanes);
  }
}

// The plan of a call, or false where the kernel above does not take it.
static bool rotary_plan(const RotaryParams& p, int cache_size, RotaryPlan* plan) {
  auto al16 = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
  const int D = p.head_size, N = p.num_tokens, HK = p.num_kv_heads, sms = sm_count();
  if (D % 16 != 0 || D > 512 || p.rot % (p.neighbours ? 8 : 16) != 0) return false;
  if (!al16(p.query_out) || !al16(p.query) || !al16(p.key) || !al16(p.value) || !al16(p.key_cache) || !al16(p.value_cache) ||
      !al16(p.table))
    return false;
  if (p.query_out_stride % 8 != 0 || p.query_stride % 8 != 0 || p.key_stride % 8 != 0 || p.value_stride % 8 != 0) return false;
  const bool flash = p.x == 0;
  if (flash ? p.block_stride % 8 != 0 || p.page_stride % 8 != 0 || p.head_stride % 8 != 0 : p.x != 16 / cache_size) return false;
  RotaryPlan r{};
  r.units = p.neighbours ? D / 8 : p.rot / 16 + (D - p.rot) / 8;
  const int rows = kRotaryThreads / r.units;
  r.tokens = 1;
  while (r.tokens * 2 <= rows && r.tokens < N) r.tokens *= 2;
  r.lanes = rows / r.tokens;
  const int64_t tiles = (int64_t(N) + r.tokens - 1) / r.tokens;
  // heads of a block: 8 to a thread (16 where a unit is one chunk), fewer while that leaves SMs without blocks
  auto divide = [&](int heads, int& per, int& parts) -> int64_t {
    per = std::min(heads, (p.neighbours ? 16 : 8) * r.lanes);
    while (per > r.lanes && tiles * ((heads + per - 1) / per) < 4 * sms) per = std::max(r.lanes, per / 2);
    parts = (heads + per - 1) / per;
    return tiles * parts;
  };
  const int64_t q = divide(p.num_heads, r.q_heads, r.q_parts), k = divide(HK, r.k_heads, r.k_parts) * (flash ? 2 : 1);
  int64_t v = 0;
  if (!flash) {
    const int64_t tiles16 = (int64_t(N) + 15) / 16;
    r.v_dims = 64;
    r.v_heads = HK;
    while (r.v_heads > 1 && tiles16 * ((HK + r.v_heads - 1) / r.v_heads) < 2 * sms) r.v_heads = (r.v_heads + 1) / 2;
    r.v_parts = (HK + r.v_heads - 1) / r.v_heads;
    v = tiles16 * r.v_parts;
    if (v < 2 * sms && r.v_heads == 1) r.v_dims = 16;  // an item to each warp
  }
  if (q + k + v > INT32_MAX) return false;
  r.q_blocks = int(q);
  r.k_blocks = int(k);
  r.v_blocks = int(v);
  r.few = q + k + v <= 3 * int64_t(sms);
  *plan = r;
  return true;
}

template <typename in_t, typename cache_t, int KV>
static int launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  bool taken = false;
  if constexpr (sizeof(in_t) == 2) {
    RotaryPlan plan;
    taken = rotary_plan(p, sizeof(cache_t), &plan);
    if (taken)
      e = launch_dependent(p.neighbours ? rotary_write_kernel<in_t, KV, false> : rotary_write_kernel<in_t, KV, true>,
                           dim3(plan.q_blocks + plan.k_blocks + plan.v_blocks), dim3(kRotaryThreads), 0, stream, p, plan);
  }
  if (!taken)
    e = launch_dependent(rotary_write_plain_kernel<in_t, cache_t, KV>, dim3(p.num_tokens), dim3(256), 0, stream, p);
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

// Whether two tensors of `rows` rows share bytes (rows of `bytes`, `stride` apart).  Of different strides only their
// extents are compared.
struct RowSpan {
  const void* ptr;
  int64_t stride, bytes;
};
static bool rows_meet(const RowSpan& a, const RowSpan& b, int64_t rows) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.ptr), pb = reinterpret_cast<uintptr_t>(b.ptr);
  if (pa + (rows - 1) * a.stride + a.bytes <= pb || pb + (rows - 1) * b.stride + b.bytes <= pa) return false;
  if (rows == 1 || a.stride != b.stride || a.stride < a.bytes || b.stride < b.bytes) return true;
  int64_t d = int64_t(pb - pa) % a.stride;  // of b's rows inside a's
  if (d < 0) d += a.stride;
  return d < a.bytes || d + b.bytes > a.stride;
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
  const int64_t es = a->in_dtype == B200PA_F32 ? 4 : 2, n = a->num_tokens, q_row = int64_t(r->num_heads) * a->head_size * es,
                kv_row = int64_t(a->num_heads) * a->head_size * es;
  B200PA_CHECK_ARG(n == 1 || r->query_out_stride * es >= q_row, "the rows of query_out must not overlap");
  const RowSpan out{r->query_out, r->query_out_stride * es, q_row};
  const bool in_place = r->query_out == r->query && (n == 1 || r->query_out_stride == r->query_stride);
  B200PA_CHECK_ARG((in_place || !rows_meet(out, {r->query, r->query_stride * es, q_row}, n)) &&
                       !rows_meet(out, {a->key, a->key_stride * es, kv_row}, n) &&
                       !rows_meet(out, {a->value, a->value_stride * es, kv_row}, n),
                   "query_out must not overlap key, value, or query (but for a rotation in place)");
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

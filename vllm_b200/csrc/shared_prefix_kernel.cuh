// Decode attention of a batch whose sequences begin with the same cache blocks: what the batch has in common is
// read once for all of it.
//
//   softmax(q K^T) V over [prefix | own tokens] = (2^(mp - M) Op + 2^(ms - M) Os) / (2^(mp - M) lp + 2^(ms - M) ls)
//
// with, for either part, the maximum m of its logits (in the log2 domain), the sum l of 2^(logit - m) and the
// weighted sum O of its values.  The launches:
//   * this kernel takes the prefix.  The queries of all sequences meet the same K and V, so it is two matrix products
//     with as many rows as there are (sequence, query head of a kv head) pairs: tcgen05 tiles of 128 rows x 128 keys,
//     the pipeline of the prefill kernel (prefill_kernel.cuh: operand layouts, softmax in two halves, roles of the
//     warps), without a causal edge and without a plan on the device: all items cost the same.
//   * a decode kernel takes every sequence's own tokens.  The one of decode_direct.cuh follows this one, adds the prefix's
//     parts to its accumulators, in fp32, and writes the result.  The one of decode_kernel.cuh runs beside this one on
//     SMs of its own and leaves its parts in the scratch; shared_prefix_combine_kernel, below, adds all of them up.
//     Which of them: shared_prefix_way (shared_prefix.cu).
// The work of this kernel is a flat list (kv head, group of row tiles, key tile), cut into equal ranges, one to a CTA;
// a range may cover the end of one item and the start of the next.  What a CTA has of an item goes to a slot of the
// scratch: item + CTA is a number of its own for every such pair, so nothing is counted and nobody waits.
//   A group is two row tiles over the same keys, which share every K and V tile; where there is only one row tile
// (few sequences: bound by HBM, and by the chain product - softmax - product of a row tile), its key tiles go to the
// two softmax warpgroups in turns, each with accumulators of its own.
// What bounds it: the exponentials and the chain product - softmax - product of a tile, under the tensor cores' rate.
// Measured on B200: 2000 sequences of 64 / 8 heads of 128 behind 2016 tokens of an fp8 cache 131 us (1.0 PFLOP/s, tensor
// pipe 52 % active, 41 MB of HBM read); 8 of 32 / 8 heads behind 65008, one row tile, bf16, 51 us (5.2 TB/s).
#pragma once

#include "prefill_kernel.cuh"

namespace b200pa {

struct SharedPrefixParams {
  const void* q;              // [num_seqs, num_heads, D], row stride q_stride
  const void* kc;
  const void* vc;
  const int* blocks;          // of the prefix
  const int* seq_lens;
  const float* alibi;
  const float* k_scale;
  unsigned char* parts;       // slots of one or two row tiles' parts
  int* status;
  int64_t q_stride;
  int64_t kv_block_stride;    // elements
  int64_t kv_head_stride;
  int num_seqs;
  int num_kv_heads;
  int group;
  int block_size;
  int prefix_len;             // a multiple of block_size
  int row_tiles;              // of a kv head
  int groups;                 // of row tiles of a kv head
  int key_tiles;              // of the prefix
  int cut;                    // key tiles of a CTA; 0: from `balance`
  int* cut_out;               // where it is written then
  SharedPrefixBalance balance;
  int tail_items;             // (kv head, head group) pairs of a sequence behind the prefix
  int turns;                  // 1: one row tile, whose key tiles the warpgroups take in turns
  float scale;
};

// A row tile's part: O as [4 dimensions][128 rows] in fp32, then (m, l) of the rows.
constexpr int shared_prefix_part_bytes(int D) { return 128 * (D * 4 + 8); }

template <typename QT, int KV, int D>
__global__ void __launch_bounds__(kPrefillThreads, 1)
pa_shared_prefix_kernel(const SharedPrefixParams p, const __grid_constant__ CUtensorMap qmap,
                        const __grid_constant__ CUtensorMap vmap) {
  using SH = PrefillShape<D>;
  constexpr bool kFp8 = KV != kCache16;
  constexpr bool kE5 = KV == kCacheE5M2;
  constexpr bool kBf = !kFp8 && std::is_same_v<QT, __nv_bfloat16>;  // operand type: bf16, else f16
  constexpr bool kWiden = kFp8 && std::is_same_v<QT, __nv_bfloat16>;  // Q becomes f16
  constexpr int DP = SH::DP, NQ = SH::NQ, KT = SH::KT, NS = SH::kSlots;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ uint64_t s_bar[2 * NS + 14];
  __shared__ uint32_t s_tmem;
  __shared__ int64_t s_blocks[kPrefillThreads / 32];

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t bar0 = smem_u32(s_bar);
  auto kv_full = [&](uint32_t s) { return bar0 + 8u * s; };
  auto kv_empty = [&](uint32_t s) { return bar0 + 8u * (NS + s); };
  auto s_full = [&](int i) { return bar0 + 8u * (2 * NS + i); };
  auto p_half = [&](int i) { return bar0 + 8u * (2 * NS + 2 + i); };
  auto p_full = [&](int i) { return bar0 + 8u * (2 * NS + 4 + i); };
  auto pv_done = [&](int i) { return bar0 + 8u * (2 * NS + 6 + i); };
  auto q_full = [&](int i) { return bar0 + 8u * (2 * NS + 8 + i); };
  auto q_empty = [&](int i) { return bar0 + 8u * (2 * NS + 10 + i); };
  auto q_land = [&](int i) { return bar0 + 8u * (2 * NS + 12 + i); };

  // (the launch behind this one may start now: it waits for this grid before it reads a part)
  grid_dependency();
  const int total = p.num_kv_heads * p.groups * p.key_tiles;
  int cut = p.cut;
  if (cut == 0) {  // SMs that are not needed here are the next launch's at once
    int64_t blocks = 0;
    for (int i = tid; i < p.num_seqs; i += kPrefillThreads)
      blocks += work_units(behind_prefix(__ldcg(p.seq_lens + i), p.prefix_len), p.block_size);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) blocks += __shfl_xor_sync(0xffffffffu, blocks, o);
    if (lane == 0) s_blocks[warp] = blocks;
    __syncthreads();
    blocks = 0;
    for (int w = 0; w < kPrefillThreads / 32; ++w) blocks += s_blocks[w];
    const int ctas = p.balance.prefix_ctas(blocks * p.tail_items);
    cut = (total + ctas - 1) / ctas;
    if (blockIdx.x == 0 && tid == 0) *p.cut_out = cut;
  }
  if (int64_t(blockIdx.x) * cut >= total) return;

  const uint32_t sq = smem_u32(smem);
  const uint32_t skv = sq + NQ * SH::kQBytes;
  if ((sq & 1023u) != 0) {  // (swizzles go by address bits)
    if (tid == 0) atomicExch(p.status, kStatusNoRing);
    return;
  }
  if (warp == 12) {
    if (lane == 0) {
      for (int s = 0; s < NS; ++s) {
        mbar_init(kv_full(s), 4);
        mbar_init(kv_empty(s), 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full(i), 1);
        mbar_init(p_half(i), 4);
        mbar_init(p_full(i), 4);
        mbar_init(pv_done(i), 1);
        mbar_init(q_full(i), kWiden ? 2 : 1);
        mbar_init(q_empty(i), 1);
        mbar_init(q_land(i), 1);
      }
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(smem_u32(&s_tmem), 512);
  }
  if constexpr (DP != D) {
    // K's padding granule takes part in the product: zero, once (K sits in the even slots of the ring)
    static_assert(DP - D == 8 && NS % 2 == 0, "one padding granule; K and V in slots of their own");
    for (int i = tid; i < NS / 2 * KT; i += kPrefillThreads)
      *reinterpret_cast<uint4*>(smem + NQ * SH::kQBytes + (i / KT) * 2 * SH::kTileBytes + ((D / 8) * KT + i % KT) * 16) =
          make_uint4(0, 0, 0, 0);
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int G = p.group, B = p.block_size, b_shift = 31 - __clz(B);
  const int T = 128 / G;  // sequences of a row tile
  const bool turns = p.turns != 0;
  // ---- this CTA's range of the list, as pieces of items
  struct Piece {
    int item, kvh, tile0;  // tile0: first row tile
    int b, e;              // key tiles
  };
  const int u_end = min(total, (int(blockIdx.x) + 1) * cut);
  int u = int(blockIdx.x) * cut;
  auto next = [&](Piece& it) -> bool {
    if (u >= u_end) return false;
    it.item = u / p.key_tiles;
    it.b = u - it.item * p.key_tiles;
    it.e = min(p.key_tiles, it.b + u_end - u);
    it.kvh = it.item / p.groups;
    it.tile0 = (it.item - it.kvh * p.groups) * (turns ? 1 : NQ);
    u += it.e - it.b;
    return true;
  };
  auto has = [&](const Piece& it, int i) { return !turns && it.tile0 + i < p.row_tiles; };  // (i < NQ)

  bool ok = true;
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    const bool got = __all_sync(0xffffffffu, mbar_spin(bar, parity));
    if (!got) {
      ok = false;
      if (lane == 0) atomicExch(p.status, kStatusMbarTimeout);
    }
    return got;
  };
  auto arrive = [&](uint32_t bar) {  // once per warp, for everything its lanes have done
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  Piece it;

  if (warp < 8) {
    // ================================================= softmax: one thread per row
    reg_inc<PrefillRegs<kFp8>::kSoftmax>();
    const int wg = warp >> 2;
    const int row = tid & 127;
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + uint32_t(wg * KT);
    const uint32_t t_o = tmem + lane_off + uint32_t(NQ * KT + wg * DP);
    const float c = p.scale * kLog2e * (kFp8 ? __ldcg(p.k_scale) : 1.f);
    const bool biased = p.alibi != nullptr || !(c > 0.f);  // the maximum is taken of the scaled values then
    const int row_seq = row / G, row_head = row % G;
    uint32_t n_s = 0, n_pv = 0;  // S tiles received, PV products issued for this warpgroup's accumulators

    while (ok && next(it)) {
      if (wg >= NQ || (!turns && !has(it, wg))) continue;
      const int tile = it.tile0 + (turns ? 0 : wg), step = turns ? 2 : 1, first = it.b + (turns ? wg : 0);
      const int seq = tile * T + row_seq;
      const bool valid = row < T * G && seq < p.num_seqs;
      const int len = valid ? __ldcg(p.seq_lens + seq) : p.prefix_len;
      const int keys = len >= p.prefix_len ? p.prefix_len : 0;  // that this row sees (see behind_prefix)
      const int keys_all = __reduce_min_sync(0xffffffffu, keys);
      const float slope = (p.alibi != nullptr && valid) ? __ldcg(p.alibi + it.kvh * G + row_head) * kLog2e : 0.f;
      float m = -INFINITY, l = 0.f;
      bool unset = true;  // a row of this warp has no maximum yet
      for (int j = first; j < it.e; j += step) {
        if (!wait(s_full(wg), n_s & 1)) break;
        ++n_s;
        tc_fence_after();
        // (as in the prefill kernel: for 16-bit caches without a bias the exponentials of the first half start with
        // the running maximum as it is; the tile is done again where that was too low, by 2^12)
        constexpr int NC = KT / 32;
        const int key0 = j * KT;
        float x[NC][32], cc = c, nm = 0.f;
        float2 sa, sb;
        uint32_t w[NC][16];
        auto exps = [&](int ch, int k) {
          const float2 t = ffma2(make_float2(x[ch][k], x[ch][k + 1]), make_float2(cc, cc), make_float2(nm, nm));
          const float2 e2 = make_float2(fast_exp2(t.x), fast_exp2(t.y));
          if (k & 2) sb = fadd2(sb, e2); else sa = fadd2(sa, e2);
          w[ch][k / 2] = pack2<kBf>(e2.x, e2.y);
        };
        for (bool look = kFp8 || biased || unset;; look = true) {
#pragma unroll
          for (int ch = 0; ch < NC; ++ch) tmem_ld32(t_s + ch * 32, x[ch]);
          int last = keys - 1 - key0;  // last column of this row that counts
          cc = c;                      // (goes through the wait for the TMEM loads, see tmem_landed)
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          tmem_landed(m4, cc, last);
          if (biased) {  // t = x c + slope (key - (len - 1))
            const float base = slope * float(key0 - (len - 1));
#pragma unroll
            for (int ch = 0; ch < NC; ++ch)
#pragma unroll
              for (int k = 0; k < 32; ++k) x[ch][k] = fmaf(slope, float(ch * 32 + k), fmaf(x[ch][k], cc, base));
            cc = 1.f;
          }
          if (key0 + KT > keys_all) {  // the end of the prefix, or of a shorter sequence
            asm volatile("");          // (a branch in fact, not 128 selects for every tile)
#pragma unroll
            for (int ch = 0; ch < NC; ++ch)
#pragma unroll
              for (int k = 0; k < 32; ++k) x[ch][k] = ch * 32 + k <= last ? x[ch][k] : -INFINITY;
          }
          if (kFp8 || look) {
            asm volatile("");
            float h4[4] = {m4[0], m4[1], m4[2], m4[3]};
#pragma unroll
            for (int ch = 0; ch < NC; ++ch)
#pragma unroll
              for (int k = 0; k < 32; k += 2) h4[k / 2 & 3] = fmax3(h4[k / 2 & 3], x[ch][k], x[ch][k + 1]);
            const float mx = fmax3(fmaxf(h4[0], h4[1]), h4[2], h4[3]) * cc;
            // raise the maximum, and rescale what has been summed
            // (a row without a sequence decides nothing: where its query would be, shared memory holds anything)
            const bool grow = valid && (mx > m + (kFp8 || biased ? 8.f : 0.f) || (m == -INFINITY && mx > m));
            if (__any_sync(0xffffffffu, grow)) {
              const float m_new = fmaxf(m, mx);
              const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m - m_new);
              m = m_new;
              l *= alpha;
              if (j > first) {
                if (!wait(pv_done(wg), (n_pv - 1) & 1)) break;
                tc_fence_after();
#pragma unroll 1
                for (int ch = 0; ch < DP / 16; ++ch) {
                  float o[16];
                  tmem_ld16(t_o + ch * 16, o);
#pragma unroll
                  for (int k = 0; k < 16; ++k) o[k] *= alpha;
                  tmem_st16(t_o + ch * 16, o);
                }
                tmem_wait_st();
              }
            }
            if (!kFp8) unset = __any_sync(0xffffffffu, valid && m == -INFINITY);
          }
          nm = m == -INFINITY ? 0.f : -m;
          sa = sb = make_float2(0.f, 0.f);
#pragma unroll
          for (int ch = 0; ch < NC / 2; ++ch)
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              exps(ch, k);
              if (!kFp8) m4[k / 2 & 3] = fmax3(m4[k / 2 & 3], x[NC / 2 + ch][k], x[NC / 2 + ch][k + 1]);
            }
          const float mx = fmax3(fmaxf(m4[0], m4[1]), m4[2], m4[3]) * cc;
          const bool low = valid && ((sa.x + sa.y) + (sb.x + sb.y) > 4096.f || mx > m + 12.f);
          if (kFp8 || look || !__any_sync(0xffffffffu, low)) break;
        }
        if (!ok) break;
        // (P's columns lie over S columns: 16 a chunk of 32)
#pragma unroll
        for (int ch = 0; ch < NC; ++ch) {
          if (ch >= NC / 2) {
#pragma unroll
            for (int k = 0; k < 32; k += 2) exps(ch, k);
          }
          tmem_st16(t_s + ch * 16, w[ch]);
          if (ch == NC / 2 - 1 || ch == NC - 1) {
            tmem_wait_st();
            tc_fence_before();
            arrive(ch == NC - 1 ? p_full(wg) : p_half(wg));
          }
        }
        l += (sa.x + sa.y) + (sb.x + sb.y);
        ++n_pv;
      }
      if (!ok) break;
      // ---- this CTA's part of the row, not divided by its sum
      const bool any = it.e > first;
      unsigned char* part = p.parts + (size_t(it.item + int(blockIdx.x)) * (turns ? 2 : NQ) + wg) * shared_prefix_part_bytes(D);
      if (any) {
        if (!wait(pv_done(wg), (n_pv - 1) & 1)) break;
        tc_fence_after();
        constexpr int NCO = DP / 16, CH = NCO % 4 == 0 ? 4 : (NCO % 3 == 0 ? 3 : NCO);  // chunks read at a time
        static_assert(CH <= 7, "registers");
#pragma unroll 1
        for (int c0 = 0; c0 < NCO; c0 += CH) {
          float o[CH][16], keep[4] = {l, 0.f, 0.f, 0.f};
          float l2 = l;
          int dummy = 0;
#pragma unroll
          for (int k = 0; k < CH; ++k) tmem_ld16_start(t_o + (c0 + k) * 16, o[k]);
          tmem_landed(keep, l2, dummy);
          if (valid) {
            float4* dst = reinterpret_cast<float4*>(part) + c0 * 4 * 128 + row;
#pragma unroll
            for (int k = 0; k < CH; ++k)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (D % 16 == 0 || (c0 + k) * 16 + i * 4 < D)
                  dst[(k * 4 + i) * 128] = make_float4(o[k][4 * i], o[k][4 * i + 1], o[k][4 * i + 2], o[k][4 * i + 3]);
          }
        }
        tc_fence_before();  // (ordered before the next piece's p_half, which frees O)
      }
      if (valid) reinterpret_cast<float2*>(part + 128 * D * 4)[row] = make_float2(m, any ? l : 0.f);
    }
  } else if (warp < 12) {
    // ================================================= producers: K and V tiles into shared memory
    reg_dec<PrefillRegs<kFp8>::kProducer>();
    const int pt = tid - 256;  // 0 .. 127
    uint32_t n_half = 0;       // halves (K or V tiles) put on their way
    const char* kb = static_cast<const char*>(p.kc);
    const char* vb = static_cast<const char*>(p.vc);
    constexpr int ES = kFp8 ? 1 : 2;
    const int P = p.prefix_len;
    // K tiles of 16-bit caches are announced when their copies have landed, up to two later; before
    // the warp waits for anything, all of them are (the MMAs may be waiting for just those).
    uint32_t n_k = 0, n_told = 0;  // K tiles put on their way, announced
    auto announce = [&]() {
      fence_proxy_async();
      arrive(kv_full(2 * n_told % NS));
      ++n_told;
    };
    auto announce_all = [&]() {
      if (n_k - n_told >= 2) {
        cp_async_wait<1>();
        while (n_k - n_told > 1) announce();
      }
      if (n_k != n_told) {
        cp_async_wait<0>();
        announce();
      }
    };
    auto wait_slot = [&](uint32_t h) -> bool {
      const uint32_t use = h / NS;  // times the slot has been filled before
      if (use == 0) return true;
      if constexpr (!kFp8) {
        if (!__all_sync(0xffffffffu, mbar_test(kv_empty(h % NS), (use - 1) & 1))) announce_all();
      }
      return wait(kv_empty(h % NS), (use - 1) & 1);
    };
    auto slot_of = [&](uint32_t h) { return skv + (h % NS) * SH::kTileBytes; };
    while (ok && next(it)) {
      const int64_t head_off = int64_t(it.kvh) * p.kv_head_stride * ES;
      auto block_of = [&](int key) { return key < P ? __ldcg(p.blocks + (key >> b_shift)) : 0; };
      auto page = [&](const char* base, int blk) {
        return base + int64_t(blk) * p.kv_block_stride * ES + head_off;
      };
      if constexpr (!kFp8) {
        // K: a thread owns one key and walks along its 16-byte granules.  V: pages of 16 keys, each one copy by
        // tensor map, issued by the first warp; the prefix ends with a page.
        constexpr int NP = KT / 16;  // pages per tile
        const int kt = pt % KT, kg = pt / KT;
        int k_blk = block_of(it.b * KT + kt), v_blk = block_of(it.b * KT + lane % NP * 16);
        for (int j = it.b; j < it.e && ok; ++j) {
          {
            const int key = j * KT + kt;
            const char* src = page(kb, k_blk) + (kg * B + (key & (B - 1))) * 16;
            const int bytes = key < P ? 16 : 0;
            if (j + 1 < it.e) k_blk = block_of(key + KT);
            if (!wait_slot(n_half)) break;
            uint32_t dst = slot_of(n_half) + (kg * KT + kt) * 16;
#pragma unroll 4
            for (int g = kg; g < D / 8; g += 128 / KT) {
              cp_async16(dst, src, bytes);
              dst += 128 * 16;
              src += (128 / KT) * B * 16;
            }
            cp_async_commit();
            ++n_half;
            ++n_k;
            if (n_k - n_told > 1) {
              cp_async_wait<1>();
              announce();
            }
          }
          const int key = j * KT + lane % NP * 16;
          const int cur = v_blk;
          if (j + 1 < it.e) v_blk = block_of(key + KT);
          if (!wait_slot(n_half)) break;
          const int pages = min(NP, (P - j * KT + 15) / 16);
          const uint32_t full = kv_full(n_half % NS);
          if (warp != 8) {
            arrive(full);
          } else {
            if (lane == 0) mbar_expect_tx(full, pages * D * 32);
            __syncwarp();
            if (lane < pages) tma_load4(slot_of(n_half) + lane * DP * 32, &vmap, key & (B - 1), 0, it.kvh, cur, full);
            __syncwarp();
          }
          ++n_half;
        }
      } else {
        // fp8: 16-byte loads into registers (the next half is always in flight), widened to two
        // 16-byte granules of f16.  K: a thread owns one key; V: 16 keys and every 16th dimension.
        const int kt = pt % KT, kg = pt / KT;
        constexpr int KN = (D / 16 + 128 / KT - 1) / (128 / KT);
        constexpr int VJ = KT / 16;
        constexpr int VDS = 128 / VJ;           // threads that share a 16-key group
        const int vj = pt / VDS, vd = pt % VDS;
        constexpr int VN = (D + VDS - 1) / VDS;
        uint4 kr[KN], vr[VN];
        auto get_k = [&](int j) {
          const int key = j * KT + kt;
          const char* src = page(kb, block_of(key)) + (key & (B - 1)) * 16;
#pragma unroll
          for (int i = 0; i < KN; ++i) {
            const int g = kg + i * (128 / KT);
            if (key < P && g < D / 16) kr[i] = __ldcg(reinterpret_cast<const uint4*>(src + int64_t(g) * B * 16));
            else kr[i] = make_uint4(0, 0, 0, 0);
          }
        };
        auto get_v = [&](int j) {
          const int key = j * KT + vj * 16;
          const char* src = page(vb, block_of(key)) + (key & (B - 1));
#pragma unroll
          for (int i = 0; i < VN; ++i) {
            const int d = vd + i * VDS;
            if (key < P && d < D) vr[i] = __ldcg(reinterpret_cast<const uint4*>(src + int64_t(d) * B));
            else vr[i] = make_uint4(0, 0, 0, 0);
          }
        };
        auto widen = [&](const uint4& x, uint4& lo, uint4& hi) {
          fp8x4_to_f16<kE5>(x.x, lo.x, lo.y);
          fp8x4_to_f16<kE5>(x.y, lo.z, lo.w);
          fp8x4_to_f16<kE5>(x.z, hi.x, hi.y);
          fp8x4_to_f16<kE5>(x.w, hi.z, hi.w);
        };
        get_k(it.b);
        get_v(it.b);
        for (int j = it.b; j < it.e && ok; ++j) {
          if (!wait_slot(n_half)) break;
          {
            const uint32_t dst = slot_of(n_half) + kt * 16;
#pragma unroll
            for (int i = 0; i < KN; ++i) {
              const int g = kg + i * (128 / KT);
              if (D / 16 % (128 / KT) == 0 || g < D / 16) {
                uint4 lo, hi;
                widen(kr[i], lo, hi);
                st_shared16(dst + (2 * g) * KT * 16, lo);
                st_shared16(dst + (2 * g + 1) * KT * 16, hi);
              }
            }
            fence_proxy_async();
            arrive(kv_full(n_half % NS));
            ++n_half;
            if (j + 1 < it.e) get_k(j + 1);
          }
          if (!wait_slot(n_half)) break;
          {
            const uint32_t dst = slot_of(n_half) + 2 * vj * DP * 16;
#pragma unroll
            for (int i = 0; i < VN; ++i) {
              const int d = vd + i * VDS;
              if (D % VDS == 0 || d < D) {
                uint4 lo, hi;
                widen(vr[i], lo, hi);
                st_shared16(dst + d * 16, lo);
                st_shared16(dst + (DP + d) * 16, hi);
              }
            }
            fence_proxy_async();
            arrive(kv_full(n_half % NS));
            ++n_half;
            if (j + 1 < it.e) get_v(j + 1);
          }
        }
      }
      if (!ok) break;
      if constexpr (!kFp8) announce_all();
    }
    if constexpr (!kFp8) {  // nobody leaves with copies on their way (after a wait that ran out, too)
      cp_async_wait_all();
      if (warp == 8)
        for (uint32_t h = n_half < NS ? 0 : n_half - NS; h < n_half; ++h) mbar_spin(kv_full(h % NS), (h / NS) & 1);
    }
  } else {
    reg_dec<PrefillRegs<kFp8>::kMma>();
    if (warp == 12) {
    // ================================================= the MMA warp (all lanes run along, one elected issues: see
    // prefill_kernel.cuh)
    const uint32_t idesc_s = mma_idesc(kBf, 128, KT);
    const uint32_t idesc_o = mma_idesc(kBf, 128, DP);
    uint32_t n_h = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};  // halves, Q tiles, P tiles
    auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
    auto commit = [&](uint32_t bar) {
      if (elect_one()) mma_commit(bar);
      __syncwarp();
    };
    const uint64_t q_desc = SH::kQBox == 64 ? smem_desc_sw128(sq) : smem_desc_sw32(sq, 256);
    auto q_step = [](int ks) {  // where K step ks lies, in 16-byte units
      return SH::kQBox == 64 ? ks / 4 * (128 * 128 / 16) + ks % 4 * 2 : ks * (128 * 32 / 16);
    };
    const uint64_t k_desc = smem_desc(skv, KT * 16, 128);
    const uint64_t v_desc = kFp8 ? smem_desc(skv, DP * 16, 128) : smem_desc_sw32(skv, 256);
    auto wait_half = [&](uint32_t h) { return wait(kv_full(h % NS), (h / NS) & 1); };
    // S of warpgroup i from Q tile qt and the K tile in half h
    auto qk = [&](int i, int qt, uint32_t h) {
      const uint64_t kd = k_desc + uniform((h % NS) * (SH::kTileBytes >> 4));
      const uint64_t qd = q_desc + qt * (SH::kQBytes >> 4);
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
          mma_ss(tmem + i * KT, qd + q_step(ks), kd + ks * 2 * KT, idesc_s, ks > 0);
        mma_commit(s_full(i));
      }
      __syncwarp();
    };
    // half of the keys of a tile (`steps`: pages of 16 keys that the tile has)
    auto pv = [&](int i, uint32_t h, int half, int steps, bool more) {
      const uint64_t vd = v_desc + uniform((h % NS) * (SH::kTileBytes >> 4));
      if (elect_one()) {
        constexpr int NK = KT / 32;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          const int ks = half * NK + k;
          if (kFp8 || ks < steps)
            mma_ts(tmem + NQ * KT + i * DP, tmem + i * KT + ks * 8, vd + ks * 2 * DP, idesc_o, more || ks > 0);
        }
        if (half == 1) mma_commit(pv_done(i));
      }
      __syncwarp();
    };
    // O of warpgroup i and the V tile j in half h
    auto pv_both = [&](int i, uint32_t h, int j, bool more) -> bool {
      const int steps = int(uniform((p.prefix_len - j * KT + 15) / 16));
      if (!wait(p_half(i), n_p[i] & 1)) return false;
      tc_fence_after();
      pv(i, h, 0, steps, more);
      if (!wait(p_full(i), n_p[i] & 1)) return false;
      ++n_p[i];
      tc_fence_after();
      pv(i, h, 1, steps, true);
      return true;
    };
    while (ok && next(it)) {
      const int b = int(uniform(it.b)), e = int(uniform(it.e));
      if (NQ == 2 && turns) {
        // halves n_h + 2 k, n_h + 2 k + 1: K and V of tile b + k, which belong to warpgroup k & 1
        const int n = e - b;
        if (!wait(q_full(0), n_q[0]++ & 1)) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!ok || i >= n) continue;
          if (!wait_half(n_h + 2 * i)) continue;
          tc_fence_after();
          qk(i, 0, n_h + 2 * i);
          commit(kv_empty((n_h + 2 * i) % NS));
        }
        if (!ok) break;
        if (n <= 2) commit(q_empty(0));
        for (int k0 = 0; k0 < n && ok; k0 += 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = k0 + i;
            if (!ok || k >= n) continue;
            if (!wait_half(n_h + 2 * k + 1)) continue;
            if (!pv_both(i, n_h + 2 * k + 1, b + k, k0 > 0)) continue;
            commit(kv_empty((n_h + 2 * k + 1) % NS));
            if (k + 2 < n) {
              if (!wait_half(n_h + 2 * k + 4)) continue;
              tc_fence_after();
              qk(i, 0, n_h + 2 * k + 4);
              commit(kv_empty((n_h + 2 * k + 4) % NS));
              if (k + 3 == n) commit(q_empty(0));
            }
          }
        }
        if (!ok) break;
        n_h += 2 * n;
        continue;
      }
      bool on[2] = {true, false};
      if constexpr (NQ == 2) on[1] = int(uniform(has(it, 1))) != 0;
      if (!wait_half(n_h)) break;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (!on[i] || !ok) continue;
        if (!wait(q_full(i), n_q[i]++ & 1)) continue;
        tc_fence_after();
        qk(i, i, n_h);
        if (b + 1 == e) commit(q_empty(i));
      }
      if (!ok) break;
      commit(kv_empty(n_h % NS));
      ++n_h;
      for (int j = b; j < e; ++j) {
        // V tile j is half n_h, K tile j + 1 half n_h + 1
        if (!wait_half(n_h)) break;
        bool have_k = false;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          if (!ok || !on[i]) continue;
          if (!pv_both(i, n_h, j, j > b)) continue;
          if (j + 1 < e) {
            if (!have_k && !wait_half(n_h + 1)) continue;
            have_k = true;
            qk(i, i, n_h + 1);
            if (j + 2 == e) commit(q_empty(i));
          }
        }
        if (!ok) break;
        commit(kv_empty(n_h % NS));
        ++n_h;
        if (have_k) {
          commit(kv_empty(n_h % NS));
          ++n_h;
        }
      }
      if (!ok) break;
    }
    } else if (warp >= 14) {
    // ================================================= Q into shared memory (warp 14): a tile's sequences and heads are
    // a box of a tensor map.  bf16 becomes f16 in place for an fp8 cache, half a tile by each of warps 14 and 15.
    uint32_t n_q[2] = {0, 0};
    while (ok && (kWiden || warp == 14) && next(it)) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (!ok || (turns ? i > 0 : !has(it, i))) continue;
        const uint32_t land = kWiden ? q_land(i) : q_full(i);
        // (in front of warp 15's first conversion of this tile, too: it follows the landing)
        if (warp == 14) {
          if (n_q[i] > 0 && !wait(q_empty(i), (n_q[i] - 1) & 1)) continue;
          constexpr int NB = DP / SH::kQBox;
          if (lane == 0) {
            mbar_expect_tx(land, NB * SH::kQBox * 2 * T * G);
#pragma unroll
            for (int x = 0; x < NB; ++x)
              tma_load3(sq + i * SH::kQBytes + x * 128 * SH::kQBox * 2, &qmap, x * SH::kQBox, it.kvh * G,
                        (it.tile0 + i) * T, land);
          }
          __syncwarp();
        }
        if constexpr (kWiden) {
          if (!wait(land, n_q[i] & 1)) continue;
          const uint32_t at = sq + i * SH::kQBytes + (warp - 14) * (SH::kQBytes / 2) + lane * 16;
#pragma unroll 4
          for (int o = 0; o < SH::kQBytes / 2; o += 512) {
            const uint4 v = ld_shared16(at + o);
            auto f16 = [](uint32_t w) { return pack2<false>(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); };
            st_shared16(at + o, make_uint4(f16(v.x), f16(v.y), f16(v.z), f16(v.w)));
          }
          fence_proxy_async();
          arrive(q_full(i));
        }
        ++n_q[i];
      }
    }
    if (warp == 14) {  // nobody leaves with copies on their way
#pragma unroll
      for (int i = 0; i < NQ; ++i)
        if (n_q[i] > 0) mbar_spin(kWiden ? q_land(i) : q_full(i), (n_q[i] - 1) & 1);
    }
    }
  }
  // ---- everything issued has been waited for by the softmax warpgroups (or a wait ran out)
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The sum of all parts of a sequence: grid.x = items, a thread to four dimensions of a head, or several, which share the
// parts between them (few sequences behind a long prefix have over a hundred).  A chain of two trips (places, parts) and a
// start, which the launch in front lets it have early: with that, 32-bit indexes ahead of its wait and blocks no larger
// than an item, 256 sequences of 32 heads of 128 behind 4096 tokens take 105 us, 109 without, in all.
constexpr int kCombineThreads = 256;

struct CombineParams {
  void* out;
  const float* v_scale;  // nullptr: 1
  float* lse;
  const int* cut;
  SharedPrefixParts pre;
  int num_seqs, num_heads, group, head_groups, heads, D;  // heads: of an item
  int share;                                              // threads to a unit
  int ranges;                                             // most that the persistent kernel can have had
};

template <typename QT>
__global__ void __launch_bounds__(kCombineThreads) shared_prefix_combine_kernel(const CombineParams p) {
  constexpr bool kBf = std::is_same_v<QT, __nv_bfloat16>;
  __shared__ float4 s_acc[kCombineThreads];
  __shared__ float2 s_ml[kCombineThreads];
  const unsigned tid = threadIdx.x, D = p.D, HPI = p.heads, item = blockIdx.x;
  const unsigned sub = item / unsigned(p.num_seqs), seq = item - sub * unsigned(p.num_seqs);
  const unsigned kvh = sub / unsigned(p.head_groups), hg = sub - kvh * unsigned(p.head_groups);
  const unsigned nheads = min(HPI, p.group - hg * HPI), units = nheads * (D / 4);
  const unsigned share = p.share, lanes = blockDim.x / share;
  const unsigned z = tid / lanes, u = blockIdx.y * lanes + tid - z * lanes;
  const bool on = u < units;
  const unsigned d4 = on ? u / nheads : 0, hl = on ? u - d4 * nheads : 0;
  // (SharedPrefixParts::row, with the cut that the prefix's kernel has chosen)
  const unsigned tile = seq / unsigned(p.pre.tokens), grp = p.pre.turns ? tile : tile / unsigned(p.pre.tiles);
  const unsigned it = kvh * unsigned(p.pre.groups) + grp, u0 = it * unsigned(p.pre.key_tiles);
  const int row = int(seq - tile * p.pre.tokens) * p.group + hg * HPI;
  const unsigned room = min(HPI, unsigned(p.group));
  const int64_t own_slot = own_part_bytes(room, D), part = 128 * (D * 4 + 8);
  grid_dependency();
  const unsigned cut = __ldcg(p.cut);
  int2 found = __ldcg(p.pre.found + item);
  const float v_scale = p.v_scale ? __ldcg(p.v_scale) : 1.f;
  // (in bounds whatever is there: a wait of the launch in front that ran out leaves items out)
  found.x = min(max(found.x, 0), p.ranges - 1);
  found.y = min(max(found.y, 0), p.ranges - found.x);
  const unsigned char* own = p.pre.own + (int64_t(item) + found.x) * own_slot;
  const unsigned c0 = u0 / cut, c1 = (u0 + p.pre.key_tiles - 1) / cut;
  const unsigned char* first =
      p.pre.parts + (int64_t(it + c0) * p.pre.tiles + (p.pre.turns ? 0 : tile - grp * p.pre.tiles)) * part;
  const int64_t step = p.pre.turns ? part : p.pre.tiles * part;
  const int np = found.y, n = np + int(c1 - c0 + 1) * (p.pre.turns ? 2 : 1);

  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = int(z); k0 < n && on; k0 += 4 * share) {
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = min(k0 + k * share, n - 1);
      const unsigned char* q = s < np ? own + s * own_slot : first + (s - np) * step;
      ml[k] = __ldcg(reinterpret_cast<const float2*>(s < np ? q + room * D * 4 + hl * 8 : q + 128 * D * 4 + (row + hl) * 8));
      v[k] = __ldcg(reinterpret_cast<const float4*>(s < np ? q + (d4 * room + hl) * 16 : q + (d4 * 128 + row + hl) * 16));
      if (k0 + k * share >= n) ml[k] = make_float2(-INFINITY, 0.f);
    }
    float m_new = m;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (ml[k].y != 0.f) m_new = fmaxf(m_new, ml[k].x);
    const float old = m_new == -INFINITY ? 0.f : fast_exp2(m - m_new);
    l *= old;
    acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
    m = m_new;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (ml[k].y != 0.f) {  // (what has no key has written no output)
        const float f = fast_exp2(ml[k].x - m);
        l += ml[k].y * f;
        acc.x += f * v[k].x;
        acc.y += f * v[k].y;
        acc.z += f * v[k].z;
        acc.w += f * v[k].w;
      }
    }
  }
  if (share > 1) {
    s_acc[tid] = acc;
    s_ml[tid] = make_float2(m, l);
    __syncthreads();
    if (z > 0 || !on) return;
    for (unsigned k = 1; k < share; ++k) {
      const float2 ml = s_ml[tid + k * lanes];
      if (ml.y == 0.f) continue;
      const float4 v = s_acc[tid + k * lanes];
      const float m_new = fmaxf(m, ml.x);
      const float old = m_new == -INFINITY ? 0.f : fast_exp2(m - m_new), f = fast_exp2(ml.x - m_new);
      l = l * old + ml.y * f;
      acc = make_float4(acc.x * old + v.x * f, acc.y * old + v.y * f, acc.z * old + v.z * f, acc.w * old + v.w * f);
      m = m_new;
    }
  }
  if (!on) return;
  const float inv = v_scale * __fdividef(1.f, l + 1e-6f);
  const int head = kvh * p.group + hg * HPI + hl;
  uint2 w;
  w.x = pack2<kBf>(acc.x * inv, acc.y * inv);
  w.y = pack2<kBf>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(static_cast<QT*>(p.out) + (int64_t(seq) * p.num_heads + head) * D + d4 * 4) = w;
  if (p.lse != nullptr && d4 == 0)
    p.lse[int64_t(head) * p.num_seqs + seq] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace b200pa

// Host entry of decode attention over a prefix that all sequences of the batch share.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "launch_state.cuh"
#include "shared_prefix_inst.cuh"
#include "tails_inst.cuh"
#include "tensor_map.cuh"

namespace b200pa {

struct SharedPrefixPlan {
  SharedPrefixKernels k;  // k.prefix null: the ordinary kernels
  int row_tiles = 0, groups = 0, key_tiles = 0, cut = 0, turns = 0, tiles = 0, grid = 0;
  // behind the prefix: the persistent kernel beside it and a third that adds up, where tails.fn is not null; else the
  // direct one in clusters, or a warp to an item
  TailsKernelInfo tails{nullptr, 0, 1};
  int warps = 0, slots = 0, min_chunk = 0;
  size_t smem = 0;
  int cluster = 1;  // 0: every warp an item of its own
  int heads = 0;                                // query heads of an item of the persistent kernel
  int64_t items = 0;                            // (sequence, kv head, head group)
  SharedPrefixBalance balance{};
  int64_t own_at = 0, found_at = 0, bytes = 0;  // scratch: the prefix's parts, partials, their places; its size
};

static TailsKernelInfo find_tails(int d, int qdt, int kv, int gp, int nt) {
  switch (d) {
    case 32: return find_tails_d32(qdt, kv, gp, nt);
    case 64: return find_tails_d64(qdt, kv, gp, nt);
    case 80: return find_tails_d80(qdt, kv, gp, nt);
    case 96: return find_tails_d96(qdt, kv, gp, nt);
    case 112: return find_tails_d112(qdt, kv, gp, nt);
    case 128: return find_tails_d128(qdt, kv, gp, nt);
    case 192: return find_tails_d192(qdt, kv, gp, nt);
    case 256: return find_tails_d256(qdt, kv, gp, nt);
  }
  return {nullptr, 0, 1};
}

// The persistent kernel's launch, as in attention_entry: two ring slots a warp, as many warps as shared memory and
// registers have room for (16-bit caches: 12).  False where the table of the sequences does not fit.
static bool plan_tails(const b200pa_attn_args& a, int gp, SharedPrefixPlan& r) {
  const int es = a.kv_dtype == B200PA_KV_AUTO ? 2 : 1;
  const TailsKernelInfo ki = find_tails(a.head_size, a.q_dtype, a.kv_dtype, gp, a.block_size / 16);
  const size_t table = size_t((a.num_seqs + 1 + 3) & ~3) * 4;
  if (ki.fn == nullptr || table > 48 * 1024) return false;
  const size_t step = size_t(a.head_size) * a.block_size * es * ki.pages_per_step;
  const int split = step >= 4096 ? 1 : 0;
  const size_t slot = split ? step : 2 * step;
  const size_t budget = 227 * 1024 - 2048 - table - 1024;
  int w = int(std::min<size_t>(size_t(ki.max_warps), budget / (2 * slot)));
  if (es == 2 && w > 12) w = 12;
  if (w >= 8) w &= ~3;
  if (w < 1) return false;
  r.slots = 2;
  const Tuning tune = tuning();
  if (tune.warps) w = std::min(w, tune.warps);
  if (tune.stages) r.slots = std::max(split ? 2 : 1, std::min(int(budget / (size_t(w) * slot)), tune.stages));
  r.tails = ki;
  r.warps = w;
  r.min_chunk = std::max(2, (64 / a.block_size + 1) & ~1);
  r.smem = table + ((size_t(w) * r.slots * 8 + 127) & ~size_t(127)) + size_t(w) * r.slots * slot;
  return true;
}

// Pieces that the persistent kernel cuts a sequence into, at most: the third launch adds them up four at a time, a trip to
// memory each.  One sequence of 30000 own tokens among 256 behind 1024 tokens, 8 / 1 heads of 128: without a bound (469
// pieces of 64 tokens) 74 us, 256 pieces 55, 128 58, 64 81 (the warps with them are last then); 32 / 8 heads 81 with 96
// and more.
constexpr int kMostPieces = 256;

static SharedPrefixKernels find_shared_prefix(const b200pa_attn_args& a) {
  const int es = a.kv_dtype == B200PA_KV_AUTO ? 2 : 1;
  auto al = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
  // (what the two kernels need: 16-byte accesses; strides that a tensor map holds)
  const bool fits = (a.block_size == 16 || a.block_size == 32) && a.num_heads / a.num_kv_heads <= 128 && al(a.key_cache) &&
                    al(a.value_cache) && al(a.query) && al(a.out) && (a.kv_block_stride * es) % 16 == 0 &&
                    (a.kv_head_stride * es) % 16 == 0 &&
                    (es == 1 || (tensor_map_stride(a.kv_block_stride) && tensor_map_stride(a.kv_head_stride))) &&
                    a.q_stride % 8 == 0 && tensor_map_stride(a.q_stride) && a.blocksparse_vert_stride <= 1;
  if (!fits) return {};
  const int group = a.num_heads / a.num_kv_heads;
  return a.head_size <= 80    ? find_shared_prefix_small(a.head_size, a.q_dtype, a.kv_dtype, group)
         : a.head_size <= 112 ? find_shared_prefix_mid(a.head_size, a.q_dtype, a.kv_dtype, group)
         : a.head_size <= 128 ? find_shared_prefix_128(a.head_size, a.q_dtype, a.kv_dtype, group)
                              : find_shared_prefix_large(a.head_size, a.q_dtype, a.kv_dtype, group);
}

// What the prefix's kernel takes for a key tile of an item, ns of an SM: two row tiles in turns on the tensor cores, or
// one by itself (measured: 128 fp8 sequences, 64 / 8 heads of 128, behind 8192 2.3 us; 8 sequences behind 65008 1.55;
// head sizes 64 and 256 2.0 and 1.8), or its K and V on the way.
static int64_t unit_ns(int head_size, int row_tiles, int turns, bool biased, bool fp8, int64_t tile_bytes) {
  int64_t work = row_tiles == 1 ? 1800 : turns ? 1000 + 4 * head_size : 1500 + 8 * std::min(head_size, 128);
  if (biased) work = work * 3 / 2;
  else if (fp8 && !turns) work = work * 41 / 50;
  return std::max(work, tile_bytes * 1000 / 60000);
}

// ... and for a piece of an item beside its key tiles: a pipeline that fills and drains, queries in, a part out.  (A prefix
// of 96 tokens is one key tile: without this its CTAs were last.  1029 sequences behind 96, 8 / 2 heads of 128, 115 -> 95
// us; 430 behind 96, 28 / 4 heads of 256, 246 -> 162; 256 behind 256, 32 / 8 heads of 128, 131 -> 97.)
static int64_t piece_ns(int head_size, int turns) { return turns ? 0 : 2500 + 14 * head_size; }

// Which way a call goes: 0 the ordinary kernels on whole sequences; behind the prefix the direct kernel (1), the same
// with a warp to an item (2), or the persistent one beside the prefix and a third launch (3).  What each takes, us:
// fitted to 410 random batches (2 to 2000 sequences, prefixes of 64 to 65000 tokens, up to 3000 own ones, all head sizes,
// cache types and ten head counts; own lengths are taken as half the bound).  Over these and 500 others the choice is
// 3.3 % from the best of the four on average, more than 25 % in 35 of the 910.  The ordinary kernels are given 5 %: that
// costs nothing on average, and 32 of the 910 are over 10 % slower than them, not 48.
//   prefix_all: the prefix's work over all SMs; prefix_cut: of its longest CTA
static int shared_prefix_way(const b200pa_attn_args& a, int prefix_len, const SharedPrefixPlan& r, double prefix_all,
                             double prefix_cut, bool tails) {
  const int group = a.num_heads / a.num_kv_heads, es = a.kv_dtype == B200PA_KV_AUTO ? 2 : 1, sms = sm_count();
  const double D = a.head_size, N = a.num_seqs, us = 1 / 6.5e6;  // (bytes to us at HBM's rate)
  const double own = std::max(a.max_seq_len - prefix_len, 1), tiles = own / 16 + 0.5;
  const double row = a.num_kv_heads * D * 2 * es, hbm = N * own / 2 * row * us;
  const double latency = (es == 1 ? 0.63 + 0.0037 * D : 0.43 + 0.0061 * D) * (group > 8 ? 1.4 : 1);  // of a tile
  const double prefix = 6.5 + prefix_cut, places = 3.0 * sms, warps = r.cluster * kDirectWarps, items = double(r.items);
  const double waves = std::max(1.0, items * r.cluster / places), solo_waves = std::max(1.0, items / places / kDirectWarps);
  // trips to the prefix's parts, of which a row of few sequences has over a hundred
  const double parts = (double(r.key_tiles) / r.cut + 1) * (r.turns ? 2 : 1);
  const double rounds = std::ceil(parts / (4 * r.cluster)) * std::ceil(std::min(group, 16) * D / 4 / 128);
  double t[4];
  t[0] = 14.2 + std::max(N * (prefix_len + own / 2) * row * us, 1.13 * (prefix_len + own / 2) / 1024 * latency) +
         (group > 8 && D > 128 ? 30 : 0);  // (two head tiles of a wide head: the persistent kernel only)
  t[1] = prefix + 6 + std::max({2.9 * hbm, 0.75 * tiles / warps * latency,
                                waves * (4 + 1.2 * std::max(own / 32 / warps, 0.5) * latency)}) +
         0.43 * std::max(rounds - 4, 0.0);
  t[2] = prefix + 5 + std::max({1.2 * hbm, 0.95 * tiles * latency, solo_waves * (5.6 + 0.8 * std::max(own / 32, 1.0) * latency)}) +
         0.43 * std::max(parts - 8, 0.0);
  const double tail_items = N * a.num_kv_heads * ((group + (group <= 8 ? 7 : 15)) / (group <= 8 ? 8 : 16));
  const double beside = (N * own / 2 * row / 65e3 + tail_items * 0.5) / sms;
  t[3] = tails ? 25 + std::max(prefix_all + beside, hbm) + 0.6e-6 * N * a.num_heads * D * 4 : 1e30;
  t[0] *= 0.95;
  return int(std::min_element(t, t + 4) - t);
}

static SharedPrefixPlan shared_prefix_plan(const b200pa_attn_args& a, int prefix_len) {
  SharedPrefixPlan r;
  if (a.num_seqs < 2 || prefix_len == 0) return r;
  const SharedPrefixKernels k = find_shared_prefix(a);
  if (k.prefix == nullptr) return r;
  const Tuning tune = tuning();
  const int sms = sm_count(), group = a.num_heads / a.num_kv_heads, T = 128 / group;
  r.row_tiles = (a.num_seqs + T - 1) / T;
  r.turns = k.row_tiles == 2 && r.row_tiles == 1;
  const int per = r.turns ? 1 : k.row_tiles;
  r.groups = (r.row_tiles + per - 1) / per;
  r.tiles = r.turns ? 2 : k.row_tiles;
  r.key_tiles = (prefix_len + k.keys - 1) / k.keys;
  const int64_t items = int64_t(a.num_kv_heads) * r.groups, units = items * r.key_tiles;
  if (units > INT32_MAX / 2) return r;
  r.cut = int((units + sms - 1) / sms);
  r.grid = int((units + r.cut - 1) / r.cut);
  const int es = a.kv_dtype == B200PA_KV_AUTO ? 2 : 1;
  auto up = [](int64_t v) { return (v + 255) & ~int64_t(255); };

  // ---- behind the prefix
  const int gp = group <= 8 ? 1 : 2, heads = 8 * gp;
  const int64_t tail_items = int64_t(a.num_seqs) * a.num_kv_heads * ((group + heads - 1) / heads);
  r.items = int64_t(a.num_seqs) * a.num_kv_heads * ((group + k.heads - 1) / k.heads);
  if (r.items > INT32_MAX / 16) return {};
  const int64_t unit = unit_ns(a.head_size, k.row_tiles, r.turns, a.alibi_slopes != nullptr, es == 1,
                               int64_t(k.keys) * a.head_size * 2 * es);
  const int64_t places = int64_t(sms) * k.ctas_per_sm;
  const int64_t own_tiles = (int64_t(std::max(a.max_seq_len - prefix_len, 1)) + 15) / 16;
  // CTAs of a sequence and head: as many as the GPU takes at once, but no more warps than there are 16-token tiles
  while (r.cluster < 8 && r.items * r.cluster * 10 <= places * 6 && r.cluster * kDirectWarps < own_tiles) r.cluster *= 2;
  if (tune.cluster) r.cluster = tune.cluster;
  const bool tails = tail_items <= INT32_MAX / 16 && sms >= 16 && plan_tails(a, gp, r);
  const int way = tune.behind ? tune.behind : shared_prefix_way(a, prefix_len, r, units * unit * 1e-3 / sms, r.cut * unit * 1e-3, tails);
  if (way == 0) return {};
  if (way != 3) r.tails.fn = nullptr;
  if (way == 2) r.cluster = 0;
  r.bytes = up((items + r.grid) * r.tiles * int64_t(k.part_bytes));
  if (r.tails.fn != nullptr) {
    r.items = tail_items;
    r.heads = heads;
    const int64_t slot = own_part_bytes(std::min(heads, group), a.head_size), ranges = int64_t(sms) * r.warps;
    r.own_at = up((items + sms) * r.tiles * int64_t(k.part_bytes));
    r.found_at = r.own_at + up((tail_items + ranges) * slot);
    r.bytes = r.found_at + up(tail_items * 8) + 256;
    r.grid = sms;
    const int64_t page = int64_t(a.head_size) * a.block_size * es * 2;  // bytes of a block and kv head
    r.balance.sms = sms;
    r.balance.prefix = units * unit + items * piece_ns(a.head_size, r.turns);
    r.balance.items = tail_items * 500;
    if (tune.prefix) r.balance.prefix = r.balance.prefix * tune.prefix / 100;
    r.balance.block = page * 1000 / 65000;
    r.balance.block_hbm = page * 1000 / 6500;
    r.balance.prefix_start = 8000;
    r.balance.behind_start = 14000;
  }
  r.k = k;
  return r;
}

static int check_shared_prefix(const b200pa_attn_args* a, int32_t prefix_len) {
  if (const int bad = attention_check(a, false); bad != B200PA_OK) return bad;
  B200PA_CHECK_ARG(prefix_len >= 0 && prefix_len % a->block_size == 0,
                   "prefix_len %d has to be a multiple of the block size %d", prefix_len, a->block_size);
  B200PA_CHECK_ARG(a->num_seqs == 0 || prefix_len / a->block_size <= a->max_num_blocks_per_seq,
                   "prefix_len %d does not fit block tables of %d blocks", prefix_len, a->max_num_blocks_per_seq);
  B200PA_CHECK_ARG(a->blocksparse_vert_stride <= 1, "a shared prefix and block-sparse attention do not go together");
  return B200PA_OK;
}

// A dimension of size 1 may come with any stride.
static b200pa_attn_args with_plain_strides(b200pa_attn_args a) {
  if (a.num_kv_heads == 1) a.kv_head_stride = int64_t(a.head_size) * a.block_size;
  if (a.num_seqs == 1) a.q_stride = int64_t(a.num_heads) * a.head_size;
  return a;
}

}  // namespace b200pa

extern "C" int b200pa_shared_prefix_route(const b200pa_attn_args* args, int32_t prefix_len, int32_t* way) {
  using namespace b200pa;
  B200PA_CHECK_ARG(way != nullptr, "way is NULL");
  if (const int bad = check_shared_prefix(args, prefix_len); bad != B200PA_OK) return bad;
  const SharedPrefixPlan plan = args->num_seqs > 0 ? shared_prefix_plan(with_plain_strides(*args), prefix_len) : SharedPrefixPlan{};
  *way = plan.k.prefix == nullptr ? 0 : plan.tails.fn != nullptr ? 3 : plan.cluster == 0 ? 2 : 1;
  return B200PA_OK;
}

extern "C" int64_t b200pa_shared_prefix_scratch_bytes(const b200pa_attn_args* args, int32_t prefix_len) {
  using namespace b200pa;
  if (const int bad = check_shared_prefix(args, prefix_len); bad != B200PA_OK) return bad;
  if (args->num_seqs == 0) return 0;
  return shared_prefix_plan(with_plain_strides(*args), prefix_len).bytes;
}

extern "C" int b200pa_paged_attention_shared_prefix(const b200pa_attn_args* args, int32_t prefix_len, void* scratch,
                                                    int64_t scratch_bytes, void* stream) {
  using namespace b200pa;
  if (const int bad = check_shared_prefix(args, prefix_len); bad != B200PA_OK || args->num_seqs == 0) return bad;
  const b200pa_attn_args plain = with_plain_strides(*args), *a = &plain;
  const SharedPrefixPlan plan = shared_prefix_plan(*a, prefix_len);
  if (plan.k.prefix == nullptr) return b200pa_paged_attention_v1(a, stream);
  B200PA_CHECK_ARG(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0 && scratch_bytes >= plan.bytes,
                   "a shared prefix needs %lld bytes of scratch on a 16-byte boundary, got %lld", (long long)plan.bytes,
                   (long long)scratch_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  SharedPrefixParams p{};
  p.q = a->query;
  p.kc = a->key_cache;
  p.vc = a->value_cache;
  p.blocks = a->block_tables;
  p.seq_lens = a->seq_lens;
  p.alibi = a->alibi_slopes;
  p.k_scale = a->k_scale;
  p.parts = static_cast<unsigned char*>(scratch);
  p.status = device_status_ptr();
  if (p.status == nullptr) {
    set_error("could not resolve the device-side status word");
    return B200PA_ECUDA;
  }
  p.q_stride = a->q_stride;
  p.kv_block_stride = a->kv_block_stride;
  p.kv_head_stride = a->kv_head_stride;
  p.num_seqs = a->num_seqs;
  p.num_kv_heads = a->num_kv_heads;
  p.group = a->num_heads / a->num_kv_heads;
  p.block_size = a->block_size;
  p.prefix_len = prefix_len;
  p.row_tiles = plan.row_tiles;
  p.groups = plan.groups;
  p.key_tiles = plan.key_tiles;
  p.cut = plan.cut;
  p.turns = plan.turns;
  p.scale = a->scale;
  if (plan.tails.fn != nullptr) {
    p.cut = 0;
    p.cut_out = reinterpret_cast<int*>(p.parts + plan.bytes - 256);
    p.balance = plan.balance;
    p.tail_items = int(plan.items / a->num_seqs);
  }
  cudaError_t e = plan.k.prefix(p, a->num_heads, plan.grid, s);
  count_launch();
  if (e != cudaSuccess) {
    set_error("shared prefix kernel launch failed: %s", cudaGetErrorString(e));
    return B200PA_ECUDA;
  }

  DecodeParams d{};
  d.out = a->out;
  d.q = a->query;
  d.kc = a->key_cache;
  d.vc = a->value_cache;
  d.block_tables = a->block_tables + prefix_len / a->block_size;
  d.seq_lens = a->seq_lens;
  d.alibi = a->alibi_slopes;
  d.k_scale = a->k_scale;
  d.v_scale = a->v_scale;
  d.q_stride = a->q_stride;
  d.kv_block_stride = a->kv_block_stride;
  d.kv_head_stride = a->kv_head_stride;
  d.num_seqs = a->num_seqs;
  d.num_heads = a->num_heads;
  d.num_kv_heads = a->num_kv_heads;
  d.block_size = a->block_size;
  d.max_blocks_per_seq = a->max_num_blocks_per_seq;
  d.len_cap = INT32_MAX;
  d.group = p.group;
  d.scale = a->scale;
  d.lse = a->out_lse;
  d.status = p.status;
  SharedPrefixParts pre{};
  pre.parts = p.parts;
  pre.prefix_len = prefix_len;
  pre.tokens = 128 / p.group;
  pre.groups = plan.groups;
  pre.key_tiles = plan.key_tiles;
  pre.cut = plan.cut;
  pre.tiles = plan.tiles;
  pre.turns = plan.turns;
  if (plan.tails.fn != nullptr) {
    d.head_groups = (p.group + plan.heads - 1) / plan.heads;
    d.nstages = plan.slots;
    d.use_table = 1;
    d.min_chunk = plan.min_chunk;
    d.max_partitions = tuning().max_parts ? tuning().max_parts : kMostPieces;  // (bounds the cuts)
    pre.own = p.parts + plan.own_at;
    pre.found = reinterpret_cast<int2*>(p.parts + plan.found_at);
    pre.balance = plan.balance;
    e = plan.tails.fn(d, pre, sm_count(), plan.warps * 32, plan.smem, s);
  } else {
    d.head_groups = (p.group + plan.k.heads - 1) / plan.k.heads;
    e = plan.cluster == 0 ? plan.k.solo(d, pre, int(plan.items), s)
                          : plan.k.behind(d, pre, int(plan.items), plan.cluster, s);
  }
  count_launch();
  if (e != cudaSuccess) {
    set_error("shared prefix decode kernel launch failed: %s", cudaGetErrorString(e));
    return B200PA_ECUDA;
  }
  if (plan.tails.fn == nullptr) return B200PA_OK;
  CombineParams c{};
  c.out = a->out;
  c.v_scale = a->kv_dtype == B200PA_KV_AUTO ? nullptr : a->v_scale;
  c.lse = a->out_lse;
  c.cut = p.cut_out;
  c.pre = pre;
  c.num_seqs = a->num_seqs;
  c.num_heads = a->num_heads;
  c.group = p.group;
  c.head_groups = d.head_groups;
  c.heads = plan.heads;
  c.ranges = sm_count() * plan.warps;
  // threads that share four dimensions of a head: 1, 2, 4 ... 32, so that each adds up a few parts
  const int64_t most = int64_t(plan.key_tiles) * p.num_kv_heads * plan.groups < sm_count() ? plan.key_tiles
                       : sm_count() / (p.num_kv_heads * plan.groups) + 2;
  c.share = 1;
  while (c.share < 32 && c.share * 6 < most * (plan.turns ? 2 : 1)) c.share *= 2;
  c.D = a->head_size;
  const int per_item = std::min(p.group, plan.heads) * (a->head_size / 4);
  const int threads = std::min(kCombineThreads, (per_item * c.share + 31) / 32 * 32), lanes = threads / c.share;
  e = launch_dependent(a->q_dtype == B200PA_BF16 ? shared_prefix_combine_kernel<__nv_bfloat16> : shared_prefix_combine_kernel<__half>,
                       dim3(unsigned(plan.items), unsigned((per_item + lanes - 1) / lanes)), dim3(threads), 0, s, c);
  count_launch();
  if (e != cudaSuccess) {
    set_error("shared prefix combine kernel launch failed: %s", cudaGetErrorString(e));
    return B200PA_ECUDA;
  }
  return B200PA_OK;
}

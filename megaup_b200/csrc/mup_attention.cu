// C ABI of the sliding-window attention with sinks (include/megaup.h):
// argument checks, tensor maps, the split of the work and the launches.
#include <algorithm>

#include "mup_attn_backward.cuh"
#include "mup_attn_forward.cuh"
#include "mup_attn_tokens.cuh"
#include "mup_host.cuh"

namespace {

using namespace mup;

constexpr int kSms = 148;
constexpr int kMaxLength = 1 << 29;  // positions plus a window side stay inside 32 bits

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

int padded_dim(const mup_window_attention& a) { return a.head_dim <= 64 ? 64 : 128; }

int64_t total_rows(const mup_window_attention& a) { return static_cast<int64_t>(a.batch) * a.heads_q * a.seq_q; }

int check_problem(const mup_window_attention* args) {
  if (args == nullptr) return host_fail(MUP_ERR_BAD_ARG, "window attention: null argument");
  const mup_window_attention& a = *args;
  if (a.head_dim < 8 || a.head_dim > 128 || a.head_dim % 8 != 0)
    return host_fail(MUP_ERR_UNSUPPORTED, "window attention: head_dim %d is not a multiple of 8 up to 128", a.head_dim);
  if (a.batch < 1 || a.heads_q < 1 || a.heads_kv < 1 || a.heads_q % a.heads_kv != 0)
    return host_fail(MUP_ERR_BAD_ARG, "window attention: batch %d, heads %d / %d", a.batch, a.heads_q, a.heads_kv);
  if (a.seq_q < 1 || a.seq_k < 1 || a.seq_q > kMaxLength || a.seq_k > kMaxLength)
    return host_fail(MUP_ERR_BAD_ARG, "window attention: %d queries and %d keys (1 .. %d)", a.seq_q, a.seq_k, kMaxLength);
  if (total_rows(a) > 0x7fffffff)
    return host_fail(MUP_ERR_UNSUPPORTED, "window attention: %d x %d x %d rows", a.batch, a.heads_q, a.seq_q);
  if (a.sinks < 0 || !(a.scale > 0.0f) || a.scale > 1e30f)
    return host_fail(MUP_ERR_BAD_ARG, "window attention: sinks %d, scale %g", a.sinks, static_cast<double>(a.scale));
  if (a.sequences != nullptr) {
    if (a.batch != 1 || a.kv_lengths != nullptr || a.n_sequences < 1 || a.longest_q < 1 || a.longest_q > a.seq_q ||
        a.longest_k < 0 || a.longest_k > a.seq_k || a.n_q_blocks_256 < 1 || a.n_q_blocks_128 < a.n_q_blocks_256 ||
        a.n_k_blocks_128 < 0)
      return host_fail(MUP_ERR_BAD_ARG, "window attention: inconsistent packed sequences");
  }
  return MUP_OK;
}

int check_tensor(const char* name, const void* base, const int64_t strides[3]) {
  if (base == nullptr || reinterpret_cast<uintptr_t>(base) % 16 != 0)
    return host_fail(MUP_ERR_BAD_ARG, "window attention: %s is null or not 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    if (strides[i] <= 0 || strides[i] % 8 != 0 || strides[i] >= (1ll << 39))
      return host_fail(MUP_ERR_BAD_ARG, "window attention: %s stride %lld is no positive multiple of 16 bytes", name,
                       static_cast<long long>(strides[i]));
  return MUP_OK;
}

// What a launch reads besides the tensors. (The counts and lengths of the lists are the caller's; a list that is too short
// for the longest sequence cannot be one of these sequences.)
int check_tables(const mup_window_attention& a, bool backward) {
  const auto misaligned = [](const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (misaligned(a.lse, 4) || misaligned(a.kv_lengths, 4) || misaligned(a.workspace, 16))
    return host_fail(MUP_ERR_BAD_ARG, "window attention: lse, kv_lengths or workspace is not aligned (4, 4, 16 bytes)");
  if (a.sequences == nullptr) return MUP_OK;
  if (misaligned(a.sequences, 16))
    return host_fail(MUP_ERR_BAD_ARG, "window attention: sequences is not 16-byte aligned");
  const struct {
    const char* name;
    const int32_t* list;
    int count, needed;
  } lists[] = {{"q_blocks_256", a.q_blocks_256, a.n_q_blocks_256, ceil_div(a.longest_q, 256)},
               {"q_blocks_128", a.q_blocks_128, a.n_q_blocks_128, ceil_div(a.longest_q, 128)},
               {"k_blocks_128", a.k_blocks_128, a.n_k_blocks_128, backward ? ceil_div(a.longest_k, 128) : 0}};
  for (const auto& l : lists) {
    if (l.count < l.needed || (l.count > 0 && (l.list == nullptr || misaligned(l.list, 32))))
      return host_fail(MUP_ERR_BAD_ARG, "window attention: %s is null, not 32-byte aligned or has fewer than %d entries",
                       l.name, l.needed);
  }
  return MUP_OK;
}

AttnShape make_shape(const mup_window_attention& a, uint32_t* status) {
  AttnShape s{};
  s.batch = a.batch, s.heads_q = a.heads_q, s.heads_kv = a.heads_kv;
  s.seq_q = a.seq_q, s.seq_k = a.seq_k, s.head_dim = a.head_dim;
  s.causal = a.causal != 0;
  s.left = a.left < 0 ? kNoLimit : std::min(a.left, kNoLimit);
  s.right = s.causal ? 0 : a.right < 0 ? kNoLimit : std::min(a.right, kNoLimit);
  // a window without a left limit holds the sinks that a causal row may see
  s.sinks = s.causal && s.left == kNoLimit ? 0 : a.sinks;
  s.scale = a.scale, s.scale_log2 = a.scale * kLog2e;
  s.kv_lengths = a.kv_lengths;
  s.sequences = reinterpret_cast<const int4*>(a.sequences);
  s.status = status;
  s.timeout_ns = a.timeout_ns != 0 ? a.timeout_ns : 5000000000ull;
  return s;
}

// How a forward pass is cut into CTAs.
struct ForwardPlan {
  int packed_heads, pair_heads, single, head_sets, blocks, splits;
  bool small_blocks;  // packed lists: blocks of 128 rows instead of 256
};

ForwardPlan plan_forward(const mup_window_attention& a) {
  ForwardPlan f{};
  const int group = a.heads_q / a.heads_kv;
  const bool packed = a.sequences != nullptr;
  const int queries = packed ? a.longest_q : a.seq_q;
  // Few queries: the heads of a group share a sub-tile's 128 rows.
  f.packed_heads = 1;
  while (group % (2 * f.packed_heads) == 0 && 2 * f.packed_heads * queries <= kTileRows) f.packed_heads *= 2;
  const int rows = kTileRows / f.packed_heads;
  const int sets = group / f.packed_heads;
  f.pair_heads = sets % 2 == 0;
  f.single = !f.pair_heads && queries <= rows;
  f.head_sets = a.heads_q / (f.packed_heads * (f.pair_heads ? 2 : 1));
  f.small_blocks = f.pair_heads || f.single;
  const int block_rows = f.small_blocks ? rows : 2 * rows;
  f.blocks = packed ? (f.small_blocks ? a.n_q_blocks_128 : a.n_q_blocks_256) : a.batch * ceil_div(a.seq_q, block_rows);
  // Too few CTAs for the GPU: several share a block's key tiles.
  const AttnShape s = make_shape(a, nullptr);
  const int keys = packed ? a.longest_k : a.seq_k;
  const int64_t window = static_cast<int64_t>(s.left) + s.right + std::min(block_rows, queries);
  const int tiles = std::max(1, std::min(ceil_div(keys, kTileRows),
                                         ceil_div(std::min<int64_t>(window, keys), kTileRows) + 1 + ceil_div(std::min(s.sinks, keys), kTileRows)));
  const int64_t ctas = static_cast<int64_t>(f.blocks) * f.head_sets;
  f.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kSms / std::max<int64_t>(ctas, 1), tiles)));
  return f;
}

// Few query rows: the kernel for tokens over a cache. Measured, few rows' kernel / 128-row kernel, 8 rows: 256 keys 5.7 /
// 8.5 us, 4096 6.9 / 10.6, 65536 13.4 / 18.3, 16 sequences of 4096 11.4 / 16.4, 64 of them 28.1 / 34.6; 16 rows, 4096
// keys: 7.3 / 9.7. It has one row tile: above 16 rows it would read the cache again for each.
bool few_rows(const mup_window_attention& a) {
  const int queries = a.sequences != nullptr ? a.longest_q : a.seq_q;
  return static_cast<int64_t>(a.heads_q / a.heads_kv) * queries <= kTokenRows;
}

// Keys of a CTA where lengths differ. Measured on 16 sequences of 8192 to 65536 keys (308 MB): 1024 56.9 us, 2048 67.8 (as
// many CTAs as places, some with less to do), 4096 55.3; smaller shares spread one long sequence among short ones better.
constexpr int kTokenShare = 1024;

constexpr int kMostTokenCtas = 4096;  // bounds the workspace: 8 KB of a CTA

struct TokenPlan {
  int splits, share;
  bool cluster;
};

TokenPlan plan_tokens(const mup_window_attention& a) {
  const bool packed = a.sequences != nullptr;
  const AttnShape s = make_shape(a, nullptr);
  const int keys = packed ? a.longest_k : a.seq_k, queries = packed ? a.longest_q : a.seq_q;
  const int64_t window = std::min<int64_t>(static_cast<int64_t>(s.left) + s.right + queries, keys);
  const int64_t visible = std::min<int64_t>(keys, window + s.sinks);
  const int64_t places = static_cast<int64_t>(packed ? a.n_sequences : a.batch) * a.heads_kv;
  const int64_t most = std::max<int64_t>(1, ceil_div(visible, kTokenKeys));
  const int64_t fill = std::max<int64_t>(1, kTokenCtas * kSms / places);
  TokenPlan t{};
  // Short: joined within a cluster, without a workspace and a second launch. Measured with 8 heads over 256 / 512 / 1024 /
  // 2000 keys: a call takes 9 us of host time instead of 13, and replays of a graph 5.6 / 6.5 / 7.1 / 8.2 us instead of
  // 6.0 / 6.1 / 6.2 / 7.0. The rule is that of calls; a graph of tokens over 512 keys and more would be better off without.
  if (most <= 4 * kTokenCluster) {
    t.splits = static_cast<int>(std::min<int64_t>({most, fill, kTokenCluster}));
    t.cluster = t.splits > 1;
    return t;
  }
  t.splits = static_cast<int>(std::min<int64_t>({most, fill, kMostSplits}));
  // Sequences of different lengths, cut for the longest: shares of one size, so that no CTA has more to do than others
  // and a short sequence leaves its last CTAs nothing.
  if (packed || a.kv_lengths != nullptr) {
    const int64_t bound = std::min<int64_t>(kMostSplits, kMostTokenCtas / places);
    t.splits = static_cast<int>(std::max<int64_t>(t.splits, std::min<int64_t>(visible / kTokenShare, bound)));
    t.share = ceil_div(visible / kTokenKeys + 3, t.splits);  // the sinks' and the window's tiles may be cut at their ends
  }
  return t;
}

uint64_t partial_bytes(const mup_window_attention& a, int splits) {
  return static_cast<uint64_t>(splits) * total_rows(a) * (padded_dim(a) + 1) * sizeof(float);
}

uint64_t forward_workspace(const mup_window_attention& a) {
  if (few_rows(a)) {
    const TokenPlan t = plan_tokens(a);
    return t.cluster || t.splits <= 1 ? 0 : partial_bytes(a, t.splits);
  }
  const ForwardPlan f = plan_forward(a);
  return f.splits <= 1 ? 0 : partial_bytes(a, f.splits);
}

int check_workspace(const mup_window_attention& a, uint64_t needed) {
  if (needed == 0 || (a.workspace != nullptr && a.workspace_bytes >= needed)) return MUP_OK;
  return host_fail(MUP_ERR_BAD_ARG, "window attention: the workspace has %llu bytes, %llu are needed",
                   static_cast<unsigned long long>(a.workspace_bytes), static_cast<unsigned long long>(needed));
}

int encode_rows(CUtensorMap* map, const mup_window_attention& a, const void* base, const int64_t strides[3], int rows,
                int heads, int box_rows, int box_heads) {
  const uint64_t dims[4] = {static_cast<uint64_t>(a.head_dim), static_cast<uint64_t>(rows),
                            static_cast<uint64_t>(heads), static_cast<uint64_t>(a.batch)};
  const int64_t order[3] = {strides[1], strides[2], strides[0]};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), static_cast<uint32_t>(box_heads), 1};
  return encode_map_4d(map, base, dims, order, box);
}

template <int DP>
int launch_combine(const mup_window_attention& a, const float* partial_out, const float* partial_lse, int splits,
                   cudaStream_t stream) {
  AttnCombine c{};
  c.partial_out = partial_out, c.partial_lse = partial_lse, c.splits = splits;
  c.head_dim = a.head_dim, c.heads_q = a.heads_q, c.seq_q = a.seq_q, c.total_rows = total_rows(a);
  c.out = static_cast<__nv_bfloat16*>(a.out), c.out_rest = static_cast<__nv_bfloat16*>(a.out_rest);
  c.out_batch = a.out_strides[0], c.out_seq = a.out_strides[1], c.out_head = a.out_strides[2], c.lse = a.lse;
  // Few rows with many parts want more threads a row (8 rows of 296 parts: 11 us with 128 threads, 3 us with 512).
  const bool wide = splits > 48;
  MUP_HOST_CUDA(launch_early(wide ? attention_combine_kernel<DP, 512> : attention_combine_kernel<DP, 128>,
                             dim3(static_cast<unsigned>(c.total_rows)), wide ? 512 : 128, 0, 1, stream, c));
  return MUP_OK;
}

template <int DP>
int launch_forward(const mup_window_attention& a, cudaStream_t stream, uint32_t* status) {
  const ForwardPlan f = plan_forward(a);
  CUtensorMap q_map, k_map, v_map;
  int rc = encode_rows(&q_map, a, a.q, a.q_strides, a.seq_q, a.heads_q, kTileRows / f.packed_heads, f.packed_heads);
  if (rc == MUP_OK) rc = encode_rows(&k_map, a, a.k, a.k_strides, a.seq_k, a.heads_kv, kTileRows, 1);
  if (rc == MUP_OK) rc = encode_rows(&v_map, a, a.v, a.v_strides, a.seq_k, a.heads_kv, kTileRows, 1);
  if (rc != MUP_OK) return rc;
  AttnForward p{};
  p.shape = make_shape(a, status);
  if (a.sequences != nullptr)
    p.tiles = reinterpret_cast<const AttnPackedBlock*>(f.small_blocks ? a.q_blocks_128 : a.q_blocks_256);
  p.blocks_per_sequence = f.blocks / a.batch;
  p.head_sets = f.head_sets, p.packed_heads = f.packed_heads, p.rows_log2 = 7;
  for (int h = f.packed_heads; h > 1; h /= 2) --p.rows_log2;
  p.pair_heads = f.pair_heads;
  p.splits = f.splits, p.single = f.single;
  p.out = static_cast<__nv_bfloat16*>(a.out), p.out_rest = static_cast<__nv_bfloat16*>(a.out_rest);
  p.out_batch = a.out_strides[0], p.out_seq = a.out_strides[1], p.out_head = a.out_strides[2];
  p.lse = a.lse;
  p.total_rows = total_rows(a);
  p.partial_out = static_cast<float*>(a.workspace);
  p.partial_lse = p.partial_out + (f.splits > 1 ? f.splits * p.total_rows * DP : 0);
  using Cfg = AttnForwardConfig<DP>;
  static uint64_t ready = 0;
  MUP_HOST_CUDA(allow_smem_once(attention_forward_kernel<DP>, Cfg::kSmemBytes, a.device, &ready));
  const int64_t grid = static_cast<int64_t>(f.blocks) * f.head_sets * f.splits;
  if (grid > 0x7fffffff) return host_fail(MUP_ERR_UNSUPPORTED, "window attention: too many row blocks");
  MUP_HOST_CUDA(launch_early(attention_forward_kernel<DP>, dim3(static_cast<unsigned>(grid)), Cfg::kThreads, Cfg::kSmemBytes, 1,
                             stream, p, q_map, k_map, v_map));
  if (f.splits > 1) return launch_combine<DP>(a, p.partial_out, p.partial_lse, f.splits, stream);
  return MUP_OK;
}

template <int DP>
int launch_tokens(const mup_window_attention& a, cudaStream_t stream, uint32_t* status) {
  const TokenPlan plan = plan_tokens(a);
  CUtensorMap k_map, v_map;
  int rc = encode_rows(&k_map, a, a.k, a.k_strides, a.seq_k, a.heads_kv, kTokenKeys, 1);
  if (rc == MUP_OK) rc = encode_rows(&v_map, a, a.v, a.v_strides, a.seq_k, a.heads_kv, kTokenKeys, 1);
  if (rc != MUP_OK) return rc;
  AttnTokens p{};
  p.shape = make_shape(a, status);
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.out = static_cast<__nv_bfloat16*>(a.out), p.out_rest = static_cast<__nv_bfloat16*>(a.out_rest);
  p.q_batch = a.q_strides[0], p.q_seq = a.q_strides[1], p.q_head = a.q_strides[2];
  p.out_batch = a.out_strides[0], p.out_seq = a.out_strides[1], p.out_head = a.out_strides[2];
  p.lse = a.lse;
  p.splits = plan.splits, p.share = plan.share, p.cluster = plan.cluster;
  p.total_rows = total_rows(a);
  p.partial_out = static_cast<float*>(a.workspace);
  p.partial_lse = p.partial_out + (plan.splits > 1 && !plan.cluster ? plan.splits * p.total_rows * DP : 0);
  using Cfg = AttnTokensConfig<DP>;
  const int64_t grid = static_cast<int64_t>(a.sequences != nullptr ? a.n_sequences : a.batch) * a.heads_kv * plan.splits;
  if (grid > 0x7fffffff) return host_fail(MUP_ERR_UNSUPPORTED, "window attention: too many sequences");
  static uint64_t ready = 0;
  MUP_HOST_CUDA(allow_smem_once(attention_tokens_kernel<DP>, Cfg::kSmemBytes, a.device, &ready));
  MUP_HOST_CUDA(launch_early(attention_tokens_kernel<DP>, dim3(static_cast<unsigned>(grid)), Cfg::kThreads, Cfg::kSmemBytes,
                             plan.cluster ? plan.splits : 1, stream, p, k_map, v_map));
  if (plan.splits > 1 && !plan.cluster) return launch_combine<DP>(a, p.partial_out, p.partial_lse, plan.splits, stream);
  return MUP_OK;
}

// How a backward pass is cut into CTAs.
struct BackwardPlan {
  int shared_tiles, shares;
};
constexpr int64_t kMostSharedJobs = 1024;

BackwardPlan plan_backward(const mup_window_attention& a) {
  const bool packed = a.sequences != nullptr;
  const AttnShape s = make_shape(a, nullptr);
  const int group = a.heads_q / a.heads_kv;
  const int queries = packed ? a.longest_q : a.seq_q, keys = packed ? a.longest_k : a.seq_k;
  const int key_tiles = ceil_div(keys, kTileRows);
  const int64_t tiles = packed ? a.n_k_blocks_128 : static_cast<int64_t>(a.batch) * key_tiles;
  const int64_t all_rows = static_cast<int64_t>(group) * ceil_div(queries, kTileRows);
  const int64_t window = static_cast<int64_t>(s.left) + s.right + kTileRows;
  const int64_t window_rows =
      std::min(all_rows, static_cast<int64_t>(group) * (ceil_div(std::min<int64_t>(window, queries), kTileRows) + 1));
  // A sink's tile is seen by every later row, other tiles by a window's rows: it is cut into shares of about as many
  // query tiles. Too few key tiles for the GPU: all of them are cut. (Packed sequences that are shorter than the longest
  // leave shares unused; their number is bounded, and with it the workspace: 128 KB a share.)
  const int64_t ctas = std::max<int64_t>(1, tiles * a.heads_kv);
  const int64_t sequences = packed ? a.n_sequences : a.batch;
  const auto bounded = [&](int64_t shares, int shared_tiles) {
    return std::min(shares, kMostSharedJobs / std::max<int64_t>(1, sequences * a.heads_kv * shared_tiles));
  };
  BackwardPlan b{};
  if (2 * ctas <= kSms) {
    b.shared_tiles = key_tiles;
    b.shares = static_cast<int>(bounded(std::min<int64_t>(kSms / ctas, ceil_div(all_rows, 2)), b.shared_tiles));
  }
  if (b.shares <= 1 && s.sinks > 0 && keys > 0) {
    const int64_t per_cta = std::max(window_rows, ctas * window_rows / (4 * kSms));
    b.shared_tiles = ceil_div(std::min(s.sinks, keys), kTileRows);
    b.shares = static_cast<int>(bounded(std::min<int64_t>(64, ceil_div(all_rows, per_cta)), b.shared_tiles));
  }
  if (b.shares <= 1 || keys == 0) b.shared_tiles = 0, b.shares = 1;
  return b;
}

uint64_t partial_floats(const mup_window_attention& a, const BackwardPlan& b) {
  const int64_t sequences = a.sequences != nullptr ? a.n_sequences : a.batch;
  return static_cast<uint64_t>(sequences) * a.heads_kv * b.shared_tiles * b.shares * 2 * kTileRows * padded_dim(a);
}

// lse2 and delta, then (16-byte aligned) the shares.
uint64_t stat_floats(const mup_window_attention& a) { return (2 * static_cast<uint64_t>(total_rows(a)) + 3) / 4 * 4; }

uint64_t backward_workspace(const mup_window_attention& a, const BackwardPlan& b) {
  return (stat_floats(a) + partial_floats(a, b)) * sizeof(float);
}

template <int DP>
int launch_backward(const mup_window_attention& a, cudaStream_t stream, uint32_t* status) {
  const BackwardPlan plan = plan_backward(a);
  const int checked = check_workspace(a, backward_workspace(a, plan));
  if (checked != MUP_OK) return checked;
  CUtensorMap q_map, k_map, v_map, do_map;
  int rc = encode_rows(&q_map, a, a.q, a.q_strides, a.seq_q, a.heads_q, kTileRows, 1);
  if (rc == MUP_OK) rc = encode_rows(&do_map, a, a.dout, a.dout_strides, a.seq_q, a.heads_q, kTileRows, 1);
  if (rc == MUP_OK) rc = encode_rows(&k_map, a, a.k, a.k_strides, a.seq_k, a.heads_kv, kTileRows, 1);
  if (rc == MUP_OK) rc = encode_rows(&v_map, a, a.v, a.v_strides, a.seq_k, a.heads_kv, kTileRows, 1);
  if (rc != MUP_OK) return rc;
  float* workspace = static_cast<float*>(a.workspace);

  AttnDelta d{};
  d.out_rest = static_cast<const __nv_bfloat16*>(a.out_rest);
  d.out = static_cast<const __nv_bfloat16*>(a.out), d.dout = static_cast<const __nv_bfloat16*>(a.dout);
  d.out_batch = a.out_strides[0], d.out_seq = a.out_strides[1], d.out_head = a.out_strides[2];
  d.dout_batch = a.dout_strides[0], d.dout_seq = a.dout_strides[1], d.dout_head = a.dout_strides[2];
  d.lse = a.lse, d.lse2 = workspace, d.delta = workspace + total_rows(a);
  d.total_rows = total_rows(a), d.heads_q = a.heads_q, d.seq_q = a.seq_q, d.head_dim = a.head_dim;

  AttnBackward p{};
  p.shape = make_shape(a, status);
  const bool packed = a.sequences != nullptr;
  p.q_blocks = reinterpret_cast<const AttnPackedBlock*>(packed ? a.q_blocks_128 : nullptr);
  p.k_blocks = reinterpret_cast<const AttnPackedBlock*>(packed ? a.k_blocks_128 : nullptr);
  p.n_q_blocks = packed ? a.n_q_blocks_128 : ceil_div(a.seq_q, kTileRows);
  p.n_k_blocks = packed ? a.n_k_blocks_128 : ceil_div(a.seq_k, kTileRows);
  p.n_sequences = packed ? a.n_sequences : a.batch;
  p.shared_tiles = plan.shared_tiles, p.shares = plan.shares;
  p.lse2 = d.lse2, p.delta = d.delta, p.partial = workspace + stat_floats(a);
  p.dq = static_cast<__nv_bfloat16*>(a.dq), p.dk = static_cast<__nv_bfloat16*>(a.dk), p.dv = static_cast<__nv_bfloat16*>(a.dv);
  p.dq_batch = a.dq_strides[0], p.dq_seq = a.dq_strides[1], p.dq_head = a.dq_strides[2];
  p.dk_batch = a.dk_strides[0], p.dk_seq = a.dk_strides[1], p.dk_head = a.dk_strides[2];
  p.dv_batch = a.dv_strides[0], p.dv_seq = a.dv_strides[1], p.dv_head = a.dv_strides[2];

  const int64_t q_grid = static_cast<int64_t>(p.n_q_blocks) * (packed ? 1 : a.batch) * a.heads_q;
  const int64_t shared_jobs = static_cast<int64_t>(p.n_sequences) * a.heads_kv * plan.shared_tiles * plan.shares;
  const int64_t k_grid = shared_jobs + static_cast<int64_t>(a.heads_kv) *
                                           (packed ? p.n_k_blocks : a.batch * (p.n_k_blocks - plan.shared_tiles));
  if (q_grid + k_grid > 0x7fffffff)
    return host_fail(MUP_ERR_UNSUPPORTED, "window attention: too many row blocks");
  const int smem = AttnBackwardConfig<DP>::kSmemBytes;
  static uint64_t ready = 0;
  MUP_HOST_CUDA(allow_smem_once(attention_backward_kernel<DP>, smem, a.device, &ready));
  p.dkv_jobs = static_cast<int>(k_grid);
  MUP_HOST_CUDA(launch_early(attention_delta_kernel, ceil_div(total_rows(a), 16 * kDeltaRows), 256, 0, 1, stream, d));
  MUP_HOST_CUDA(launch_early(attention_backward_kernel<DP>, dim3(static_cast<unsigned>(k_grid + q_grid)), 384, smem, 1, stream, p, q_map, k_map, v_map, do_map));
  if (plan.shared_tiles > 0) {
    const int64_t quads = static_cast<int64_t>(p.n_sequences) * a.heads_kv * plan.shared_tiles * 2 * kTileRows * (DP / 4);
    MUP_HOST_CUDA(launch_early(attention_dkv_join_kernel<DP>, ceil_div(quads, 256), 256, 0, 1, stream, p));
  }
  return MUP_OK;
}

}  // namespace

extern "C" {

int mup_window_attention_workspace(const mup_window_attention* args, uint64_t* forward_bytes,
                                   uint64_t* backward_bytes) {
  const int rc = check_problem(args);
  if (rc != MUP_OK) return rc;
  if (forward_bytes != nullptr) *forward_bytes = forward_workspace(*args);
  if (backward_bytes != nullptr) *backward_bytes = backward_workspace(*args, plan_backward(*args));
  return MUP_OK;
}

int mup_window_attention_forward(const mup_window_attention* args, void* stream) {
  int rc = check_problem(args);
  if (rc == MUP_OK) rc = check_tensor("q", args->q, args->q_strides);
  if (rc == MUP_OK) rc = check_tensor("k", args->k, args->k_strides);
  if (rc == MUP_OK) rc = check_tensor("v", args->v, args->v_strides);
  if (rc == MUP_OK) rc = check_tensor("out", args->out, args->out_strides);
  if (rc == MUP_OK && args->out_rest != nullptr) rc = check_tensor("out_rest", args->out_rest, args->out_strides);
  if (rc == MUP_OK) rc = check_tables(*args, false);
  if (rc == MUP_OK) rc = check_workspace(*args, forward_workspace(*args));
  if (rc != MUP_OK) return rc;
  DeviceScope scope(args->device);
  MUP_HOST_CUDA(scope.error());
  uint32_t* status = nullptr;
  rc = device_status_word(args->device, &status);
  if (rc != MUP_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (few_rows(*args)) return args->head_dim <= 64 ? launch_tokens<64>(*args, s, status) : launch_tokens<128>(*args, s, status);
  return args->head_dim <= 64 ? launch_forward<64>(*args, s, status) : launch_forward<128>(*args, s, status);
}

int mup_window_attention_backward(const mup_window_attention* args, void* stream) {
  int rc = check_problem(args);
  if (rc != MUP_OK) return rc;
  if (args->kv_lengths != nullptr) return host_fail(MUP_ERR_UNSUPPORTED, "window attention: no gradient with kv_lengths");
  if (args->lse == nullptr) return host_fail(MUP_ERR_BAD_ARG, "window attention: the backward pass needs lse");
  rc = check_tensor("q", args->q, args->q_strides);
  if (rc == MUP_OK) rc = check_tensor("k", args->k, args->k_strides);
  if (rc == MUP_OK) rc = check_tensor("v", args->v, args->v_strides);
  if (rc == MUP_OK) rc = check_tensor("out", args->out, args->out_strides);
  if (rc == MUP_OK && args->out_rest != nullptr) rc = check_tensor("out_rest", args->out_rest, args->out_strides);
  if (rc == MUP_OK) rc = check_tensor("dout", args->dout, args->dout_strides);
  if (rc == MUP_OK) rc = check_tensor("dq", args->dq, args->dq_strides);
  if (rc == MUP_OK) rc = check_tensor("dk", args->dk, args->dk_strides);
  if (rc == MUP_OK) rc = check_tensor("dv", args->dv, args->dv_strides);
  if (rc == MUP_OK) rc = check_tables(*args, true);
  if (rc != MUP_OK) return rc;
  DeviceScope scope(args->device);
  MUP_HOST_CUDA(scope.error());
  uint32_t* status = nullptr;
  rc = device_status_word(args->device, &status);
  if (rc != MUP_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return args->head_dim <= 64 ? launch_backward<64>(*args, s, status) : launch_backward<128>(*args, s, status);
}

}  // extern "C"

// Forward pass of the sliding-window attention with sinks.
//
// A CTA computes two sub-tiles of 128 query rows against one stream of key and
// value tiles of 128 rows: S = Q K^T and O += P V are tcgen05 products with
// their accumulators in TMEM (2 x 128 columns of S, 2 x DP of O), P stays in
// TMEM as the second product's left operand. While four warps turn one
// sub-tile's S into P, the tensor pipe works on the other's.
//
// Bound by the tensor pipe and the exponentials together (a step of two 128 x 128 x 128 sub-tiles takes about 3030 cycles,
// 2048 of them products, 2048 the special function units' exponentials), on long windows by the board's power: 756 GFLOP of
// a video window over 32768 rows 604 us cold (1.25 PFLOP/s), 700 at the 1000 W cap. Short windows lose 20 % to a CTA's start
// and end: packed prompts under a window of 1024 158 us for 112 GFLOP of visible pairs.
// Two sub-tiles rather than one: with one nothing fills the pipe during the exponentials. TMEM rather than shared memory for
// P: 32 KB a step less through shared memory, which the products' right operands keep busy.
//
// P is rounded to BF16 for the second product, whose operands have one type, V's: off by at most 2^-8 of itself, as the
// result's own rounding (relative error against 64 bits 2.1e-3 to 2.4e-3, with FP32 weights 1.6e-3). The row's sum takes the
// FP32 values. Weights below 2^-126 become 0.
#pragma once

#include "mup_attn_common.cuh"

namespace mup {

struct AttnForward {
  AttnShape shape;
  const AttnPackedBlock* tiles;  // packed: the row blocks; null when dense
  int blocks_per_sequence;  // dense: row blocks per sequence
  int head_sets;            // heads_q / heads per CTA
  int packed_heads;         // heads per sub-tile, a power of two: its 128 rows are heads x rows of a head
  int rows_log2;            // of a head in a sub-tile
  int pair_heads;           // sub-tile 1 holds the next heads (1) or the next rows (0)
  int splits;               // CTAs that share one block's key tiles
  int single;               // only sub-tile 0 exists
  __nv_bfloat16 *out, *out_rest;  // out_rest: what out's rounding leaves, or null
  int64_t out_batch, out_seq, out_head;
  float* lse;               // [batch, heads, rows] or null
  float* partial_out;       // [splits, total rows, DP], splits > 1
  float* partial_lse;       // [splits, total rows], base 2
  int64_t total_rows;       // batch * heads_q * seq_q
};

template <int DP>
struct AttnForwardConfig {
  static constexpr int kPanels = DP / 64;
  static constexpr int kTileBytes = kPanels * kPanelBytes;
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kOffQ = 0;
  static constexpr int kOffStages = 2 * kTileBytes;
  static constexpr int kOffBars = kOffStages + kStages * kTileBytes;
  // q full [2], stage full, stage empty, s full [2], half of p full [2][2], done [2], drain [2], started
  static constexpr int kBars = 2 + 2 * kStages + 8 + 2 + 1;
  static constexpr int kOffWords = kOffBars + kBars * 8;
  static constexpr int kSmemBytes = kOffWords + 16;  // TMEM's address, abort, copies of K and V, sub-tiles with a Q
  static constexpr int kThreads = 384;
  static constexpr int kTmemO = 256;
};

// What a CTA computes: decoded by each role for itself, so that no role holds what only another needs.
struct ForwardBlock {
  AttnSeq seq;
  int batch, head0, kv_head, rows, rows_log2, row0, row_step, head_step, split;

  __device__ __forceinline__ explicit ForwardBlock(const AttnForward& p) {
    int w = blockIdx.x;
    split = w % p.splits;
    w /= p.splits;
    const int head_set = w % p.head_sets;
    w /= p.head_sets;
    int sequence;
    rows_log2 = p.rows_log2;
    rows = 1 << rows_log2;
    row_step = p.pair_heads ? 0 : rows;
    head_step = p.pair_heads ? p.packed_heads : 0;
    if (p.tiles != nullptr) {
      seq = load_block(p.tiles, w, sequence, row0);
    } else {
      // the last rows first: under a causal mask they have the most keys
      sequence = w % p.shape.batch;
      row0 = (p.blocks_per_sequence - 1 - w / p.shape.batch) * (p.single || p.pair_heads ? rows : 2 * rows);
      seq = load_sequence(p.shape, sequence);
    }
    batch = p.shape.sequences != nullptr ? 0 : sequence;
    head0 = head_set * p.packed_heads * (p.pair_heads ? 2 : 1);
    kv_head = head0 / (p.shape.heads_q / p.shape.heads_kv);
  }
  // the second sub-tile may lie behind the sequence's end
  __device__ __forceinline__ bool exists(const AttnForward& p, int t) const {
    return row0 + t * row_step < seq.nq && !(t == 1 && p.single);
  }
  __device__ __forceinline__ RowSpan first(const AttnForward& p, int t) const {
    return row_span(p.shape, seq, row0 + t * row_step);
  }
  __device__ __forceinline__ RowSpan last(const AttnForward& p, int t) const {
    return row_span(p.shape, seq, min(row0 + t * row_step + rows, seq.nq) - 1);
  }
  __device__ __forceinline__ TileList tiles(const AttnForward& p, int t) const {
    return make_tile_list(first(p, t), last(p, t));
  }
  // the key tiles of both sub-tiles
  __device__ __forceinline__ TileList all(const AttnForward& p) const {
    return make_tile_list(first(p, 0), last(p, exists(p, 1) ? 1 : 0));
  }
  // this CTA's share of them
  __device__ __forceinline__ void share(const AttnForward& p, int count, int& begin, int& end) const {
    const int each = (count + p.splits - 1) / p.splits;
    begin = min(split * each, count);
    end = min(begin + each, count);
  }
};

// Raise of the row maximum, in powers of two, up to which the old reference is kept: P is then at most 2^8, which
// neither its BF16 rounding (relative) nor the FP32 sums mind, and O is rescaled only where it has to be.
constexpr float kKeepMaximum = 8.0f;

template <int DP>
__global__ void __launch_bounds__(384, 1)
    attention_forward_kernel(const __grid_constant__ AttnForward p, const __grid_constant__ CUtensorMap q_map,
                             const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using Cfg = AttnForwardConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto bar = [&](int i) { return base + Cfg::kOffBars + i * 8; };
  const auto q_full = [&](int t) { return bar(t); };
  const auto full = [&](int s) { return bar(2 + s); };
  const auto empty = [&](int s) { return bar(2 + Cfg::kStages + s); };
  const auto s_full = [&](int t) { return bar(2 + 2 * Cfg::kStages + t); };
  const auto p_full = [&](int t, int half) { return bar(4 + 2 * Cfg::kStages + 2 * t + half); };
  const auto done = [&](int t) { return bar(8 + 2 * Cfg::kStages + t); };
  const auto drain = [&](int t) { return bar(10 + 2 * Cfg::kStages + t); };
  const uint32_t started = bar(12 + 2 * Cfg::kStages);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffWords);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffWords + 4);
  volatile uint32_t* copies = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffWords + 8);
  const WaitControl ctl{abort_flag, p.shape.status, p.shape.timeout_ns};

  grid_dep_launch();
  grid_dep_wait();
  // The copies of this CTA, in the order of the products: for step i K of tile i, then V of the tile before it.
  const auto load_tile = [&](const ForwardBlock& block, const CUtensorMap& map, int kt, int s) {
    mbar_arrive_expect_tx(full(s), Cfg::kTileBytes);
    const uint32_t dst = base + Cfg::kOffStages + s * Cfg::kTileBytes;
#pragma unroll
    for (int panel = 0; panel < Cfg::kPanels; ++panel)
      tma_load_4d(dst + panel * kPanelBytes, &map, panel * 64, block.seq.k0 + kt * kTileRows, block.kv_head, block.batch,
                  full(s));
  };
  // Both kinds of warps change their registers first and meet when barriers and TMEM are there.
  if (warp >= 8) {
    fewer_registers<72>();
    const bool loads_here = warp == 8 && elect_one_sync();
    const ForwardBlock block(p);
    if (loads_here) {
      const TileList all = block.all(p);
      int begin, end;
      block.share(p, all.count, begin, end);
      *abort_flag = 0u, copies[0] = copies[1] = 0u;
      const int users = block.exists(p, 1) ? 2 : 1;  // warps that read a stage
      for (int s = 0; s < Cfg::kStages; ++s) {
        mbar_init(full(s), 1);
        mbar_init(empty(s), users);
      }
      mbar_init(started, 1);
      for (int t = 0; t < 2; ++t) {
        mbar_init(q_full(t), 1);
        mbar_init(drain(t), 1);
        mbar_init(s_full(t), 1);
        mbar_init(p_full(t, 0), 128);
        mbar_init(p_full(t, 1), 128);
        mbar_init(done(t), 1);
      }
      fence_mbar_init();
      fence_proxy_async_smem();
      // the first copies do not wait for the other warps
      if (begin < end) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!block.exists(p, t)) continue;
          mbar_arrive_expect_tx(q_full(t), Cfg::kTileBytes);
#pragma unroll
          for (int panel = 0; panel < Cfg::kPanels; ++panel)
            tma_load_4d(base + Cfg::kOffQ + t * Cfg::kTileBytes + panel * kPanelBytes, &q_map, panel * 64,
                        block.seq.q0 + block.row0 + t * block.row_step, block.head0 + t * block.head_step, block.batch,
                        q_full(t));
          if (t == 0) load_tile(block, k_map, all.tile(begin), 0);
        }
      }
    }
    if (warp == 9) {
      tmem_alloc<1>(smem_u32(tmem_slot), 512);
      tmem_relinquish<1>();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    if (loads_here) {
      // ------------------------------------------------------------ TMA loads
      const TileList all = block.all(p);
      int begin, end;
      block.share(p, all.count, begin, end);
      int loads = 1;
      bool ok = true;
      const auto load = [&](const CUtensorMap& map, int kt) {
        const int s = loads % Cfg::kStages, use = loads / Cfg::kStages;
        if (use > 0 && !ctl.wait_alone(empty(s), (use - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT)) return false;
        load_tile(block, map, kt, s);
        ++loads;
        return true;
      };
      for (int i = begin + 1; ok && i <= end; ++i) {
        if (i < end) ok = load(k_map, all.tile(i));
        if (ok) ok = load(v_map, all.tile(i - 1));
      }
      if (begin < end) copies[0] = loads, copies[1] = block.exists(p, 1) ? 2 : 1;
    } else if (warp == 9 || (warp == 10 && block.exists(p, 1))) {
      // ------------------------------------------------------------ products
      // One warp per sub-tile: the issue of a product waits for room in the tensor pipe's short queue, so with one
      // warp for both every barrier between two issues left the pipe empty.
      const int t = warp - 9;
      const bool leader = elect_one_sync();
      const TileList all = block.all(p), mine = block.tiles(p, t);
      const bool exists = block.exists(p, t);
      int begin, end;
      block.share(p, all.count, begin, end);
      const uint32_t s_tmem = tmem + t * kTileRows, o_tmem = tmem + Cfg::kTmemO + t * DP;
      const uint32_t q_tile = base + Cfg::kOffQ + t * Cfg::kTileBytes;
      int stage = 0, steps = 0;  // the ring's next stage and its phase
      uint32_t phase = 0;
      const auto advance = [&] {
        if (++stage == Cfg::kStages) stage = 0, phase ^= 1;
      };
      bool ok = true, pending = false;
      for (int i = begin; begin < end && i <= end; ++i) {
        // Step i: K of tile i arrives, then V of the tile before it. Everything that does not depend on the softmax
        // warps comes before the waits for them, so that the products follow each other without a pause.
        bool active = false;
        int ks = 0;
        if (i < end) {
          ks = stage;
          ok = ctl.wait(full(ks), phase, MUP_ST_MMA_FULL_TIMEOUT);
          advance();
          active = exists && sees_tile(mine, all.tile(i));
          if (active && steps == 0) {
            ok = ok && ctl.wait(q_full(t), 0, MUP_ST_MMA_FULL_TIMEOUT);
            // Behind the first sub-tile's first product: the one's exponentials then run beside the other's products, and
            // both stay so (3030 cycles a step). Started together they stay together for ten steps and more, at 4700 to
            // 5800 cycles a step. (A barrier of its own with one phase: this warp may look late, when s_full is phases on.)
            if (t == 1 && i == begin && block.exists(p, 0) && sees_tile(block.tiles(p, 0), all.tile(i)))
              ok = ok && ctl.wait(started, 0, MUP_ST_MMA_ACC_TIMEOUT);
          }
        }
        if (ok && i > begin) {
          const int vs = stage;
          const uint32_t v_tile = base + Cfg::kOffStages + vs * Cfg::kTileBytes;
          ok = ctl.wait(full(vs), phase, MUP_ST_MMA_FULL_TIMEOUT);
          advance();
          if (ok && pending) {
            // (both warps clear the same rows: whichever comes second writes the zeros that are there)
            zero_unseen_rows<DP>(smem + Cfg::kOffStages + vs * Cfg::kTileBytes, all, all.tile(i - 1) * kTileRows, lane);
            const uint32_t parity = (steps - 1) & 1;
            ok = ctl.wait(p_full(t, 0), parity, MUP_ST_MMA_ACC_TIMEOUT);
            if (!ok) break;
            tc_fence_after_sync();
            // the first 64 keys while the softmax warps are at the others
            if (leader) umma_tmem_by_cols<DP, 0, 4>(o_tmem, s_tmem, 32, v_tile, steps > 1);
            ok = ctl.wait(p_full(t, 1), parity, MUP_ST_MMA_ACC_TIMEOUT);
            if (!ok) break;
            tc_fence_after_sync();
            if (leader) {
              umma_tmem_by_cols<DP, 4, 8>(o_tmem, s_tmem, 32, v_tile, true);
              umma_commit_1(empty(vs));
              umma_commit_1(done(t));  // the last arrival from a product: nothing reaches this CTA's barriers after it
            }
          } else if (ok && leader) {
            mbar_arrive(empty(vs));
          }
        }
        if (!ok) break;
        pending = active;
        if (active) {
          tc_fence_after_sync();
          if (leader) {
            umma_rows_by_rows<DP>(s_tmem, q_tile, base + Cfg::kOffStages + ks * Cfg::kTileBytes);
            umma_commit_1(s_full(t));
            umma_commit_1(empty(ks));
            if (t == 0 && i == begin) umma_commit_1(started);
          }
          ++steps;
        } else if (i < end && leader) {
          mbar_arrive(empty(ks));
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    more_registers<216>();
    const int t = warp / 4;
    const int quarter = warp % 4;
    const int r = quarter * 32 + lane;
    const ForwardBlock block(p);
    const TileList all = block.all(p), mine = block.tiles(p, t);
    const RowSpan first = block.first(p, t), last = block.last(p, t);
    int begin, end;
    block.share(p, all.count, begin, end);
    const int row = block.row0 + t * block.row_step + (r & (block.rows - 1));
    const bool exists = block.exists(p, t);
    const RowSpan span = row_span(p.shape, block.seq, row);
    const float c = p.shape.scale_log2;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + t * kTileRows + lane_base;
    const uint32_t o_tmem = tmem + Cfg::kTmemO + t * DP + lane_base;
    float top = -INFINITY, sum = 0.0f;
    int steps = 0;
    bool ok = true;
    for (int i = begin; exists && i < end; ++i) {
      const int j0 = all.tile(i) * kTileRows;
      if (!sees_tile(mine, all.tile(i))) continue;
      if (!ctl.wait(s_full(t), steps & 1, MUP_ST_EPILOGUE_TIMEOUT)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      uint32_t raw[4][32];
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld_32x32(s_tmem + b * 32, raw[b]);
      tmem_ld_wait();
      if (!tile_is_full(first, last, j0)) {
        const int low = span.low - j0, high = span.high - j0, sink = span.sink - j0;
#pragma unroll
        for (int b = 0; b < 4; ++b) hide_scores(raw[b], span_bits(low - b * 32, high - b * 32, sink - b * 32));
      }
      const float seen_top = fmaxf(max3(max32(raw[0]), max32(raw[1]), max32(raw[2])), max32(raw[3]));
      // the reference of the exponents: kept while the maximum grows little
      float factor = 1.0f;
      bool rescale = false;
      if (top == -INFINITY) {
        top = seen_top;  // nothing was added yet
      } else if ((seen_top - top) * c > kKeepMaximum) {
        factor = exp2_sfu((top - seen_top) * c);
        top = seen_top;
        rescale = true;
      }
      if (__any_sync(0xffffffffu, rescale)) {
        // S of this step was issued behind the last product into O: that has ended as well
        sum *= factor;
#pragma unroll 1
        for (int b = 0; b < DP / 16; ++b) {
          uint32_t o[16];
          tmem_ld_32x16(o_tmem + b * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
          tmem_st_32x16(o_tmem + b * 16, o);
        }
      }
      const float shift = top == -INFINITY ? 0.0f : -top * c;
      const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift);
      float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t(&packed)[16] = reinterpret_cast<uint32_t(&)[16]>(raw[b]);  // in place: entry x replaces a used one
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          float2 e = fma2(make_float2(__uint_as_float(raw[b][2 * x]), __uint_as_float(raw[b][2 * x + 1])), c2, shift2);
          e.x = exp2_sfu(e.x);
          e.y = exp2_sfu(e.y);
          sums[x & 1] = add2(sums[x & 1], e);
          packed[x] = pack_bf16(e.x, e.y);
        }
        tmem_st_32x16(s_tmem + b * 16, packed);
        if (b & 1) {
          tmem_st_wait();
          tc_fence_before_sync();
          mbar_arrive(p_full(t, b >> 1));
        }
      }
      sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
      ++steps;
    }
    // (the phases before the last one have ended with their successors' S; a sub-tile that saw nothing has no product
    // that waited for its Q, whose place is used again below)
    if (ok && steps > 0)
      ok = ctl.wait(done(t), (steps - 1) & 1, MUP_ST_EPILOGUE_TIMEOUT);
    else if (ok && exists && begin < end)
      ok = ctl.wait(q_full(t), 0, MUP_ST_EPILOGUE_TIMEOUT);
    // ---- O / sum, rounded once
    if (ok && exists) {
      tc_fence_after_sync();
      const int head0 = block.head0 + t * block.head_step, tile_row0 = block.row0 + t * block.row_step;
      const auto index_of = [&](int x) {  // of row x of the sub-tile
        return (static_cast<int64_t>(block.batch) * p.shape.heads_q + head0 + (x >> block.rows_log2)) * p.shape.seq_q +
               block.seq.q0 + tile_row0 + (x & (block.rows - 1));
      };
      const auto is_row = [&](int x) { return tile_row0 + (x & (block.rows - 1)) < block.seq.nq; };
      const bool empty_row = sum == 0.0f;
      if (is_row(r)) {
        const float lse2 = empty_row ? -INFINITY : top * c + log2f(sum);
        if (p.splits > 1)
          p.partial_lse[block.split * p.total_rows + index_of(r)] = lse2;
        else if (p.lse != nullptr)
          p.lse[index_of(r)] = lse2 * 0.69314718055994531f;
      }
      const float scale = empty_row ? 0.0f : 1.0f / sum;
      uint8_t* staged = smem + Cfg::kOffQ + t * Cfg::kTileBytes;
      constexpr int kRowBytes = DP * 2;
      const auto load_o = [&](int b, uint32_t(&o)[32]) {
        if (steps > 0) {
          tmem_ld_32x32(o_tmem + b * 32, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int x = 0; x < 32; ++x) o[x] = steps > 0 && !empty_row ? o[x] : 0u;
      };
      if (p.splits > 1) {  // half of the FP32 columns at a time
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
#pragma unroll 1
          for (int b = 0; b < DP / 64; ++b) {
            uint32_t o[32];
            load_o(half * (DP / 64) + b, o);
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<float4*>(staged_piece<kRowBytes>(staged, r, b * 8 + x / 4)) =
                  make_float4(__uint_as_float(o[x]) * scale, __uint_as_float(o[x + 1]) * scale,
                              __uint_as_float(o[x + 2]) * scale, __uint_as_float(o[x + 3]) * scale);
          }
          if (p.packed_heads == 1)
            write_staged_rows<kRowBytes>(staged, quarter * 32, lane, kRowBytes,
                                         reinterpret_cast<uint8_t*>(p.partial_out + (block.split * p.total_rows + index_of(0)) * DP +
                                                                    half * (DP / 2)),
                                         DP * 4, block.seq.nq - tile_row0);
          else
            write_staged_rows<kRowBytes>(staged, quarter * 32, lane, kRowBytes, [&](int x) {
            return !is_row(x) ? nullptr
                              : reinterpret_cast<uint8_t*>(p.partial_out + (block.split * p.total_rows + index_of(x)) * DP +
                                                           half * (DP / 2));
          });
        }
      } else {
        const auto write = [&](__nv_bfloat16* out, bool rest) {
#pragma unroll 1
          for (int b = 0; b < DP / 32; ++b) {
            uint32_t o[32];
            load_o(b, o);
#pragma unroll
            for (int x = 0; x < 32; x += 8)
              *staged_piece<kRowBytes>(staged, r, b * 4 + x / 8) =
                  rest ? pack_bf16x8_rest(o + x, scale) : pack_bf16x8(o + x, scale);
          }
          __nv_bfloat16* to = out + block.batch * p.out_batch + (block.seq.q0 + tile_row0) * p.out_seq + head0 * p.out_head;
          if (p.packed_heads == 1)
            write_staged_rows<kRowBytes>(staged, quarter * 32, lane, p.shape.head_dim * 2, reinterpret_cast<uint8_t*>(to),
                                         p.out_seq * 2, block.seq.nq - tile_row0);
          else
            write_staged_rows<kRowBytes>(staged, quarter * 32, lane, p.shape.head_dim * 2, [&](int x) {
              return !is_row(x) ? nullptr
                                : reinterpret_cast<uint8_t*>(to + (x & (block.rows - 1)) * p.out_seq +
                                                             (x >> block.rows_log2) * p.out_head);
            });
        };
        write(p.out, false);
        if (p.out_rest != nullptr) write(p.out_rest, true);
      }
    }
    tc_fence_before_sync();
  }
  __syncthreads();
  if (*abort_flag != 0u) {  // (nobody sets it any more: all threads take this branch or none)
    // a role may have issued its last product or copy before another gave up
    if (warp == 9 || warp == 10) drain_products(drain(warp - 9));
    if (threadIdx.x == 0) {
      for (int t = 0; t < static_cast<int>(copies[1]); ++t) drain_barrier(q_full(t), 0);
      drain_ring(full(0), Cfg::kStages, copies[0]);
    }
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc<1>(*tmem_slot, 512);
  }
}

// Joins the partial results of `splits` CTAs per row, always in the same order: a block per row, THREADS / (DP / 4)
// threads per four columns, each with every so-many-th split.
struct AttnCombine {
  const float* partial_out;
  const float* partial_lse;
  int splits, head_dim, heads_q, seq_q;
  int64_t total_rows;
  __nv_bfloat16 *out, *out_rest;
  int64_t out_batch, out_seq, out_head;
  float* lse;
};
constexpr int kMostSplits = 512;

template <int DP, int THREADS>
__global__ void __launch_bounds__(THREADS) attention_combine_kernel(const __grid_constant__ AttnCombine p) {
  constexpr int kQuads = DP / 4, kLanes = THREADS / kQuads, kWarps = THREADS / 32;
  __shared__ float weight[kMostSplits];
  __shared__ float warp_top[kWarps], warp_sum[kWarps];
  __shared__ float4 shared_acc[kLanes][kQuads];
  const int64_t row = blockIdx.x;
  const int thread = threadIdx.x, warp = thread / 32, lane = thread % 32;
  grid_dep_wait();  // the partial results are there
  float top = -INFINITY;
  for (int s = thread; s < p.splits; s += THREADS) {
    const float l = p.partial_lse[s * p.total_rows + row];
    weight[s] = l;
    top = fmaxf(top, l);
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_top[w]);
  float sum = 0.0f;
  for (int s = thread; s < p.splits; s += THREADS) {
    const float l = weight[s];
    weight[s] = l == -INFINITY ? 0.0f : exp2_sfu(l - top);
    sum += weight[s];
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += warp_sum[w];
  const int quad = thread % kQuads, part = thread / kQuads;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const float4* src = reinterpret_cast<const float4*>(p.partial_out + row * DP) + quad;
#pragma unroll 4
  for (int s = part; s < p.splits; s += kLanes) {
    const float w = weight[s];
    if (w == 0.0f) continue;  // such a split may have written nothing
    const float4 v = src[s * p.total_rows * kQuads];
    acc.x += w * v.x, acc.y += w * v.y, acc.z += w * v.z, acc.w += w * v.w;
  }
  shared_acc[part][quad] = acc;
  __syncthreads();
  if (part != 0 || quad * 4 >= p.head_dim) return;
#pragma unroll
  for (int i = 1; i < kLanes; ++i) {
    const float4 v = shared_acc[i][quad];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
  }
  const int seq = static_cast<int>(row % p.seq_q);
  const int64_t bh = row / p.seq_q;
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t at = (bh / p.heads_q) * p.out_batch + seq * p.out_seq + (bh % p.heads_q) * p.out_head + quad * 4;
  *reinterpret_cast<uint2*>(p.out + at) =
      make_uint2(pack_bf16(acc.x * scale, acc.y * scale), pack_bf16(acc.z * scale, acc.w * scale));
  if (p.out_rest != nullptr)
    *reinterpret_cast<uint2*>(p.out_rest + at) =
        make_uint2(pack_bf16_rest(acc.x * scale, acc.y * scale), pack_bf16_rest(acc.z * scale, acc.w * scale));
  if (quad == 0 && p.lse != nullptr) p.lse[row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace mup

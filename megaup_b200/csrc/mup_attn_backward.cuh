// Backward pass of the sliding-window attention with sinks. With P = exp(S - lse) and delta = rowsum(dO * O):
//     dP = dO V^T,  dS = P (dP - delta),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
//
// One launch of two kinds of CTAs, which both recompute S and dP: one walks the key tiles of a block of query rows and sums
// dQ, one walks the query tiles of a block of key rows (over all heads of the group) and sums dK and dV. That is seven
// products per pair of tiles where CTAs that share dQ would need five, but every sum stays in one CTA's TMEM: no atomics,
// no FP32 gradient in memory, the same bits every time. (A shared dQ to which key tiles add in a fixed order would have
// the same bits too; it was neither built nor measured.)
//
// Rounded to 16 bits: P for dV's product and dS for dK's and dQ's, whose other operands are BF16 and whose type is both
// operands'. Each is off by at most 2^-8 of itself, as the gradients' own rounding; the FP32 values of P make dS.
//
// Bound by the board's power on long sequences: 65536 rows, window 4096, 4 heads of one group, 128 wide take 1632 us in
// one launch (two launches 1770: the first one's last wave left SMs idle), seven products at 1.14 PFLOP/s.
#pragma once

#include "mup_attn_common.cuh"

namespace mup {

struct AttnBackward {
  AttnShape shape;
  const AttnPackedBlock* q_blocks;  // packed: blocks of 128 query rows; null when dense
  const AttnPackedBlock* k_blocks;  // packed: blocks of 128 key rows
  int n_q_blocks, n_k_blocks;  // packed: of the lists; dense: per sequence
  int n_sequences;
  int dkv_jobs;  // CTAs of dK and dV
  // The first `shared_tiles` key tiles of every sequence are each computed by `shares` CTAs.
  int shared_tiles, shares;
  const float* lse2;   // [batch, heads, rows], base 2; +inf where a row sees nothing
  const float* delta;  // the same shape
  float* partial;      // [sequence, kv head, shared tile, share, {dV, dK}, 128, DP]
  __nv_bfloat16 *dq, *dk, *dv;
  int64_t dq_batch, dq_seq, dq_head, dk_batch, dk_seq, dk_head, dv_batch, dv_seq, dv_head;
};

// ---------------------------------------------------------------------------
// delta and the base-2 log-sum-exp of every row: 16 lanes per row. Bound by memory: O, its rest and dO are read once.
// ---------------------------------------------------------------------------

struct AttnDelta {
  const __nv_bfloat16 *out, *out_rest, *dout;  // out_rest may be null
  int64_t out_batch, out_seq, out_head, dout_batch, dout_seq, dout_head;
  const float* lse;
  float *lse2, *delta;
  int64_t total_rows;
  int heads_q, seq_q, head_dim;
};

__device__ __forceinline__ float dot_bf16x2(uint32_t a, uint32_t b, float sum) {
  sum = fmaf(__uint_as_float(a << 16), __uint_as_float(b << 16), sum);
  return fmaf(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u), sum);
}

constexpr int kDeltaRows = 4;  // of 16 lanes: all their loads are in flight at once; a warp's 8 rows follow each other

__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ AttnDelta p) {
  // the kernel after this one reads what the ones before it wrote as well: it may begin once those have ended
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x % 32, part = lane % 16;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32) * 2 * kDeltaRows;
  uint4 x[kDeltaRows], y[kDeltaRows], z[kDeltaRows];
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    const int64_t item = first + i * 2 + lane / 16;
    x[i] = y[i] = z[i] = make_uint4(0, 0, 0, 0);
    if (item >= p.total_rows || part * 8 >= p.head_dim) continue;
    const uint32_t bh = static_cast<uint32_t>(item) / p.seq_q, row = static_cast<uint32_t>(item) - bh * p.seq_q;
    const uint32_t b = bh / p.heads_q, head = bh - b * p.heads_q;
    x[i] = ld_stream_v4(p.out + b * p.out_batch + row * p.out_seq + head * p.out_head + part * 8);
    y[i] = ld_stream_v4(p.dout + b * p.dout_batch + row * p.dout_seq + head * p.dout_head + part * 8);
    if (p.out_rest != nullptr)
      z[i] = ld_stream_v4(p.out_rest + b * p.out_batch + row * p.out_seq + head * p.out_head + part * 8);
  }
  float mine = 0.0f;  // of row `first + lane`, in the first eight lanes
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    float sum = dot_bf16x2(x[i].x, y[i].x, 0.0f);
    sum = dot_bf16x2(x[i].y, y[i].y, sum);
    sum = dot_bf16x2(x[i].z, y[i].z, sum);
    sum = dot_bf16x2(x[i].w, y[i].w, sum);
    float rest = dot_bf16x2(z[i].x, y[i].x, 0.0f);
    rest = dot_bf16x2(z[i].y, y[i].y, rest);
    rest = dot_bf16x2(z[i].z, y[i].z, rest);
    sum += dot_bf16x2(z[i].w, y[i].w, rest);
#pragma unroll
    for (int d = 8; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float there = __shfl_sync(0xffffffffu, sum, lane % 2 * 16);
    if (lane / 2 == i) mine = there;
  }
  if (lane < 2 * kDeltaRows && first + lane < p.total_rows) {
    const float l = p.lse[first + lane];
    p.delta[first + lane] = l == -INFINITY ? 0.0f : mine;  // whatever dO is where the row sees nothing
    p.lse2[first + lane] = l == -INFINITY ? INFINITY : l * kLog2e;
  }
}

// ---------------------------------------------------------------------------
// dQ
// ---------------------------------------------------------------------------

template <int DP>
struct AttnDqConfig {
  static constexpr int kPanels = DP / 64;
  static constexpr int kTileBytes = kPanels * kPanelBytes;
  static constexpr int kKStages = 3, kVStages = 2;
  static constexpr int kOffQ = 0, kOffDo = kTileBytes, kOffK = 2 * kTileBytes;
  static constexpr int kOffV = kOffK + kKStages * kTileBytes;
  static constexpr int kOffBars = kOffV + kVStages * kTileBytes;
  // q and dO full, k full/empty, v full/empty, s full [2], dp full, ds full, done, drain
  static constexpr int kBars = 1 + 2 * kKStages + 2 * kVStages + 6;
  static constexpr int kOffWords = kOffBars + kBars * 8;
  static constexpr int kSmemBytes = kOffWords + 16;  // TMEM's address, abort, copies into the two rings
  static constexpr int kTmemDp = 256, kTmemDq = 384;
};

template <int DP>
__device__ __forceinline__ void attention_dq(const AttnBackward& p, const CUtensorMap& q_map, const CUtensorMap& k_map,
                                             const CUtensorMap& v_map, const CUtensorMap& do_map, uint8_t* smem,
                                             int job) {
  using Cfg = AttnDqConfig<DP>;
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto bar = [&](int i) { return base + Cfg::kOffBars + i * 8; };
  const uint32_t q_full = bar(0);
  const auto k_full = [&](int s) { return bar(1 + s); };
  const auto k_empty = [&](int s) { return bar(1 + Cfg::kKStages + s); };
  constexpr int kV = 1 + 2 * Cfg::kKStages;
  const auto v_full = [&](int s) { return bar(kV + s); };
  const auto v_empty = [&](int s) { return bar(kV + Cfg::kVStages + s); };
  constexpr int kS = kV + 2 * Cfg::kVStages;
  const auto s_full = [&](int b) { return bar(kS + b); };
  const uint32_t dp_full = bar(kS + 2), ds_full = bar(kS + 3), done = bar(kS + 4), drain = bar(kS + 5);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffWords);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffWords + 4);
  volatile uint32_t* copies = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffWords + 8);
  const WaitControl ctl{abort_flag, p.shape.status, p.shape.timeout_ns};

  const int head = job % p.shape.heads_q;
  const int w = job / p.shape.heads_q;
  int sequence, row0;
  AttnSeq seq;
  if (p.q_blocks != nullptr) {
    seq = load_block(p.q_blocks, w, sequence, row0);
  } else {
    sequence = w % p.shape.batch, row0 = (p.n_q_blocks - 1 - w / p.shape.batch) * kTileRows;
    seq = load_sequence(p.shape, sequence);
  }
  const int batch = p.shape.sequences != nullptr ? 0 : sequence;
  const int kv_head = head / (p.shape.heads_q / p.shape.heads_kv);
  const RowSpan first = row_span(p.shape, seq, row0);
  const RowSpan last = row_span(p.shape, seq, min(row0 + kTileRows, seq.nq) - 1);
  const TileList tiles = make_tile_list(first, last);
  const int n = tiles.count;

  if (threadIdx.x == 0) {
    *abort_flag = 0u, copies[0] = copies[1] = 0u;
    for (int i = 0; i < Cfg::kBars; ++i) mbar_init(bar(i), bar(i) == ds_full ? 256 : 1);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    fewer_registers<72>();
    if (warp == 8 && elect_one_sync() && n > 0) {
      int i = 0, key_copies = 0;
      auto load = [&](const CUtensorMap& map, uint32_t dst, uint32_t full, int row, int h) {
#pragma unroll
        for (int panel = 0; panel < Cfg::kPanels; ++panel)
          tma_load_4d(dst + panel * kPanelBytes, &map, panel * 64, row, h, batch, full);
      };
      mbar_arrive_expect_tx(q_full, 2 * Cfg::kTileBytes);
      load(q_map, base + Cfg::kOffQ, q_full, seq.q0 + row0, head);
      load(do_map, base + Cfg::kOffDo, q_full, seq.q0 + row0, head);
      for (; i < n; ++i) {
        const int ks = i % Cfg::kKStages, vs = i % Cfg::kVStages;
        const int row = seq.k0 + tiles.tile(i) * kTileRows;
        if (i >= Cfg::kKStages && !ctl.wait_alone(k_empty(ks), (i / Cfg::kKStages - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT)) break;
        mbar_arrive_expect_tx(k_full(ks), Cfg::kTileBytes);
        load(k_map, base + Cfg::kOffK + ks * Cfg::kTileBytes, k_full(ks), row, kv_head);
        ++key_copies;
        if (i >= Cfg::kVStages && !ctl.wait_alone(v_empty(vs), (i / Cfg::kVStages - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT)) break;
        mbar_arrive_expect_tx(v_full(vs), Cfg::kTileBytes);
        load(v_map, base + Cfg::kOffV + vs * Cfg::kTileBytes, v_full(vs), row, kv_head);
      }
      copies[0] = key_copies, copies[1] = i;
    } else if (warp == 9 && n > 0) {
      const bool leader = elect_one_sync();
      // S of tile i goes to buffer i % 2, where dS replaces it; dP has one buffer.
      auto score = [&](int i) {
        const int ks = i % Cfg::kKStages;
        if (!ctl.wait(k_full(ks), (i / Cfg::kKStages) & 1, MUP_ST_MMA_FULL_TIMEOUT)) return false;
        zero_unseen_rows<DP>(smem + Cfg::kOffK + ks * Cfg::kTileBytes, tiles, tiles.tile(i) * kTileRows, lane);
        tc_fence_after_sync();
        if (leader) {
          umma_rows_by_rows<DP>(tmem + (i & 1) * kTileRows, base + Cfg::kOffQ, base + Cfg::kOffK + ks * Cfg::kTileBytes);
          umma_commit_1(s_full(i & 1));
        }
        return true;
      };
      auto score_gradient = [&](int i) {
        const int vs = i % Cfg::kVStages;
        if (!ctl.wait(v_full(vs), (i / Cfg::kVStages) & 1, MUP_ST_MMA_FULL_TIMEOUT)) return false;
        tc_fence_after_sync();
        if (leader) {
          umma_rows_by_rows<DP>(tmem + Cfg::kTmemDp, base + Cfg::kOffDo, base + Cfg::kOffV + vs * Cfg::kTileBytes);
          umma_commit_1(dp_full);
          umma_commit_1(v_empty(vs));
        }
        return true;
      };
      bool ok = ctl.wait(q_full, 0, MUP_ST_MMA_FULL_TIMEOUT);
      ok = ok && score(0) && score_gradient(0);
      for (int i = 0; ok && i < n; ++i) {
        if (i + 1 < n) ok = score(i + 1);
        ok = ok && ctl.wait(ds_full, i & 1, MUP_ST_MMA_ACC_TIMEOUT);
        if (ok && i + 1 < n) ok = score_gradient(i + 1);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          const int ks = i % Cfg::kKStages;
          umma_tmem_by_cols<DP>(tmem + Cfg::kTmemDq, tmem + (i & 1) * kTileRows, 64,
                                base + Cfg::kOffK + ks * Cfg::kTileBytes, i > 0);
          umma_commit_1(k_empty(ks));
          if (i + 1 == n) umma_commit_1(done);
        }
      }
    }
  } else {
    more_registers<216>();
    // Two warpgroups share a tile's columns: thread = query row, 64 keys each.
    const int half = warp / 4, quarter = warp % 4;
    const int row = row0 + quarter * 32 + lane;
    const bool valid = row < seq.nq;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const RowSpan span = row_span(p.shape, seq, row);
    const int64_t index = (static_cast<int64_t>(batch) * p.shape.heads_q + head) * p.shape.seq_q + seq.q0 + row;
    const float c = p.shape.scale_log2;
    grid_dep_wait();
    const float shift = valid ? -p.lse2[index] : -INFINITY;
    const float delta = valid ? p.delta[index] : 0.0f;
    const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift), delta2 = make_float2(-delta, -delta);
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int j0 = tiles.tile(i) * kTileRows + half * 64;
      const uint32_t s_tmem = tmem + (i & 1) * kTileRows + half * 64 + lane_base;
      if (!ctl.wait(s_full(i & 1), (i >> 1) & 1, MUP_ST_EPILOGUE_TIMEOUT)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const bool full = tile_is_full(first, last, tiles.tile(i) * kTileRows);
      uint32_t s[2][32];
      tmem_ld_32x32(s_tmem, s[0]);
      tmem_ld_32x32(s_tmem + 32, s[1]);
      tmem_ld_wait();
      if (!full) {
        const int low = span.low - j0, high = span.high - j0, sink = span.sink - j0;
#pragma unroll
        for (int b = 0; b < 2; ++b) hide_scores(s[b], span_bits(low - b * 32, high - b * 32, sink - b * 32));
      }
#pragma unroll
      for (int x = 0; x < 64; x += 2) {
        uint32_t& s0 = s[x / 32][x % 32];
        uint32_t& s1 = s[x / 32][x % 32 + 1];
        const float2 e = fma2(make_float2(__uint_as_float(s0), __uint_as_float(s1)), c2, shift2);
        s0 = __float_as_uint(exp2_sfu(e.x));
        s1 = __float_as_uint(exp2_sfu(e.y));
      }
      if (!ctl.wait(dp_full, i & 1, MUP_ST_EPILOGUE_TIMEOUT)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t g[32];
        tmem_ld_32x32(tmem + Cfg::kTmemDp + half * 64 + b * 32 + lane_base, g);
        tmem_ld_wait();
        if (!full) {  // where P is 0 the value row may hold anything
#pragma unroll
          for (int x = 0; x < 32; ++x) g[x] = s[b][x] == 0u ? 0u : g[x];
        }
        uint32_t packed[16];
#pragma unroll
        for (int x = 0; x < 32; x += 2) {
          const float2 d = mul2(make_float2(__uint_as_float(s[b][x]), __uint_as_float(s[b][x + 1])),
                                add2(make_float2(__uint_as_float(g[x]), __uint_as_float(g[x + 1])), delta2));
          packed[x / 2] = pack_bf16(d.x, d.y);
        }
        tmem_st_32x16(s_tmem + b * 16, packed);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(ds_full);
    }
    if (ok && n > 0) ok = ctl.wait(done, 0, MUP_ST_EPILOGUE_TIMEOUT);
    if (ok) {
      tc_fence_after_sync();
      // both warpgroups' columns of a row are written in halves of a row, through Q's place (no product reads it now)
      uint8_t* staged = smem + Cfg::kOffQ + half * (kTileRows * DP);
      const int r = quarter * 32 + lane;
#pragma unroll 1
      for (int b = 0; b < DP / 64; ++b) {
        uint32_t g[32];
        if (n > 0) {
          tmem_ld_32x32(tmem + Cfg::kTmemDq + half * (DP / 2) + b * 32 + lane_base, g);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) g[x] = 0u;
        }
#pragma unroll
        for (int x = 0; x < 32; x += 8) *staged_piece<DP>(staged, r, b * 4 + x / 8) = pack_bf16x8(g + x, p.shape.scale);
      }
      write_staged_rows<DP>(staged, quarter * 32, lane, p.shape.head_dim * 2 - half * DP, [&](int x) {
        return row0 + x >= seq.nq ? nullptr
                                  : reinterpret_cast<uint8_t*>(p.dq + batch * p.dq_batch + (seq.q0 + row0 + x) * p.dq_seq +
                                                               head * p.dq_head + half * (DP / 2));
      });
    }
    tc_fence_before_sync();
  }
  __syncthreads();
  if (*abort_flag != 0u) {  // (nobody sets it any more: all threads take this branch or none)
    // a role may have issued its last product or copy before another gave up
    if (warp == 9) drain_products(drain);
    if (threadIdx.x == 0 && n > 0) {
      drain_barrier(q_full, 0);
      drain_ring(k_full(0), Cfg::kKStages, copies[0]);
      drain_ring(v_full(0), Cfg::kVStages, copies[1]);
    }
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// dK, dV
// ---------------------------------------------------------------------------

// The query tiles that see something of a key tile, times the heads of the group, and how they are cut into shares.
struct KeyTileSteps {
  int q_tile0, q_tiles, steps;
  __device__ __forceinline__ KeyTileSteps(const AttnShape& p, const AttnSeq& seq, int tile) {
    const int j0 = tile * kTileRows, j1 = min(j0 + kTileRows, seq.nk) - 1;
    const bool has_sinks = j0 < p.sinks;
    const int low = has_sinks ? (p.causal ? max(0, j0 - seq.off) : 0) : max(0, j0 - p.right - seq.off);
    const int high = has_sinks ? seq.nq - 1 : min(seq.nq - 1, j1 + p.left - seq.off);
    q_tile0 = low / kTileRows;
    q_tiles = high < low ? 0 : high / kTileRows - q_tile0 + 1;
    steps = q_tiles * (p.heads_q / p.heads_kv);
  }
  __device__ __forceinline__ int per_share(int shares) const { return (steps + shares - 1) / shares; }
  // shares that have steps (the first one counts as such: it writes zeros where nothing sees the tile)
  __device__ __forceinline__ int used(int shares) const {
    const int each = per_share(shares);
    return each == 0 ? 1 : (steps + each - 1) / each;
  }
};

template <int DP>
struct AttnDkvConfig {
  static constexpr int kPanels = DP / 64;
  static constexpr int kTileBytes = kPanels * kPanelBytes;
  static constexpr int kQStages = 3, kDoStages = 2, kStatStages = 2;
  static constexpr int kOffK = 0, kOffV = kTileBytes, kOffQ = 2 * kTileBytes;
  static constexpr int kOffDo = kOffQ + kQStages * kTileBytes;
  static constexpr int kOffStats = kOffDo + kDoStages * kTileBytes;  // per stage: 128 lse2, 128 delta
  static constexpr int kOffBars = kOffStats + kStatStages * 1024;
  // k and v full, q full/empty, dO full/empty, stats full/empty, s, dp, p, ds full, done, drain
  static constexpr int kBars = 1 + 2 * kQStages + 2 * kDoStages + 2 * kStatStages + 6;
  static constexpr int kOffWords = kOffBars + kBars * 8;
  static constexpr int kSmemBytes = kOffWords + 16;  // TMEM's address, abort, copies into the two rings
  static constexpr int kTmemDp = 128, kTmemDv = 256, kTmemDk = 384;
};

template <int DP>
__device__ __forceinline__ void attention_dkv(const AttnBackward& p, const CUtensorMap& q_map, const CUtensorMap& k_map,
                                              const CUtensorMap& v_map, const CUtensorMap& do_map, uint8_t* smem,
                                              int job) {
  using Cfg = AttnDkvConfig<DP>;
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto bar = [&](int i) { return base + Cfg::kOffBars + i * 8; };
  const uint32_t kv_full = bar(0);
  const auto q_full = [&](int s) { return bar(1 + s); };
  const auto q_empty = [&](int s) { return bar(1 + Cfg::kQStages + s); };
  constexpr int kD = 1 + 2 * Cfg::kQStages;
  const auto do_full = [&](int s) { return bar(kD + s); };
  const auto do_empty = [&](int s) { return bar(kD + Cfg::kDoStages + s); };
  constexpr int kT = kD + 2 * Cfg::kDoStages;
  const auto stat_full = [&](int s) { return bar(kT + s); };
  const auto stat_empty = [&](int s) { return bar(kT + Cfg::kStatStages + s); };
  constexpr int kS = kT + 2 * Cfg::kStatStages;
  const uint32_t s_full = bar(kS), dp_full = bar(kS + 1), p_full = bar(kS + 2), ds_full = bar(kS + 3);
  const uint32_t done = bar(kS + 4), drain = bar(kS + 5);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffWords);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffWords + 4);
  volatile uint32_t* copies = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffWords + 8);
  const WaitControl ctl{abort_flag, p.shape.status, p.shape.timeout_ns};

  // ---- the key tile, and this CTA's share of the query tiles that see it
  const int heads_kv = p.shape.heads_kv, group = p.shape.heads_q / heads_kv;
  const int shared_jobs = p.n_sequences * heads_kv * p.shared_tiles * p.shares;
  int sequence, tile, kv_head, share = 0, shares = 1;
  AttnSeq seq;
  if (job < shared_jobs) {
    share = job % p.shares, shares = p.shares;
    job /= p.shares;
    tile = job % p.shared_tiles;
    kv_head = job / p.shared_tiles % heads_kv;
    sequence = job / p.shared_tiles / heads_kv;
    seq = load_sequence(p.shape, sequence);
  } else {
    job -= shared_jobs;
    kv_head = job % heads_kv;
    job /= heads_kv;
    if (p.k_blocks != nullptr) {
      int row0;
      seq = load_block(p.k_blocks, job, sequence, row0);
      tile = row0 / kTileRows;
      if (tile < p.shared_tiles) return;
    } else {
      sequence = job % p.shape.batch, tile = p.shared_tiles + job / p.shape.batch;
      seq = load_sequence(p.shape, sequence);
    }
  }
  const int batch = p.shape.sequences != nullptr ? 0 : sequence;
  const int j0 = tile * kTileRows;
  if (j0 >= seq.nk) return;  // packed: a shared tile that this sequence does not have
  const bool has_sinks = j0 < p.shape.sinks;
  const KeyTileSteps work(p.shape, seq, tile);
  const int q_tile0 = work.q_tile0, q_tiles = work.q_tiles;
  const int per_share = work.per_share(shares);
  const int begin = min(share * per_share, work.steps), n = min(begin + per_share, work.steps) - begin;
  if (share > 0 && n == 0) return;  // (the joining kernel knows)

  if (threadIdx.x == 0) {
    *abort_flag = 0u, copies[0] = copies[1] = 0u;
    for (int i = 0; i < Cfg::kBars; ++i) {
      const uint32_t b = bar(i);
      const bool all_threads = b == p_full || b == ds_full || (b >= stat_empty(0) && b < s_full);
      mbar_init(b, all_threads ? 256 : b >= stat_full(0) && b < stat_empty(0) ? 32 : 1);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    fewer_registers<72>();
    if (warp == 8 && elect_one_sync() && n > 0) {
      int i = 0, query_copies = 0;
      auto load = [&](const CUtensorMap& map, uint32_t dst, uint32_t full, int row, int h) {
#pragma unroll
        for (int panel = 0; panel < Cfg::kPanels; ++panel)
          tma_load_4d(dst + panel * kPanelBytes, &map, panel * 64, row, h, batch, full);
      };
      mbar_arrive_expect_tx(kv_full, 2 * Cfg::kTileBytes);
      load(k_map, base + Cfg::kOffK, kv_full, seq.k0 + j0, kv_head);
      load(v_map, base + Cfg::kOffV, kv_full, seq.k0 + j0, kv_head);
      for (; i < n; ++i) {
        const int qs = i % Cfg::kQStages, ds = i % Cfg::kDoStages;
        const int head = kv_head * group + (begin + i) / q_tiles;
        const int row = seq.q0 + (q_tile0 + (begin + i) % q_tiles) * kTileRows;
        if (i >= Cfg::kQStages && !ctl.wait_alone(q_empty(qs), (i / Cfg::kQStages - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT)) break;
        mbar_arrive_expect_tx(q_full(qs), Cfg::kTileBytes);
        load(q_map, base + Cfg::kOffQ + qs * Cfg::kTileBytes, q_full(qs), row, head);
        ++query_copies;
        if (i >= Cfg::kDoStages && !ctl.wait_alone(do_empty(ds), (i / Cfg::kDoStages - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT)) break;
        mbar_arrive_expect_tx(do_full(ds), Cfg::kTileBytes);
        load(do_map, base + Cfg::kOffDo + ds * Cfg::kTileBytes, do_full(ds), row, head);
      }
      copies[0] = query_copies, copies[1] = i;
    } else if (warp == 10) {
      // ------------------------------------------- lse and delta of the query rows
      grid_dep_wait();
      for (int i = 0; i < n; ++i) {
        const int st = i % Cfg::kStatStages;
        const int head = kv_head * group + (begin + i) / q_tiles;
        const int row0 = (q_tile0 + (begin + i) % q_tiles) * kTileRows;
        const int64_t index = (static_cast<int64_t>(batch) * p.shape.heads_q + head) * p.shape.seq_q + seq.q0 + row0;
        float lse2[4], delta[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // rows behind the sequence's end weigh nothing
          const bool valid = row0 + x * 32 + lane < seq.nq;
          lse2[x] = valid ? p.lse2[index + x * 32 + lane] : INFINITY;
          delta[x] = valid ? p.delta[index + x * 32 + lane] : 0.0f;
        }
        if (i >= Cfg::kStatStages && !ctl.wait(stat_empty(st), (i / Cfg::kStatStages - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT))
          break;
        float* dst = reinterpret_cast<float*>(smem + Cfg::kOffStats + st * 1024);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          dst[x * 32 + lane] = -lse2[x];
          dst[128 + x * 32 + lane] = -delta[x];
        }
        mbar_arrive(stat_full(st));
      }
    } else if (warp == 9 && n > 0) {
      const bool leader = elect_one_sync();
      // rows that see nothing, and those of a query tile behind the sequence's end (packed: the next sequence's), become 0
      const int blind = !p.shape.causal && has_sinks ? 0 : -seq.off - p.shape.right;  // so many first ones
      auto clean = [&](int i, uint8_t* where) {
        const int row0 = (q_tile0 + (begin + i) % q_tiles) * kTileRows;
        const bool ends = p.shape.sequences != nullptr && row0 + kTileRows > seq.nq;
        if (row0 >= blind && !ends) return;
        if (row0 < blind) zero_tile_rows<DP>(where, 0, min(blind - row0, kTileRows), lane);
        if (ends) zero_tile_rows<DP>(where, seq.nq - row0, kTileRows, lane);
        fence_proxy_async_smem();
        __syncwarp();
      };
      auto score = [&](int i) {
        const int qs = i % Cfg::kQStages;
        if (!ctl.wait(q_full(qs), (i / Cfg::kQStages) & 1, MUP_ST_MMA_FULL_TIMEOUT)) return false;
        clean(i, smem + Cfg::kOffQ + qs * Cfg::kTileBytes);
        tc_fence_after_sync();
        if (leader) {
          umma_rows_by_rows<DP>(tmem, base + Cfg::kOffK, base + Cfg::kOffQ + qs * Cfg::kTileBytes);
          umma_commit_1(s_full);
        }
        return true;
      };
      auto score_gradient = [&](int i) {
        const int ds = i % Cfg::kDoStages;
        if (!ctl.wait(do_full(ds), (i / Cfg::kDoStages) & 1, MUP_ST_MMA_FULL_TIMEOUT)) return false;
        clean(i, smem + Cfg::kOffDo + ds * Cfg::kTileBytes);
        tc_fence_after_sync();
        if (leader) {
          umma_rows_by_rows<DP>(tmem + Cfg::kTmemDp, base + Cfg::kOffV, base + Cfg::kOffDo + ds * Cfg::kTileBytes);
          umma_commit_1(dp_full);
        }
        return true;
      };
      bool ok = ctl.wait(kv_full, 0, MUP_ST_MMA_FULL_TIMEOUT);
      ok = ok && score(0) && score_gradient(0);
      for (int i = 0; ok && i < n; ++i) {
        const int qs = i % Cfg::kQStages, ds = i % Cfg::kDoStages;
        // P(i) -> dV and S(i + 1) while dS(i) is computed, dS(i) -> dK and dP(i + 1) while P(i + 1) is
        ok = ctl.wait(p_full, i & 1, MUP_ST_MMA_ACC_TIMEOUT);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          umma_tmem_by_cols<DP>(tmem + Cfg::kTmemDv, tmem, 64, base + Cfg::kOffDo + ds * Cfg::kTileBytes, i > 0);
          umma_commit_1(do_empty(ds));
        }
        if (i + 1 < n) ok = score(i + 1);
        ok = ok && ctl.wait(ds_full, i & 1, MUP_ST_MMA_ACC_TIMEOUT);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          umma_tmem_by_cols<DP>(tmem + Cfg::kTmemDk, tmem + Cfg::kTmemDp, 64, base + Cfg::kOffQ + qs * Cfg::kTileBytes, i > 0);
          umma_commit_1(q_empty(qs));
          if (i + 1 == n) umma_commit_1(done);
        }
        if (i + 1 < n) ok = score_gradient(i + 1);
      }
    }
  } else {
    more_registers<216>();
    // Two warpgroups share a tile's columns: thread = key row, 64 queries each.
    const int half = warp / 4, quarter = warp % 4;
    const int j = j0 + quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const float2 c2 = make_float2(p.shape.scale_log2, p.shape.scale_log2);
    // the query rows that see key j: [see_low, see_high]
    const bool is_sink = j < p.shape.sinks;
    int see_low = (is_sink && !p.shape.causal ? -kNoLimit : j - (is_sink ? 0 : p.shape.right)) - seq.off;
    int see_high = is_sink ? kNoLimit : j - seq.off + p.shape.left;
    if (j >= seq.nk) see_low = kNoLimit, see_high = -1;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int row0 = (q_tile0 + (begin + i) % q_tiles) * kTileRows;
      // every row of the query tile sees every key of the tile
      const int at_first = row0 + seq.off, at_last = min(row0 + kTileRows, seq.nq) - 1 + seq.off;
      bool full = j0 + kTileRows <= seq.nk;
      if (j0 + kTileRows <= p.shape.sinks)
        full = full && (!p.shape.causal || at_first >= j0 + kTileRows - 1);
      else
        full = full && !has_sinks && at_first + p.shape.right >= j0 + kTileRows - 1 && at_last - p.shape.left <= j0;
      const int st = i % Cfg::kStatStages;
      const float4* stats = reinterpret_cast<const float4*>(smem + Cfg::kOffStats + st * 1024) + half * 16;
      if (!ctl.wait(stat_full(st), (i / Cfg::kStatStages) & 1, MUP_ST_EPILOGUE_TIMEOUT) ||
          !ctl.wait(s_full, i & 1, MUP_ST_EPILOGUE_TIMEOUT)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      uint32_t s[2][32];
      tmem_ld_32x32(tmem + half * 64 + lane_base, s[0]);
      tmem_ld_32x32(tmem + half * 64 + 32 + lane_base, s[1]);
      tmem_ld_wait();
      if (!full) {
        const int low = see_low - row0 - half * 64, high = see_high - row0 - half * 64;
#pragma unroll
        for (int b = 0; b < 2; ++b) hide_scores(s[b], span_bits(low - b * 32, high - b * 32, 0));
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t packed[16];
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
          const float4 shift = stats[b * 8 + x / 4];
          const float2 e0 = fma2(make_float2(__uint_as_float(s[b][x]), __uint_as_float(s[b][x + 1])), c2, make_float2(shift.x, shift.y));
          const float2 e1 = fma2(make_float2(__uint_as_float(s[b][x + 2]), __uint_as_float(s[b][x + 3])), c2, make_float2(shift.z, shift.w));
          const float p0 = exp2_sfu(e0.x), p1 = exp2_sfu(e0.y), p2 = exp2_sfu(e1.x), p3 = exp2_sfu(e1.y);
          s[b][x] = __float_as_uint(p0), s[b][x + 1] = __float_as_uint(p1);
          s[b][x + 2] = __float_as_uint(p2), s[b][x + 3] = __float_as_uint(p3);
          packed[x / 2] = pack_bf16(p0, p1);
          packed[x / 2 + 1] = pack_bf16(p2, p3);
        }
        tmem_st_32x16(tmem + half * 64 + b * 16 + lane_base, packed);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(p_full);
      if (!ctl.wait(dp_full, i & 1, MUP_ST_EPILOGUE_TIMEOUT)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t g[32];
        tmem_ld_32x32(tmem + Cfg::kTmemDp + half * 64 + b * 32 + lane_base, g);
        tmem_ld_wait();
        if (!full) {  // where P is 0 the key's value row may hold anything
#pragma unroll
          for (int x = 0; x < 32; ++x) g[x] = s[b][x] == 0u ? 0u : g[x];
        }
        uint32_t packed[16];
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
          const float4 delta = stats[32 + b * 8 + x / 4];
          const float2 d0 = mul2(make_float2(__uint_as_float(s[b][x]), __uint_as_float(s[b][x + 1])),
                                 add2(make_float2(__uint_as_float(g[x]), __uint_as_float(g[x + 1])), make_float2(delta.x, delta.y)));
          const float2 d1 = mul2(make_float2(__uint_as_float(s[b][x + 2]), __uint_as_float(s[b][x + 3])),
                                 add2(make_float2(__uint_as_float(g[x + 2]), __uint_as_float(g[x + 3])), make_float2(delta.z, delta.w)));
          packed[x / 2] = pack_bf16(d0.x, d0.y);
          packed[x / 2 + 1] = pack_bf16(d1.x, d1.y);
        }
        tmem_st_32x16(tmem + Cfg::kTmemDp + half * 64 + b * 16 + lane_base, packed);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(ds_full);
      mbar_arrive(stat_empty(st));
    }
    if (ok && n > 0) ok = ctl.wait(done, 0, MUP_ST_EPILOGUE_TIMEOUT);
    if (ok) {
      tc_fence_after_sync();
      // one warpgroup writes dV, the other dK
      const float scale = half == 0 ? 1.0f : p.shape.scale;
      const uint32_t src = tmem + (half == 0 ? Cfg::kTmemDv : Cfg::kTmemDk) + lane_base;
      const int64_t slot = ((static_cast<int64_t>(sequence) * heads_kv + kv_head) * p.shared_tiles + tile) * shares + share;
      // through V's and K's places: no product reads them now
      uint8_t* staged = smem + (half == 0 ? Cfg::kOffV : Cfg::kOffK);
      constexpr int kRowBytes = DP * 2;
      const int r = quarter * 32 + lane;
      const auto load_sum = [&](int b, uint32_t(&g)[32]) {
        if (n > 0) {
          tmem_ld_32x32(src + b * 32, g);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) g[x] = 0u;
        }
      };
      if (shares > 1) {  // half of the FP32 columns at a time
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
#pragma unroll 1
          for (int b = 0; b < DP / 64; ++b) {
            uint32_t g[32];
            load_sum(part * (DP / 64) + b, g);
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *staged_piece<kRowBytes>(staged, r, b * 8 + x / 4) = make_uint4(g[x], g[x + 1], g[x + 2], g[x + 3]);
          }
          write_staged_rows<kRowBytes>(staged, quarter * 32, lane, kRowBytes, [&](int x) {
            return reinterpret_cast<uint8_t*>(p.partial + ((slot * 2 + half) * kTileRows + x) * DP + part * (DP / 2));
          });
        }
      } else {
#pragma unroll 1
        for (int b = 0; b < DP / 32; ++b) {
          uint32_t g[32];
          load_sum(b, g);
#pragma unroll
          for (int x = 0; x < 32; x += 8) *staged_piece<kRowBytes>(staged, r, b * 4 + x / 8) = pack_bf16x8(g + x, scale);
        }
        write_staged_rows<kRowBytes>(staged, quarter * 32, lane, p.shape.head_dim * 2, [&](int x) {
          if (j0 + x >= seq.nk) return static_cast<uint8_t*>(nullptr);
          return reinterpret_cast<uint8_t*>(
              half == 0 ? p.dv + batch * p.dv_batch + (seq.k0 + j0 + x) * p.dv_seq + kv_head * p.dv_head
                        : p.dk + batch * p.dk_batch + (seq.k0 + j0 + x) * p.dk_seq + kv_head * p.dk_head);
        });
      }
    }
    tc_fence_before_sync();
  }
  __syncthreads();
  if (*abort_flag != 0u) {  // (nobody sets it any more: all threads take this branch or none)
    // a role may have issued its last product or copy before another gave up
    if (warp == 9) drain_products(drain);
    if (threadIdx.x == 0 && n > 0) {
      drain_barrier(kv_full, 0);
      drain_ring(q_full(0), Cfg::kQStages, copies[0]);
      drain_ring(do_full(0), Cfg::kDoStages, copies[1]);
    }
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, 512);
  }
}

// Both in one launch, the CTAs of dK and dV (the longer ones) first: neither needs the other, and small problems fill the
// GPU better together. Launched while the delta kernel runs; the warps that read its results wait for it.
template <int DP>
struct AttnBackwardConfig {
  static constexpr int kSmemBytes = AttnDqConfig<DP>::kSmemBytes > AttnDkvConfig<DP>::kSmemBytes
                                        ? AttnDqConfig<DP>::kSmemBytes
                                        : AttnDkvConfig<DP>::kSmemBytes;
};

template <int DP>
__global__ void __launch_bounds__(384, 1)
    attention_backward_kernel(const __grid_constant__ AttnBackward p, const __grid_constant__ CUtensorMap q_map,
                              const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                              const __grid_constant__ CUtensorMap do_map) {
  extern __shared__ __align__(1024) uint8_t smem[];
  grid_dep_launch();
  const int job = blockIdx.x;
  if (job < p.dkv_jobs)
    attention_dkv<DP>(p, q_map, k_map, v_map, do_map, smem, job);
  else
    attention_dq<DP>(p, q_map, k_map, v_map, do_map, smem, job - p.dkv_jobs);
}

// Sums the shares of the shared key tiles, always in the same order: one thread per four columns of dV or dK.
template <int DP>
__global__ void __launch_bounds__(256) attention_dkv_join_kernel(const __grid_constant__ AttnBackward p) {
  constexpr int kQuads = DP / 4;
  grid_dep_wait();
  int64_t item = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x);
  const int quad = static_cast<int>(item % kQuads);
  item /= kQuads;
  const int r = static_cast<int>(item % kTileRows);
  item /= kTileRows;
  const int which = static_cast<int>(item % 2);
  item /= 2;
  const int tile = static_cast<int>(item % p.shared_tiles);
  item /= p.shared_tiles;
  const int kv_head = static_cast<int>(item % p.shape.heads_kv);
  const int sequence = static_cast<int>(item / p.shape.heads_kv);
  if (sequence >= p.n_sequences || quad * 4 >= p.shape.head_dim) return;
  const AttnSeq seq = load_sequence(p.shape, sequence);
  const int j = tile * kTileRows + r;
  if (j >= seq.nk) return;
  const int64_t slot = ((static_cast<int64_t>(sequence) * p.shape.heads_kv + kv_head) * p.shared_tiles + tile) * p.shares;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const int used = KeyTileSteps(p.shape, seq, tile).used(p.shares);
  for (int s = 0; s < used; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(p.partial + (((slot + s) * 2 + which) * kTileRows + r) * DP + quad * 4);
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  const float scale = which == 0 ? 1.0f : p.shape.scale;
  const int batch = p.shape.sequences != nullptr ? 0 : sequence;
  __nv_bfloat16* dst = which == 0 ? p.dv + batch * p.dv_batch + (seq.k0 + j) * p.dv_seq + kv_head * p.dv_head
                                  : p.dk + batch * p.dk_batch + (seq.k0 + j) * p.dk_seq + kv_head * p.dk_head;
  *reinterpret_cast<uint2*>(dst + quad * 4) =
      make_uint2(pack_bf16(sum.x * scale, sum.y * scale), pack_bf16(sum.z * scale, sum.w * scale));
}

}  // namespace mup

// Forward pass for few query rows (tokens over a cache): at most 16 rows of a key/value head's group.
//
// Bound by reading the visible keys and values once, and for short windows by latency. One 16-row tile of mma.sync
// products holds all rows: the tensor work is negligible, and tcgen05's 128-row tiles would be empty for the most part.
// One warp keeps a ring of 64-key tiles filled by TMA, so that many tiles are in flight whatever the others do; four warps
// take 16 keys of every tile each: S = Q K^T (m16n8k16, K by ldmatrix), softmax in registers, O += P V (V by
// ldmatrix.trans). The warps of a CTA join their (maximum, sum, O) in shared memory; CTAs that share a sequence join
// through the shared memory of their cluster where there are few, else through the workspace and the combining kernel.
// Roundings are those of the 128-row kernel: P to BF16 for the second product, then the result.
//
// Measured on B200: one token of 4 heads over a window of 1024 keys 7.1 us; 16 tokens of 8 heads over caches of 8192 to
// 65536 keys (308 MB) 57 us, 5.4 TB/s, 82 % of the copy rate. Two CTAs of three 32 KB tiles per SM; one of six 60 us, two of
// two 70 us, three of two 58 us (registers spill). Before, with every lane loading its own fragments and no ring: 67 us,
// and with a ring of 16-byte cp.async copies 71 us.
#pragma once

#include "mup_attn_forward.cuh"

namespace mup {

constexpr int kTokenRows = 16, kTokenKeys = 64, kTokenWarps = 4, kTokenCluster = 8;
constexpr int kTokenCtas = 2;  // per SM: one's start and end beside the other's stream

struct AttnTokens {
  AttnShape shape;
  const __nv_bfloat16* q;
  int64_t q_batch, q_seq, q_head;
  int splits;   // CTAs per sequence and key/value head
  int share;    // key tiles of a CTA, or 0: a splits-th of its sequence's
  int cluster;  // the CTAs of a sequence and head are one cluster
  __nv_bfloat16 *out, *out_rest;  // out_rest: what out's rounding leaves, or null
  int64_t out_batch, out_seq, out_head;
  float* lse;          // [batch, heads, rows] or null
  float* partial_out;  // [splits, total rows, DP] and
  float* partial_lse;  // [splits, total rows], base 2, when splits > 1 and not a cluster
  int64_t total_rows;
};

template <int DP>
struct AttnTokensConfig {
  static constexpr int kPanels = DP / 64;
  static constexpr int kPanelBytes = kTokenKeys * 128;
  static constexpr int kTileBytes = kPanels * kPanelBytes;  // of K or V
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int kRowFloats = DP + 4;  // rows start in different banks
  static constexpr int kJoinFloats = kTokenWarps * kTokenRows * (kRowFloats + 2);  // in the ring's place afterwards
  static constexpr int kOffBars = kStages * 2 * kTileBytes;
  static constexpr int kOffAbort = kOffBars + 2 * kStages * 8;
  static constexpr int kSmemBytes = kOffAbort + 16;
  static constexpr int kThreads = 32 * (kTokenWarps + 1);
  static_assert(kJoinFloats * 4 <= kOffBars);
};

// D[16 x 8] += A[16 x 16] B[16 x 8], BF16 in, FP32 out.
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four 8 x 8 matrices of 16-bit elements; lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

template <int DP>
__global__ void __launch_bounds__(AttnTokensConfig<DP>::kThreads, kTokenCtas)
    attention_tokens_kernel(const __grid_constant__ AttnTokens p, const __grid_constant__ CUtensorMap k_map,
                            const __grid_constant__ CUtensorMap v_map) {
  using Cfg = AttnTokensConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const auto full = [&](int s) { return base + Cfg::kOffBars + s * 8; };
  const auto empty = [&](int s) { return base + Cfg::kOffBars + (Cfg::kStages + s) * 8; };
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + Cfg::kOffAbort);
  const WaitControl ctl{abort_flag, p.shape.status, p.shape.timeout_ns};
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  grid_dep_launch();
  grid_dep_wait();
  int w = blockIdx.x;
  const int split = w % p.splits;
  w /= p.splits;
  const int kv_head = w % p.shape.heads_kv, sequence = w / p.shape.heads_kv;
  const AttnSeq seq = load_sequence(p.shape, sequence);
  const int batch = p.shape.sequences != nullptr ? 0 : sequence;
  const int group = p.shape.heads_q / p.shape.heads_kv;
  const int rows = group * seq.nq;  // row r: query r % nq of head r / nq
  const int dim = p.shape.head_dim;

  // ---- this CTA's key tiles
  const RowSpan first = row_span(p.shape, seq, 0), last = row_span(p.shape, seq, max(seq.nq, 1) - 1);
  const TileList tiles = make_tile_list(first, last, kTokenKeys);
  const int count = rows > 0 ? tiles.count : 0;
  const int each = p.share > 0 ? p.share : (count + p.splits - 1) / p.splits;
  const int begin = min(split * each, count), end = min(begin + each, count);
  if (p.share > 0 && split > 0 && begin == count) {  // a sequence shorter than the longest
    if (threadIdx.x < rows) {
      const int head = kv_head * group + threadIdx.x / seq.nq, query = seq.q0 + threadIdx.x % seq.nq;
      p.partial_lse[split * p.total_rows + (static_cast<int64_t>(batch) * p.shape.heads_q + head) * p.shape.seq_q + query] =
          -INFINITY;
    }
    return;
  }

  const bool loads_here = warp == kTokenWarps && elect_one_sync();
  const auto load_tile = [&](int i) {
    const int s = (i - begin) % Cfg::kStages;
    const uint32_t dst = base + s * 2 * Cfg::kTileBytes;
    const int row = seq.k0 + tiles.tile(i) * kTokenKeys;
    mbar_arrive_expect_tx(full(s), 2 * Cfg::kTileBytes);
#pragma unroll
    for (int panel = 0; panel < Cfg::kPanels; ++panel)
      tma_load_4d(dst + panel * Cfg::kPanelBytes, &k_map, panel * 64, row, kv_head, batch, full(s));
#pragma unroll
    for (int panel = 0; panel < Cfg::kPanels; ++panel)
      tma_load_4d(dst + Cfg::kTileBytes + panel * Cfg::kPanelBytes, &v_map, panel * 64, row, kv_head, batch, full(s));
  };
  if (loads_here) {
    *abort_flag = 0u;
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), kTokenWarps);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
    for (int i = begin; i < min(end, begin + Cfg::kStages); ++i) load_tile(i);  // these wait for nobody
  }

  float o[DP / 8][4] = {};
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  int loads = min(end - begin, Cfg::kStages);
  const float c2 = p.shape.scale_log2;
  if (warp == kTokenWarps) {
    __syncthreads();
    if (loads_here) {
      for (int i = begin + Cfg::kStages; i < end; ++i) {
        const int n = i - begin;
        if (!ctl.wait_alone(empty(n % Cfg::kStages), (n / Cfg::kStages - 1) & 1, MUP_ST_PRODUCER_SLOT_TIMEOUT)) break;
        load_tile(i);
        ++loads;
      }
    }
  } else {
    // ---- the query rows g and g + 8, as the products' left fragments
    uint32_t q_frag[DP / 16][4];
    RowSpan span[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + h * 8;
      const int head = kv_head * group + (rows > 0 ? r / seq.nq : 0), row = rows > 0 ? r % seq.nq : 0;
      span[h] = row_span(p.shape, seq, row);
      const __nv_bfloat16* src = p.q + batch * p.q_batch + (seq.q0 + row) * p.q_seq + head * p.q_head + t * 2;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          q_frag[s][h + 2 * e] = r < rows && s * 16 + e * 8 < dim ? *reinterpret_cast<const uint32_t*>(src + s * 16 + e * 8) : 0u;
    }
    __syncthreads();
    // a lane's row addresses inside a panel, for K and for V
    const int matrix = lane / 8;
    const int k_row = warp * 16 + (matrix >> 1) * 8 + lane % 8, v_row = warp * 16 + (matrix & 1) * 8 + lane % 8;
    int stage = 0;
    uint32_t phase = 0;
    for (int i = begin; i < end; ++i) {
      const int j0 = tiles.tile(i) * kTokenKeys + warp * 16;
      if (!ctl.wait(full(stage), phase, MUP_ST_MMA_FULL_TIMEOUT)) break;
      if (j0 < tiles.sink_end || (j0 <= tiles.high && j0 + 16 > tiles.low)) {
        const uint32_t k_tile = base + stage * 2 * Cfg::kTileBytes + k_row * 128;
        const uint32_t v_tile = base + stage * 2 * Cfg::kTileBytes + Cfg::kTileBytes + v_row * 128;
        const bool all_seen = tile_is_full(first, last, j0, 16);
        float s[2][4] = {}, s_odd[2][4] = {};  // two sums each: shorter chains of dependent products
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          const int chunk = x * 2 + (matrix & 1);
          uint32_t b[4];
          ldmatrix_x4(b, k_tile + chunk / 8 * Cfg::kPanelBytes + (((chunk % 8) ^ (k_row & 7)) * 16));
          mma_16x8x16(x & 1 ? s_odd[0] : s[0], q_frag[x], b[0], b[1]);
          mma_16x8x16(x & 1 ? s_odd[1] : s[1], q_frag[x], b[2], b[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] += s_odd[n][x];
        uint32_t keep[2] = {~0u, ~0u};  // the value rows that some row sees: others may hold anything
        if (!all_seen) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int j = j0 + n * 8 + t * 2 + (x & 1);
              const RowSpan& r = span[x >> 1];
              if (!(j < r.sink || (j >= r.low && j <= r.high))) s[n][x] = -INFINITY;
              const bool seen = j < tiles.sink_end || (j >= tiles.low && j <= tiles.high);
              if (!seen) keep[n] &= x & 1 ? 0x0000ffffu : 0xffff0000u;
            }
        }
        bool moved = false;
        float factor[2] = {1.0f, 1.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          if (top[h] == -INFINITY) {
            top[h] = m;  // nothing was added yet
          } else if ((m - top[h]) * c2 > kKeepMaximum) {
            factor[h] = exp2_sfu((top[h] - m) * c2);
            top[h] = m;
            moved = true;
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) sum[h] *= factor[h];
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[n][x] *= factor[x >> 1];
        }
        uint32_t weight[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float shift = top[h] == -INFINITY ? 0.0f : -top[h] * c2;
            const float e0 = exp2_sfu(fmaf(s[n][2 * h], c2, shift)), e1 = exp2_sfu(fmaf(s[n][2 * h + 1], c2, shift));
            sum[h] += e0 + e1;
            weight[n * 2 + h] = pack_bf16(e0, e1);
          }
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          const int chunk = n * 2 + (matrix >> 1);
          uint32_t b[4];
          ldmatrix_x4_trans(b, v_tile + chunk / 8 * Cfg::kPanelBytes + (((chunk % 8) ^ (v_row & 7)) * 16));
          if (!all_seen) b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
          mma_16x8x16(o[2 * n], weight, b[0], b[1]);
          mma_16x8x16(o[2 * n + 1], weight, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(stage));
      if (++stage == Cfg::kStages) stage = 0, phase ^= 1;
    }
  }
  __syncthreads();  // every tile has been read: the ring's place is used again
  if (*abort_flag != 0u) {
    if (loads_here) drain_ring(full(0), Cfg::kStages, loads);
    __syncthreads();
  }

  // ---- join the warps
  float* smem_o = reinterpret_cast<float*>(smem);  // [warps, rows, row floats]
  float* smem_top = smem_o + kTokenWarps * kTokenRows * Cfg::kRowFloats;
  float* smem_sum = smem_top + kTokenWarps * kTokenRows;
  if (warp < kTokenWarps) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      float* dst = smem_o + (warp * kTokenRows + g + h * 8) * Cfg::kRowFloats + t * 2;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
      if (t == 0) {
        smem_top[warp * kTokenRows + g + h * 8] = top[h] * c2;  // base 2
        smem_sum[warp * kTokenRows + g + h * 8] = sum[h];
      }
    }
  }
  __syncthreads();
  // kEach threads per row, each DP / kEach columns in steps of kEach (the loading warp has none)
  constexpr int kEach = 32 * kTokenWarps / kTokenRows;
  const bool joins = warp < kTokenWarps;
  const int r = joins ? threadIdx.x / kEach : 0, column = threadIdx.x % kEach;
  float whole_top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kTokenWarps; ++i) whole_top = fmaxf(whole_top, smem_top[i * kTokenRows + r]);
  float whole_sum = 0.0f, joined[DP / kEach] = {};
#pragma unroll
  for (int i = 0; i < kTokenWarps; ++i) {
    const float mine = smem_top[i * kTokenRows + r];
    const float scale = mine == -INFINITY ? 0.0f : exp2_sfu(mine - whole_top);
    whole_sum += scale * smem_sum[i * kTokenRows + r];
#pragma unroll
    for (int x = 0; x < DP / kEach; ++x)
      joined[x] += scale * smem_o[(i * kTokenRows + r) * Cfg::kRowFloats + x * kEach + column];
  }
  if (p.cluster) {
    // this CTA's result takes the place of its first warp's; then every CTA joins its share of the rows of all
    __syncthreads();
    if (joins) {
#pragma unroll
      for (int x = 0; x < DP / kEach; ++x) smem_o[r * Cfg::kRowFloats + x * kEach + column] = joined[x];
      if (column == 0) smem_top[r] = whole_top, smem_sum[r] = whole_sum;
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    // one warp per row, DP / 32 columns per lane
    const int rank = static_cast<int>(cluster_ctarank());
    for (int row = rank + warp * p.splits; joins && row < rows; row += p.splits * kTokenWarps) {
      float tops[kTokenCluster], all_top = -INFINITY, all_sum = 0.0f, acc[DP / 32] = {};
#pragma unroll
      for (int i = 0; i < kTokenCluster; ++i) {
        tops[i] = i < p.splits ? ld_cluster_f32(mapa_cluster(smem_u32(smem_top + row), i)) : -INFINITY;
        all_top = fmaxf(all_top, tops[i]);
      }
#pragma unroll
      for (int i = 0; i < kTokenCluster; ++i) {
        if (i >= p.splits) break;
        const float scale = tops[i] == -INFINITY ? 0.0f : exp2_sfu(tops[i] - all_top);
        all_sum += scale * ld_cluster_f32(mapa_cluster(smem_u32(smem_sum + row), i));
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
          acc[x] += scale * ld_cluster_f32(mapa_cluster(smem_u32(smem_o + row * Cfg::kRowFloats + lane * (DP / 32) + x), i));
      }
      const int head = kv_head * group + row / seq.nq, query = seq.q0 + row % seq.nq;
      const float scale = all_sum == 0.0f ? 0.0f : 1.0f / all_sum;
      const int64_t at = batch * p.out_batch + query * p.out_seq + head * p.out_head + lane * (DP / 32);
#pragma unroll
      for (int x = 0; x < DP / 32; x += 2) {
        if (lane * (DP / 32) + x >= dim) continue;
        *reinterpret_cast<uint32_t*>(p.out + at + x) = pack_bf16(acc[x] * scale, acc[x + 1] * scale);
        if (p.out_rest != nullptr)
          *reinterpret_cast<uint32_t*>(p.out_rest + at + x) = pack_bf16_rest(acc[x] * scale, acc[x + 1] * scale);
      }
      if (p.lse != nullptr && lane == 0)
        p.lse[(static_cast<int64_t>(batch) * p.shape.heads_q + head) * p.shape.seq_q + query] =
            all_sum == 0.0f ? -INFINITY : (all_top + log2f(all_sum)) * 0.69314718055994531f;
    }
    // nobody leaves while another reads its shared memory
    cluster_arrive_release();
    cluster_wait_acquire();
    return;
  }
  if (!joins || r >= rows) return;
  const int head = kv_head * group + r / seq.nq, query = seq.q0 + r % seq.nq;
  const int64_t index = (static_cast<int64_t>(batch) * p.shape.heads_q + head) * p.shape.seq_q + query;
  const float scale = whole_sum == 0.0f ? 0.0f : 1.0f / whole_sum;
  const float lse2 = whole_sum == 0.0f ? -INFINITY : whole_top + log2f(whole_sum);
  if (p.splits > 1) {
    float* dst = p.partial_out + (split * p.total_rows + index) * DP;
#pragma unroll
    for (int x = 0; x < DP / kEach; ++x) dst[x * kEach + column] = joined[x] * scale;
    if (column == 0) p.partial_lse[split * p.total_rows + index] = lse2;
  } else {
    const int64_t at = batch * p.out_batch + query * p.out_seq + head * p.out_head + column;
#pragma unroll
    for (int x = 0; x < DP / kEach; ++x) {
      if (x * kEach + column >= dim) continue;
      const float v = joined[x] * scale;
      const __nv_bfloat16 rounded = __float2bfloat16_rn(v);
      p.out[at + x * kEach] = rounded;
      if (p.out_rest != nullptr) p.out_rest[at + x * kEach] = __float2bfloat16_rn(v - __bfloat162float(rounded));
    }
    if (column == 0 && p.lse != nullptr) p.lse[index] = lse2 * 0.69314718055994531f;
  }
}

}  // namespace mup

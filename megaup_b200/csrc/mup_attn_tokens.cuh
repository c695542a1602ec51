// Forward pass for few query rows (tokens over a cache): at most 16 rows of a key/value head's group.
//
// Bound by reading the visible keys and values once, and for short windows by latency. One 16-row tile of mma.sync
// products holds all rows, so the tensor work is negligible and the 128-row tiles of tcgen05 would be empty for the
// most part; nothing goes through shared memory on the way in: every warp walks 16-key steps of its own, and both operands
// are loaded straight into the fragments of the products, 16 bytes per lane, by choosing which head element each
// index of a product stands for:
//   S = Q K^T, m16n8k16: lane (g, t) = (lane / 4, lane % 4) loads elements 32c + 8t .. + 7 of key g (and of query rows g
//     and g + 8): its 8 elements are the K indices 2t, 2t + 1, 2t + 8, 2t + 9 of two steps, in any order as long as Q's
//     is the same.
//   O += P V: the lane loads elements 64b + 8g .. + 7 of keys 2t, 2t + 1, 2t + 8 and 2t + 9, and N index g of product i
//     stands for element 64b + 8g + i; pairs of keys are joined by byte permutes.
// The warps of a CTA join their (maximum, sum, O) in shared memory; CTAs that share a sequence join through the shared
// memory of their cluster where there are few, else through the workspace and the combining kernel.
//
// Measured on B200: one token of 4 heads over a window of 1024 keys 6.9 us (the 128-row kernel and its join: 11.9 us);
// 16 tokens of 8 heads over caches of 8192 to 65536 keys (300 MB) 67 us, 4.5 TB/s (128-row kernel: 107 us). Two
// CTAs of four warps per SM, this step's and the next one's tiles in registers; with one step in flight 78 us, with
// CTAs of eight warps 86 us.
#pragma once

#include "mup_attn_forward.cuh"

namespace mup {

constexpr int kTokenRows = 16, kTokenStep = 16, kTokenWarps = 4, kTokenCluster = 8;
constexpr int kTokenCtas = 8 / kTokenWarps;  // per SM

struct AttnTokens {
  AttnShape shape;
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_batch, q_seq, q_head, k_batch, k_seq, k_head, v_batch, v_seq, v_head;
  int splits;   // CTAs per sequence and key/value head
  int share;    // steps of a CTA, or 0: a splits-th of its sequence's
  int cluster;  // they are one cluster
  __nv_bfloat16 *out, *out_rest;  // out_rest: what out's rounding leaves, or null
  int64_t out_batch, out_seq, out_head;
  float* lse;          // [batch, heads, rows] or null
  float* partial_out;  // [splits, total rows, DP] and
  float* partial_lse;  // [splits, total rows], base 2, when splits > 1 and not a cluster
  int64_t total_rows;
};

template <int DP>
struct AttnTokensConfig {
  static constexpr int kRowFloats = DP + 4;  // rows start in different banks
  static constexpr int kSmemBytes = kTokenWarps * kTokenRows * (kRowFloats + 2) * 4;  // more than the query fragments
};

// D[16 x 8] += A[16 x 16] B[16 x 8], BF16 in, FP32 out.
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

template <int DP>
__global__ void __launch_bounds__(32 * kTokenWarps, kTokenCtas) attention_tokens_kernel(const __grid_constant__ AttnTokens p) {
  using Cfg = AttnTokensConfig<DP>;
  constexpr int kChunks = DP / 32, kBlocks = DP / 64;
  extern __shared__ __align__(16) float token_smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  int w = blockIdx.x;
  const int split = w % p.splits;
  w /= p.splits;
  const int kv_head = w % p.shape.heads_kv, sequence = w / p.shape.heads_kv;
  grid_dep_launch();
  grid_dep_wait();
  const AttnSeq seq = load_sequence(p.shape, sequence);
  const int batch = p.shape.sequences != nullptr ? 0 : sequence;
  const int group = p.shape.heads_q / p.shape.heads_kv;
  const int rows = group * seq.nq;  // row r: query r % nq of head r / nq
  const int dim = p.shape.head_dim;

  // ---- this warp's steps of 16 keys
  const RowSpan first = row_span(p.shape, seq, 0), last = row_span(p.shape, seq, max(seq.nq, 1) - 1);
  const TileList steps = make_tile_list(first, last, kTokenStep);
  const int count = rows > 0 ? steps.count : 0;
  const int each = ((p.share > 0 ? p.share : (count + p.splits - 1) / p.splits) + kTokenWarps - 1) / kTokenWarps;
  if (p.share > 0 && split * kTokenWarps * each >= count) {  // a sequence shorter than the longest
    if (threadIdx.x < rows) {
      const int head = kv_head * group + threadIdx.x / seq.nq, query = seq.q0 + threadIdx.x % seq.nq;
      p.partial_lse[split * p.total_rows + (static_cast<int64_t>(batch) * p.shape.heads_q + head) * p.shape.seq_q + query] =
          -INFINITY;
    }
    return;
  }
  const int begin = min((split * kTokenWarps + warp) * each, count), end = min(begin + each, count);

  const __nv_bfloat16* k_base = p.k + batch * p.k_batch + seq.k0 * p.k_seq + kv_head * p.k_head + t * 8;
  const __nv_bfloat16* v_base = p.v + batch * p.v_batch + seq.k0 * p.v_seq + kv_head * p.v_head + g * 8;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // keys that no row sees are not read
  const auto seen = [&](int j) { return j < steps.sink_end || (j >= steps.low && j <= steps.high); };
  uint4 k_frag[2][2][kChunks], v_frag[2][kBlocks][4];  // this step's and the next one's
  // where every row sees all of a step's keys, nothing is tested
  const auto is_full = [&](int i) { return tile_is_full(first, last, steps.tile(i) * kTokenStep, kTokenStep); };
  const auto load_keys = [&](int i, uint4(&k)[2][kChunks]) {
    const int j0 = steps.tile(i) * kTokenStep;
    const __nv_bfloat16* src = k_base + (j0 + g) * p.k_seq;
    if (dim == DP && is_full(i)) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) k[n][c] = ld_stream_v4(src + n * 8 * p.k_seq + c * 32);
      return;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const bool there = seen(j0 + n * 8 + g);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        k[n][c] = there && c * 32 + t * 8 < dim ? ld_stream_v4(src + n * 8 * p.k_seq + c * 32) : zero;
    }
  };
  const auto load_values = [&](int i, uint4(&v)[kBlocks][4]) {
    const int j0 = steps.tile(i) * kTokenStep;
    const __nv_bfloat16* src = v_base + (j0 + t * 2) * p.v_seq;
    if (dim == DP && is_full(i)) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) v[b][x] = ld_stream_v4(src + ((x & 1) + (x >> 1) * 8) * p.v_seq + b * 64);
      return;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int row = (x & 1) + (x >> 1) * 8;
      const bool there = seen(j0 + t * 2 + row);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        v[b][x] = there && b * 64 + g * 8 < dim ? ld_stream_v4(src + row * p.v_seq + b * 64) : zero;
    }
  };
  if (begin < end) {
    load_keys(begin, k_frag[0]);
    load_values(begin, v_frag[0]);
  }

  // ---- the query rows g and g + 8
  // (in shared memory, as every lane's fragments: the registers hold the tiles in flight)
  uint4* q_frag = reinterpret_cast<uint4*>(token_smem) + warp * 2 * kChunks * 32 + lane;
  RowSpan span[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + h * 8;
    const int head = kv_head * group + (rows > 0 ? r / seq.nq : 0), row = rows > 0 ? r % seq.nq : 0;
    span[h] = row_span(p.shape, seq, row);
    const __nv_bfloat16* src = p.q + batch * p.q_batch + (seq.q0 + row) * p.q_seq + head * p.q_head + t * 8;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      q_frag[(h * kChunks + c) * 32] = r < rows && c * 32 + t * 8 < dim ? ld_stream_v4(src + c * 32) : zero;
  }

  const float c2 = p.shape.scale_log2;
  float o[kBlocks][8][4] = {};
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  const auto step = [&](int i, const uint4(&k)[2][kChunks], const uint4(&v)[kBlocks][4], uint4(&k_next)[2][kChunks],
                        uint4(&v_next)[kBlocks][4]) {
    if (i + 1 < end) {
      load_keys(i + 1, k_next);
      load_values(i + 1, v_next);
    }
    float s[2][4] = {}, s_odd[2][4] = {};  // two sums each: shorter chains of dependent products
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const uint4 q0 = q_frag[c * 32], q1 = q_frag[(kChunks + c) * 32];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma_16x8x16(s[n], q0.x, q1.x, q0.y, q1.y, k[n][c].x, k[n][c].y);
        mma_16x8x16(s_odd[n], q0.z, q1.z, q0.w, q1.w, k[n][c].z, k[n][c].w);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] += s_odd[n][x];
    if (!is_full(i)) {
      const int j0 = steps.tile(i) * kTokenStep;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int j = j0 + n * 8 + t * 2 + (x & 1);
          const RowSpan& r = span[x >> 1];
          if (!(j < r.sink || (j >= r.low && j <= r.high))) s[n][x] = -INFINITY;
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
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[b][n][x] *= factor[x >> 1];
    }
    uint32_t weight[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float shift = top[h] == -INFINITY ? 0.0f : -top[h] * c2;
        const float e0 = exp2_sfu(fmaf(s[n][2 * h], c2, shift)), e1 = exp2_sfu(fmaf(s[n][2 * h + 1], c2, shift));
        sum[h] += e0 + e1;
        weight[n][h] = pack_bf16(e0, e1);
      }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const uint32_t *v0 = &v[b][0].x, *v1 = &v[b][1].x, *v2 = &v[b][2].x, *v3 = &v[b][3].x;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const uint32_t pick = n & 1 ? 0x7632 : 0x5410;
        mma_16x8x16(o[b][n], weight[0][0], weight[0][1], weight[1][0], weight[1][1], __byte_perm(v0[n / 2], v1[n / 2], pick),
                    __byte_perm(v2[n / 2], v3[n / 2], pick));
      }
    }
  };
  for (int i = begin; i < end; i += 2) {
    step(i, k_frag[0], v_frag[0], k_frag[1], v_frag[1]);
    if (i + 1 < end) step(i + 1, k_frag[1], v_frag[1], k_frag[0], v_frag[0]);
  }
  __syncthreads();  // the query fragments' place is used again

  // ---- join the warps
  float* smem_o = token_smem;  // [warps, rows, row floats]
  float* smem_top = token_smem + kTokenWarps * kTokenRows * Cfg::kRowFloats;
  float* smem_sum = smem_top + kTokenWarps * kTokenRows;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    float* dst = smem_o + (warp * kTokenRows + g + h * 8) * Cfg::kRowFloats + t * 16;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int n = 0; n < 8; n += 4)
          *reinterpret_cast<float4*>(dst + b * 64 + e * 8 + n) =
              make_float4(o[b][n][2 * h + e], o[b][n + 1][2 * h + e], o[b][n + 2][2 * h + e], o[b][n + 3][2 * h + e]);
    if (t == 0) {
      smem_top[warp * kTokenRows + g + h * 8] = top[h] * c2;  // base 2
      smem_sum[warp * kTokenRows + g + h * 8] = sum[h];
    }
  }
  __syncthreads();
  // kEach threads per row, each DP / kEach columns in steps of kEach
  constexpr int kEach = 32 * kTokenWarps / kTokenRows;
  const int r = threadIdx.x / kEach, column = threadIdx.x % kEach;
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
    // this CTA's result takes the place of its first warp's; then every CTA joins the columns of all
    __syncthreads();
#pragma unroll
    for (int x = 0; x < DP / kEach; ++x) smem_o[r * Cfg::kRowFloats + x * kEach + column] = joined[x];
    if (column == 0) smem_top[r] = whole_top, smem_sum[r] = whole_sum;
    cluster_arrive_release();
    cluster_wait_acquire();
    // rows of the cluster's CTAs in turn: the rank's share of them, one warp per row, DP / 32 columns per lane
    const int rank = static_cast<int>(cluster_ctarank());
    for (int row = rank + warp * p.splits; row < rows; row += p.splits * kTokenWarps) {
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
  if (r >= rows) return;
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

// What the sliding-window attention kernels share: which keys a row sees, the
// list of key tiles of a block of rows, and the PTX they need beyond mup_ptx.cuh.
//
// Row i of a sequence with Lq queries and Lk keys stands at position
// at = i + Lk - Lq. It sees key j when
//     j < Lk, (not causal or j <= at), and (j < sinks or at - left <= j <= at + right)
// so per row the visible keys are [0, sink) and [low, high]; all three bounds
// only grow with the row, which makes the keys that a block of rows sees two
// ranges as well, bounded by its first and last row.
#pragma once

#include "../../include/megaup.h"
#include "mup_ptx.cuh"

namespace mup {

constexpr int kTileRows = 128;       // rows of a Q, K, V or dO tile, lanes of TMEM
constexpr int kPanelBytes = 16384;   // 128 rows of 64 BF16 with the 128-byte swizzle
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNoLimit = 1 << 30;    // a window side without a limit

struct AttnShape {
  int batch, heads_q, heads_kv, seq_q, seq_k, head_dim;
  int causal, left, right, sinks;  // left, right already kNoLimit where unlimited; right 0 when causal
  float scale, scale_log2;
  const int* kv_lengths;   // [batch] or null (then every sequence has seq_k keys)
  const int4* sequences;   // packed: {first query row, queries, first key row, keys}; null when dense
  uint32_t* status;
  uint64_t timeout_ns;
};

struct AttnSeq {
  int q0, nq, k0, nk, off;  // off = nk - nq
};

__device__ __forceinline__ AttnSeq load_sequence(const AttnShape& p, int sequence) {
  AttnSeq s;
  if (p.sequences != nullptr) {
    const int4 v = p.sequences[sequence];
    s.q0 = v.x, s.nq = v.y, s.k0 = v.z, s.nk = v.w;
  } else {
    s.q0 = 0, s.nq = p.seq_q, s.k0 = 0, s.nk = p.seq_k;
    // a length outside [0, seq_k] would name rows that are not there
    if (p.kv_lengths != nullptr) s.nk = min(max(p.kv_lengths[sequence], 0), p.seq_k);
  }
  s.off = s.nk - s.nq;
  return s;
}

// An entry of a packed block list: a block of rows and the sequence it belongs to, read at once.
struct alignas(32) AttnPackedBlock {
  int sequence, row0, q0, nq, k0, nk, unused[2];
};
__device__ __forceinline__ AttnSeq load_block(const AttnPackedBlock* list, int i, int& sequence, int& row0) {
  const int4 a = reinterpret_cast<const int4*>(list + i)[0], b = reinterpret_cast<const int4*>(list + i)[1];
  sequence = a.x, row0 = a.y;
  AttnSeq s;
  s.q0 = a.z, s.nq = a.w, s.k0 = b.x, s.nk = b.y;
  s.off = s.nk - s.nq;
  return s;
}

struct RowSpan {
  int sink, low, high;  // [0, sink) and [low, high]
};

__device__ __forceinline__ RowSpan row_span(const AttnShape& p, const AttnSeq& s, int row) {
  RowSpan r;
  const int at = row + s.off;
  r.low = max(at - p.left, 0);
  r.high = min(at + p.right, s.nk - 1);
  r.sink = min(p.sinks, s.nk);
  if (p.causal) r.sink = max(min(r.sink, at + 1), 0);
  return r;
}

// The key tiles (of kTileRows keys, or another size) that the rows [first, last] see, in ascending order.
struct TileList {
  int split, second, count;  // entries [0, split) are tiles 0.., the rest start at tile `second`
  int sink_end, low, high;   // the rows' union of keys
  __device__ __forceinline__ int tile(int i) const { return i < split ? i : second + (i - split); }
};

__device__ __forceinline__ TileList make_tile_list(const RowSpan& first, const RowSpan& last, int size = kTileRows) {
  TileList t;
  t.sink_end = last.sink, t.low = first.low, t.high = last.high;
  const int sink_tiles = (last.sink + size - 1) / size;
  if (last.high < first.low) {
    t.split = 0, t.second = 0, t.count = sink_tiles;
    return t;
  }
  const int w0 = first.low / size, w1 = last.high / size;
  if (sink_tiles == 0) {
    t.split = 0, t.second = w0, t.count = w1 - w0 + 1;
  } else if (w0 <= sink_tiles) {
    t.split = 0, t.second = 0, t.count = max(w1 + 1, sink_tiles);
  } else {
    t.split = sink_tiles, t.second = w0, t.count = sink_tiles + w1 - w0 + 1;
  }
  return t;
}

// Whether a block of rows with this union of keys sees anything of key tile `kt`.
__device__ __forceinline__ bool sees_tile(const TileList& t, int kt) {
  const int j0 = kt * kTileRows;
  return j0 < t.sink_end || (j0 <= t.high && j0 + kTileRows > t.low);
}

// Whether every key of the tile is seen by every row between `first` and `last`.
__device__ __forceinline__ bool tile_is_full(const RowSpan& first, const RowSpan& last, int j0, int size = kTileRows) {
  return (j0 >= last.low && j0 + size - 1 <= first.high) || j0 + size <= first.sink;
}

// Bit x of the result: x < n (n may be anything).
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// Bit x: x < sink or low <= x <= high.
__device__ __forceinline__ uint32_t span_bits(int low, int high, int sink) {
  return (bits_below(high + 1) & ~bits_below(low)) | bits_below(sink);
}
// Scores whose bit is not set become -inf.
__device__ __forceinline__ void hide_scores(uint32_t (&score)[32], uint32_t seen) {
#pragma unroll
  for (int x = 0; x < 32; ++x) score[x] = (seen >> x) & 1u ? score[x] : 0xff800000u;
}

// ---------------------------------------------------------------------------
// PTX
// ---------------------------------------------------------------------------

__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// D[tmem] (+)= A[tmem, 16-bit pairs per column] * B[smem].
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 2^x of the special-function unit (results below 2^-126 become 0; -inf gives 0).
__device__ __forceinline__ float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The largest of three (a NaN only where all are).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The largest of 32 scores, in four chains.
__device__ __forceinline__ float max32(const uint32_t (&v)[32]) {
  float m[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    m[b] = max3(__uint_as_float(v[b * 8]), __uint_as_float(v[b * 8 + 1]), __uint_as_float(v[b * 8 + 2]));
    m[b] = max3(m[b], __uint_as_float(v[b * 8 + 3]), __uint_as_float(v[b * 8 + 4]));
    m[b] = max3(m[b], __uint_as_float(v[b * 8 + 5]), __uint_as_float(v[b * 8 + 6]));
    m[b] = fmaxf(m[b], __uint_as_float(v[b * 8 + 7]));
  }
  return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

// Two FP32 lanes in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// {lo, hi} rounded to BF16, lo in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Shared-memory descriptor of a tile of rows of 64 BF16 (128-byte swizzle) read
// with the row as the K index of the product (the contiguous index is N): 8-row
// groups are 1024 bytes apart (stride offset), the next 64 columns one panel on
// (leading offset).
__device__ __forceinline__ uint64_t make_mnmajor_sw128_desc(uint32_t smem_addr, uint32_t panel_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(panel_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
constexpr uint32_t kIdescTransposeB = 1u << 16;  // B is stored with N contiguous

// D[128 x 128] = A B^T over the head dimension, both tiles K-major: one issue sequence of DP / 16 products.
template <int DP>
__device__ __forceinline__ void umma_rows_by_rows(uint32_t d_tmem, uint32_t a_smem, uint32_t b_smem) {
  constexpr uint32_t idesc = make_idesc_bf16(kTileRows, kTileRows);
  const uint64_t a = make_kmajor_sw128_desc(a_smem), b = make_kmajor_sw128_desc(b_smem);
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const uint64_t step = static_cast<uint64_t>(((kk >> 2) * kPanelBytes + (kk & 3) * 32) >> 4);
    umma_bf16<1>(d_tmem, a + step, b + step, idesc, kk != 0);
  }
}

// D[128 x DP] (+)= A[128 x 128, TMEM] B[128 x DP], B's rows being the summed index. The A columns of K step kk start
// at kk / 4 * half_stride + kk % 4 * 8 (half_stride 32: packed without a gap).
template <int DP, int BEGIN = 0, int END = 8>
__device__ __forceinline__ void umma_tmem_by_cols(uint32_t d_tmem, uint32_t a_tmem, int half_stride, uint32_t b_smem,
                                                  bool accumulate) {
  constexpr uint32_t idesc = make_idesc_bf16(kTileRows, DP) | kIdescTransposeB;
  const uint64_t b = make_mnmajor_sw128_desc(b_smem, kPanelBytes);
#pragma unroll
  for (int kk = BEGIN; kk < END; ++kk)
    umma_bf16_ts(d_tmem, a_tmem + (kk >> 2) * half_stride + (kk & 3) * 8, b + static_cast<uint64_t>((kk * 2048) >> 4),
                 idesc, accumulate || kk != 0);
}

// ---------------------------------------------------------------------------
// Bounded waits: a wait that runs out records its cause once, raises the CTA's
// abort flag (every other wait then gives up too) and returns false; the role
// leaves its loop and meets the others at the CTA's last barrier. What is in
// flight then ends (drain_products, drain_ring) before TMEM and shared memory
// are given up.
// ---------------------------------------------------------------------------

struct WaitControl {
  volatile uint32_t* abort_flag;
  uint32_t* status;
  uint64_t timeout_ns;

  // The whole warp calls this, converged, and every lane leaves with the same result: a phase that ends just as the limit
  // is reached must not send some lanes into the aligned instructions behind the wait and others out of the loop. Where a
  // lane saw the phase's end at the first look, the others see it at poll's first one; where none did, all are here and
  // vote. (A vote at the first look as well costs 3 to 4 % of a backward pass: it stands between the barrier and the issue.)
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t code) const {
    if (mbar_try_wait(bar, parity)) return true;
    const uint32_t lanes = __activemask();
    if (__all_sync(lanes, poll(bar, parity))) return true;
    give_up(code);
    return false;
  }
  // One thread of a warp (the copies' issuer).
  __device__ __forceinline__ bool wait_alone(uint32_t bar, uint32_t parity, uint32_t code) const {
    if (mbar_try_wait(bar, parity) || poll(bar, parity)) return true;
    give_up(code);
    return false;
  }
  // (a failed try_wait has suspended the thread for about 5 us, measured: the clock and the flag may be read each time)
  __device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) const {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity))
      if (*abort_flag != 0u || globaltimer_ns() - t0 > timeout_ns) return false;
    return true;
  }
  __device__ __forceinline__ void give_up(uint32_t code) const {
    if (*abort_flag == 0u) {
      *abort_flag = 1u;
      if (status != nullptr) {
        *reinterpret_cast<volatile uint32_t*>(status) = (code << 24) | (blockIdx.x & 0xffffffu);
        __threadfence_system();
      }
    }
  }
};

// After an abort: waits for a copy or product in flight, whatever the abort flag says, but no longer than a fifth of a
// second (they end within microseconds).
constexpr uint64_t kDrainNs = 200000000;
__device__ __forceinline__ void drain_barrier(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kDrainNs) return;
}

// After an abort, in a warp whose elected thread issued products (elect.sync chooses the same one every time): they end.
__device__ __forceinline__ void drain_products(uint32_t bar) {
  if (elect_one_sync()) umma_commit_1(bar);
  __syncwarp();
  drain_barrier(bar, 0);
}

// The last of `loads` copies into a ring of `stages` end: a wait ran out, and their places are about to be given up.
__device__ __forceinline__ void drain_ring(uint32_t full, int stages, int loads) {
  for (int n = max(0, loads - stages); n < loads; ++n) drain_barrier(full + n % stages * 8, (n / stages) & 1);
}

// Rows [from, to) of a tile that is in shared memory become zero. The whole warp calls it; the tile's next reader is
// a product (async proxy).
template <int DP>
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int from, int to, int lane) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int i = lane; i < (to - from) * 8; i += 32) {
#pragma unroll
    for (int panel = 0; panel < DP / 64; ++panel)
      *reinterpret_cast<uint4*>(tile + panel * kPanelBytes + from * 128 + i * 16) = zero;
  }
}

// Results leave through shared memory: a thread holds a row, and rows written by their threads would touch 32 lines per
// instruction. Piece `chunk` (16 bytes) of row r of a tile with RB bytes per row, its place permuted so that neither
// side has bank conflicts.
template <int RB>
__device__ __forceinline__ uint4* staged_piece(uint8_t* tile, int r, int chunk) {
  constexpr int kMask = RB >= 128 ? 7 : RB / 16 - 1;
  return reinterpret_cast<uint4*>(tile + r * RB + ((chunk ^ (r & kMask)) * 16));
}
// The warp's 32 rows, from `first`, whole rows at a time to where dst(r) points (null: nowhere), `bytes` of each.
template <int RB, typename Dst>
__device__ __forceinline__ void write_staged_rows(uint8_t* tile, int first, int lane, int bytes, Dst dst) {
  constexpr int kLanes = RB / 16;
  __syncwarp();
#pragma unroll 4
  for (int k = 0; k < kLanes; ++k) {
    const int r = first + k * (32 / kLanes) + lane / kLanes, chunk = lane % kLanes;
    const uint4 v = *staged_piece<RB>(tile, r, chunk);
    uint8_t* to = dst(r);
    if (to != nullptr && chunk * 16 < bytes) *reinterpret_cast<uint4*>(to + chunk * 16) = v;
  }
  __syncwarp();
}
// The same where row r goes to `to` + r * stride, rows from `end` on nowhere.
template <int RB>
__device__ __forceinline__ void write_staged_rows(uint8_t* tile, int first, int lane, int bytes, uint8_t* to,
                                                  int64_t stride, int end) {
  constexpr int kLanes = RB / 16, kRows = 32 / kLanes;
  __syncwarp();
  const int chunk = lane % kLanes, r0 = first + lane / kLanes;
  uint8_t* dst = to + r0 * stride + chunk * 16;
  if (chunk * 16 >= bytes) end = 0;
#pragma unroll 8
  for (int k = 0; k < kLanes; ++k, dst += kRows * stride) {
    const uint4 v = *staged_piece<RB>(tile, r0 + k * kRows, chunk);
    if (r0 + k * kRows < end) *reinterpret_cast<uint4*>(dst) = v;
  }
  __syncwarp();
}
__device__ __forceinline__ uint4 pack_bf16x8(const uint32_t* v, float scale) {
  uint4 p;
  p.x = pack_bf16(__uint_as_float(v[0]) * scale, __uint_as_float(v[1]) * scale);
  p.y = pack_bf16(__uint_as_float(v[2]) * scale, __uint_as_float(v[3]) * scale);
  p.z = pack_bf16(__uint_as_float(v[4]) * scale, __uint_as_float(v[5]) * scale);
  p.w = pack_bf16(__uint_as_float(v[6]) * scale, __uint_as_float(v[7]) * scale);
  return p;
}

// What the rounding of pack_bf16x8 leaves.
__device__ __forceinline__ uint32_t pack_bf16_rest(float lo, float hi) {
  const uint32_t p = pack_bf16(lo, hi);
  return pack_bf16(lo - __uint_as_float(p << 16), hi - __uint_as_float(p & 0xffff0000u));
}
__device__ __forceinline__ uint4 pack_bf16x8_rest(const uint32_t* v, float scale) {
  uint4 p;
  p.x = pack_bf16_rest(__uint_as_float(v[0]) * scale, __uint_as_float(v[1]) * scale);
  p.y = pack_bf16_rest(__uint_as_float(v[2]) * scale, __uint_as_float(v[3]) * scale);
  p.z = pack_bf16_rest(__uint_as_float(v[4]) * scale, __uint_as_float(v[5]) * scale);
  p.w = pack_bf16_rest(__uint_as_float(v[6]) * scale, __uint_as_float(v[7]) * scale);
  return p;
}

// A row of a key or value tile that none of the block's rows sees (another sequence's, one behind the filled part of a
// cache, one between the sinks and the window) has to be finite where its weight is 0: it becomes 0. The whole warp
// calls this between the tile's arrival and its first product.
template <int DP>
__device__ __forceinline__ void zero_unseen_rows(uint8_t* tile, const TileList& seen, int j0, int lane) {
  if ((j0 >= seen.low && j0 + kTileRows - 1 <= seen.high) || j0 + kTileRows <= seen.sink_end) return;
  const bool window = seen.high >= seen.low;
  const int sinks = min(max(seen.sink_end - j0, 0), kTileRows);
  const int from = window ? min(max(seen.low - j0, 0), kTileRows) : kTileRows;
  const int to = window ? min(max(seen.high + 1 - j0, 0), kTileRows) : kTileRows;
  zero_tile_rows<DP>(tile, sinks, max(sinks, from), lane);
  zero_tile_rows<DP>(tile, max(sinks, to), kTileRows, lane);
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace mup

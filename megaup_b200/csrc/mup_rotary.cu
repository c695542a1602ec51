// Rotary positions with several axes (include/megaup.h, mup_axial_rotary).
//
// Bound by memory: every element of q and k is read and written once. A warp
// owns a row of the sequence: each lane holds the
// sines and cosines of the pairs of its 16-byte columns and walks the row's
// heads of both tensors with them, so an angle is computed once per row and
// not once per head, and no table of angles is read.
//
// An angle is position * frequency, for a far position many turns. Its
// fraction of a turn is what counts: the product is taken in turns and in 64
// bits (position * frequency / 2 pi, error 2^-53 of the number of turns), the
// whole turns are dropped there, and sine and cosine of the rest are taken in
// 32 bits.
//
// Measured on B200 (32768 rows, 5 + 5 heads of 128, interleaved: 168 MB moved): 55 us with a warp per row and no
// work kept between rows, 44 us with all loads of a row ahead of its angles, 35 us with resident warps and angles shared
// between a warp's lanes, 31 us (5.4 TB/s, 82 % of the copy rate) with the heads' offsets kept as well. Two resident blocks
// of 256 threads beat three (33 us, registers spill) and four (41 us). Rotated halves, 65536 rows of 8 + 2 heads in a fused
// projection (335 MB): 123 us at first, 69 us (4.9 TB/s) with the two halves in two lanes.
#include <algorithm>

#include "mup_host.cuh"
#include "mup_ptx.cuh"

namespace {

using namespace mup;

struct RotaryParams {
  const __nv_bfloat16* x[2];
  __nv_bfloat16* y[2];
  int64_t x_batch[2], x_row[2], x_head[2], y_batch[2], y_row[2], y_head[2];
  int heads[2];
  const void* positions;
  int64_t pos_axis, pos_batch, pos_row;
  const double* turns;
  const int* pair_axis;
  uint32_t rows, items;  // of a sequence, of the batch
  int head_dim, pairs, position_type;
  int heads_each;  // heads that a group takes of a row, at most kHeads
  float sign;
};

__device__ __forceinline__ double load_position(const RotaryParams& p, int64_t at) {
  if (p.position_type == MUP_ROTARY_INT64) return static_cast<double>(static_cast<const long long*>(p.positions)[at]);
  if (p.position_type == MUP_ROTARY_INT32) return static_cast<double>(static_cast<const int*>(p.positions)[at]);
  return static_cast<double>(static_cast<const float*>(p.positions)[at]);
}

__device__ __forceinline__ float low_bf16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

struct Turn {
  float cos, sin;
};

// The angles of a lane's N neighbouring pairs. Several lanes of a warp hold the same pairs (of different heads, and of
// both halves of one): the first SHARED of them compute N / SHARED pairs each and hand them to the others. A lane keeps
// the frequencies of those it computes and where their axes lie in `positions`.
template <int N, int SHARED>
struct LanePairs {
  static constexpr int kEach = N / SHARED;
  double turns[kEach];
  int64_t axis[kEach];

  // `first`: the lane's first pair; `copy`: its place among the lanes with the same pairs.
  __device__ __forceinline__ LanePairs(const RotaryParams& p, int first, int copy) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int pair = first + i * SHARED + copy % SHARED;
      const bool turned = pair < p.pairs;
      turns[i] = turned ? p.turns[pair] : 0.0;
      axis[i] = turned ? p.pair_axis[pair] * p.pos_axis : 0;
    }
  }
  // The whole warp calls this; `lane_of(c)` is the lane that is copy c of the caller's pairs.
  template <typename LaneOf>
  __device__ __forceinline__ void turn(const RotaryParams& p, int64_t at, LaneOf lane_of, Turn (&t)[N]) const {
    double position[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) position[i] = load_position(p, at + axis[i]);
    Turn mine[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const double all = position[i] * turns[i];
      const float rest = static_cast<float>(all - rint(all));
      sincospif(2.0f * rest, &mine[i].sin, &mine[i].cos);
      mine[i].sin *= p.sign;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      t[i] = mine[i / SHARED];
      if constexpr (SHARED > 1) {
        const int from = lane_of(i % SHARED);
        t[i].cos = __shfl_sync(0xffffffffu, t[i].cos, from);
        t[i].sin = __shfl_sync(0xffffffffu, t[i].sin, from);
      }
    }
  }
};

// A lane holds 16 bytes of a head, `lanes` lanes (a power of two up to 32) a head, and the 32 / lanes groups of a warp take
// every 32 / lanes-th head of a row: up to kHeads heads each, whose loads are in flight while the angles are computed.
// Rows with more heads are cut along the grid's second dimension (and their angles computed again, a third of the
// instructions). Interleaved, the 16 bytes are four pairs. Otherwise they are one half of eight pairs, whose other half
// lies pairs / 8 lanes away and is exchanged by shuffles: loads and stores stay those of the interleaved form.
constexpr int kHeads = 6;
constexpr int kResident = 2;  // blocks per SM

template <bool INTERLEAVED, int SHARED>
__global__ void __launch_bounds__(256, kResident) rotary_kernel(const __grid_constant__ RotaryParams p, int lanes) {
  constexpr int kPairs = INTERLEAVED ? 4 : 8;
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x % 32;
  const int groups = 32 / lanes, group = lane / lanes, place = lane % lanes;
  const int column = place * 8;
  const int half_lanes = p.pairs / 8;  // not interleaved: lanes of a half
  const bool second = !INTERLEAVED && place >= half_lanes;
  const int pair0 = INTERLEAVED ? place * 4 : (place - (second ? half_lanes : 0)) * 8;
  const int other = lane + (second ? -half_lanes : half_lanes);
  const int copies = INTERLEAVED ? 1 : 2;
  const auto lane_of = [&](int copy) {
    return INTERLEAVED ? copy * lanes + place : copy / 2 * lanes + min(pair0 / 8 + copy % 2 * half_lanes, lanes - 1);
  };
  const LanePairs<kPairs, SHARED> pairs(p, pair0, group * copies + (second ? 1 : 0));
  // the group's heads of both tensors, as offsets of 16 bytes from a row's start
  const int heads = p.heads[0] + p.heads[1];
  uint32_t x_at[kHeads], y_at[kHeads], used = 0, second_tensor = 0;
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    int head = (blockIdx.y * p.heads_each + h) * groups + group;
    if (h >= p.heads_each || head >= heads || column >= p.head_dim) continue;
    const int t = head >= p.heads[0];
    head -= t ? p.heads[0] : 0;
    used |= 1u << h;
    second_tensor |= t << h;
    x_at[h] = static_cast<uint32_t>((head * p.x_head[t] + column) / 8);
    y_at[h] = static_cast<uint32_t>((head * p.y_head[t] + column) / 8);
  }
  for (uint32_t item = blockIdx.x * 8 + threadIdx.x / 32; item < p.items; item += gridDim.x * 8) {
    const uint32_t b = p.rows == p.items ? 0 : item / p.rows, row = item - b * p.rows;
    const uint4* x[2];
    uint4* y[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x[t] = reinterpret_cast<const uint4*>(p.x[t] + b * p.x_batch[t] + row * p.x_row[t]);
      y[t] = reinterpret_cast<uint4*>(p.y[t] + b * p.y_batch[t] + row * p.y_row[t]);
    }
    uint4 v[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
      if (used >> h & 1) v[h] = ld_stream_v4(((second_tensor >> h & 1) ? x[1] : x[0]) + x_at[h]);
    Turn turn[kPairs];
    pairs.turn(p, b * p.pos_batch + row * p.pos_row, lane_of, turn);
    if constexpr (!INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn[i].sin = second ? turn[i].sin : -turn[i].sin;
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (h >= p.heads_each) break;
      uint32_t* words = &v[h].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lo = low_bf16(words[i]), hi = high_bf16(words[i]);
        if constexpr (INTERLEAVED) {
          if (pair0 + i < p.pairs)
            words[i] = two_bf16(lo * turn[i].cos - hi * turn[i].sin, lo * turn[i].sin + hi * turn[i].cos);
        } else {
          const uint32_t there = __shfl_sync(0xffffffffu, words[i], other);
          const Turn t0 = turn[2 * i], t1 = turn[2 * i + 1];
          if (pair0 < p.pairs)
            words[i] = two_bf16(lo * t0.cos + low_bf16(there) * t0.sin, hi * t1.cos + high_bf16(there) * t1.sin);
        }
      }
      if (used >> h & 1) ((second_tensor >> h & 1) ? y[1] : y[0])[y_at[h]] = v[h];
    }
  }
}

int check_rows(const char* name, const void* base, const int64_t strides[3]) {
  if (base == nullptr || reinterpret_cast<uintptr_t>(base) % 16 != 0)
    return host_fail(MUP_ERR_BAD_ARG, "axial rotary: %s is null or not 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0)
      return host_fail(MUP_ERR_BAD_ARG, "axial rotary: %s stride %lld is no multiple of 16 bytes", name,
                       static_cast<long long>(strides[i]));
  return MUP_OK;
}

constexpr unsigned kBlocks = 148 * kResident;

cudaError_t launch(RotaryParams& p, bool interleaved, cudaStream_t stream) {
  int lanes = 1;
  while (lanes * 8 < p.head_dim) lanes *= 2;
  const int per_group = (p.heads[0] + p.heads[1] + 32 / lanes - 1) / (32 / lanes);
  const int parts = (per_group + kHeads - 1) / kHeads;
  p.heads_each = (per_group + parts - 1) / parts;
  const int copies = 32 / lanes * (interleaved ? 1 : 2);
  // Warps stay for several rows: a lane's frequencies are read once, and a block's start is paid once.
  const dim3 grid(std::min((p.items + 7) / 8, kBlocks), parts);
  void (*kernel)(RotaryParams, int);
  if (interleaved)
    kernel = copies >= 4 ? rotary_kernel<true, 4> : copies == 2 ? rotary_kernel<true, 2> : rotary_kernel<true, 1>;
  else
    kernel = copies >= 8 ? rotary_kernel<false, 8> : copies == 4 ? rotary_kernel<false, 4> : rotary_kernel<false, 2>;
  return launch_early(kernel, grid, 256, 0, 1, stream, p, lanes);
}

}  // namespace

extern "C" int mup_axial_rotary_launch(const mup_axial_rotary* args, void* stream) {
  if (args == nullptr) return host_fail(MUP_ERR_BAD_ARG, "axial rotary: null argument");
  const mup_axial_rotary& a = *args;
  if (a.head_dim < 8 || a.head_dim > 256 || a.head_dim % 8 != 0)
    return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: head_dim %d is not a multiple of 8 up to 256", a.head_dim);
  if (a.pairs < 1 || 2 * a.pairs > a.head_dim || (!a.interleaved && a.pairs % 8 != 0))
    return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: %d pairs in heads of %d", a.pairs, a.head_dim);
  if (a.batch < 1 || a.rows < 1 || a.axes < 1 || a.heads[0] < 1 || a.heads[1] < 0)
    return host_fail(MUP_ERR_BAD_ARG, "axial rotary: batch %d, rows %d, axes %d, heads %d and %d", a.batch, a.rows,
                     a.axes, a.heads[0], a.heads[1]);
  if (a.positions == nullptr || a.turns == nullptr || a.pair_axis == nullptr || a.position_type < 0 || a.position_type > 2)
    return host_fail(MUP_ERR_BAD_ARG, "axial rotary: positions or frequencies are missing");
  if (reinterpret_cast<uintptr_t>(a.positions) % (a.position_type == MUP_ROTARY_INT64 ? 8 : 4) != 0 ||
      reinterpret_cast<uintptr_t>(a.turns) % 8 != 0 || reinterpret_cast<uintptr_t>(a.pair_axis) % 4 != 0)
    return host_fail(MUP_ERR_BAD_ARG, "axial rotary: positions or frequencies are not aligned to their type");
  RotaryParams p{};
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    const void* x = t == 0 ? a.q : a.k;
    void* y = t == 0 ? a.q_out : a.k_out;
    int rc = check_rows(t == 0 ? "q" : "k", x, a.x_strides[t]);
    if (rc == MUP_OK) rc = check_rows(t == 0 ? "q's output" : "k's output", y, a.y_strides[t]);
    if (rc != MUP_OK) return rc;
    p.x[t] = static_cast<const __nv_bfloat16*>(x), p.y[t] = static_cast<__nv_bfloat16*>(y);
    p.x_batch[t] = a.x_strides[t][0], p.x_row[t] = a.x_strides[t][1], p.x_head[t] = a.x_strides[t][2];
    p.y_batch[t] = a.y_strides[t][0], p.y_row[t] = a.y_strides[t][1], p.y_head[t] = a.y_strides[t][2];
    p.heads[t] = a.heads[t];
    // a head's place in a row is kept as 32 bits of 16-byte units
    for (int64_t stride : {a.x_strides[t][2], a.y_strides[t][2]})
      if (a.heads[t] > 65536 || stride / 8 * a.heads[t] > 0xffffffffll)
        return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: %d heads at a stride of %lld", a.heads[t],
                         static_cast<long long>(stride));
  }
  p.positions = a.positions;
  p.pos_axis = a.pos_strides[0], p.pos_batch = a.pos_strides[1], p.pos_row = a.pos_strides[2];
  p.turns = a.turns, p.pair_axis = a.pair_axis;
  p.rows = a.rows, p.head_dim = a.head_dim, p.pairs = a.pairs, p.position_type = a.position_type;
  const int64_t items = static_cast<int64_t>(a.batch) * a.rows;
  if (items > 0x7fffffff) return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: %lld rows", static_cast<long long>(items));
  p.items = static_cast<uint32_t>(items);
  p.sign = a.inverse ? -1.0f : 1.0f;
  DeviceScope scope(a.device);
  MUP_HOST_CUDA(scope.error());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  MUP_HOST_CUDA(launch(p, a.interleaved != 0, s));
  return MUP_OK;
}

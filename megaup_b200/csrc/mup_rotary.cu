// Rotary positions with several axes (include/megaup.h, mup_axial_rotary).
//
// Bound by memory: every element of q and k is read and written once. A warp
// owns a row of the sequence (or a share of its heads): each lane holds the
// sines and cosines of the pairs of its 16-byte columns and walks the row's
// heads of both tensors with them, so an angle is computed once per row and
// not once per head, and no table of angles is read.
//
// An angle is position * frequency, for a far position many turns. Its
// fraction of a turn is what counts: the product is taken in turns and in 64
// bits (position * frequency / 2 pi, error 2^-53 of the number of turns), the
// whole turns are dropped there, and sine and cosine of the rest are taken in
// 32 bits.
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
  int rows, head_dim, pairs, head_shares;
  int64_t items;  // batch * rows * head_shares
  float sign;
};

template <int TYPE>
__device__ __forceinline__ double load_position(const void* positions, int64_t at) {
  if constexpr (TYPE == MUP_ROTARY_INT32) return static_cast<double>(static_cast<const int*>(positions)[at]);
  if constexpr (TYPE == MUP_ROTARY_INT64) return static_cast<double>(static_cast<const long long*>(positions)[at]);
  return static_cast<double>(static_cast<const float*>(positions)[at]);
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

// Pairs from `pairs` on are not turned: cosine 1, sine 0 mark them.
template <int TYPE>
__device__ __forceinline__ Turn turn_of(const RotaryParams& p, int pair, int64_t at) {
  const double position = load_position<TYPE>(p.positions, at + p.pair_axis[pair] * p.pos_axis);
  const double turns = position * p.turns[pair];
  const float rest = static_cast<float>(turns - rint(turns));
  Turn t;
  sincospif(2.0f * rest, &t.sin, &t.cos);
  t.sin *= p.sign;
  return t;
}

// Interleaved pairs: a lane's 16 bytes are four pairs. `lanes` lanes cover a head (a power of two up to 32), a warp's
// 32 / lanes groups take every 32 / lanes-th head; heads wider than 256 take several passes of columns.
template <int TYPE>
__global__ void __launch_bounds__(256) rotary_interleaved_kernel(const RotaryParams p, int lanes) {
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  if (item >= p.items) return;
  const int lane = threadIdx.x % 32;
  const int share = static_cast<int>(item % p.head_shares);
  const int64_t place = item / p.head_shares;
  const int64_t b = place / p.rows, row = place - b * p.rows;
  const int groups = 32 / lanes, group = lane / lanes;
  const int64_t at = b * p.pos_batch + row * p.pos_row;
  for (int column = (lane % lanes) * 8; column < p.head_dim; column += lanes * 8) {
    Turn turn[4];
    bool turned[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pair = column / 2 + i;
      turned[i] = pair < p.pairs;
      if (turned[i]) turn[i] = turn_of<TYPE>(p, pair, at);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const __nv_bfloat16* x = p.x[which] + b * p.x_batch[which] + row * p.x_row[which] + column;
      __nv_bfloat16* y = p.y[which] + b * p.y_batch[which] + row * p.y_row[which] + column;
#pragma unroll 4
      for (int head = share * groups + group; head < p.heads[which]; head += p.head_shares * groups) {
        uint4 v = *reinterpret_cast<const uint4*>(x + head * p.x_head[which]);
        uint32_t* words = &v.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = low_bf16(words[i]), c = high_bf16(words[i]);
          if (turned[i]) words[i] = two_bf16(a * turn[i].cos - c * turn[i].sin, a * turn[i].sin + c * turn[i].cos);
        }
        *reinterpret_cast<uint4*>(y + head * p.y_head[which]) = v;
      }
    }
  }
}

// Halves: pair p is (p, p + pairs); a lane holds eight pairs as 16 bytes of each half. The columns behind 2 * pairs
// are copied by the lanes behind the pairs'.
template <int TYPE>
__global__ void __launch_bounds__(256) rotary_halves_kernel(const RotaryParams p, int lanes) {
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  if (item >= p.items) return;
  const int lane = threadIdx.x % 32;
  const int share = static_cast<int>(item % p.head_shares);
  const int64_t place = item / p.head_shares;
  const int64_t b = place / p.rows, row = place - b * p.rows;
  const int groups = 32 / lanes, group = lane / lanes;
  const int64_t at = b * p.pos_batch + row * p.pos_row;
  const int units = p.pairs / 8 + (p.head_dim - 2 * p.pairs) / 8;
  for (int unit = lane % lanes; unit < units; unit += lanes) {
    const bool turned = unit < p.pairs / 8;
    const int column = turned ? unit * 8 : p.pairs + unit * 8;
    Turn turn[8];
    if (turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn[i] = turn_of<TYPE>(p, column + i, at);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const __nv_bfloat16* x = p.x[which] + b * p.x_batch[which] + row * p.x_row[which] + column;
      __nv_bfloat16* y = p.y[which] + b * p.y_batch[which] + row * p.y_row[which] + column;
#pragma unroll 2
      for (int head = share * groups + group; head < p.heads[which]; head += p.head_shares * groups) {
        uint4 v = *reinterpret_cast<const uint4*>(x + head * p.x_head[which]);
        if (turned) {
          uint4 w = *reinterpret_cast<const uint4*>(x + head * p.x_head[which] + p.pairs);
          uint32_t *first = &v.x, *second = &w.x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a0 = low_bf16(first[i]), a1 = high_bf16(first[i]);
            const float c0 = low_bf16(second[i]), c1 = high_bf16(second[i]);
            const Turn t0 = turn[2 * i], t1 = turn[2 * i + 1];
            first[i] = two_bf16(a0 * t0.cos - c0 * t0.sin, a1 * t1.cos - c1 * t1.sin);
            second[i] = two_bf16(a0 * t0.sin + c0 * t0.cos, a1 * t1.sin + c1 * t1.cos);
          }
          *reinterpret_cast<uint4*>(y + head * p.y_head[which] + p.pairs) = w;
        }
        *reinterpret_cast<uint4*>(y + head * p.y_head[which]) = v;
      }
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

template <int TYPE>
void launch(const RotaryParams& p, bool interleaved, cudaStream_t stream) {
  const int units = interleaved ? p.head_dim / 8 : p.pairs / 8 + (p.head_dim - 2 * p.pairs) / 8;
  int lanes = 1;
  while (lanes < units && lanes < 32) lanes *= 2;
  const unsigned grid = static_cast<unsigned>((p.items + 7) / 8);
  if (interleaved)
    rotary_interleaved_kernel<TYPE><<<grid, 256, 0, stream>>>(p, lanes);
  else
    rotary_halves_kernel<TYPE><<<grid, 256, 0, stream>>>(p, lanes);
}

}  // namespace

extern "C" int mup_axial_rotary_launch(const mup_axial_rotary* args, void* stream) {
  if (args == nullptr) return host_fail(MUP_ERR_BAD_ARG, "axial rotary: null argument");
  const mup_axial_rotary& a = *args;
  if (a.head_dim < 8 || a.head_dim > 512 || a.head_dim % 8 != 0)
    return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: head_dim %d is not a multiple of 8 up to 512", a.head_dim);
  if (a.pairs < 1 || 2 * a.pairs > a.head_dim || (!a.interleaved && a.pairs % 8 != 0))
    return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: %d pairs in heads of %d", a.pairs, a.head_dim);
  if (a.batch < 1 || a.rows < 1 || a.axes < 1 || a.heads[0] < 1 || a.heads[1] < 0)
    return host_fail(MUP_ERR_BAD_ARG, "axial rotary: batch %d, rows %d, axes %d, heads %d and %d", a.batch, a.rows,
                     a.axes, a.heads[0], a.heads[1]);
  if (a.positions == nullptr || a.turns == nullptr || a.pair_axis == nullptr || a.position_type < 0 || a.position_type > 2)
    return host_fail(MUP_ERR_BAD_ARG, "axial rotary: positions or frequencies are missing");
  RotaryParams p{};
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    int rc = check_rows(t == 0 ? "q" : "k", a.x[t], a.x_strides[t]);
    if (rc == MUP_OK) rc = check_rows(t == 0 ? "q's output" : "k's output", a.y[t], a.y_strides[t]);
    if (rc != MUP_OK) return rc;
    p.x[t] = static_cast<const __nv_bfloat16*>(a.x[t]), p.y[t] = static_cast<__nv_bfloat16*>(a.y[t]);
    p.x_batch[t] = a.x_strides[t][0], p.x_row[t] = a.x_strides[t][1], p.x_head[t] = a.x_strides[t][2];
    p.y_batch[t] = a.y_strides[t][0], p.y_row[t] = a.y_strides[t][1], p.y_head[t] = a.y_strides[t][2];
    p.heads[t] = a.heads[t];
  }
  p.positions = a.positions;
  p.pos_axis = a.pos_strides[0], p.pos_batch = a.pos_strides[1], p.pos_row = a.pos_strides[2];
  p.turns = a.turns, p.pair_axis = a.pair_axis;
  p.rows = a.rows, p.head_dim = a.head_dim, p.pairs = a.pairs;
  p.head_shares = 1;
  p.items = static_cast<int64_t>(a.batch) * a.rows * p.head_shares;
  if (p.items / 8 >= 0x7fffffff) return host_fail(MUP_ERR_UNSUPPORTED, "axial rotary: too many rows");
  p.sign = a.inverse ? -1.0f : 1.0f;
  DeviceScope scope(a.device);
  MUP_HOST_CUDA(scope.error());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.position_type == MUP_ROTARY_INT32)
    launch<MUP_ROTARY_INT32>(p, a.interleaved != 0, s);
  else if (a.position_type == MUP_ROTARY_INT64)
    launch<MUP_ROTARY_INT64>(p, a.interleaved != 0, s);
  else
    launch<MUP_ROTARY_FLOAT32>(p, a.interleaved != 0, s);
  MUP_HOST_CUDA(cudaGetLastError());
  return MUP_OK;
}

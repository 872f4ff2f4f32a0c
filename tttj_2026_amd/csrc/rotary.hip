// Rotary positions: in every head, pairs (a, b) of features are turned by position times the pair's frequency,
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),
// or back (transposed), which is the gradient.  Pairs are halves of the turned part (i, i + pairs) or neighbours
// (2 i, 2 i + 1); features behind the turned part stay.
//
// The angle is worked out in turns in 64 bits, whose whole part is dropped exactly; what is left, less the nearest quarter,
// is at most an eighth of a turn, where the Taylor sums of sine and cosine to the 9th and 8th power are off by 2^-25.
#include "cache_checks.hpp"
#include "kernels.hpp"
#include "seq_attention.hpp"

namespace tt {

struct RotaryArgs {
  const uint16_t* x;
  uint16_t* out;
  const double* frequencies;
  const int32_t *positions, *starts, *lengths;
  int64_t x_row, x_head, out_row, out_head;
  int tokens, batch, heads, head_dim, pairs;
  int units, per_pass, waves;  // V pairs each, of a head; heads of a wave's pass; waves per token
  float magnitude, sign;       // sign -1: transposed
};

// Cosine and sine of 2 pi t.
__device__ __forceinline__ float2 cos_sin_turns(double t) {
  t -= rint(t);
  const double quarter = rint(4.0 * t);
  const float x = (float)(t - 0.25 * quarter) * 6.2831853071795865f, y = x * x;
  const float s = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f);
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int q = (int)quarter & 3;
  const float co = (q & 1) ? s : c, si = (q & 1) ? c : s;
  return make_float2((q == 1 || q == 2) ? -co : co, (q & 2) ? -si : si);
}

// `waves` waves per token, each of which works out the token's cosines and sines for itself (a pair per lane, through LDS)
// and turns every waves-th group of heads; a lane has the same V pairs in all of them.  Bound by HBM: 36207 tokens on 40 heads
// of 128 137 us, 5.4 TB/s read and written; 8192 tokens on 32 heads of 64, half of each turned, 14.5 us (16.3 with no load
// before the position, 18 with the pieces that stay read at the end).
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  typedef T vec __attribute__((ext_vector_type(V)));
  __shared__ float2 s_turn[4][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int task = (int)blockIdx.x * 4 + wave, token = task / a.waves, share = task - token * a.waves;
  if (token >= a.tokens) return;
  const T* const x = reinterpret_cast<const T*>(a.x) + token * a.x_row;
  T* const out = reinterpret_cast<T*>(a.out) + token * a.out_row;
  const int in = lane / a.units, head0 = share * a.per_pass + in;
  int unit = lane - in * a.units;
  const auto first = [&]() { return INTERLEAVED ? 2 * V * unit : V * unit; };
  const auto second = [&]() { return INTERLEAVED ? 2 * V * unit + V : a.pairs + V * unit; };
  const auto load = [&](int head, int at) { return *reinterpret_cast<const vec*>(x + head * a.x_head + at); };
  // The first heads are asked for before the position, which takes several loads that wait for one another.
  vec y, z;
  bool live = in < a.per_pass && unit < a.units && head0 < a.heads;
  if (live) y = load(head0, first()), z = load(head0, second());
  // Pieces of the heads that stay as they are, the lane's first two as well: they lie in the lines that are read for the rest
  // of their heads, and later those may have gone from the caches.
  const int rest = (a.head_dim - 2 * a.pairs) / V, pieces = a.out == a.x ? 0 : a.heads * rest;
  const auto piece = [&](int e) { return make_int2(e / rest, 2 * a.pairs + e % rest * V); };  // its head, and where
  vec kept[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = share * 64 + lane + 64 * a.waves * i;
    if (e < pieces) kept[i] = load(piece(e).x, piece(e).y);
  }
  int64_t position;
  if (a.positions != nullptr) {
    position = a.positions[token];
  } else {
    int seq = token, i = 0, count = 1;
    if (a.starts != nullptr) {
      seq = seq_search(a.batch, token, [&](int b) { return seq_start(a.starts, b, a.tokens); });
      const int first = seq_start(a.starts, seq, a.tokens);
      i = token - first;
      count = seq_start(a.starts, seq + 1, a.tokens) - first;
      if (i < 0 || i >= count) return;
    }
    position = (int64_t)a.lengths[seq] - count + i;
  }
  for (int p = lane; p < a.pairs; p += 64) {
    const float2 t = cos_sin_turns((double)position * (a.frequencies[p] * 0.15915494309189533577));
    s_turn[wave][p] = make_float2(t.x * a.magnitude, t.y * a.magnitude * a.sign);
  }
  lds_done();
  while (live) {
    float2 turn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) turn[i] = s_turn[wave][unit * V + i];
    for (int head = head0; head < a.heads;) {
      const int next = head + a.waves * a.per_pass;
      vec y1 = y, z1 = z;
      if (next < a.heads) y1 = load(next, first()), z1 = load(next, second());
      T from[2 * V], to[2 * V];
#pragma unroll
      for (int i = 0; i < V; ++i) from[i] = y[i], from[V + i] = z[i];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int p = INTERLEAVED ? 2 * i : i, q = INTERLEAVED ? 2 * i + 1 : V + i;
        const float u = (float)from[p], v = (float)from[q];
        to[p] = (T)(u * turn[i].x - v * turn[i].y);
        to[q] = (T)(u * turn[i].y + v * turn[i].x);
      }
      vec r, s;
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = to[i], s[i] = to[V + i];
      *reinterpret_cast<vec*>(out + head * a.out_head + first()) = r;
      *reinterpret_cast<vec*>(out + head * a.out_head + second()) = s;
      head = next;
      y = y1, z = z1;
    }
    unit += 64;  // (more than 64 units of a head: one wave has them all)
    live = unit < a.units && a.units > 64;
    if (live) y = load(head0, first()), z = load(head0, second());
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = share * 64 + lane + 64 * a.waves * i;
    if (e < pieces) *reinterpret_cast<vec*>(out + piece(e).x * a.out_head + piece(e).y) = kept[i];
  }
  for (int e = share * 64 + lane + 64 * a.waves * 2; e < pieces; e += 64 * a.waves)
    *reinterpret_cast<vec*>(out + piece(e).x * a.out_head + piece(e).y) = load(piece(e).x, piece(e).y);
}

template <typename T, int V>
static void launch_rotary_as(const RotaryArgs& a, bool interleaved, int blocks, hipStream_t stream) {
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, V, true>), dim3(blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, V, false>), dim3(blocks), dim3(256), 0, stream, a);
}

template <typename T>
static int launch_rotary(RotaryArgs& a, int width, bool interleaved, hipStream_t stream) {
  a.units = a.pairs / width;
  a.per_pass = a.units < 64 ? 64 / a.units : 1;
  const int passes = (a.heads + a.per_pass - 1) / a.per_pass;
  // Few tokens are spread over the chip, up to a pass per wave.
  a.waves = 1;
  while (2 * a.waves <= passes && (int64_t)a.tokens * a.waves < 4 * (int64_t)device_cus()) a.waves *= 2;
  const int blocks = (int)(((int64_t)a.tokens * a.waves + 3) / 4);
  if (width == 8) launch_rotary_as<T, 8>(a, interleaved, blocks, stream);
  else if (width == 4) launch_rotary_as<T, 4>(a, interleaved, blocks, stream);
  else if (width == 2) launch_rotary_as<T, 2>(a, interleaved, blocks, stream);
  else launch_rotary_as<T, 1>(a, interleaved, blocks, stream);
  return launch_status("rotary_kernel");
}

}  // namespace tt

extern "C" int tt_rotary(const tt_rotary_rows* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_rotary_rows, "rotary");
  TT_REQUIRE(c.tokens >= 0 && c.batch >= 0 && c.heads > 0, "rotary: bad shape (tokens %d, batch %d, heads %d)", c.tokens,
             c.batch, c.heads);
  TT_REQUIRE(c.pairs > 0 && c.head_dim <= 256 && 2 * (int64_t)c.pairs <= c.head_dim,
             "rotary: %d pairs of features in heads of %d (256 at most)", c.pairs, c.head_dim);
  TT_REQUIRE((int64_t)c.tokens * c.heads < (1LL << 31) && c.tokens < (1 << 26) &&
                 (int64_t)c.heads * c.head_dim <= (1LL << 30),
             "rotary: %d tokens of %d heads of %d", c.tokens, c.heads, c.head_dim);
  TT_REQUIRE(c.dtype == TT_FP16 || c.dtype == TT_BF16, "rotary: bad dtype %d", c.dtype);
  TT_REQUIRE(c.magnitude == c.magnitude && fabsf(c.magnitude) < INFINITY, "rotary: magnitude %g is not finite", c.magnitude);
  TT_REQUIRE((c.positions != nullptr) != (c.lengths != nullptr), "rotary: either positions or lengths are needed");
  TT_REQUIRE(c.starts == nullptr || c.positions == nullptr, "rotary: starts come with lengths");
  if (c.tokens == 0) return TT_OK;
  if (c.positions == nullptr) {
    TT_REQUIRE(c.starts != nullptr || c.tokens == c.batch, "rotary: %d tokens for %d sequences without starts", c.tokens,
               c.batch);
    if (c.batch == 0) return TT_OK;
  }
  TT_REQUIRE(c.x && c.out && c.frequencies, "rotary: null pointer");
  TT_REQUIRE(c.x_row >= 0 && c.x_head >= 0 && (c.out_row > 0 || c.tokens == 1) && (c.out_head > 0 || c.heads == 1),
             "rotary: strides %lld, %lld of x and %lld, %lld of out", (long long)c.x_row, (long long)c.x_head,
             (long long)c.out_row, (long long)c.out_head);
  TT_REQUIRE(c.out_row >= 0 && c.out_head >= 0, "rotary: strides %lld, %lld of out", (long long)c.out_row,
             (long long)c.out_head);
  TT_REQUIRE(c.x != c.out || (c.x_row == c.out_row && c.x_head == c.out_head), "rotary: in place with other strides");
  const uint64_t grain = ((uintptr_t)c.x | (uintptr_t)c.out) / 2 | (uint64_t)c.x_row | (uint64_t)c.x_head |
                         (uint64_t)c.out_row | (uint64_t)c.out_head | (uint64_t)c.pairs | (uint64_t)c.head_dim;
  TT_REQUIRE((((uintptr_t)c.x | (uintptr_t)c.out) & 1) == 0 && ((uintptr_t)c.frequencies & 7) == 0, "rotary: not aligned");
  // Lanes read and write as many features at once as all addresses are aligned to.
  const int width = (grain & 7) == 0 ? 8 : (grain & 3) == 0 ? 4 : (grain & 1) == 0 ? 2 : 1;
  RotaryArgs a{};
  a.x = static_cast<const uint16_t*>(c.x), a.out = static_cast<uint16_t*>(c.out), a.frequencies = c.frequencies;
  a.positions = c.positions, a.starts = c.starts, a.lengths = c.lengths;
  a.x_row = c.x_row, a.x_head = c.x_head, a.out_row = c.out_row, a.out_head = c.out_head;
  a.tokens = c.tokens, a.batch = c.batch, a.heads = c.heads, a.head_dim = c.head_dim, a.pairs = c.pairs;
  a.magnitude = c.magnitude, a.sign = c.transpose ? -1.f : 1.f;
  return c.dtype == TT_FP16 ? launch_rotary<half>(a, width, c.interleaved != 0, (hipStream_t)stream)
                            : launch_rotary<bf16>(a, width, c.interleaved != 0, (hipStream_t)stream);
}

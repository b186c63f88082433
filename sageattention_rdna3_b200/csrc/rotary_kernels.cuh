// Rotary positions, by themselves and on the way into a paged cache.
//
// Pair (x, y) of a head becomes (x cos a - y sin a, x sin a + y cos a), a = frequency of the pair * position of the token on
// the pair's axis.  Both kernels read every value once and write it once: they are bound by HBM, and by the latency of a
// launch when there are few tokens.
//
// The angle.  A position of 10^6 times a frequency in fp32 is off by up to 0.06 radians.  Here the frequency is a
// fraction of a turn in units of 2^-64; a 64-bit product with the integer position wraps at whole turns by itself, and
// its upper 32 bits are the angle, to 2^-32 turns of that product, without a range reduction.  The frequency itself is rounded to 2^-64:
// at position p that is p 2^-65 turns more.
//
// The split.  A thread owns 8 pairs of a token (16-byte loads of both halves), computes their 8 angles once and walks over
// a slice of the heads with them, two heads in flight: with one head per thread the sines take longer than the memory.
// us, 4213 tokens, 48 + 12 heads of 128 (floor 20.1) / 24576 tokens, 32 heads of 64 (31.2) / append of 8404 tokens, 48 + 24 heads (48):
// slices of 2 heads 31.7 / 43.6 / 72.3, of 4 26.1 / 35.2 / 60.2, of 8 26.1 / 35.1 / 58.3, of 16 29.5 / 39.2 / 59.7; four heads in flight
// (three blocks per SM instead of four) in slices of 8 26.9 / 39.0 / 60.1; one 30.0 / 39.2 / 63.7.  sincospif in place of the
// polynomials below 26.6 / 35.6 / 62.4.  fp32, 24576 tokens, 32 heads of 64: 76.4 us, 82 % of the copy rate (15 registers spill).
#pragma once

#include "paged_common.cuh"

namespace sage {
namespace paged {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryBlocks = 4;                      // per SM
constexpr int kHeadsInFlight = 2;

struct Rotary {
  const uint64_t* freq;         // null: nothing is turned
  const int32_t* axis;
  int pairs, n_axes, interleaved;
  const void* positions;        // null (append only): the position in the sequence
  int positions_64;
  long long stride_b, stride_s;
  int inverse;
};

struct HeadSpan {               // rows of one tensor, [.., head, D]
  const void* in;
  void* out;
  long long in_b, in_h, in_s, out_b, out_h, out_s;
};

// 16 elements of a head as two groups of 8: those of the lower and of the upper half of the pairs (or 16 neighbours).
template <typename T>
struct Group {
  static constexpr int kVec = sizeof(T) / 2;          // 16-byte vectors per 8 elements
  uint4 a[kVec], b[kVec];
  __device__ __forceinline__ void load(const T* lo, const T* hi) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      a[i] = reinterpret_cast<const uint4*>(lo)[i];   // (not through the read-only path: an output may be its input)
      b[i] = reinterpret_cast<const uint4*>(hi)[i];
    }
  }
  __device__ __forceinline__ void store(T* lo, T* hi) const {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      reinterpret_cast<uint4*>(lo)[i] = a[i];
      reinterpret_cast<uint4*>(hi)[i] = b[i];
    }
  }
  __device__ __forceinline__ void turn(const float (&c)[8], const float (&s)[8], bool interleaved) {
    uint32_t* wa = reinterpret_cast<uint32_t*>(a);
    uint32_t* wb = reinterpret_cast<uint32_t*>(b);
    if constexpr (sizeof(T) == 4) {
      float* fa = reinterpret_cast<float*>(a);
      float* fb = reinterpret_cast<float*>(b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float& x = interleaved ? (i < 4 ? fa[2 * i] : fb[2 * i - 8]) : fa[i];
        float& y = interleaved ? (i < 4 ? fa[2 * i + 1] : fb[2 * i - 7]) : fb[i];
        const float x0 = x, y0 = y;
        x = x0 * c[i] - y0 * s[i];
        y = x0 * s[i] + y0 * c[i];
      }
    } else if (interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t& w = i < 4 ? wa[i] : wb[i - 4];
        const float2 v = to_float2(w, static_cast<const T*>(nullptr));
        w = from_float2(v.x * c[i] - v.y * s[i], v.x * s[i] + v.y * c[i], static_cast<const T*>(nullptr));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 xf = to_float2(wa[i], static_cast<const T*>(nullptr)), yf = to_float2(wb[i], static_cast<const T*>(nullptr));
        const f32x2_t x = pack2(xf.x, xf.y), y = pack2(yf.x, yf.y);
        const f32x2_t cc = pack2(c[2 * i], c[2 * i + 1]), ss = pack2(s[2 * i], s[2 * i + 1]);
        const float2 lo = unpack2(ffma2(y, pack2(-s[2 * i], -s[2 * i + 1]), fmul2(x, cc)));
        const float2 hi = unpack2(ffma2(y, cc, fmul2(x, ss)));
        wa[i] = from_float2(lo.x, lo.y, static_cast<const T*>(nullptr));
        wb[i] = from_float2(hi.x, hi.y, static_cast<const T*>(nullptr));
      }
    }
  }
};

// Offsets of the two groups of chunk `c` (16 elements) of a head, and whether it holds pairs at all.
__device__ __forceinline__ bool chunk_offsets(int c, const Rotary& r, int* lo, int* hi) {
  const bool turned = c < r.pairs / 8;                // (2 * pairs is a multiple of 16)
  if (turned && !r.interleaved) {
    *lo = 8 * c;
    *hi = r.pairs + 8 * c;
  } else {
    *lo = 16 * c;
    *hi = 16 * c + 8;
  }
  return turned;
}

__device__ __forceinline__ long long position_at(const Rotary& r, long long offset, int axis) {
  return r.positions_64 ? static_cast<const long long*>(r.positions)[offset + axis]
                        : static_cast<const int32_t*>(r.positions)[offset + axis];
}

// cos and sin of 2 pi t / 2^32 for two angles.  The nearest quarter turn is taken off in integers, which leaves r in
// [-1/8, 1/8] turns, exact to fp32; there sin(2 pi r) = r S(r^2) and cos(2 pi r) = C(r^2) with polynomials of degree 3 and 4, fitted for
// the smallest largest error (1.2e-9 and 9.5e-11; 1e-7 with fp32 arithmetic).  Two angles at a time in packed arithmetic this is
// half the instructions of sincospif, and the sines are what the kernel computes most.
__device__ __forceinline__ void sincos_turns(uint32_t t0, uint32_t t1, float* s0, float* s1, float* c0, float* c1) {
  const uint32_t q0 = (t0 + 0x20000000u) >> 30, q1 = (t1 + 0x20000000u) >> 30;
  const f32x2_t r = fmul2(pack2(static_cast<float>(static_cast<int32_t>(t0 - (q0 << 30))), static_cast<float>(static_cast<int32_t>(t1 - (q1 << 30)))),
                          pack2(2.3283064365386963e-10f, 2.3283064365386963e-10f));
  const f32x2_t u = fmul2(r, r);
  auto both = [](float x) { return pack2(x, x); };
  f32x2_t s = ffma2(u, both(-75.24006420070805f), both(81.58812464087775f));
  s = ffma2(u, s, both(-41.34162804270634f));
  s = fmul2(r, ffma2(u, s, both(6.28318522034183f)));
  f32x2_t c = ffma2(u, both(59.22040756857688f), both(-85.44285212867844f));
  c = ffma2(u, c, both(64.93931620850677f));
  c = ffma2(u, c, both(-19.739208650358023f));
  c = ffma2(u, c, both(1.0f));
  const float2 ss = unpack2(s), cc = unpack2(c);
  // quarter turns: (sin, cos) -> (cos, -sin) -> (-sin, -cos) -> (-cos, sin)
  auto place = [](uint32_t q, float sn, float cs, float* s_out, float* c_out) {
    const float a = q & 1u ? cs : sn, b = q & 1u ? sn : cs;
    *s_out = __uint_as_float(__float_as_uint(a) ^ (q << 30 & 0x80000000u));
    *c_out = __uint_as_float(__float_as_uint(b) ^ ((q + 1u) << 30 & 0x80000000u));
  };
  place(q0, ss.x, cc.x, s0, c0);
  place(q1, ss.y, cc.y, s1, c1);
}

// cos and sin of the 8 pairs of a chunk; `pos` holds the token's position on every axis.
__device__ __forceinline__ void chunk_angles(const Rotary& r, int chunk, const long long (&pos)[SAGE_MAX_ROTARY_AXES], float (&c)[8],
                                             float (&s)[8]) {
  const ulonglong2* freq = reinterpret_cast<const ulonglong2*>(r.freq + 8 * chunk);
  const int4* axes = reinterpret_cast<const int4*>(r.axis + 8 * chunk);
  uint32_t turns[8];
  auto turn = [&](int axis, unsigned long long f) -> uint32_t {
    long long at = pos[0];
    if (r.n_axes > 1) {
      at = axis == 1 ? pos[1] : at;
      at = axis == 2 ? pos[2] : at;
      at = axis == 3 ? pos[3] : at;
    }
    return static_cast<uint32_t>(static_cast<unsigned long long>(at) * f >> 32);
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int4 a = r.n_axes > 1 ? __ldg(axes + i) : make_int4(0, 0, 0, 0);
    const ulonglong2 f = __ldg(freq + 2 * i), g = __ldg(freq + 2 * i + 1);
    turns[4 * i] = turn(a.x, f.x);
    turns[4 * i + 1] = turn(a.y, f.y);
    turns[4 * i + 2] = turn(a.z, g.x);
    turns[4 * i + 3] = turn(a.w, g.y);
  }
#pragma unroll
  for (int i = 0; i < 8; i += 2) sincos_turns(turns[i], turns[i + 1], &s[i], &s[i + 1], &c[i], &c[i + 1]);
  if (r.inverse) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = -s[i];
  }
}

struct RotaryParams {
  HeadSpan q, k;
  Rotary rotary;
  int B, S, Hq, Hkv;
  int heads_per_block;
};

// grid: (token blocks, slices of the Hq + Hkv heads)
template <typename T, int D>
__global__ void __launch_bounds__(kRotaryThreads, kRotaryBlocks) sage_rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int kChunks = D / 16;
  constexpr int kTokens = kRotaryThreads / kChunks;
  const int chunk = threadIdx.x % kChunks;
  const long long token = static_cast<long long>(blockIdx.x) * kTokens + threadIdx.x / kChunks;
  grid_dependency_wait();
  grid_launch_dependents();
  if (token >= static_cast<long long>(p.B) * p.S) return;
  const int b = static_cast<int>(token / p.S), at = static_cast<int>(token - static_cast<long long>(b) * p.S);
  int lo, hi;
  const bool turned = chunk_offsets(chunk, p.rotary, &lo, &hi);
  const int h0 = blockIdx.y * p.heads_per_block, h1 = min(h0 + p.heads_per_block, p.Hq + p.Hkv);

  auto span_of = [&](int h, const T** in, T** out) {
    const bool is_q = h < p.Hq;
    const HeadSpan& x = is_q ? p.q : p.k;
    const int hh = is_q ? h : h - p.Hq;
    *in = static_cast<const T*>(x.in) + b * x.in_b + hh * x.in_h + at * x.in_s;
    *out = static_cast<T*>(x.out) + b * x.out_b + hh * x.out_h + at * x.out_s;
  };
  float c[8], s[8];
#pragma unroll 1
  for (int h = h0; h < h1; h += kHeadsInFlight) {
    Group<T> g[kHeadsInFlight];
    T* out[kHeadsInFlight];
#pragma unroll
    for (int u = 0; u < kHeadsInFlight; ++u) {
      const T* in;
      span_of(min(h + u, h1 - 1), &in, &out[u]);
      g[u].load(in + lo, in + hi);
    }
    if (h == h0 && turned) {                          // under the first loads
      long long pos[SAGE_MAX_ROTARY_AXES];
      const long long offset = b * p.rotary.stride_b + at * p.rotary.stride_s;
#pragma unroll
      for (int a = 0; a < SAGE_MAX_ROTARY_AXES; ++a) pos[a] = a < p.rotary.n_axes ? position_at(p.rotary, offset, a) : 0;
      chunk_angles(p.rotary, chunk, pos, c, s);
    }
#pragma unroll
    for (int u = 0; u < kHeadsInFlight; ++u) {
      if (h + u >= h1) break;
      if (turned) g[u].turn(c, s, p.rotary.interleaved != 0);
      g[u].store(out[u] + lo, out[u] + hi);
    }
  }
}

struct AppendParams {
  HeadSpan q, k, v;             // strides _b unused; the outputs of k and v are the pages (out_b page, out_s slot)
  Rotary rotary;
  Batch batch;
  Status status;
  int Hq, Hkv;
  int heads_per_block;
};

constexpr int kAppendCuMax = 1024;                    // sequences whose cu_q is searched in shared memory

// Heads in the order q, k, v.  grid: (token blocks, slices of the Hq + 2 Hkv heads)
template <typename T, int D>
__global__ void __launch_bounds__(kRotaryThreads, kRotaryBlocks) sage_paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kChunks = D / 16;
  constexpr int kTokens = kRotaryThreads / kChunks;
  __shared__ int s_cu[kAppendCuMax + 1];
  const int chunk = threadIdx.x % kChunks;
  const long long token_ll = static_cast<long long>(blockIdx.x) * kTokens + threadIdx.x / kChunks;
  grid_dependency_wait();
  grid_launch_dependents();
  const bool searched = p.batch.cu_q != nullptr, in_shared = p.batch.B <= kAppendCuMax;
  if (searched && in_shared) {
    for (int i = threadIdx.x; i <= p.batch.B; i += kRotaryThreads) s_cu[i] = p.batch.cu_q[i];
    __syncthreads();
  }
  if (token_ll >= p.batch.T) return;
  const int token = static_cast<int>(token_ll);

  // The sequence of the token: the last one that starts at or before it.
  int b = token;
  if (searched) {
    const int32_t* cu = p.batch.cu_q;
    int lo = 0, hi = p.batch.B;                       // cu[lo] <= token < cu[hi], as far as that holds at all
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if ((in_shared ? s_cu[mid] : cu[mid]) <= token) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  int q0, q1;
  p.batch.tokens(b, &q0, &q1);
  // (without cu_q a sequence of length 0 is a slot that is not in use: its row belongs to no sequence)
  const bool belongs = token >= q0 && token < q1 && (searched || p.batch.kv_lens[b] != 0);
  const long long at = belongs ? static_cast<long long>(p.batch.kv_lens[b]) - (q1 - token) : 0;
  long long page = -1;
  int slot = 0;
  if (belongs) {
    const long long col = at >> p.batch.page_log2;
    slot = static_cast<int>(at & ((1 << p.batch.page_log2) - 1));
    int code = 0;
    if (at < 0 || col >= p.batch.table_width) {
      code = kStatusBadLength;
    } else {
      page = p.batch.table[b * p.batch.table_stride + col];
      if (page < 0 || page >= p.batch.num_pages) {
        page = -1;
        code = kStatusBadPage;
      }
    }
    if (code != 0 && chunk == 0 && blockIdx.y == 0) p.status.report(code);
  }

  int lo = 16 * chunk, hi = lo + 8;
  const bool turned = p.rotary.freq != nullptr && chunk_offsets(chunk, p.rotary, &lo, &hi);
  const int heads_turned = p.Hq + p.Hkv, heads = heads_turned + p.Hkv;
  const int h0 = blockIdx.y * p.heads_per_block, h1 = min(h0 + p.heads_per_block, heads);
  auto span_of = [&](int h, const T** in, T** out) {
    const HeadSpan& x = h < p.Hq ? p.q : h < heads_turned ? p.k : p.v;
    const int hh = h < p.Hq ? h : h < heads_turned ? h - p.Hq : h - heads_turned;
    *in = static_cast<const T*>(x.in) + hh * x.in_h + token * x.in_s;
    if (h < p.Hq) *out = static_cast<T*>(x.out) + hh * x.out_h + token * x.out_s;
    else *out = page < 0 ? nullptr : static_cast<T*>(x.out) + page * x.out_b + hh * x.out_h + slot * x.out_s;
  };
  float c[8], s[8];
#pragma unroll 1
  for (int h = h0; h < h1; h += kHeadsInFlight) {
    Group<T> g[kHeadsInFlight];
    T* out[kHeadsInFlight];
#pragma unroll
    for (int u = 0; u < kHeadsInFlight; ++u) {
      const T* in;
      span_of(min(h + u, h1 - 1), &in, &out[u]);
      g[u].load(in + lo, in + hi);
    }
    if (h == h0 && turned && h0 < heads_turned) {     // under the first loads
      long long pos[SAGE_MAX_ROTARY_AXES];
#pragma unroll
      for (int a = 0; a < SAGE_MAX_ROTARY_AXES; ++a) {
        pos[a] = p.rotary.positions == nullptr ? at : a < p.rotary.n_axes ? position_at(p.rotary, token * p.rotary.stride_s, a) : 0;
      }
      chunk_angles(p.rotary, chunk, pos, c, s);
    }
#pragma unroll
    for (int u = 0; u < kHeadsInFlight; ++u) {
      if (h + u >= h1 || out[u] == nullptr) continue;
      if (!belongs) {                                 // a row of q that belongs to no sequence
#pragma unroll
        for (int i = 0; i < Group<T>::kVec; ++i) g[u].a[i] = g[u].b[i] = make_uint4(0, 0, 0, 0);
      } else if (turned && h + u < heads_turned) {
        g[u].turn(c, s, p.rotary.interleaved != 0);
      }
      g[u].store(out[u] + lo, out[u] + hi);
    }
  }
}

}  // namespace paged
}  // namespace sage

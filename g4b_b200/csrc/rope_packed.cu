// Per-head RMS norm, rotary embedding over several position axes, V norm and the paged append,
// for rows packed behind one another (prompts and chunks of different lengths, no padding).
//
// What rope_append.cu does for a [B, H, Tq, D] chunk whose positions count up, done for N rows
// of which slot b owns [q_starts[b], q_starts[b + 1]): the rotation pair i of a row turns by
// positions[axis(i)][row] * freqs[i] -- one axis for text; time, height and width for the patches
// of an image or a video -- while the row's place in the cache still counts up.
//
// The angle is reduced in 64 bits: at position 131072 a 32-bit product is off by up to
// 2^-8 rad, as much as a bf16 rounding.  A lane needs four angles per token against rows of hundreds of
// elements: 98.8 us for 32768 tokens of 8 + 2 + 2 heads of 256, 98.2 us with 32-bit angles.
//
// Pure streaming: reads N (H + 2G) D input elements, writes as many 16-bit ones.  A one-warp
// block takes one token with all its heads at prefill sizes (its sines and cosines are computed
// once), or a few heads of it at decode sizes, for parallelism.  kLanes lanes hold a row, each
// four consecutive rotation pairs (i, i + D/2) per pass, so a warp holds 32 / kLanes rows at a
// time; loads of four such sets go out before any is processed.
//
// Measured (f32 in, 16 bits out, 8 + 2 + 2 heads of 256, three sets of inputs in turn; 97 to 104 us by the way the passes are
// timed): 32768 tokens 97.5 us = 6190 GB/s, 0.95 of the copy; 4417 tokens of three axes 20.1 us (launches alone 18.2; 13.1
// with one set, which stays in L2).  32 / 28 / 24 warps an SM: 97.5 / 100.8 / 106.6 and 20.1 / 24.1 / 24.3 us; 4300 tokens at head dim
// 128, where 32 warps leave 64 registers and 48 to 72 bytes of spills, 13.9 / 15.4 / 15.8 us.  What bounds it is the issue rate (2.4 of 4
// instructions a cycle) next to HBM, as in rope_append.cu.
#include "common.cuh"

namespace g4b {
namespace {

struct RopePackedParams {
  const void* q; const void* k; const void* v;
  void* q_out;
  const float* freqs;
  const void* positions;            // [A, N] int32 or int64, or null: the row's place in the cache
  const uint8_t* pair_axis;         // [D/2], or null: axis 0
  const int32_t* q_starts; const int32_t* times;
  const float* q_w; const float* k_w;
  void* k_pool; void* v_pool;
  const int32_t* block_tables;
  int64_t qs[2], ks[2], vs[2], qos[2];           // strides (elements) of row and head
  int64_t pos_s0, pos_s1, axis_s, starts_s, time_s, bt_s0, bt_s1, freq_s, qw_s, kw_s;
  int q_out_dtype, cache_dtype;
  int N, B, H, G, D, axes, n_heads, heads_per_warp;
  uint32_t n_slots;                 // warps per token
  int page_shift, num_pages, max_pages;
  int pos_i64, norm_qk, norm_v;
  int starts_quads;                 // q_starts can be read four at a time
  float eps;
  int32_t* status;
};

enum : int32_t { kErrOutside = 0x101, kErrBadEntry = 0x102, kErrAxis = 0x106, kErrStarts = 0x107 };

__device__ __forceinline__ float4 widen4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 widen4(const __half* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 widen4(const __nv_bfloat16* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                     __uint_as_float(raw.y & 0xffff0000u));
}
__device__ __forceinline__ void narrow4(void* base, int dtype, int64_t at, float4 x) {
  if (dtype == G4B_F32) {
    *reinterpret_cast<float4*>((float*)base + at) = x;
    return;
  }
  uint2 raw;
  if (dtype == G4B_F16) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    raw = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    raw = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  *reinterpret_cast<uint2*>((uint16_t*)base + at) = raw;
}

// The slot that owns packed row `row`, and where its rows end; -1: no slot's row, kContradiction: starts that decrease or
// leave [0, N], for which nothing is computed (what they would append could lie anywhere in live pages).  A warp looks at
// all of them, since one that finds its slot by a search does not see whether the others agree: one a lane, or 128 a
// load, so that up to 127 slots are one trip to L2.  Against a 32-way search that trusts them (single tokens, one a slot): 8
// slots 3.3 us for 3.6, 64 slots 3.5 for 3.5, 256 slots 4.7 for 4.4, 1000 slots 14.1 for 10.7; 32768 rows of 5 the same.
constexpr int kContradiction = -2;
__device__ __forceinline__ int slot_of_row(const RopePackedParams& p, int row, int lane, int& end) {
  if (p.B < 32) {
    const int x = lane <= p.B ? p.q_starts[lane * p.starts_s] : p.N;
    const int prev = __shfl_up_sync(0xffffffffu, x, 1);
    if (__any_sync(0xffffffffu, x < (lane == 0 ? 0 : prev) || x > p.N)) return kContradiction;
    const int slot = __popc(__ballot_sync(0xffffffffu, x <= row)) - 1;   // (of slots that start there, the last: it has rows)
    if (slot >= p.B) return -1;
    end = __shfl_sync(0xffffffffu, x, slot + 1);
    return slot;
  }
  int up_to_row = 0, behind_row = p.N, before = 0;     // starts at or in front of the row; the first behind it
  bool bad = false;
#pragma unroll 2
  for (int first = 0; first <= p.B; first += 128) {
    const int at = first + lane * 4;
    int x[4] = {p.N, p.N, p.N, p.N};
    if (p.starts_quads && at + 3 <= p.B) {
      const int4 v = *reinterpret_cast<const int4*>(p.q_starts + at);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i <= p.B) x[i] = p.q_starts[(int64_t)(at + i) * p.starts_s];
    }
    int prev = __shfl_up_sync(0xffffffffu, x[3], 1);
    if (lane == 0) prev = before;
    before = __shfl_sync(0xffffffffu, x[3], 31);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bad |= x[i] < prev;
      prev = x[i];
      if (x[i] <= row) ++up_to_row;
      else behind_row = min(behind_row, x[i]);
    }
  }
  if (__any_sync(0xffffffffu, bad || before > p.N)) return kContradiction;
  end = __reduce_min_sync(0xffffffffu, behind_row);
  const int slot = __reduce_add_sync(0xffffffffu, up_to_row) - 1;
  return slot < p.B ? slot : -1;
}

// KIND 0 q, 1 k, 2 v.  kOut: the 16-bit type of q_out and the pools, or 0 for run-time types.
template <int KIND, typename In, int kLanes, int kIters, bool kExact, int kOut>
__device__ __forceinline__ void rows_of_kind(const RopePackedParams& p, int h_begin, int h_end, int row, int64_t page_row,
                                             int lane, const float4 (&sn)[kIters], const float4 (&cs)[kIters]) {
  constexpr int kSets = 4, kRows = 32 / kLanes;
  const int sub = lane / kLanes, l = lane % kLanes;
  const int half = p.D >> 1;
  const In* src = (const In*)(KIND == 0 ? p.q : (KIND == 1 ? p.k : p.v));
  const int64_t* ss = KIND == 0 ? p.qs : (KIND == 1 ? p.ks : p.vs);
  src += row * ss[0];
  if (KIND != 0 && page_row < 0) return;
  void* out = KIND == 0 ? p.q_out : (KIND == 1 ? p.k_pool : p.v_pool);
  const int dtype = kOut != 0 ? kOut : (KIND == 0 ? p.q_out_dtype : p.cache_dtype);
  const int64_t out_row = KIND == 0 ? row * p.qos[0] : page_row * p.D;
  const int64_t out_hs = KIND == 0 ? p.qos[1] : ((int64_t)p.D << p.page_shift);
  const bool norm = KIND == 2 ? p.norm_v != 0 : p.norm_qk != 0;
  const float* w = KIND == 0 ? p.q_w : (KIND == 1 ? p.k_w : nullptr);
  const int64_t ws = KIND == 0 ? p.qw_s : p.kw_s;
  const float inv_d = 1.f / (float)p.D;
  for (int h0 = h_begin; h0 < h_end; h0 += kSets * kRows) {
    float4 x1[kSets][kIters], x2[kSets][kIters];
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      const int h = h0 + i * kRows + sub;
      if (h < h_end) {
        const In* r = src + h * ss[1];
#pragma unroll
        for (int it = 0; it < kIters; ++it) {
          const int d = it * kLanes * 4 + l * 4;
          if (kExact || d < half) { x1[i][it] = widen4(r + d); x2[i][it] = widen4(r + d + half); }
          else { x1[i][it] = x2[i][it] = make_float4(0.f, 0.f, 0.f, 0.f); }
        }
      } else {
#pragma unroll
        for (int it = 0; it < kIters; ++it) x1[i][it] = x2[i][it] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      if (h0 + i * kRows >= h_end) break;      // (warp-uniform)
      const int h = h0 + i * kRows + sub;
      float inv = 1.f;
      if (norm) {
        float sq = 0.f;
#pragma unroll
        for (int it = 0; it < kIters; ++it) {
          const float4 a = x1[i][it], c = x2[i][it];
          sq += (a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w) + (c.x * c.x + c.y * c.y + c.z * c.z + c.w * c.w);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        inv = rsqrtf(sq * inv_d + p.eps);
      }
      if (h >= h_end) continue;
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        const int d = it * kLanes * 4 + l * 4;
        if (!kExact && d >= half) continue;
        float4 a = x1[i][it], c = x2[i][it];
        float4 wa = make_float4(inv, inv, inv, inv), wc = wa;
        if (KIND != 2 && norm && w != nullptr) {
          if (ws == 1) {
            const float4 u = *reinterpret_cast<const float4*>(w + d), t = *reinterpret_cast<const float4*>(w + d + half);
            wa = make_float4(inv * u.x, inv * u.y, inv * u.z, inv * u.w);
            wc = make_float4(inv * t.x, inv * t.y, inv * t.z, inv * t.w);
          } else {
            wa = make_float4(inv * w[d * ws], inv * w[(d + 1) * ws], inv * w[(d + 2) * ws], inv * w[(d + 3) * ws]);
            const int e = d + half;
            wc = make_float4(inv * w[e * ws], inv * w[(e + 1) * ws], inv * w[(e + 2) * ws], inv * w[(e + 3) * ws]);
          }
        }
        a = make_float4(a.x * wa.x, a.y * wa.y, a.z * wa.z, a.w * wa.w);
        c = make_float4(c.x * wc.x, c.y * wc.y, c.z * wc.z, c.w * wc.w);
        if (KIND != 2) {
          const float4 s = sn[it], o = cs[it];
          const float4 y = make_float4(o.x * a.x - s.x * c.x, o.y * a.y - s.y * c.y, o.z * a.z - s.z * c.z, o.w * a.w - s.w * c.w);
          c = make_float4(o.x * c.x + s.x * a.x, o.y * c.y + s.y * a.y, o.z * c.z + s.z * a.z, o.w * c.w + s.w * a.w);
          a = y;
        }
        const int64_t at = out_row + h * out_hs + d;
        narrow4(out, dtype, at, a);
        narrow4(out, dtype, at + half, c);
      }
    }
  }
}

template <typename In, int kLanes, int kIters, bool kExact, int kOut>
__global__ void __launch_bounds__(32, kIters == 1 ? 32 : 16) rope_packed_kernel(const __grid_constant__ RopePackedParams p) {
  const int lane = threadIdx.x;
  const int row = (int)(p.n_slots == 1 ? blockIdx.x : blockIdx.x / p.n_slots);
  const int part = (int)(blockIdx.x - (uint32_t)row * p.n_slots);
  const int half = p.D >> 1;
  int end = 0;
  const int b = slot_of_row(p, row, lane, end);
  if (b < 0) {                                        // rows that no slot owns stay as they are
    if (b == kContradiction && lane == 0) atomicCAS(p.status, 0, kErrStarts);
    return;
  }
  const int place = p.times[b * p.time_s] - (end - row);

  const int h_begin = part * p.heads_per_warp, h_end = min(h_begin + p.heads_per_warp, p.n_heads);
  const int q0 = min(h_begin, p.H), q1 = min(h_end, p.H);
  const int k0 = min(max(h_begin, p.H), p.H + p.G) - p.H, k1 = min(max(h_end, p.H), p.H + p.G) - p.H;
  const int v0 = max(h_begin, p.H + p.G) - p.H - p.G, v1 = max(h_end, p.H + p.G) - p.H - p.G;

  int64_t page_row = -1;                              // row of kv head 0 in the pools
  if (h_end > p.H) {
    const int pg = place >> p.page_shift;
    if (place < 0 || pg >= p.max_pages) {
      if (lane == 0) atomicCAS(p.status, 0, kErrOutside);
    } else {
      const int page = p.block_tables[b * p.bt_s0 + pg * p.bt_s1];
      if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicCAS(p.status, 0, kErrBadEntry);
      } else {
        page_row = (((int64_t)page * p.G) << p.page_shift) + (place & ((1 << p.page_shift) - 1));
      }
    }
  }
  float4 sn[kIters], cs[kIters];
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    sn[it] = make_float4(0.f, 0.f, 0.f, 0.f);
    cs[it] = make_float4(1.f, 1.f, 1.f, 1.f);
    const int d = it * kLanes * 4 + (lane % kLanes) * 4;
    if (h_begin < p.H + p.G && (kExact || d < half)) {
      float s4[4], c4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int axis = p.pair_axis != nullptr ? p.pair_axis[(d + i) * p.axis_s] : 0;
        if (axis >= p.axes) { atomicCAS(p.status, 0, kErrAxis); axis = 0; }
        int64_t pos = place;
        if (p.positions != nullptr) {
          const int64_t at = axis * p.pos_s0 + row * p.pos_s1;
          pos = p.pos_i64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
        }
        // turns, reduced to [-1/2, 1/2] before they become 32 bits
        double turns = (double)pos * ((double)p.freqs[(d + i) * p.freq_s] * 0.15915494309189533577);
        turns -= rint(turns);
        // the reduced angle is in [-pi, pi], where the fast functions are off by at most 2^-21.  An output is off by that
        // much of its pair's magnitude: 1/500 of a 16-bit rounding where it is about as large as the pair; more of its own rounding
        // where the two products cancel, as any 32-bit rotation's is (32768 tokens: 98.8 -> 97.5 us, 4417 of three axes: 20.8 -> 20.1)
        if constexpr (kOut != 0) __sincosf(6.2831853f * (float)turns, &s4[i], &c4[i]);
        else sincospif(2.f * (float)turns, &s4[i], &c4[i]);
      }
      sn[it] = make_float4(s4[0], s4[1], s4[2], s4[3]);
      cs[it] = make_float4(c4[0], c4[1], c4[2], c4[3]);
    }
  }
  if (q1 > q0) rows_of_kind<0, In, kLanes, kIters, kExact, kOut>(p, q0, q1, row, page_row, lane, sn, cs);
  if (k1 > k0) rows_of_kind<1, In, kLanes, kIters, kExact, kOut>(p, k0, k1, row, page_row, lane, sn, cs);
  if (v1 > v0) rows_of_kind<2, In, kLanes, kIters, kExact, kOut>(p, v0, v1, row, page_row, lane, sn, cs);
}

// An absent optional tensor has rank 0; one without elements (a step without rows) has no pointer.
bool given(const G4bTensor& t) { return t.ptr != nullptr || t.ndim != 0; }

int check_rank(const G4bTensor& t, const char* name, int ndim) {
  if (t.ndim != ndim) return fail(G4B_ERR_BAD_ARG, "%s: expected rank %d, got %d", name, ndim, t.ndim);
  bool empty = false;
  for (int i = 0; i < ndim; ++i) {
    if (t.shape[i] < 0) return fail(G4B_ERR_BAD_ARG, "%s: negative extent", name);
    empty |= t.shape[i] == 0;
  }
  if (t.ptr == nullptr && !empty) return fail(G4B_ERR_BAD_ARG, "%s: null pointer", name);
  return G4B_OK;
}

// [N, heads, D] rows a lane can read or write four elements of at a time
int check_rows(const G4bTensor& t, const char* name, int64_t N, int64_t heads, int64_t D) {
  int rc;
  if ((rc = check_rank(t, name, 3))) return rc;
  if ((N >= 0 && t.shape[0] != N) || (heads >= 0 && t.shape[1] != heads) || (D >= 0 && t.shape[2] != D))
    return fail(G4B_ERR_BAD_ARG, "%s: rows, heads or head dim do not agree", name);
  if (!is_float_dtype(t.dtype)) return fail(G4B_ERR_BAD_DTYPE, "%s must be f32, f16 or bf16", name);
  if (t.shape[2] > 1 && t.stride[2] != 1) return fail(G4B_ERR_BAD_STRIDE, "%s: innermost stride must be 1", name);
  if (((uintptr_t)t.ptr & 15) != 0) return fail(G4B_ERR_BAD_STRIDE, "%s: base must be 16-byte aligned", name);
  for (int i = 0; i < 2; ++i)
    if (t.shape[i] > 1 && (t.stride[i] % 4) != 0)
      return fail(G4B_ERR_BAD_STRIDE, "%s: strides must be multiples of 4 elements", name);
  return G4B_OK;
}

template <typename In, int kLanes, int kIters, bool kExact>
void launch_out(const RopePackedParams& p, unsigned blocks, int out16, cudaStream_t st) {
  if (out16 == G4B_F16) rope_packed_kernel<In, kLanes, kIters, kExact, G4B_F16><<<blocks, 32, 0, st>>>(p);
  else if (out16 == G4B_BF16) rope_packed_kernel<In, kLanes, kIters, kExact, G4B_BF16><<<blocks, 32, 0, st>>>(p);
  else rope_packed_kernel<In, kLanes, kIters, kExact, 0><<<blocks, 32, 0, st>>>(p);
}

template <typename In>
void launch_in(const RopePackedParams& p, unsigned blocks, int out16, cudaStream_t st) {
  if (p.D == 256) launch_out<In, 32, 1, true>(p, blocks, out16, st);
  else if (p.D == 512) launch_out<In, 32, 2, true>(p, blocks, out16, st);
  else if (p.D == 128) launch_out<In, 16, 1, true>(p, blocks, out16, st);
  else if (p.D <= 256) launch_out<In, 32, 1, false>(p, blocks, 0, st);
  else launch_out<In, 32, 2, false>(p, blocks, 0, st);
}

}  // namespace

int launch_rope_norm_append_packed(const G4bRopePackedArgs& a, cudaStream_t st) {
  int rc;
  if ((rc = check_rows(a.q, "q", -1, -1, -1))) return rc;
  const int64_t N = a.q.shape[0], H = a.q.shape[1], D = a.q.shape[2];
  if ((rc = check_rows(a.k, "k", N, -1, D))) return rc;
  const int64_t G = a.k.shape[1];
  if ((rc = check_rows(a.v, "v", N, G, D))) return rc;
  if (a.k.dtype != a.q.dtype || a.v.dtype != a.q.dtype) return fail(G4B_ERR_BAD_DTYPE, "q, k and v must have one dtype");
  if (D % 8 != 0 || D < 8 || D > 512) return fail(G4B_ERR_UNSUPPORTED, "head dim must be a multiple of 8, at most 512");
  if (H < 1 || G < 1) return fail(G4B_ERR_BAD_ARG, "at least one query head and one kv head");
  if (given(a.q_out) && (rc = check_rows(a.q_out, "q_out", N, H, D))) return rc;
  if (rows_overlap(given(a.q_out) ? a.q_out : a.q))
    return fail(G4B_ERR_BAD_STRIDE, "%s: rows that are written must not overlap", given(a.q_out) ? "q_out" : "q");
  if ((rc = check_rank(a.rope_freqs, "rope_freqs", 1))) return rc;
  if (a.rope_freqs.shape[0] != D / 2) return fail(G4B_ERR_BAD_ARG, "rope_freqs must have D/2 entries");
  if (a.rope_freqs.dtype != G4B_F32) return fail(G4B_ERR_BAD_DTYPE, "rope_freqs must be f32");
  int64_t axes = 1;
  if (given(a.positions)) {
    if ((rc = check_rank(a.positions, "positions", 2))) return rc;
    if (a.positions.dtype != G4B_I32 && a.positions.dtype != G4B_I64) return fail(G4B_ERR_BAD_DTYPE, "positions must be int32 or int64");
    if (a.positions.shape[1] != N || a.positions.shape[0] < 1) return fail(G4B_ERR_BAD_ARG, "positions must be [axes, N]");
    axes = a.positions.shape[0];
    if (axes > 255) return fail(G4B_ERR_UNSUPPORTED, "at most 255 position axes");
  }
  if (given(a.pair_axis)) {
    if ((rc = check_rank(a.pair_axis, "pair_axis", 1))) return rc;
    if (a.pair_axis.dtype != G4B_U8) return fail(G4B_ERR_BAD_DTYPE, "pair_axis must be uint8");
    if (a.pair_axis.shape[0] != D / 2) return fail(G4B_ERR_BAD_ARG, "pair_axis must have D/2 entries");
    if (!given(a.positions)) return fail(G4B_ERR_BAD_ARG, "pair_axis needs positions");
  } else if (axes > 1) {
    return fail(G4B_ERR_BAD_ARG, "positions over several axes need pair_axis");
  }
  if ((rc = check_rank(a.q_starts, "q_starts", 1)) || (rc = check_rank(a.time_dim_sizes, "time_dim_sizes", 1)) ||
      (rc = check_rank(a.block_tables, "block_tables", 2))) return rc;
  if (a.q_starts.dtype != G4B_I32 || a.time_dim_sizes.dtype != G4B_I32 || a.block_tables.dtype != G4B_I32)
    return fail(G4B_ERR_BAD_DTYPE, "q_starts, time_dim_sizes and block_tables must be int32");
  const int64_t B = a.time_dim_sizes.shape[0];
  if (a.q_starts.shape[0] != B + 1 || a.block_tables.shape[0] != B)
    return fail(G4B_ERR_BAD_ARG, "q_starts must have B + 1 entries and block_tables B rows");
  const G4bTensor* w[2] = {&a.q_norm_w, &a.k_norm_w};
  for (int i = 0; i < 2; ++i) {
    if (!given(*w[i])) continue;
    if ((rc = check_rank(*w[i], i == 0 ? "q_norm_w" : "k_norm_w", 1))) return rc;
    if (w[i]->shape[0] != D) return fail(G4B_ERR_BAD_ARG, "norm weights must have D entries");
    if (w[i]->dtype != G4B_F32) return fail(G4B_ERR_BAD_DTYPE, "norm weights must be f32");
    if (((uintptr_t)w[i]->ptr & 15) != 0) return fail(G4B_ERR_BAD_STRIDE, "norm weights must be 16-byte aligned");
  }
  const G4bTensor* pools[2] = {&a.k_pool, &a.v_pool};
  for (int i = 0; i < 2; ++i) {
    const G4bTensor& c = *pools[i];
    const char* nm = i == 0 ? "k_pool" : "v_pool";
    if ((rc = check_rank(c, nm, 4))) return rc;
    if (c.shape[1] != G || c.shape[2] != a.page_size || c.shape[3] != D)
      return fail(G4B_ERR_BAD_ARG, "%s must be [num_pages, G, page_size, D]", nm);
    if (!is_float_dtype(c.dtype)) return fail(G4B_ERR_BAD_DTYPE, "%s must be f32, f16 or bf16", nm);
    if (!contiguous_from(c, 0)) return fail(G4B_ERR_BAD_STRIDE, "%s must be contiguous", nm);
    if (((uintptr_t)c.ptr & 15) != 0) return fail(G4B_ERR_BAD_STRIDE, "%s must be 16-byte aligned", nm);
  }
  if (a.k_pool.dtype != a.v_pool.dtype || a.k_pool.shape[0] != a.v_pool.shape[0])
    return fail(G4B_ERR_BAD_ARG, "k_pool and v_pool must have one dtype and shape");
  if (a.page_size <= 0 || (a.page_size & (a.page_size - 1)) != 0) return fail(G4B_ERR_BAD_ARG, "page_size must be a power of two");
  if (a.k_pool.shape[0] > 0x7fffffffLL || a.block_tables.shape[1] > 0x7fffffffLL)
    return fail(G4B_ERR_TOO_LARGE, "pages are counted in 31 bits");
  if (B > 1 << 24) return fail(G4B_ERR_TOO_LARGE, "at most %d slots", 1 << 24);      // (every warp looks at all of their starts)
  if ((a.norm_qk != 0 || a.norm_v != 0) && !(a.rmsnorm_eps > -INFINITY && a.rmsnorm_eps < INFINITY))
    return fail(G4B_ERR_BAD_ARG, "rmsnorm_eps must be finite");
  G4B_STOP_IF_VALIDATE_ONLY();
  if (N == 0 || B == 0) return G4B_OK;

  RopePackedParams p{};
  p.q = a.q.ptr; p.k = a.k.ptr; p.v = a.v.ptr;
  const G4bTensor& qo = a.q_out.ptr != nullptr ? a.q_out : a.q;
  p.q_out = qo.ptr; p.q_out_dtype = qo.dtype;
  p.freqs = (const float*)a.rope_freqs.ptr; p.freq_s = a.rope_freqs.stride[0];
  p.positions = a.positions.ptr; p.pos_s0 = a.positions.stride[0]; p.pos_s1 = a.positions.stride[1];
  p.pos_i64 = a.positions.dtype == G4B_I64;
  p.pair_axis = (const uint8_t*)a.pair_axis.ptr; p.axis_s = a.pair_axis.stride[0];
  p.q_starts = (const int32_t*)a.q_starts.ptr; p.starts_s = a.q_starts.stride[0];
  p.starts_quads = p.starts_s == 1 && ((uintptr_t)p.q_starts & 15) == 0;
  p.times = (const int32_t*)a.time_dim_sizes.ptr; p.time_s = a.time_dim_sizes.stride[0];
  p.q_w = (const float*)a.q_norm_w.ptr; p.qw_s = a.q_norm_w.stride[0];
  p.k_w = (const float*)a.k_norm_w.ptr; p.kw_s = a.k_norm_w.stride[0];
  p.k_pool = a.k_pool.ptr; p.v_pool = a.v_pool.ptr; p.cache_dtype = a.k_pool.dtype;
  p.block_tables = (const int32_t*)a.block_tables.ptr;
  p.bt_s0 = a.block_tables.stride[0]; p.bt_s1 = a.block_tables.stride[1];
  for (int i = 0; i < 2; ++i) { p.qs[i] = a.q.stride[i]; p.ks[i] = a.k.stride[i]; p.vs[i] = a.v.stride[i]; p.qos[i] = qo.stride[i]; }
  p.N = (int)N; p.B = (int)B; p.H = (int)H; p.G = (int)G; p.D = (int)D; p.axes = (int)axes;
  p.n_heads = (int)(H + 2 * G);
  while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
  p.num_pages = (int)a.k_pool.shape[0]; p.max_pages = (int)a.block_tables.shape[1];
  p.norm_qk = a.norm_qk; p.norm_v = a.norm_v; p.eps = a.rmsnorm_eps;
  p.status = device_status_ptr();
  if (p.status == nullptr) return G4B_ERR_CUDA;
  // Few rows (decode): the rows a warp holds at a time, for parallelism.  Many (prefill): a warp
  // takes all heads of a token and computes the token's sines and cosines once.  All heads / the former: 12 heads of 256, 512
  // tokens 7.3 / 6.1 us, 1024 tokens 7.7 / 9.4, 1365 tokens 8.6 / 11.9, 4096 tokens 17.8 / 32.5; 12 heads of 128, 512 tokens 5.9 / 4.4,
  // 1365 tokens 6.5 / 7.5.
  p.heads_per_warp = N * p.n_heads >= 16384 ? p.n_heads : (D == 128 ? 2 : 1);
  p.n_slots = (uint32_t)((p.n_heads + p.heads_per_warp - 1) / p.heads_per_warp);
  const int64_t blocks = N * (int64_t)p.n_slots;
  if (N > 0x7fffffffLL || blocks > 0x7fffffffLL) return fail(G4B_ERR_TOO_LARGE, "rope_norm_append_packed: too many rows");
  const int out16 = p.q_out_dtype == p.cache_dtype && p.cache_dtype != G4B_F32 ? p.cache_dtype : 0;
  G4B_DISPATCH_FLOAT(a.q.dtype, T, launch_in<T>(p, (unsigned)blocks, out16, st));
  G4B_CUDA_CHECK(cudaGetLastError());
  return G4B_OK;
}

}  // namespace g4b

extern "C" int g4b_rope_norm_append_packed(const G4bRopePackedArgs* args, void* cuda_stream) {
  if (args == nullptr) return g4b::fail(G4B_ERR_BAD_ARG, "args is null");
  return g4b::launch_rope_norm_append_packed(*args, (cudaStream_t)cuda_stream);
}

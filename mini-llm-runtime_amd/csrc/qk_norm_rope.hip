// RMSNorm of each query and key head, rotary positions, and the append of keys
// and values to the paged cache, in one launch.
//
// Input: one row per token of [q heads | k heads | v heads] x head_dim. For a
// head x of D elements, R of them rotated, i < R/2:
//   n_j  = x_j w_j / sqrt(mean(x^2) + eps)            (n = x without weights)
//   a_i  = position * inv_freq[i],  c = f cos a_i,  s = f sin a_i
//   lo' = lo c - hi s,  hi' = hi c + lo s
// on the pairs (lo, hi) = (n_i, n_{i+R/2}) (half layout) or (n_2i, n_2i+1)
// (interleaved); elements from R on are n_j. Everything is FP32 and rounded
// once, as it is stored. q goes to q_out, k and v to the token's cache slot.
//
// Angles: an FP32 product position * inv_freq is off by up to position * 2^-24
// radians (0.06 at a million), so the angle is taken in turns in 64 bits,
// reduced to (-1/2, 1/2] exactly, and only then rounded to FP32 (off by at
// most 2^-25 turns); the sine and cosine are of that multiple of pi.
//
// Layout: a head is 64 / HPW lanes wide, a lane holds VEC pairs as two vectors
// of VEC elements (half layout: VEC elements at i and VEC at i + R/2, or, from
// R on, the two halves of the rest; interleaved: 2 VEC neighbours), so the
// rotation needs no exchange between lanes and the norm's sum is a butterfly
// over the head's lanes. A head's lanes keep their place from head to head,
// so a lane reads its cosines, sines and weights once per token or once at all.
// A wave takes a token, or a token's heads are dealt over several waves (few
// tokens); the next head is loaded while one is worked on. The token's angles are computed one per lane and exchanged through
// the wave's own LDS rows.
//
// Bound by memory: each element is read and written once (bf16, 4,096 tokens of
// 28/4 heads of 128: 75.6 MB in 14.6 us, 5.2 TB/s, the rate of a large copy; the
// kernel that loaded two heads and then worked on both took 16.4 us).
#include "mlr_common.h"

#include <algorithm>

namespace mlr {
namespace {

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

struct NormRopeParams {
  const void *qkv, *qw, *kw, *slots;
  const int64_t *positions;
  const float *inv_freq;
  void *q_out, *kc, *vc;
  int64_t qkv_st, q_st, num_slots, num_tokens;
  float eps, factor;
  int hq, hkv, d, half;  // half: rotated pairs, R / 2
  int parts;             // waves a token's heads are dealt to
};

// Sum over the `width` (a power of two) neighbouring lanes of each head. Every
// step adds two lanes' equal partial sums, so all lanes hold the same bits.
__device__ __forceinline__ float sum_lanes(float x, int width) {
  auto dpp = [](float v, auto ctrl) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  if (width > 1) x += dpp(x, std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  if (width > 2) x += dpp(x, std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  if (width > 4) x += dpp(x, std::integral_constant<int, 0x141>{});  // row_half_mirror
  if (width > 8) x += dpp(x, std::integral_constant<int, 0x140>{});  // row_mirror
  if (width > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (width > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

template <typename T, typename I, int VEC, bool kInter, bool kNorm>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeParams p, int width) {
  using V = Pack<T, VEC>;
  extern __shared__ float cs_all[];  // per wave: [half] cos, [half] sin
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float *cs = cs_all + wv * 2 * p.half;
  const int d = p.d, half = p.half;
  const int hpw = 64 / width;              // heads per pass of a wave
  const int chunks = d / 2 / VEC;          // lanes of a head that hold elements
  const int ch = lane & (width - 1), hl = lane / width;
  const bool live = ch < chunks;
  const int pair = (live ? ch : 0) * VEC;  // the lane's first pair
  // Where its two vectors start in the head, and whether they are rotated.
  int e_lo, e_hi;
  const bool rot = pair < half;
  if constexpr (kInter) {
    e_lo = 2 * pair;
    e_hi = e_lo + VEC;
  } else if (rot) {
    e_lo = pair;
    e_hi = pair + half;
  } else {
    e_lo = pair + half;  // 2 half + (pair - half)
    e_hi = e_lo + (d / 2 - half);
  }
  const int heads = p.hq + 2 * p.hkv;
  const int64_t items = p.num_tokens * p.parts;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 6);
  V qw_lo, qw_hi, kw_lo, kw_hi;
  if constexpr (kNorm) {
    const T *qw = static_cast<const T *>(p.qw), *kw = static_cast<const T *>(p.kw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {  // the weights' own alignment is an element's
      qw_lo.v[j] = qw[e_lo + j];
      qw_hi.v[j] = qw[e_hi + j];
      kw_lo.v[j] = kw[e_lo + j];
      kw_hi.v[j] = kw[e_hi + j];
    }
  }
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 6) + wv; it < items;
       it += stride) {
    const int64_t t = it / p.parts;
    const int part = static_cast<int>(it - t * p.parts);
    const T *row = static_cast<const T *>(p.qkv) + t * p.qkv_st;
    V lo, hi;
    auto load = [&](int h0) {
      const T *src = row + static_cast<int64_t>(min(h0 + hl, heads - 1)) * d;
      lo = *reinterpret_cast<const V *>(src + e_lo);
      hi = *reinterpret_cast<const V *>(src + e_hi);
    };
    load(part * hpw);
    const int64_t slot = static_cast<int64_t>(static_cast<const I *>(p.slots)[t]);
    const bool write_kv = slot >= 0 && slot < p.num_slots;
    const double pos = static_cast<double>(p.positions[t]);
    for (int i = lane; i < half; i += 64) {
      const double turns = pos * (static_cast<double>(p.inv_freq[i]) * 0.15915494309189535);
      const float x = static_cast<float>(turns - rint(turns));
      float sv, cv;
      sincospif(2.f * x, &sv, &cv);
      cs[i] = cv * p.factor;
      cs[half + i] = sv * p.factor;
    }
    __builtin_amdgcn_wave_barrier();
    float c[VEC], s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      c[j] = rot ? cs[pair + j] : 1.f;
      s[j] = rot ? cs[half + pair + j] : 0.f;
    }
    const int step = p.parts * hpw;
    for (int h0 = part * hpw; h0 < heads; h0 += step) {
      const int h = h0 + hl;
      const V now_lo = lo, now_hi = hi;
      if (h0 + step < heads) load(h0 + step);  // in flight while this head is worked on
      const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
      float a[VEC], b[VEC];  // lo and hi
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if constexpr (kInter) {
          a[j] = Elem<T>::to_f32(2 * j < VEC ? now_lo.v[2 * j % VEC] : now_hi.v[2 * j % VEC]);
          b[j] = Elem<T>::to_f32(2 * j + 1 < VEC ? now_lo.v[(2 * j + 1) % VEC]
                                                 : now_hi.v[(2 * j + 1) % VEC]);
        } else {
          a[j] = Elem<T>::to_f32(now_lo.v[j]);
          b[j] = Elem<T>::to_f32(now_hi.v[j]);
        }
      }
      if constexpr (kNorm) {
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sq += a[j] * a[j] + b[j] * b[j];
        sq = sum_lanes(live ? sq : 0.f, width);
        const float r = rsqrtf(sq / static_cast<float>(d) + p.eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int lo_at = kInter ? 2 * j : j, hi_at = kInter ? 2 * j + 1 : j;
          const V &wl = is_q ? qw_lo : kw_lo, &wh = is_q ? qw_hi : kw_hi;
          const T w_a = kInter ? (lo_at < VEC ? wl.v[lo_at % VEC] : wh.v[lo_at % VEC])
                               : wl.v[j];
          const T w_b = kInter ? (hi_at < VEC ? wl.v[hi_at % VEC] : wh.v[hi_at % VEC])
                               : wh.v[j];
          a[j] = a[j] * r * Elem<T>::to_f32(w_a);
          b[j] = b[j] * r * Elem<T>::to_f32(w_b);
        }
      }
      V olo = now_lo, ohi = now_hi;
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          // Beyond the rotated part the values pass as they are, so that one
          // that is not finite stays alone.
          const T x = Elem<T>::from_f32(rot ? a[j] * c[j] - b[j] * s[j] : a[j]);
          const T y = Elem<T>::from_f32(rot ? b[j] * c[j] + a[j] * s[j] : b[j]);
          if constexpr (kInter) {
            (2 * j < VEC ? olo : ohi).v[2 * j % VEC] = x;
            (2 * j + 1 < VEC ? olo : ohi).v[(2 * j + 1) % VEC] = y;
          } else {
            olo.v[j] = x;
            ohi.v[j] = y;
          }
        }
      }
      if (live && h < heads && (is_q || write_kv)) {
        T *o = is_q ? static_cast<T *>(p.q_out) + t * p.q_st + static_cast<int64_t>(h) * d
               : is_v
                   ? static_cast<T *>(p.vc) + (slot * p.hkv + (h - p.hq - p.hkv)) * d
                   : static_cast<T *>(p.kc) + (slot * p.hkv + (h - p.hq)) * d;
        *reinterpret_cast<V *>(o + e_lo) = olo;
        *reinterpret_cast<V *>(o + e_hi) = ohi;
      }
    }
    __builtin_amdgcn_wave_barrier();  // cs is rewritten for the next token
  }
}

template <typename T, typename I, int VEC, bool kInter, bool kNorm>
int launch(NormRopeParams p, hipStream_t stream) {
  int width = 1;
  while (width * VEC < p.d / 2) width *= 2;
  MLR_REQUIRE(width <= 64,
              "mlr_qk_norm_rope_write: head_dim %d needs rows aligned to more than %d elements",
              p.d, VEC);
  const int heads = p.hq + 2 * p.hkv;
  const int passes = (heads + 64 / width - 1) / (64 / width);
  // Heads of a token are dealt over so many waves that the call has about sixteen
  // for every CU, a pass of the heads at least each. 32/8 heads of 128, us, a wave per
  // token and this rule: bf16, 1 token 7.0 and 3.9, 512 tokens 8.8 and 5.8, 2,048
  // tokens 13.2 and 12.5; FP32 7.9 and 3.7, 10.9 and 7.0, 19.2 and 18.2. At 4,096
  // tokens two waves each would take 22.1 in place of 19.9 (bf16).
  const int cus = current_device_cus() > 0 ? current_device_cus() : 256;
  p.parts = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({16 * static_cast<int64_t>(cus) / p.num_tokens, passes, 16})));
  const int waves = 4;
  const int64_t wgs = ceil_div(p.num_tokens * p.parts, waves);
  const unsigned blocks = static_cast<unsigned>(wgs < 65536 ? wgs : 65536);
  const size_t lds = static_cast<size_t>(waves) * 2 * p.half * sizeof(float);
  qk_norm_rope_kernel<T, I, VEC, kInter, kNorm><<<blocks, 64 * waves, lds, stream>>>(p, width);
  return check_launch("mlr_qk_norm_rope_write");
}

template <typename T, typename I, int VEC>
int launch_layout(const NormRopeParams &p, bool inter, hipStream_t stream) {
  if (p.qw != nullptr)
    return inter ? launch<T, I, VEC, true, true>(p, stream)
                 : launch<T, I, VEC, false, true>(p, stream);
  return inter ? launch<T, I, VEC, true, false>(p, stream)
               : launch<T, I, VEC, false, false>(p, stream);
}

template <typename T, typename I>
int launch_type(const NormRopeParams &p, bool inter, hipStream_t stream) {
  // Vectors of 16 bytes, of 4 elements, or single elements: the two vectors of
  // every lane must lie inside the rotated part or outside it, and all rows
  // start at multiples of the vector.
  auto fits = [&](int vec) {
    const uintptr_t mask = vec * sizeof(T) - 1;
    return p.d / 2 % vec == 0 && p.half % vec == 0 && p.qkv_st % vec == 0 && p.q_st % vec == 0 &&
           ((reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.q_out) |
             reinterpret_cast<uintptr_t>(p.kc) | reinterpret_cast<uintptr_t>(p.vc)) & mask) == 0;
  };
  constexpr int kWide = 16 / sizeof(T);
  if (fits(kWide)) return launch_layout<T, I, kWide>(p, inter, stream);
  if (kWide != 4 && fits(4)) return launch_layout<T, I, 4>(p, inter, stream);
  return launch_layout<T, I, 1>(p, inter, stream);
}

}  // namespace
}  // namespace mlr

extern "C" int mlr_qk_norm_rope_write(
    const void *qkv, int64_t qkv_stride_t, const void *q_weight, const void *k_weight, double eps,
    const int64_t *positions, const float *inv_freq, int64_t rotary_dim, int interleaved,
    double attention_factor, const void *slot_mapping, int index_dtype, void *q_out,
    int64_t q_out_stride_t, void *k_cache, void *v_cache, int64_t num_slots, int64_t num_tokens,
    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int dtype, void *stream) {
  using namespace mlr;
  clear_error();
  MLR_REQUIRE(num_tokens >= 0, "mlr_qk_norm_rope_write: num_tokens must be >= 0");
  MLR_REQUIRE(num_q_heads > 0 && num_kv_heads > 0,
              "mlr_qk_norm_rope_write: head counts must be positive");
  MLR_REQUIRE(head_dim > 0 && head_dim % 2 == 0 && head_dim <= 1024,
              "mlr_qk_norm_rope_write: head_dim must be even and in (0, 1024]");
  MLR_REQUIRE(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
              "mlr_qk_norm_rope_write: rotary_dim must be even and in (0, head_dim]");
  MLR_REQUIRE(num_q_heads < (int64_t(1) << 24) && num_kv_heads < (int64_t(1) << 24) &&
                  (num_q_heads + 2 * num_kv_heads) * head_dim < (int64_t(1) << 30),
              "mlr_qk_norm_rope_write: row too wide");
  MLR_REQUIRE(qkv_stride_t >= (num_q_heads + 2 * num_kv_heads) * head_dim,
              "mlr_qk_norm_rope_write: qkv row stride smaller than its row");
  MLR_REQUIRE(q_out_stride_t >= num_q_heads * head_dim,
              "mlr_qk_norm_rope_write: q_out row stride smaller than its row");
  MLR_REQUIRE(num_slots >= 0, "mlr_qk_norm_rope_write: num_slots must be >= 0");
  MLR_REQUIRE(index_dtype == MLR_INDEX_I32 || index_dtype == MLR_INDEX_I64,
              "mlr_qk_norm_rope_write: unknown index dtype %d", index_dtype);
  MLR_REQUIRE((q_weight == nullptr) == (k_weight == nullptr),
              "mlr_qk_norm_rope_write: q_weight and k_weight come together");
  if (num_tokens == 0) return MLR_OK;
  MLR_REQUIRE(qkv && positions && inv_freq && slot_mapping && q_out && k_cache && v_cache,
              "mlr_qk_norm_rope_write: null pointer");
  NormRopeParams p;
  p.qkv = qkv;
  p.qw = q_weight;
  p.kw = k_weight;
  p.slots = slot_mapping;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.q_out = q_out;
  p.kc = k_cache;
  p.vc = v_cache;
  p.qkv_st = qkv_stride_t;
  p.q_st = q_out_stride_t;
  p.num_slots = num_slots;
  p.num_tokens = num_tokens;
  p.eps = static_cast<float>(eps);
  p.factor = static_cast<float>(attention_factor);
  p.hq = static_cast<int>(num_q_heads);
  p.hkv = static_cast<int>(num_kv_heads);
  p.d = static_cast<int>(head_dim);
  p.half = static_cast<int>(rotary_dim / 2);
  p.parts = 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool inter = interleaved != 0, i32 = index_dtype == MLR_INDEX_I32;
  switch (dtype) {
    case MLR_DTYPE_F32:
      return i32 ? launch_type<float, int32_t>(p, inter, s)
                 : launch_type<float, int64_t>(p, inter, s);
    case MLR_DTYPE_F16:
      return i32 ? launch_type<f16_t, int32_t>(p, inter, s)
                 : launch_type<f16_t, int64_t>(p, inter, s);
    case MLR_DTYPE_BF16:
      return i32 ? launch_type<bf16_t, int32_t>(p, inter, s)
                 : launch_type<bf16_t, int64_t>(p, inter, s);
    default:
      return set_error(MLR_ERR_UNSUPPORTED, "mlr_qk_norm_rope_write: unsupported dtype %d", dtype);
  }
}

// Rotary positions of packed tokens, keys and values going into a paged cache.
//
//   f = position * turns[i] in fp64, reduced to [-1/2, 1/2];  c, s = magnitude * cos, sin(2 pi f) in fp32
//   (a, b) -> (a c - b s, b c + a s) for the feature pairs (2i, 2i+1), or (i, i + rot/2) with ODIT_FLAG_NEOX, i < rot/2;
//   features from rot on pass through. One rounding, at the store.
//
// The angle is reduced in 64 bits because positions are whole numbers up to a million and beyond: in fp32 the product of such a
// position and a turn has lost the fraction that is all that counts. Behind the reduction 24 bits are enough.
//
// Bound by memory: every element of q, k and v is read once and written once. A workgroup has one token: its threads first make the token's
// (cos, sin) pairs in LDS, once for all heads, then move 16 bytes each. us, one / two / four tokens of a workgroup: 65536 tokens, 32 heads on 8
// of 128 into a cache 291 (5.5 TB/s) / 296 / 306, 8191 tokens, 24 heads on 24, a quarter of 128 rotated, 36.6 / 36.3 / 40.7, 4096 tokens as the
// first 19.8 / 22.2 / 21.7. Several pieces of a thread in flight at a time gave nothing, loads and stores past the caches 287 of the 306 but
// 12.0 where 2000 tokens take 9.6.
#include "odit_common.h"
#include "quotient.h"

namespace odit {

struct RopeAppendParams {
  const void *q, *k, *v;
  void *q_out, *k_out, *k_cache, *v_cache;
  const int64_t *positions, *slots;
  const double* turns;
  int64_t T, n_slots;
  int H, Hkv, D, rot, page;
  int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h;
  int64_t kc_p, kc_r, kc_h, vc_p, vc_r, vc_h;  // cache strides: page, row in the page, head
  float magnitude;
  Quotient by_units, by_pieces;  // by a rotated head's pieces (or features), by D / 8
};

// features [8 c, 8 c + 8) of a head, or pairs (i, i + rot/2) for i in [8 c, 8 c + 8)
template <typename T, bool NEOX>
__device__ __forceinline__ void rope_unit(const T* src, T* dst, const float2* cs, int u, int rot) {
  using R = Raw<T>;
  if constexpr (NEOX) {
    const int pairs = rot / 16;
    if (u < pairs) {
      const u32x4 a = load_raw(src + u * 8), b = load_raw(src + rot / 2 + u * 8);
      u32x4 x, y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t0 = cs[u * 8 + 2 * j], t1 = cs[u * 8 + 2 * j + 1];
        const float a0 = R::get(a, 2 * j), a1 = R::get(a, 2 * j + 1), b0 = R::get(b, 2 * j), b1 = R::get(b, 2 * j + 1);
        R::set2(x, j, fmaf(a0, t0.x, -b0 * t0.y), fmaf(a1, t1.x, -b1 * t1.y));
        R::set2(y, j, fmaf(b0, t0.x, a0 * t0.y), fmaf(b1, t1.x, a1 * t1.y));
      }
      store_raw(dst + u * 8, x);
      store_raw(dst + rot / 2 + u * 8, y);
    } else {
      store_raw(dst + (u + pairs) * 8, load_raw(src + (u + pairs) * 8));
    }
  } else {
    u32x4 a = load_raw(src + u * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = u * 4 + j;
      if (2 * i < rot) {
        const float2 t = cs[i];
        const float x = R::get(a, 2 * j), y = R::get(a, 2 * j + 1);
        R::set2(a, j, fmaf(x, t.x, -y * t.y), fmaf(y, t.x, x * t.y));
      }
    }
    store_raw(dst + u * 8, a);
  }
}

// the same for halves that are no whole number of 16-byte pieces: feature u of the head
template <typename T>
__device__ __forceinline__ void rope_feature(const T* src, T* dst, const float2* cs, int u, int rot) {
  const int half = rot / 2;
  float x = to_float(src[u]);
  if (u < half) x = fmaf(x, cs[u].x, -to_float(src[u + half]) * cs[u].y);
  else if (u < rot) x = fmaf(x, cs[u - half].x, to_float(src[u - half]) * cs[u - half].y);
  dst[u] = from_float<T>(x);
}

// FORM 0: interleaved, 1: halves in 16-byte pieces, 2: halves feature by feature
template <typename T, int FORM>
__global__ __launch_bounds__(256) void rope_append_kernel(const RopeAppendParams p) {
  extern __shared__ float2 cs[];  // [rot / 2]
  const int64_t token = blockIdx.x;
  for (int i = threadIdx.x; i < p.rot / 2; i += 256) {
    double f = static_cast<double>(p.positions[token]) * p.turns[i];
    f -= rint(f);
    float s, c;
    sincospif(2.f * static_cast<float>(f), &s, &c);
    cs[i] = make_float2(c * p.magnitude, s * p.magnitude);
  }
  int64_t page = 0, row = 0;
  bool stored = true;
  if (p.slots != nullptr) {
    const int64_t slot = p.slots[token];
    stored = slot >= 0 && slot < p.n_slots;  // (a padded token has none)
    page = stored ? slot / p.page : 0;
    row = stored ? slot - page * p.page : 0;
  }
  __syncthreads();
  const int units = FORM == 0 ? p.D / 8 : FORM == 1 ? p.D / 8 - p.rot / 16 : p.D;  // of a head that is rotated
  const int turned = (p.H + p.Hkv) * units, copies = p.v != nullptr ? p.Hkv * (p.D / 8) : 0;  // (16-byte pieces of the token's values)
  for (int i = threadIdx.x; i < turned + copies; i += 256) {
    if (i < turned) {
      const int h = p.by_units(i), u = i - h * units;
      const T* src;
      T* dst;
      if (h < p.H) {
        src = static_cast<const T*>(p.q) + token * p.qs_t + h * p.qs_h;
        dst = static_cast<T*>(p.q_out) + (token * p.H + h) * p.D;
      } else {
        if (!stored) continue;
        src = static_cast<const T*>(p.k) + token * p.ks_t + (h - p.H) * p.ks_h;
        dst = p.slots != nullptr ? static_cast<T*>(p.k_cache) + page * p.kc_p + row * p.kc_r + (h - p.H) * p.kc_h
                                 : static_cast<T*>(p.k_out) + (token * p.Hkv + (h - p.H)) * p.D;
      }
      if constexpr (FORM == 2) rope_feature<T>(src, dst, cs, u, p.rot);
      else rope_unit<T, FORM == 1>(src, dst, cs, u, p.rot);
    } else if (stored) {
      const int c = i - turned, h = p.by_pieces(c), u = c - h * (p.D / 8);
      store_raw(static_cast<T*>(p.v_cache) + page * p.vc_p + row * p.vc_r + h * p.vc_h + u * 8,
                load_raw(static_cast<const T*>(p.v) + token * p.vs_t + h * p.vs_h + u * 8));
    }
  }
}

}  // namespace odit

extern "C" int odit_rope_append(const void* q, const void* k, const void* v, const int64_t* positions, const double* turns, void* q_out,
                                void* k_out, const int64_t* slots, void* key_cache, void* value_cache, int64_t T, int H, int Hkv, int D,
                                int rot, int64_t pages, int page_size, const int64_t q_strides[2], const int64_t k_strides[2],
                                const int64_t v_strides[2], const int64_t key_cache_strides[3], const int64_t value_cache_strides[3],
                                float magnitude, int dtype, unsigned flags, void* stream) {
  using namespace odit;
  if (dtype != ODIT_BF16 && dtype != ODIT_F16) {
    set_error("odit_rope_append: dtype code %d unsupported (bf16 and fp16 only)", dtype);
    return ODIT_ENOTSUP;
  }
  ODIT_CHECK_ARG(T >= 0 && H > 0 && Hkv > 0 && H <= 65536 && Hkv <= 65536, "odit_rope_append: bad shape");
  ODIT_CHECK_ARG(D > 0 && D % 8 == 0 && D <= 1024, "odit_rope_append: head size %d must be a multiple of 8 up to 1024", D);
  ODIT_CHECK_ARG(rot > 0 && rot % 2 == 0 && rot <= D, "odit_rope_append: rotary width %d must be even and in (0, D=%d]", rot, D);
  const bool cached = slots != nullptr;
  ODIT_CHECK_ARG(q_strides && k_strides, "odit_rope_append: null strides");
  ODIT_CHECK_ARG(cached ? v_strides && key_cache_strides && value_cache_strides && k_out == nullptr && pages >= 0 && page_size > 0
                        : v == nullptr && key_cache == nullptr && value_cache == nullptr,
                 "odit_rope_append: slots come with v, both caches and no k_out; without slots there are none of them");
  for (int i = 0; i < 2; ++i)
    ODIT_CHECK_ARG(q_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && (!cached || v_strides[i] % 8 == 0),
                   "odit_rope_append: strides must be multiples of 8 elements");
  for (int i = 0; cached && i < 3; ++i)
    ODIT_CHECK_ARG(key_cache_strides[i] % 8 == 0 && value_cache_strides[i] % 8 == 0,
                   "odit_rope_append: cache strides must be multiples of 8 elements");
  const int64_t cache_sizes[3] = {pages, page_size, Hkv};
  for (int i = 0; cached && i < 3; ++i)
    ODIT_CHECK_ARG(cache_sizes[i] <= 1 || (key_cache_strides[i] != 0 && value_cache_strides[i] != 0),
                   "odit_rope_append: cache rows must not share memory (a stride of 0)");
  if (T == 0) return ODIT_OK;
  ODIT_CHECK_ARG(q && k && positions && turns && q_out && (cached ? v != nullptr : k_out != nullptr), "odit_rope_append: null tensors");
  ODIT_CHECK_ARG(!cached || pages == 0 || (key_cache && value_cache), "odit_rope_append: null caches");
  ODIT_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_out) && aligned16(key_cache) &&
                     aligned16(value_cache),
                 "odit_rope_append: tensors must be 16-byte aligned");

  RopeAppendParams p;
  p.q = q; p.k = k; p.v = v;
  p.q_out = q_out; p.k_out = k_out; p.k_cache = key_cache; p.v_cache = value_cache;
  p.positions = positions; p.slots = slots; p.turns = turns;
  p.T = T; p.n_slots = cached ? pages * page_size : 0;
  p.H = H; p.Hkv = Hkv; p.D = D; p.rot = rot; p.page = cached ? page_size : 1;
  p.qs_t = q_strides[0]; p.qs_h = q_strides[1]; p.ks_t = k_strides[0]; p.ks_h = k_strides[1];
  p.vs_t = cached ? v_strides[0] : 0; p.vs_h = cached ? v_strides[1] : 0;
  p.kc_p = cached ? key_cache_strides[0] : 0; p.kc_r = cached ? key_cache_strides[1] : 0; p.kc_h = cached ? key_cache_strides[2] : 0;
  p.vc_p = cached ? value_cache_strides[0] : 0; p.vc_r = cached ? value_cache_strides[1] : 0; p.vc_h = cached ? value_cache_strides[2] : 0;
  p.magnitude = magnitude;
  ODIT_CHECK_ARG(T < (1ll << 24), "odit_rope_append: %lld tokens are too many", static_cast<long long>(T));
  const size_t lds = static_cast<size_t>(rot / 2) * sizeof(float2);
  const int form = !(flags & ODIT_FLAG_NEOX) ? 0 : rot % 16 == 0 ? 1 : 2;
  p.by_units = quotient(form == 0 ? D / 8 : form == 1 ? D / 8 - rot / 16 : D);
  p.by_pieces = quotient(D / 8);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define ODIT_ROPE_GO(E)                                                                                                  \
  if (form == 0) hipLaunchKernelGGL((rope_append_kernel<E, 0>), dim3(T), dim3(256), lds, st, p);                      \
  else if (form == 1) hipLaunchKernelGGL((rope_append_kernel<E, 1>), dim3(T), dim3(256), lds, st, p);                 \
  else hipLaunchKernelGGL((rope_append_kernel<E, 2>), dim3(T), dim3(256), lds, st, p);
  if (dtype == ODIT_BF16) { ODIT_ROPE_GO(bf16_t) }
  else { ODIT_ROPE_GO(f16_t) }
#undef ODIT_ROPE_GO
  return check_launch("odit_rope_append");
}

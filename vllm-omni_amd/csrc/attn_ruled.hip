// Attention of whole prompts under rules for what a query sees (documents, a causal order, a window, a prefix) and what its scores become
// (a tanh cap, slopes or a table by distance).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2(x_ij - m_i),  x_ij in attn_rules.h
//
// The formulation is that of attn_fwd.hip: S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_32x32x16, a lane owns one query (and the lane 32
// further the other keys of it), P never leaves its registers, one pass with a running maximum and sum. What a query sees is two ranges
// of keys: the band [blo, bhi) that its document, the order and the window leave, and its document's prefix [plo, phi). They are worked out
// once, per lane; a tile's mask is then the two ranges' bits, formed only for tiles that some query sees in part. The tiles that a workgroup
// visits are the union of its queries' ranges (two runs where a gap lies between).
//
// A value that is NaN or infinite spoils its tile's product also for queries that do not see its key (0 times it is NaN). Rows that come out
// NaN with a finite sum are therefore done again at the end, over their own keys alone.
#include "attn_rules.h"

namespace odit {

typedef short s16x4_r __attribute__((ext_vector_type(4)));
typedef short s16x8_r __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4_r* lds_s16x4_rp;
typedef __attribute__((address_space(3))) void* lds_void_rp;

struct RuledParams {
  const void *q, *k, *v;
  void* o;
  const int *q_starts, *k_starts, *prefix;
  const float *slopes, *distance;
  int docs, causal, window, radius;  // docs 0: one document per batch row; window 0: none
  int B, Sq, Sk, H, Hkv;
  int64_t qs_b, qs_s, qs_h, ks_b, ks_s, ks_h, vs_b, vs_s, vs_h, os_b, os_s, os_h;
  float scale_log2;
  Cap cap;
  int n_qblocks, units;  // units: heads of all batch rows
};

// the document of row r: the last one that starts at or before it (the search ends whatever the starts hold)
__device__ __forceinline__ int doc_of(const int* starts, int docs, int r) {
  int lo = 0, hi = docs;  // starts[lo] <= r < starts[hi], if anywhere
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= r) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// bits of the keys of [t0, t0 + 64) in [lo, hi)
__device__ __forceinline__ uint64_t range_bits(int lo, int hi, int t0) {
  const int a = clampi(lo - t0, 0, 64), b = clampi(hi - t0, 0, 64);
  if (b <= a) return 0;
  const uint64_t upto = b == 64 ? ~0ull : (1ull << b) - 1;
  return upto & (~0ull << a);
}

// BIAS 0: none, 1: slopes, 2: table
template <typename T, int D, bool CAP, int BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void attn_ruled_kernel(const RuledParams p) {
  using M = Mma<T>;
  using frag = typename M::frag;
  constexpr int NW = 4, BM = NW * 32, BN = 64;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPI = 64 / CPR, TILEB = BN * ROWB;
  constexpr int IPW = BN / RPI / NW;  // wave instructions of a tile's load, per wavefront

  __shared__ __attribute__((aligned(1024))) char lds[4 * TILEB];  // K0 K1 V0 V1
  __shared__ int bounds[NW][4];
  __shared__ float table[BIAS == 2 ? 2 * kMaxRadius + 1 : 1];  // the head's biases in units of log2

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  // the last query blocks, which see most under a causal order, begin first; where the heads divide over the XCDs, an XCD keeps its heads
  int unit, qb;
  if (p.units % kNumXcd == 0) {
    const int per = p.units / kNumXcd, local = blockIdx.x / kNumXcd;
    unit = blockIdx.x % kNumXcd * per + local % per;
    qb = p.n_qblocks - 1 - local / per;
  } else {
    unit = blockIdx.x % p.units;
    qb = p.n_qblocks - 1 - blockIdx.x / p.units;
  }
  const int h = unit % p.H, b = unit / p.H, hkv = h / (p.H / p.Hkv);
  const int q0 = qb * BM + wave * 32;
  const int row = q0 + l32 < p.Sq ? q0 + l32 : p.Sq - 1;

  // ---- what this lane's query sees ----
  int blo, bhi, plo = 0, phi = 0, pos;  // pos: the key at the query's own place
  {
    int ks = 0, kn = p.Sk, qs = 0, qe = p.Sq, doc = b;
    bool in = true;
    if (p.docs > 0) {
      doc = doc_of(p.q_starts, p.docs, row);
      qs = p.q_starts[doc];
      qe = p.q_starts[doc + 1];
      in = row >= qs && row < qe;
      ks = clampi(p.k_starts[doc], 0, p.Sk);
      kn = clampi(p.k_starts[doc + 1], ks, p.Sk) - ks;
    }
    // the query's place from the document's first key (cut to what sums with a window keep in 32 bits, whatever the starts hold)
    constexpr int64_t kFar = (1 << 30) - 1;
    const int64_t place = static_cast<int64_t>(row) + kn - qe;
    const int at = static_cast<int>(place < -kFar ? -kFar : place > kFar ? kFar : place);
    const int lo = p.window > 0 ? clampi(at - p.window + 1, 0, kn) : 0;
    const int hi = p.causal ? clampi(at + 1, 0, kn) : p.window > 0 ? clampi(at + p.window, 0, kn) : kn;
    pos = ks + at;
    blo = ks + lo;
    bhi = in && hi > lo ? ks + hi : blo;
    if (p.prefix != nullptr && in) {
      plo = ks;
      phi = ks + clampi(p.prefix[doc], 0, kn);
    }
  }
  // the wavefront's ranges: from the smallest begin to the largest end, and what all of its queries see
  auto wave_min = [](int x) { for (int s = 1; s < 64; s <<= 1) { const int y = __shfl_xor(x, s, 64); x = y < x ? y : x; } return __builtin_amdgcn_readfirstlane(x); };
  auto wave_max = [](int x) { for (int s = 1; s < 64; s <<= 1) { const int y = __shfl_xor(x, s, 64); x = y > x ? y : x; } return __builtin_amdgcn_readfirstlane(x); };
  constexpr int kNone = 0x7fffffff;
  const int b_first = wave_min(bhi > blo ? blo : kNone), b_end = wave_max(bhi > blo ? bhi : 0);
  const int p_first = wave_min(phi > plo ? plo : kNone), p_end = wave_max(phi > plo ? phi : 0);
  const int b_all0 = wave_max(blo), b_all1 = wave_min(bhi), p_all0 = wave_max(plo), p_all1 = wave_min(phi);
  const int pos_min = wave_min(pos), pos_max = wave_max(pos);
  if (lane == 0) { bounds[wave][0] = b_first; bounds[wave][1] = b_end; bounds[wave][2] = p_first; bounds[wave][3] = p_end; }
  if constexpr (BIAS == 2) {
    const float* from = p.distance + static_cast<int64_t>(h) * (2 * p.radius + 1);
    for (int i = tid; i <= 2 * p.radius; i += 256) table[i] = from[i] * kLog2e;
  }
  __syncthreads();
  // the workgroup's tiles: up to two runs
  int s1, n1, s2, n2;
  {
    int lo[2] = {kNone, kNone}, hi[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[i] = min(lo[i], bounds[w][2 * i]);
        hi[i] = max(hi[i], bounds[w][2 * i + 1]);
      }
    int a0 = lo[0] / BN, a1 = hi[0] > lo[0] ? (hi[0] + BN - 1) / BN : a0, c0 = lo[1] / BN, c1 = hi[1] > lo[1] ? (hi[1] + BN - 1) / BN : c0;
    if (a1 == a0) { a0 = c0; a1 = c1; c1 = c0; }                                                    // one run or none
    if (c1 > c0 && c0 <= a1 && a0 <= c1) { a0 = min(a0, c0); a1 = max(a1, c1); c0 = c1 = 0; }        // they touch
    s1 = __builtin_amdgcn_readfirstlane(a0); n1 = __builtin_amdgcn_readfirstlane(a1 - a0);
    s2 = __builtin_amdgcn_readfirstlane(c0); n2 = __builtin_amdgcn_readfirstlane(c1 - c0);
  }
  const int n_tiles = n1 + n2;
  auto tile_at = [&](int i) { return i < n1 ? s1 + i : s2 + i - n1; };

  // ---- tile loads: as in attn_fwd_dma.hip, but with a buffer descriptor for each tile, so that offsets stay small in any tensor ----
  const T* const kbase = static_cast<const T*>(p.k) + b * p.ks_b + hkv * p.ks_h;
  const T* const vbase = static_cast<const T*>(p.v) + b * p.vs_b + hkv * p.vs_h;
  const int r0 = wave * IPW * RPI + lane / CPR, pc0 = lane % CPR;
  uint32_t kvoff[IPW], vvoff[IPW];
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int r = r0 + RPI * i;
    kvoff[i] = static_cast<uint32_t>(r * p.ks_s * 2) + static_cast<uint32_t>(((pc0 ^ (r % 16)) % CPR) * 16);
    vvoff[i] = static_cast<uint32_t>(r * p.vs_s * 2) + static_cast<uint32_t>(((pc0 ^ (4 * (r % 4))) % CPR) * 16);
  }
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_rp)lds));
  auto load_tile = [&](const T* base, int64_t stride, const uint32_t(&off)[IPW], int t, int dst) {
    const uint64_t a = reinterpret_cast<uint64_t>(base + static_cast<int64_t>(t) * BN * stride);
    const int rows = min(BN, p.Sk - t * BN);  // rows behind the last key read as zeros
    u32x4_v r;
    r.x = static_cast<uint32_t>(a); r.y = static_cast<uint32_t>(a >> 32) & 0xffffu;
    r.z = static_cast<uint32_t>(((rows - 1) * stride + D) * 2); r.w = 0x00020000u;
#pragma unroll
    for (int i = 0; i < IPW; ++i) load_lds16(lds_base + dst + (wave * IPW + i) * 1024, off[i], r, 0);
  };
  auto load_k = [&](int i) { load_tile(kbase, p.ks_s, kvoff, tile_at(i), (i & 1) * TILEB); };
  auto load_v = [&](int i) { load_tile(vbase, p.vs_s, vvoff, tile_at(i), (2 + (i & 1)) * TILEB); };

  const T* const qrow = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h + row * p.qs_s;
  frag qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = __builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(qrow + hh * 8 + ks * 16));

  f32x16_v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
  constexpr bool MADE = CAP || BIAS != 0;  // scores are turned into units of log2 before their maximum is taken
  const float c = MADE ? 1.f : p.scale_log2;
  float m_run = -INFINITY, l_run = 0.f, mc = 0.f;
  const float slope = BIAS == 1 ? p.slopes[h] * kLog2e : 0.f;

  const int k_lane = l32 * ROWB + (((hh ^ (l32 % 16)) % CPR) << 4);
  const int sq = (lane & 15) >> 2, dh = (lane >> 4) & 1;
  const int v_lane = (4 * hh + sq) * ROWB + ((((4 * sq) % CPR) ^ (2 * dh + ((lane & 3) >> 1))) << 4) + ((lane & 1) << 3);
  auto swapped = [&](float x) __attribute__((always_inline)) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(hh ? r[0] : r[1]);
  };

  // bias of key `key` for this lane's query, and the whole way from a product to units of log2
  auto made = [&](float s, int key) __attribute__((always_inline)) {
    float x = CAP ? p.cap(s) : s * p.scale_log2;
    if constexpr (BIAS == 1) x = fmaf(-slope, fabsf(static_cast<float>(key - pos)), x);
    if constexpr (BIAS == 2) x += table[clampi(key - pos, -p.radius, p.radius) + p.radius];
    return x;
  };

  if (n_tiles > 0) {
    load_k(0);
    load_v(0);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  for (int i = 0; i < n_tiles; ++i) {
    const int buf = i & 1, t0 = tile_at(i) * BN;
    if (i + 1 < n_tiles) {
      load_k(i + 1);
      load_v(i + 1);
    }
    if ((t0 < b_end && t0 + BN > b_first) || (t0 < p_end && t0 + BN > p_first)) {  // (wave-uniform) some query sees some key
      f32x16_v s[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kt][e] = 0.f;
      const char* kb = lds + buf * TILEB;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
          s[kt] = M::run(__builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(kb + kt * 32 * ROWB + (k_lane ^ (ks * 32)))), qf[ks], s[kt]);
      if constexpr (MADE) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kt][e] = made(s[kt][e], t0 + kt * 32 + (e >> 2) * 8 + hh * 4 + (e & 3));
      }
      if (!((t0 >= b_all0 && t0 + BN <= b_all1) || (t0 >= p_all0 && t0 + BN <= p_all1))) {
        const uint64_t w = range_bits(blo, bhi, t0) | range_bits(plo, phi, t0);
        const uint32_t half[2] = {static_cast<uint32_t>(w) >> (4 * hh), static_cast<uint32_t>(w >> 32) >> (4 * hh)};
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kt][e] = (half[kt] & (1u << ((e >> 2) * 8 + (e & 3)))) ? s[kt][e] : -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = __builtin_elementwise_maximum(mx, s[kt][e]);
      if (__any((mx - m_run) * c > 8.f)) {
        const float m_new = fmaxf(m_run, fmaxf(mx, swapped(mx)));
        const float m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f((m_run - m_safe) * c);
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        m_run = m_new;
        mc = m_safe * c;
      }
      uint32_t pf[2][2][4];
      float sum = 0.f;
#pragma unroll
      for (int pi = 0; pi < 16; ++pi) {
        const int kt = pi >> 3, e = (pi & 7) * 2;
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt][e], c, -mc)), p1 = __builtin_amdgcn_exp2f(fmaf(s[kt][e + 1], c, -mc));
        sum += p0 + p1;
        pf[kt][(pi & 7) >> 2][pi & 3] = M::pack2(p0, p1);
      }
      l_run += sum;
      const char* vb = lds + (2 + buf) * TILEB;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const char* vp = vb + (kt * 32 + g * 16) * ROWB + (v_lane ^ ((dt * 64) % ROWB));
            const s16x4_r lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_rp)(vp));
            const s16x4_r hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_rp)(vp + 8 * ROWB));
            u32x4_v pb;
            pb.x = pf[kt][g][0]; pb.y = pf[kt][g][1]; pb.z = pf[kt][g][2]; pb.w = pf[kt][g][3];
            o[dt] = M::run(__builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), __builtin_bit_cast(frag, pb), o[dt]);
          }
    }
    __builtin_amdgcn_s_waitcnt(0);  // the next tile has landed
    __syncthreads();
  }

  // ---- epilogue ----
  const float l_tot = l_run + swapped(l_run);
  const float inv = l_tot > 0.f ? 1.f / l_tot : l_tot == 0.f ? 0.f : l_tot;  // (a NaN sum is a NaN row)
  T* const orow = static_cast<T*>(p.o) + b * p.os_b + h * p.os_h;
  float probe = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = l_tot == 0.f ? 0.f : o[dt][g * 4 + e] * inv;
        probe = fmaf(x[e], 0.f, probe);  // NaN once anything is NaN or infinite
      }
      auto pair = [&](int e) __attribute__((always_inline)) {
        return __builtin_amdgcn_permlane32_swap(M::pack2(x[e], x[e + 1]), M::pack2(x[e + 4], x[e + 5]), false, false);
      };
      const auto lo = pair(0), hi = pair(2);
      u32x4_v w;
      w.x = lo[0]; w.y = hi[0]; w.z = lo[1]; w.w = hi[1];
      if (q0 + l32 < p.Sq) *reinterpret_cast<u32x4_v*>(orow + row * p.os_s + dt * 32 + g * 8 + hh * 8) = w;
    }
  // rows to be done again: finite sums, but values that are not. (l_tot == 0: nothing was seen, zeros are right)
  const bool again = q0 + l32 < p.Sq && l_tot > 0.f && l_tot < INFINITY && probe != 0.f;
  uint64_t bad = __ballot(again);
  bad = (bad | (bad >> 32)) & 0xffffffffull;
  while (bad != 0) {  // (wave-uniform)
    const int who = __builtin_ctzll(bad);
    bad &= bad - 1;
    const int r = q0 + who, at = __builtin_amdgcn_readlane(pos, who);
    const int from[2] = {__builtin_amdgcn_readlane(blo, who), __builtin_amdgcn_readlane(plo, who)};
    const int to[2] = {__builtin_amdgcn_readlane(bhi, who), __builtin_amdgcn_readlane(phi, who)};
    const T* const qp = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h + r * p.qs_s;
    float m = -INFINITY, l = 0.f, acc[D / 64] = {};
    for (int range = 0; range < 2; ++range)
      for (int j0 = from[range]; j0 < to[range]; j0 += 64) {
        const int key = j0 + lane;
        const bool live = key < to[range] && !(range == 1 && key >= from[0] && key < to[0]);  // (the band's keys have been)
        float x = -INFINITY;
        if (live) {
          const T* const kp = kbase + key * p.ks_s;
          float s = 0.f;
          for (int d = 0; d < D; d += 8) {
            const u32x4 qv = load_raw(qp + d), kv = load_raw(kp + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(Raw<T>::get(qv, e), Raw<T>::get(kv, e), s);
          }
          x = CAP ? p.cap(s) : s * p.scale_log2;
          if constexpr (BIAS == 1) x = fmaf(-slope, fabsf(static_cast<float>(key - at)), x);
          if constexpr (BIAS == 2) x += table[clampi(key - at, -p.radius, p.radius) + p.radius];
        }
        float mx = x;
        for (int sft = 1; sft < 64; sft <<= 1) mx = fmaxf(mx, __shfl_xor(mx, sft, 64));
        const float m_new = fmaxf(m, mx), m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - m_safe), w = __builtin_amdgcn_exp2f(x - m_safe);
        m = m_new;
        l = l * alpha + group_sum<64>(w);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) acc[e] *= alpha;
        const uint64_t some = __ballot(live);
        for (int u = 0; u < 64; ++u) {
          if (!((some >> u) & 1)) continue;
          const float pw = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), u));
          const T* const vp = vbase + (j0 + u) * p.vs_s + lane * (D / 64);
#pragma unroll
          for (int e = 0; e < D / 64; ++e) acc[e] = fmaf(pw, to_float(vp[e]), acc[e]);
        }
      }
    T* const op = orow + r * p.os_s + lane * (D / 64);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) op[e] = from_float<T>(acc[e] / l);
  }
}

template <typename T, int D>
static int launch_ruled(RuledParams& p, bool cap, int bias, hipStream_t stream) {
  p.n_qblocks = (p.Sq + 127) / 128;
  p.units = p.H * p.B;
  const int64_t total = static_cast<int64_t>(p.n_qblocks) * p.H * p.B;
  ODIT_CHECK_ARG(total <= 0x7fffffffll, "odit_attn_ruled: grid of %lld workgroups is too large", static_cast<long long>(total));
#define ODIT_RULED_GO(C, X) hipLaunchKernelGGL((attn_ruled_kernel<T, D, C, X>), dim3(total), dim3(256), 0, stream, p)
  if (cap) {
    if (bias == 0) ODIT_RULED_GO(true, 0); else if (bias == 1) ODIT_RULED_GO(true, 1); else ODIT_RULED_GO(true, 2);
  } else {
    if (bias == 0) ODIT_RULED_GO(false, 0); else if (bias == 1) ODIT_RULED_GO(false, 1); else ODIT_RULED_GO(false, 2);
  }
#undef ODIT_RULED_GO
  return check_launch("odit_attn_ruled");
}

}  // namespace odit

extern "C" int odit_attn_ruled(const void* q, const void* k, const void* v, void* o, int B, int Sq, int Sk, int H, int Hkv, int D,
                               const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                               const int64_t o_strides[3], float scale, const odit_attn_rules* rules, int dtype, void* stream) {
  using namespace odit;
  ODIT_CHECK_ARG(rules != nullptr, "odit_attn_ruled: null rules");
  const odit_attn_rules& r = *rules;
  if (dtype != ODIT_BF16 && dtype != ODIT_F16) {
    set_error("odit_attn_ruled: dtype code %d unsupported (bf16 and fp16 only)", dtype);
    return ODIT_ENOTSUP;
  }
  if (D != 64 && D != 128) {
    set_error("odit_attn_ruled: head size %d unsupported (64 and 128 only)", D);
    return ODIT_ENOTSUP;
  }
  ODIT_CHECK_ARG(q_strides && k_strides && v_strides && o_strides, "odit_attn_ruled: null strides");
  constexpr int kMost = 1 << 30;  // (sums of two positions stay in 32 bits)
  ODIT_CHECK_ARG(B >= 0 && Sq >= 0 && Sk >= 0 && H > 0 && Hkv > 0 && Sq <= kMost && Sk <= kMost, "odit_attn_ruled: bad shape");
  ODIT_CHECK_ARG(static_cast<int64_t>(B) * H <= 0x7fffffffll, "odit_attn_ruled: %d batch rows of %d heads are too many", B, H);
  ODIT_CHECK_ARG(H % Hkv == 0, "odit_attn_ruled: H=%d is not a multiple of Hkv=%d", H, Hkv);
  ODIT_CHECK_ARG(scale > 0.f, "odit_attn_ruled: softmax scale must be positive (got %g)", scale);
  ODIT_CHECK_ARG(r.window >= 0 && r.window <= kMost, "odit_attn_ruled: window=%d outside [0, %d]", r.window, kMost);
  ODIT_CHECK_ARG(r.docs >= 0 && (r.docs == 0 || (r.q_starts && r.k_starts)), "odit_attn_ruled: documents need q_starts and k_starts");
  ODIT_CHECK_ARG(r.cap >= 0.f && r.cap <= kMaxCap, "odit_attn_ruled: cap=%g outside [0, %g]", r.cap, kMaxCap);
  ODIT_CHECK_ARG(r.slopes == nullptr || r.distance == nullptr, "odit_attn_ruled: slopes and a table exclude each other");
  ODIT_CHECK_ARG(r.distance == nullptr || (r.radius >= 0 && r.radius <= kMaxRadius), "odit_attn_ruled: radius=%d outside [0, %d]", r.radius,
                 kMaxRadius);
  ODIT_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o), "odit_attn_ruled: q/k/v/o must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    ODIT_CHECK_ARG(q_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0 && o_strides[i] % 8 == 0,
                   "odit_attn_ruled: strides must be multiples of 8 elements");
  ODIT_CHECK_ARG(k_strides[1] >= 0 && v_strides[1] >= 0 && k_strides[1] < (1ll << 23) && v_strides[1] < (1ll << 23),
                 "odit_attn_ruled: key and value rows must lie less than %d elements apart", 1 << 23);
  if (B == 0 || Sq == 0) return ODIT_OK;
  ODIT_CHECK_ARG(q && o && (Sk == 0 || (k && v)), "odit_attn_ruled: q/k/v/o must not be null");

  RuledParams p;
  p.q = q; p.k = k; p.v = v; p.o = o;
  p.q_starts = r.q_starts; p.k_starts = r.k_starts; p.prefix = r.prefix; p.slopes = r.slopes; p.distance = r.distance;
  p.docs = r.docs; p.causal = r.causal != 0; p.window = r.window; p.radius = r.radius;
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.H = H; p.Hkv = Hkv;
  p.qs_b = q_strides[0]; p.qs_s = q_strides[1]; p.qs_h = q_strides[2];
  p.ks_b = k_strides[0]; p.ks_s = k_strides[1]; p.ks_h = k_strides[2];
  p.vs_b = v_strides[0]; p.vs_s = v_strides[1]; p.vs_h = v_strides[2];
  p.os_b = o_strides[0]; p.os_s = o_strides[1]; p.os_h = o_strides[2];
  p.scale_log2 = scale * kLog2e;
  p.cap.in = r.cap > 0.f ? 2.f * kLog2e * scale / r.cap : 0.f;
  p.cap.out = r.cap * kLog2e;
  const int bias = r.slopes != nullptr ? 1 : r.distance != nullptr ? 2 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODIT_BF16) return D == 128 ? launch_ruled<bf16_t, 128>(p, r.cap > 0.f, bias, st) : launch_ruled<bf16_t, 64>(p, r.cap > 0.f, bias, st);
  return D == 128 ? launch_ruled<f16_t, 128>(p, r.cap > 0.f, bias, st) : launch_ruled<f16_t, 64>(p, r.cap > 0.f, bias, st);
}

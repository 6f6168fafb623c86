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
// A value that is NaN or infinite spoils its tile's product also for queries that do not see its key (0 times it is NaN). Where a wavefront's rows come
// out so with a finite sum, and there are such values in tiles that its queries see in part, its rows are therefore done again at the end, with
// values and what is not finite among them apart.
#include <type_traits>

#include "attn_rules.h"
#include "quotient.h"

namespace odit {

typedef short s16x4_r __attribute__((ext_vector_type(4)));
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
  float scale_log2, bias_scale;  // scale log2(e) and 1 / scale
  float unit;                    // from what scores are kept in to units of log2: scale log2(e), or 1 behind a cap
  Cap cap;
  int n_qblocks, units;  // units: heads of all batch rows
  int group;             // query heads of a key head
  Quotient by_blocks, by_units, by_heads, by_group;  // by n_qblocks * units, by the units of a row of blocks (of an XCD), by H, by group
  int bm;                // queries of a block
  int chunks;            // workgroups that share a query block's tiles; with more than one, their sums go to ws
  const float* norms;    // [B][Hkv][kNormParts]: the largest squared length of a part's keys, by which far tiles are left out (nullptr: none is)
  float* ws;             // [units][n_qblocks][chunks][bm][D] sums, then [...][bm] (maximum in units of scores, sum)
};

// Among 64 documents from `base` on, whose starts the lanes hold: the last one that starts at or before the lane's row, one of the 32 from
// row0 on; `doc` where there is none. *past: whether a later start lies behind all the rows.
__device__ __forceinline__ int doc_among(int mine, int base, int row0, int row, int doc, bool* past) {
  const uint64_t before = __ballot(mine <= row0);
  bool end = false;
  for (int i = before == 0 ? 0 : __popcll(before) - 1; i < 64 && !end; ++i) {
    const int start = __builtin_amdgcn_readlane(mine, i);
    end = start > row0 + 31;
    if (start <= row) doc = base + i;
  }
  if (past != nullptr) *past = end;
  return doc;
}
// The documents of 32 rows from row0 on, lane l's row being row0 + l % 32: the last one that starts at or before it. The wavefront reads 64
// starts at a time: searches by halves would be log2(docs) dependent trips to memory.
// (Whatever the starts hold, the search ends and stays inside them.)
__device__ __forceinline__ int doc_of(const int* starts, int docs, int row0, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = docs;  // the first row's document is one of [lo, lo + n)
  while (n > 64) {
    const int step = (n + 63) / 64, at = lane * step;
    const uint64_t before = __ballot(at < n && starts[lo + (at < n ? at : 0)] <= row0);
    const int skip = (before == 0 ? 0 : __popcll(before) - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  int doc = lo;
  for (int base = lo; base < docs; base += 64) {
    bool past;
    doc = doc_among(base + lane < docs ? starts[base + lane] : 0x7fffffff, base, row0, row, doc, &past);
    if (past) break;
  }
  return doc;
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// of the 32 lanes of each half of a wavefront, which hold the same
template <int CTRL> __device__ __forceinline__ int dpp_int(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
__device__ __forceinline__ int half_min(int v) {
  v = min(v, dpp_int<0xB1>(v)); v = min(v, dpp_int<0x4E>(v)); v = min(v, dpp_int<0x141>(v)); v = min(v, dpp_int<0x140>(v));
  return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}
__device__ __forceinline__ int half_max(int v) { return ~half_min(~v); }

// bits of the keys of [t0, t0 + 64) in [lo, hi)
__device__ __forceinline__ uint64_t range_bits(int lo, int hi, int t0) {
  const int a = clampi(lo - t0, 0, 64), b = clampi(hi - t0, 0, 64);
  if (b <= a) return 0;
  const uint64_t upto = b == 64 ? ~0ull : (1ull << b) - 1;
  return upto & (~0ull << a);
}

// a value's bits: not finite (all of the exponent's bits are set)
template <typename T> __device__ __forceinline__ bool not_finite(uint32_t v);
template <> __device__ __forceinline__ bool not_finite<bf16_t>(uint32_t v) { return (v & 0x7f80u) == 0x7f80u; }
template <> __device__ __forceinline__ bool not_finite<f16_t>(uint32_t v) { return (v & 0x7c00u) == 0x7c00u; }
template <typename T> __device__ __forceinline__ bool is_nan(uint32_t v) { return not_finite<T>(v) && (v & (std::is_same<T, bf16_t>::value ? 0x7fu : 0x3ffu)) != 0; }

constexpr int kTablePad = 63;  // a tile's keys but one
// The keys' largest squared lengths, in kNormParts parts of each head's: a lane of the kernel below reads each. A workgroup has a part; D / 8 lanes a key.
constexpr int kNormParts = 64;
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_ruled_norms_kernel(const RuledParams p, float* norms) {
  constexpr int LPK = D / 8, KPI = 256 / LPK;
  __shared__ float waves[4];
  const int part = blockIdx.x % kNormParts, head = blockIdx.x / kNormParts, b = head / p.Hkv, hkv = head % p.Hkv;
  const int each = (p.Sk + kNormParts - 1) / kNormParts, begin = min(part * each, p.Sk), end = min(begin + each, p.Sk);
  const T* const base = static_cast<const T*>(p.k) + b * p.ks_b + hkv * p.ks_h + threadIdx.x % LPK * 8;
  float most = 0.f;
  for (int first = begin; first < end; first += 4 * KPI) {  // (for all lanes alike: they exchange sums)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = min(first + i * KPI + static_cast<int>(threadIdx.x) / LPK, end - 1);
      const u32x4 x = load_raw(base + key * p.ks_s);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(Raw<T>::get(x, e), Raw<T>::get(x, e), sum);
#pragma unroll
      for (int s = 1; s < LPK; s <<= 1) sum += __shfl_xor(sum, s, 64);
      most = __builtin_elementwise_maximum(most, sum);
    }
  }
#pragma unroll
  for (int s = LPK; s < 64; s <<= 1) most = __builtin_elementwise_maximum(most, __shfl_xor(most, s, 64));
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 4; ++w) most = __builtin_elementwise_maximum(most, waves[w]);
    norms[blockIdx.x] = most;
  }
}

// BIAS 0: none, 1: slopes, 2: table. KH: the 32-key halves of a tile that a wavefront has. With both, the workgroup's 4 wavefronts have 32
// queries each; with one, two wavefronts share 32 queries, a half of each tile each, and join at the end (ruled_plan says when).
constexpr int ruled_waves(int D, int KH) { return D == 128 ? 2 : KH == 1 ? 4 : 3; }  // wavefronts of a SIMD, workgroups of a compute unit
template <typename T, int D, bool CAP, int BIAS, int KH>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(ruled_waves(D, KH), ruled_waves(D, KH))))
void attn_ruled_kernel(const RuledParams p) {
  using M = Mma<T>;
  using frag = typename M::frag;
  constexpr int NW = 4, BM = NW * 16 * KH, BN = 64, NS = 16 * KH;  // NS: scores of a lane
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPI = 64 / CPR, TILEB = BN * ROWB;
  constexpr int IPW = BN / RPI / NW;  // wave instructions of a tile's load, per wavefront

  __shared__ __attribute__((aligned(1024))) char lds[4 * TILEB];  // K0 K1 V0 V1
  __shared__ int bounds[NW][4];
  __shared__ int places[BIAS != 0 ? NW * 32 : 1];  // pos of each lane's query
  __shared__ int4 ranges[NW * 32];  // blo, bhi, plo, phi of each lane's query: read again at each tile, which has no registers to hold them
  // BIAS 2: the head's biases, with the outermost ones once more for each further key of a tile that some distance inside begins or ends
  constexpr int kPad = kTablePad;
  extern __shared__ float table[];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  // the last query blocks, which see most under a causal order, begin first; where the heads divide over the XCDs, an XCD keeps its heads
  // (steep slopes leave a head little to do: with slopes the heads go round the XCDs and back again, so that each has steep and shallow ones, and an XCD
  // begins its rows of blocks with each of its heads in turn: it hands workgroups to its shader engines in a fixed order, so that those which
  // would get steep heads alone stood empty while the others were full. us of 16384 causal tokens, 16 heads of 128: while all tiles were visited, 1040 with
  // neighbours on an XCD, 929 going round, 910 there and back; with far tiles left out 828, and 632 with the heads in turn on the same card, 435 and 360 of 8192, 32 on 8)
  const int chunk = p.chunks > 1 ? p.by_blocks(blockIdx.x) : 0, block = blockIdx.x - chunk * (p.units * p.n_qblocks);
  int unit, qb;
  if (BIAS != 1 && p.units % kNumXcd == 0) {
    const int per = p.units / kNumXcd, local = block / kNumXcd, at = p.by_units(local);
    unit = block % kNumXcd * per + local - at * per;
    qb = p.n_qblocks - 1 - at;
  } else {
    const int at = p.by_units(block);
    unit = block - at * p.units;
    qb = p.n_qblocks - 1 - at;
    if (BIAS == 1 && p.units % kNumXcd == 0) {
      const int per = p.units / kNumXcd, j = (unit / kNumXcd + at / 2) % per, xcd = unit % kNumXcd;
      unit = j * kNumXcd + (j & 1 ? kNumXcd - 1 - xcd : xcd);
    }
  }
  // (ahead of the queries' loads: they come back in the order of their issue)
  int q_start = 0, k_start = 0, first_keys = 0;  // docs < 64: the lanes hold all starts, in one trip to memory
  if (p.docs > 0 && p.docs < 64) {
    const int at = lane <= p.docs ? lane : p.docs;
    q_start = p.q_starts[at];
    k_start = p.k_starts[at];
    if (p.prefix != nullptr) first_keys = p.prefix[min(at, p.docs - 1)];
  }
  const int b = p.by_heads(unit), h = unit - b * p.H, hkv = p.by_group(h);
  const int kt0 = KH == 1 ? wave >> 1 : 0;  // the first of this wavefront's halves
  const int q0 = qb * BM + (KH == 1 ? wave & 1 : wave) * 32;
  const int row = q0 + l32 < p.Sq ? q0 + l32 : p.Sq - 1;

  const T* const qrow = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h + row * p.qs_s;
  frag qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = __builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(qrow + hh * 8 + ks * 16));
  // (three or four workgroups to a compute unit: some fragments are read again at each tile, for want of a few registers)
  constexpr int QL = D != 64 ? 0 : KH == 1 ? (BIAS == 2 ? 0 : 1) : CAP && BIAS != 2 ? 4 : 2;
  __shared__ u32x4_v q_lds[QL > 0 ? QL * NW * 64 : 1];
  auto q_at = [&](int ks) __attribute__((always_inline)) {
    if (ks >= QL) return qf[ks];
    uint32_t from = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_rp)(q_lds + ks * NW * 64 + tid)));
    asm volatile("" : "+v"(from) : : "memory");  // (opaque, or the compiler keeps what was stored there in registers after all)
    return __builtin_bit_cast(frag, *(__attribute__((address_space(3))) const u32x4_v*)(from));
  };

  // Biases join a product at its first addition, as the accumulator's first value, where a zero would stand otherwise: they cost nothing
  // and are kept in units of products (x / scale). Behind a cap they are in units of log2.
  const float bias_unit = CAP ? kLog2e : p.bias_scale;
  if constexpr (BIAS == 2) {
    const float* from = p.distance + static_cast<int64_t>(h) * (2 * p.radius + 1);
    for (int i = tid; i <= 2 * p.radius + 2 * kPad; i += 256) table[i] = in_units(from[clampi(i - kPad, 0, 2 * p.radius)], bias_unit);
  }

  // ---- what this lane's query sees ----
  constexpr int kNone = 0x7fffffff;
  // the band of a query at place `at` of a document of kn keys
  const auto band_begin = [&](int at, int kn) { return p.window > 0 ? clampi(at - p.window + 1, 0, kn) : 0; };
  const auto band_end = [&](int at, int kn) { return p.causal ? clampi(at + 1, 0, kn) : p.window > 0 ? clampi(at + p.window, 0, kn) : kn; };
  int blo, bhi, plo = 0, phi = 0, pos;  // pos: the key at the query's own place
  {
    int ks = 0, kn = p.Sk, qs = 0, qe = p.Sq, doc = 0, prefix = 0;
    bool in = true;
    if (p.docs > 0) {
      const int row0 = q0 < p.Sq ? q0 : p.Sq - 1;
      if (p.docs < 64) {
        doc = doc_among(lane < p.docs ? q_start : kNone, 0, row0, row, 0, nullptr);
        qs = __shfl(q_start, doc, 64);
        qe = __shfl(q_start, doc + 1, 64);
        ks = __shfl(k_start, doc, 64);
        kn = __shfl(k_start, doc + 1, 64);
        prefix = __shfl(first_keys, doc, 64);
      } else {
        doc = doc_of(p.q_starts, p.docs, row0, row);
        qs = p.q_starts[doc];
        qe = p.q_starts[doc + 1];
        ks = p.k_starts[doc];
        kn = p.k_starts[doc + 1];
        prefix = p.prefix != nullptr ? p.prefix[doc] : 0;
      }
      in = row >= qs && row < qe;
      ks = clampi(ks, 0, p.Sk);
      kn = clampi(kn, ks, p.Sk) - ks;
    } else if (p.prefix != nullptr) {
      prefix = p.prefix[b];
    }
    // the query's place from the document's first key (cut to what sums with a window keep in 32 bits, whatever the starts hold)
    constexpr int64_t kFar = (1 << 30) - 1;
    const int64_t place = static_cast<int64_t>(row) + kn - qe;
    const int at = static_cast<int>(place < -kFar ? -kFar : place > kFar ? kFar : place);
    const int lo = band_begin(at, kn), hi = band_end(at, kn);
    pos = ks + at;
    blo = in && hi > lo ? ks + lo : 0;  // (nothing: [0, 0))
    bhi = in && hi > lo ? ks + hi : 0;
    if (in && prefix > 0 && kn > 0) {
      plo = ks;
      phi = ks + min(prefix, kn);
    }
  }
  int all0, all1;  // the keys that all queries of the wavefront have in their bands (none: all1 <= all0)
  {
    if (hh == 0) ranges[wave * 32 + l32] = make_int4(blo, bhi, plo, phi);
    if (BIAS != 0 && hh == 0) places[wave * 32 + l32] = pos;
    if (p.docs > 0) {
      all0 = half_max(blo);
      all1 = half_min(bhi);
      const int b0 = half_min(bhi > 0 ? blo : kNone), b1 = half_max(bhi), p0 = half_min(phi > 0 ? plo : kNone), p1 = half_max(phi);
      if (lane == 0) { bounds[wave][0] = b0; bounds[wave][1] = b1; bounds[wave][2] = p0; bounds[wave][3] = p1; }
    }
  }
  // the workgroup's tiles: up to two runs
  int s1, n1, s2, n2;
  {
    int lo[2] = {kNone, kNone}, hi[2] = {0, 0};
    if (p.docs > 0) {
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          lo[i] = min(lo[i], bounds[w][2 * i]);
          hi[i] = max(hi[i], bounds[w][2 * i + 1]);
        }
    } else {  // one document: both ends of the band rise with the row
      const int row0 = min(q0, p.Sq - 1) + p.Sk - p.Sq, row1 = min(q0 + 31, p.Sq - 1) + p.Sk - p.Sq;
      all0 = band_begin(row1, p.Sk);
      all1 = band_end(row0, p.Sk);
      const int last = min(qb * BM + BM, p.Sq) - 1;
      lo[0] = band_begin(qb * BM + p.Sk - p.Sq, p.Sk);
      hi[0] = band_end(last + p.Sk - p.Sq, p.Sk);
      lo[1] = 0;
      hi[1] = p.prefix != nullptr ? clampi(p.prefix[b], 0, p.Sk) : 0;
    }
    int a0 = lo[0] / BN, a1 = hi[0] > lo[0] ? (hi[0] + BN - 1) / BN : a0, c0 = lo[1] / BN, c1 = hi[1] > lo[1] ? (hi[1] + BN - 1) / BN : c0;
    if (a1 == a0) { a0 = c0; a1 = c1; c1 = c0; }                                                    // one run or none
    if (c1 > c0 && c0 <= a1 && a0 <= c1) { a0 = min(a0, c0); a1 = max(a1, c1); c0 = c1 = 0; }        // they touch
    s1 = __builtin_amdgcn_readfirstlane(a0); n1 = __builtin_amdgcn_readfirstlane(a1 - a0);
    s2 = __builtin_amdgcn_readfirstlane(c0); n2 = __builtin_amdgcn_readfirstlane(c1 - c0);
  }
  if constexpr (BIAS == 1) {
    // Slopes: no score exceeds |q| |k| in size, nor the cap, a query's own key has no bias, so its maximum is at least the negative of that, and a key
    // `reach` away has a probability of 2^-160 at most beside it, which is zero in 32 bits (2^-8 of that is what the running maximum may lag). Tiles
    // farther off than that from all queries are left out: of 16384 causal tokens, 16 heads with slopes of 2^-1/2 to 2^-8, more than half.
    const float steep = p.slopes[h] * kLog2e;
    if (p.norms != nullptr && steep > 0.f) {
      float q2 = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 x = __builtin_bit_cast(u32x4, qf[ks]);
#pragma unroll
        for (int e = 0; e < 8; ++e) q2 = fmaf(Raw<T>::get(x, e), Raw<T>::get(x, e), q2);
      }
      q2 += __shfl_xor(q2, 32, 64);
      float k2 = p.norms[(static_cast<int64_t>(b) * p.Hkv + hkv) * kNormParts + lane];
#pragma unroll
      for (int sft = 1; sft < 64; sft <<= 1) {  // (NaN stays NaN)
        q2 = __builtin_elementwise_maximum(q2, __shfl_xor(q2, sft, 64));
        k2 = __builtin_elementwise_maximum(k2, __shfl_xor(k2, sft, 64));
      }
      __shared__ float lengths[NW];
      if (lane == 0) lengths[wave] = q2;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) q2 = __builtin_elementwise_maximum(q2, lengths[w]);
      const float product = p.scale_log2 * sqrtf(q2) * sqrtf(k2) * 1.001f, most = CAP ? fminf(product, p.cap.out) : product;
      const float reach = (2.f * most + 160.f) / steep * 1.001f + 1.f;
      // (-1: nothing is left out. NaN and infinities in queries or keys, behind a cap too: a score may then be NaN however far its key is)
      const int far = __builtin_amdgcn_readfirstlane(product < INFINITY && reach < 1e9f ? static_cast<int>(reach) + 1 : -1);
      if (far >= 0) {
        const int row0 = qb * BM + p.Sk - p.Sq, row1 = min(qb * BM + BM, p.Sq) - 1 + p.Sk - p.Sq;
        const int from = max(row0 - far, 0) / BN, to = (row1 + far) / BN + 1;
        const auto trim = [&](int& first, int& n) {
          const int end = min(first + n, to);
          first = max(first, from);
          n = max(end - first, 0);
        };
        trim(s1, n1);
        trim(s2, n2);
      }
    }
  }
  // this workgroup's of them: tile i is number last - i of both runs together
  int last = n1 + n2 - 1, n_tiles = n1 + n2;
  if (p.chunks > 1) {
    const int begin = static_cast<int>(static_cast<int64_t>(n_tiles) * chunk / p.chunks);
    n_tiles = static_cast<int>(static_cast<int64_t>(n_tiles) * (chunk + 1) / p.chunks) - begin;
    last -= begin;
  }
  // From the last key back: under a causal order the nearest keys come first. Where distance takes from the scores, the running maximum is
  // then near its end from the first tile on (slopes at 16384 tokens, 16 heads: 1203 us forwards, 1040 backwards).
  auto tile_at = [&](int i) { return last - i < n1 ? s1 + last - i : s2 + last - i - n1; };

  // ---- tile loads: as in attn_fwd_dma.hip, but with a buffer descriptor for each tile, so that offsets stay small in any tensor ----
  const T* const kbase = static_cast<const T*>(p.k) + b * p.ks_b + hkv * p.ks_h;
  const T* const vbase = static_cast<const T*>(p.v) + b * p.vs_b + hkv * p.vs_h;
  const int r0 = wave * IPW * RPI + lane / CPR, pc0 = lane % CPR;
  constexpr auto k_swizzle = [](int r) { return D == 128 ? r % 16 : r / 2 % 8; };
  constexpr auto v_swizzle = [](int r) { return D == 128 ? 4 * (r % 4) : 4 * (r / 2 % 2); };
  // Byte offsets of the lane's first instruction; the others' rows lie a whole number of rows further down, which is the load's scalar
  // offset. The chunk of 16 bytes that a lane fetches is swizzled by its row, so that the reads of fragments touch all banks: keys by row, or by
  // row / 2 at head size 64, where two rows share the banks (by row there, as in attn_fwd_dma.hip, 43 % of the reads' cycles were conflicts);
  // values so that the 4 keys of a transposed read do. An instruction's rows are a multiple of 4 further down: another constant for keys, none for values.
  const uint32_t krow = static_cast<uint32_t>(r0 * p.ks_s * 2), kswz = static_cast<uint32_t>((pc0 ^ k_swizzle(r0)) * 16);
  const uint32_t vvoff = static_cast<uint32_t>(r0 * p.vs_s * 2) + static_cast<uint32_t>((pc0 ^ v_swizzle(r0)) * 16);
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_rp)lds));
  const uint32_t k_bytes = static_cast<uint32_t>(((BN - 1) * p.ks_s + D) * 2), v_bytes = static_cast<uint32_t>(((BN - 1) * p.vs_s + D) * 2);
  auto load_tile = [&](const T* base, int64_t stride, bool keys, int t, int dst) __attribute__((always_inline)) {
    const uint64_t a = reinterpret_cast<uint64_t>(base) + static_cast<uint64_t>(static_cast<uint32_t>(t)) * static_cast<uint32_t>(BN * 2 * stride);
    const int over = t * BN + BN - p.Sk;  // rows behind the last key read as zeros
    u32x4_v r;
    r.x = static_cast<uint32_t>(a); r.y = static_cast<uint32_t>(a >> 32) & 0xffffu;
    r.z = (keys ? k_bytes : v_bytes) - (over > 0 ? static_cast<uint32_t>(over * 2) * static_cast<uint32_t>(stride) : 0); r.w = 0x00020000u;
    uint32_t row = keys ? krow : vvoff, swz = keys ? kswz : 0;
    asm volatile("" : "+v"(swz));  // (the sums are formed here, not held in registers across the loop)
#pragma unroll
    for (int i = 0; i < IPW; ++i)
      load_lds16(lds_base + dst + (wave * IPW + i) * 1024, row + (keys ? swz ^ static_cast<uint32_t>(k_swizzle(RPI * i) * 16) : 0), r,
                 static_cast<uint32_t>(RPI * i * stride * 2));
  };
  auto load_k = [&](int i, const int buf) { load_tile(kbase, p.ks_s, true, tile_at(i), buf * TILEB); };
  auto load_v = [&](int i, const int buf) { load_tile(vbase, p.vs_s, false, tile_at(i), (2 + buf) * TILEB); };

  f32x16_v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
  const float c = CAP ? 1.f : p.scale_log2;  // from what m_run is in to units of log2
  float m_run = -INFINITY, l_run = 0.f, mc = 0.f;
  // An exponent is s c - mc in one instruction, mc being m c rounded. What that rounding loses is the same for all of a row's keys, but it grows with
  // the maximum (past 2^31 an exponent of zero comes out above 128). So where m c is past kFar, scores are made differences from the maximum ahead of
  // the exponent, and mc is zero. Scores of that size are rare (biases that forbid are: -1e10 at every key that a query sees so far), so it is
  // a branch by a scalar.
  constexpr float kFar = 1024.f;
  bool far_max = false;  // some query of the wavefront is there
  const auto is_far = [&]() __attribute__((always_inline)) { return fabsf(m_run * c) > kFar && fabsf(m_run) < INFINITY; };
  const float slope = BIAS == 1 ? in_units(p.slopes[h], bias_unit) : 0.f;

  const int k_lane = (32 * kt0 + l32) * ROWB + ((hh ^ k_swizzle(l32)) << 4);
  const int sq = (lane & 15) >> 2, dh = (lane >> 4) & 1;
  const int v_lane = (32 * kt0 + 4 * hh + sq) * ROWB + ((v_swizzle(sq) ^ (2 * dh + ((lane & 3) >> 1))) << 4) + ((lane & 1) << 3);
  auto swapped = [&](float x) __attribute__((always_inline)) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(hh ? r[0] : r[1]);
  };

  constexpr bool POLY = CAP && BIAS == 0;
  // Where a tile's probabilities are made: between the matrix instructions of the next one's scores, or where the compiler would have them, in the branch
  // that takes them, beside the second product. us, there / pinned: 4096 tokens, 24 heads of 64, all keys 125 / 117, causal 82.8 / 85.7; capped window of
  // 4096 in 8192 tokens, 32 heads of 128, 533 / 526; a table in 12 documents, 24 heads of 128, 109 / 106. With slopes many tiles have none: 940 / 974.
  constexpr bool PINNED = BIAS == 0 || (BIAS == 2 && D == 128);
  // the score of a key that is not seen (POLY: finite, as are all capped ones, for the polynomial 1 + 0 s^2 + ..; its exp2 is zero all the same)
  const float kOut = POLY ? -1e18f : -INFINITY;
  // whether some query of the wavefront sees a key of the tile from t0 on, and whether all of them see all
  auto own = [&]() __attribute__((always_inline)) { return ranges[wave * 32 + l32]; };
  constexpr int WN = 32 * KH;  // the wavefront's keys of a tile, from t0 + 32 kt0 on
  auto some_see = [&](int t0) {
    const int k0 = t0 + 32 * kt0;
    if (k0 >= all0 && k0 + WN <= all1) return true;  // (most tiles of a long prompt)
    const int4 r = own();
    return __any((k0 < r.y && k0 + WN > r.x) || (k0 < r.w && k0 + WN > r.z)) != 0;
  };
  auto all_see = [&](int t0) {
    const int k0 = t0 + 32 * kt0;
    if (k0 >= all0 && k0 + WN <= all1) return true;
    const int4 r = own();
    return __all((k0 >= r.x && k0 + WN <= r.y) || (k0 >= r.z && k0 + WN <= r.w)) != 0;
  };
  constexpr auto key_of = [](int e) { return (e >> 4) * 32 + ((e & 15) >> 2) * 8 + (e & 3); };  // of the lane's score e: t0 + 32 kt0 + key_of(e) + 4 hh

  // biases of the lane's keys of the tile from t0 on: the scores' first values, or added to what a cap has made of them
  auto biases = [&](int t0, f32x16_v(&s)[KH]) __attribute__((always_inline)) {
    const auto put = [&](int e, float bias) __attribute__((always_inline)) { s[e >> 4][e & 15] = CAP ? s[e >> 4][e & 15] + bias : bias; };
    const int pos = places[wave * 32 + l32], k0 = t0 + 32 * kt0, first = k0 + 4 * hh - pos;
    if constexpr (BIAS == 1) {
      const float at = static_cast<float>(first);
      const bool before = __all(k0 + WN - 1 <= pos), behind = __all(k0 >= pos);
      if (before || behind) {  // (linear: one instruction each)
        const float sl = before ? slope : -slope, b0 = sl * at;
#pragma unroll
        for (int e = 0; e < NS; ++e) put(e, fmaf(sl, static_cast<float>(key_of(e)), b0));
      } else {
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          put(e, -slope * fabsf(at + static_cast<float>(key_of(e))));
          if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      const bool before = __all(k0 + WN - 1 - pos <= -p.radius), behind = __all(k0 - pos >= p.radius);
      if (before || behind) {
        const float far = table[before ? 0 : 2 * p.radius + 2 * kPad];
#pragma unroll
        for (int e = 0; e < NS; ++e) put(e, far);
      } else {
        const float* const from = table + clampi(first, -p.radius - kPad, p.radius) + p.radius + kPad;
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          put(e, from[key_of(e)]);
          if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // (not all at once: there are no registers for it)
        }
      }
    }
  };
  auto first_values = [&](int t0, f32x16_v(&s)[KH]) __attribute__((always_inline)) {
    if constexpr (BIAS != 0 && !CAP) {
      biases(t0, s);
    } else {
#pragma unroll
      for (int e = 0; e < NS; ++e) s[e >> 4][e & 15] = 0.f;
    }
  };
  auto lane_max = [&](const f32x16_v(&s)[KH]) __attribute__((always_inline)) {
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < NS; ++e) mx = __builtin_elementwise_maximum(mx, s[e >> 4][e & 15]);
    return mx;
  };
  // Behind the products: the cap by its own formula and the biases behind it (CAP, unless the tile's scores stay as they are: see below),
  // keys that some query does not see; returns the lane's maximum
  auto finish_scores = [&](int t0, bool all, f32x16_v(&s)[KH]) {
    if constexpr (CAP) {
      if (__builtin_expect(p.cap.large, 0)) {
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          float x = s[e >> 4][e & 15];
          asm volatile("" : "+v"(x));  // (one after the other: there are no registers for more)
          x = p.cap.of_large(x);
          asm volatile("" : "+v"(x));
          s[e >> 4][e & 15] = x;
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          s[e >> 4][e & 15] = p.cap(s[e >> 4][e & 15]);
          if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (BIAS != 0) biases(t0, s);
    }
    if (!all) {
      const int4 r = own();
      const uint64_t w = range_bits(r.x, r.y, t0) | range_bits(r.z, r.w, t0);
      const uint32_t lower = static_cast<uint32_t>(w) >> (4 * hh), upper = static_cast<uint32_t>(w >> 32) >> (4 * hh);
      const uint32_t half[2] = {KH == 1 && kt0 == 1 ? upper : lower, upper};
#pragma unroll
      for (int e = 0; e < NS; ++e) s[e >> 4][e & 15] = (half[e >> 4] & (1u << (key_of(e) & 31))) ? s[e >> 4][e & 15] : kOut;
    }
    const float mx = lane_max(s);
    return POLY && mx == kOut ? -INFINITY : mx;
  };
  auto settle_max = [&](float mx) __attribute__((always_inline)) {
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
      if constexpr (!CAP) {
        const bool here = is_far();
        if (here) mc = 0.f;
        far_max = __any(here) != 0;
      }
    }
  };
  auto less_far_max = [&](f32x16_v(&s)[KH]) __attribute__((always_inline)) {
    if (CAP || !far_max) return;
    const float m = is_far() ? m_run : 0.f;
#pragma unroll
    for (int e = 0; e < NS; ++e) s[e >> 4][e & 15] -= m;
  };

  // Tile i of the workgroup: its probabilities from s_cur while the next tile's products are formed (stage A), then its part of the output
  // while the next scores' maximum is taken (stage B). `buf` is i % 2, a literal at every call.
  // With a cap and no bias, scores that all queries see and that are small against the cap stay products until stage A, where the cap's
  // polynomial is part of the exponent: the tanh rises, so their maximum is the capped ones'. Other tiles' scores are made at once
  // (finish_scores), and their polynomial is the score itself.
  bool seen = false, live = false;  // tile i: seen by some query of this wavefront (s_cur holds its scores), with some weight
  float c0 = 1.f, c1 = 0.f, c2 = 0.f, c3 = 0.f;  // POLY: of s_cur
  auto k_at = [&](const char* kb, int i) { return *reinterpret_cast<const u32x4_v*>(kb + i % KH * 32 * ROWB + (k_lane ^ (i / KH * 32))); };
  auto tile = [&](int i, const int buf, f32x16_v(&s_cur)[KH], f32x16_v(&s_next)[KH]) {
    const bool has_next = i + 1 < n_tiles;
    if (i + 2 < n_tiles) load_k(i + 2, buf);
    if (has_next) load_v(i + 1, buf ^ 1);
    const int tn = has_next ? tile_at(i + 1) * BN : 0;
    const bool seen_next = has_next && some_see(tn);
    float mx = -INFINITY, most = 0.f;  // the next scores' maximum and their sizes', of this lane
    if (seen || seen_next) {
      // Everything of a tile in one piece: branches around its parts would have the scores of both their ways brought together by copies
      // (32 at every tile, 10 % of a long prompt). So the next products are formed where nothing of them is seen, and probabilities of
      // scores that do not count (`live` says so), once each at the ends of a run of tiles.
      uint32_t pf[KH][2][4];
      float sum = 0.f;
      auto exponent = [&](float s) __attribute__((always_inline)) {
        if constexpr (!POLY) return fmaf(s, c, -mc);
        const float z = s * s;
        return fmaf(s, fmaf(z, fmaf(z, fmaf(z, c3, c2), c1), c0), -mc);
      };
      auto probabilities = [&](int pi) __attribute__((always_inline)) {
        const int kt = pi >> 3, e = (pi & 7) * 2;
        const float p0 = __builtin_amdgcn_exp2f(exponent(s_cur[kt][e])), p1 = __builtin_amdgcn_exp2f(exponent(s_cur[kt][e + 1]));
        sum += p0 + p1;
        uint32_t both = M::pack2(p0, p1);
        if constexpr (PINNED) asm volatile("" : "+v"(both), "+v"(sum));
        pf[kt][(pi & 7) >> 2][pi & 3] = both;
      };
      __builtin_amdgcn_s_setprio(2);
      const char* const kb = lds + (buf ^ 1) * TILEB;
      first_values(tn, s_next);
      constexpr int KPF = CAP || D == 64 ? 2 : 3;  // fragments on their way ahead of the instruction that takes them
      u32x4_v kfr[KPF + 1];
#pragma unroll
      for (int n = 0; n < KPF; ++n) kfr[n] = k_at(kb, n);
      frag qn = q_at(0);
#pragma unroll
      for (int n = 0; n < KH * KS; ++n) {
        if (n + KPF < KH * KS) kfr[(n + KPF) % (KPF + 1)] = k_at(kb, n + KPF);
        s_next[n % KH] = M::run(__builtin_bit_cast(frag, kfr[n % (KPF + 1)]), qn, s_next[n % KH]);
        if (n % KH == KH - 1 && n + 1 < KH * KS) qn = q_at((n + 1) / KH);
        constexpr int EACH = 8 / KS;
#pragma unroll
        for (int m = 0; m < EACH; ++m) probabilities(n * EACH + m);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      auto max_step = [&](int e) __attribute__((always_inline)) {
        const float x0 = s_next[e >> 4][e & 15], x1 = s_next[e >> 4][(e + 1) & 15];
        mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, x0), x1);
        if constexpr (CAP) most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, fabsf(x0)), fabsf(x1));
      };
      if (live) {
        l_run += sum;
        const char* const vb = lds + (2 + buf) * TILEB;
        constexpr int NSTEP = 2 * KH * DT, VPF = CAP || D == 64 ? 2 : 3, EACH = NS / NSTEP;
        s16x4_r vlo[VPF + 1], vhi[VPF + 1];
        auto v_fetch = [&](int st) {
          const char* const vp = vb + (st / DT) * 16 * ROWB + (v_lane ^ ((st % DT * 64) % ROWB));
          vlo[st % (VPF + 1)] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_rp)(vp));
          vhi[st % (VPF + 1)] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_rp)(vp + 8 * ROWB));
        };
#pragma unroll
        for (int st = 0; st < VPF; ++st) v_fetch(st);
#pragma unroll
        for (int st = 0; st < NSTEP; ++st) {
          if (st + VPF < NSTEP) v_fetch(st + VPF);
          const int dt = st % DT, kt = (st / DT) >> 1, g = (st / DT) & 1;
          u32x4_v pb;
          pb.x = pf[kt][g][0]; pb.y = pf[kt][g][1]; pb.z = pf[kt][g][2]; pb.w = pf[kt][g][3];
          o[dt] = M::run(__builtin_bit_cast(frag, __builtin_shufflevector(vlo[st % (VPF + 1)], vhi[st % (VPF + 1)], 0, 1, 2, 3, 4, 5, 6, 7)),
                         __builtin_bit_cast(frag, pb), o[dt]);
          if constexpr (!CAP || BIAS == 0) {
#pragma unroll
            for (int e = st * EACH; e < st * EACH + EACH; e += 2) max_step(e);
            asm volatile("" : "+v"(mx));  // (where it is: it would sink below the test behind the loop otherwise)
            if constexpr (CAP) asm volatile("" : "+v"(most));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else if constexpr (!CAP || BIAS == 0) {
#pragma unroll
        for (int e = 0; e < NS; e += 2) max_step(e);
      }
      if (seen_next) {  // the next scores made ready, as far as they are not
        const bool all = all_see(tn);
        if constexpr (POLY) {
          const bool small = all && __all(most < p.cap.few);
          if (small) mx = p.cap(mx);
          else mx = finish_scores(tn, all, s_next);
          c0 = small ? p.cap.c0 : 1.f;
          c1 = small ? p.cap.c1 : 0.f;
          c2 = small ? p.cap.c2 : 0.f;
          c3 = small ? p.cap.c3 : 0.f;
        } else if (CAP || !all) {
          mx = finish_scores(tn, all, s_next);
        }
      }
    }
    if (!seen_next) mx = -INFINITY;
    __builtin_amdgcn_s_waitcnt(0);  // this wavefront's tile loads have landed
    __syncthreads();
    settle_max(mx);
    less_far_max(s_next);
    seen = seen_next;
    // (with biases, scores may lie so far below that all of a tile's probabilities are zero in 32 bits: nothing to add)
    live = seen_next && (BIAS == 0 || __any(!((mx - m_run) * c < -150.f)));
  };

  if (n_tiles > 0) {
    load_k(0, 0);
    load_v(0, 0);
    if (n_tiles > 1) load_k(1, 1);
#pragma unroll
    for (int ks = 0; ks < QL; ++ks) q_lds[ks * NW * 64 + tid] = __builtin_bit_cast(u32x4_v, qf[ks]);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    f32x16_v sa[KH], sb[KH];
    {
      const int t0 = tile_at(0) * BN;
      seen = some_see(t0);
      first_values(t0, sa);
#pragma unroll
      for (int i = 0; i < KH * KS; ++i) sa[i % KH] = M::run(__builtin_bit_cast(frag, k_at(lds, i)), q_at(i / KH), sa[i % KH]);
      settle_max(finish_scores(t0, all_see(t0), sa));
      less_far_max(sa);
      live = seen;
    }
    __syncthreads();  // (the loop's first load goes where the first keys were)
    for (int i = 0; i < n_tiles; i += 2) {
      tile(i, 0, sa, sb);
      if (i + 1 < n_tiles) tile(i + 1, 1, sb, sa);
    }
  }

  // ---- epilogue ----
  {
    // (what follows from the lane anew: the loop has no registers to hold it)
    const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), l32 = lane & 31, hh = lane >> 5;
    const int row = min(q0 + l32, p.Sq - 1);
    auto swapped = [&](float x) __attribute__((always_inline)) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      return __uint_as_float(hh ? r[0] : r[1]);
    };
    float l_tot = l_run + swapped(l_run);
    if constexpr (KH == 1) {  // the upper halves' sums join the lower ones' (behind the loop's last barrier nothing is read from the tiles)
      f32x4_v* const jo = reinterpret_cast<f32x4_v*>(lds) + (wave & 1) * (DT * 4 * 64);
      float2* const jm = reinterpret_cast<float2*>(lds + 2 * DT * 4 * 64 * 16) + (wave & 1) * 64;
      static_assert(2 * (DT * 4 * 64 * 16 + 64 * 8) <= 4 * TILEB, "the join fits the tiles' memory");
      if (wave >= 2) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g) jo[(dt * 4 + g) * 64 + lane] = f32x4_v{o[dt][g * 4], o[dt][g * 4 + 1], o[dt][g * 4 + 2], o[dt][g * 4 + 3]};
        jm[lane] = make_float2(m_run, l_tot);
      }
      __syncthreads();
      if (wave >= 2) return;
      const float2 other = jm[lane];
      const float m = fmaxf(m_run, other.x), m_safe = m == -INFINITY ? 0.f : m;
      const float a = __builtin_amdgcn_exp2f((m_run - m_safe) * c), b = __builtin_amdgcn_exp2f((other.x - m_safe) * c);
      m_run = m;
      // (a side that saw nothing has a sum of zero, but what it multiplied by zero may be NaN)
      l_tot = (l_tot == 0.f ? 0.f : l_tot * a) + (other.y == 0.f ? 0.f : other.y * b);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4_v x = jo[(dt * 4 + g) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[dt][g * 4 + e] = o[dt][g * 4 + e] * a + x[e] * b;
        }
    }
    const bool mine = q0 + l32 < p.Sq;
    const int64_t part = (static_cast<int64_t>(unit) * p.n_qblocks + qb) * p.chunks + chunk;
    float* const po = p.ws + part * BM * D;
    float* const pml = p.ws + static_cast<int64_t>(p.units) * p.n_qblocks * p.chunks * BM * D + part * BM * 2;
    T* const orow = static_cast<T*>(p.o) + b * p.os_b + h * p.os_h;
    // stores the rows of the lanes that have one; returns the largest value in size, NaN once anything is
    auto store = [&](bool mine) __attribute__((always_inline)) {
      float probe = 0.f;
      if (p.chunks > 1) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4_v x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = l_tot == 0.f ? 0.f : o[dt][g * 4 + e];
              if (e & 1) probe = __builtin_elementwise_maximum(__builtin_elementwise_maximum(probe, fabsf(x[e - 1])), fabsf(x[e]));
            }
            if (mine) *reinterpret_cast<f32x4_v*>(po + (q0 - qb * BM + l32) * D + dt * 32 + g * 8 + hh * 4) = x;
          }
        if (mine && hh == 0) *reinterpret_cast<float2*>(pml + (q0 - qb * BM + l32) * 2) = make_float2(m_run, l_tot);
      } else {
        const float inv = 1.f / l_tot;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[e] = l_tot == 0.f ? 0.f : o[dt][g * 4 + e] * inv;
              if (e & 1) probe = __builtin_elementwise_maximum(__builtin_elementwise_maximum(probe, fabsf(x[e - 1])), fabsf(x[e]));
            }
            auto pair = [&](int e) __attribute__((always_inline)) {
              return __builtin_amdgcn_permlane32_swap(M::pack2(x[e], x[e + 1]), M::pack2(x[e + 4], x[e + 5]), false, false);
            };
            const auto lo = pair(0), hi = pair(2);
            u32x4_v w;
            w.x = lo[0]; w.y = hi[0]; w.z = lo[1]; w.w = hi[1];
            if (mine) *reinterpret_cast<u32x4_v*>(orow + row * p.os_s + dt * 32 + g * 8 + hh * 8) = w;
          }
      }
      return probe;
    };
    const float probe = store(mine);
    // rows with finite sums, but values that are not. (l_tot == 0: nothing was seen, zeros are right)
    uint64_t bad = __ballot(mine && l_tot > 0.f && l_tot < INFINITY && !(probe < INFINITY));
    bad = (bad | (bad >> 32)) & 0xffffffffull;
    if (__builtin_expect(bad == 0, 1)) return;
    const int4 its = ranges[wave * 32 + l32];
    const auto see_some = [&](int k0, int n) { return __any((k0 < its.y && k0 + n > its.x) || (k0 < its.w && k0 + n > its.z)) != 0; };
    const auto see_all = [&](int k0, int n) { return __all((k0 >= its.x && k0 + n <= its.y) || (k0 >= its.z && k0 + n <= its.w)) != 0; };
    // Whether a value that is not finite lies in what was multiplied by a zero for some row: in keys of one product that not all rows see. Elsewhere
    // such values are seen, and the rows are right as they are.
    bool spoiled = false;
    for (int i = 0; i < n_tiles && !spoiled; ++i)
      for (int k0 = tile_at(i) * BN, n = 0; n < BN && !spoiled; n += WN, k0 += WN) {
        if (!see_some(k0, WN) || see_all(k0, WN)) continue;
        bool found = false;
        for (int r = lane / CPR; r < WN; r += RPI) {
          const u32x4 x = load_raw(vbase + min(k0 + r, p.Sk - 1) * p.vs_s + lane % CPR * 8);
#pragma unroll
          for (int e = 0; e < 4; ++e) found |= not_finite<T>(x[e]) || not_finite<T>(x[e] >> 16);
        }
        spoiled = __any(found) != 0;
      }
    if (!spoiled) return;
    // The rows of the wavefront once more, 32 keys at a time, straight from memory. A product takes the values that are finite, zeros for the others; where there
    // are others, a second product counts for each feature and row those that the row sees, by kind (1, 64 and 4096 each, of 16 keys: its sum
    // says how many of which), and they are added as what they are. us, 4096 causal tokens, 16 heads of 128 on 4: all finite 91, one infinite value at the
    // head, which all rows see, 115, one NaN in the middle 250, a feature that is infinite at every key 846 (row by row, any of them took 20000).
    l_run = 0.f;
    m_run = -INFINITY;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    const int at = BIAS != 0 ? places[wave * 32 + l32] : 0;
    const T* const qp = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h + row * p.qs_s + hh * 8;
    for (int i = 0; i < 2 * n_tiles; ++i) {
      const int t0 = tile_at(i >> 1) * BN, k0 = t0 + (i & 1) * 32;
      if (!see_some(k0, 32)) continue;
      f32x16_v x;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
      const T* const kp = kbase + min(k0 + l32, p.Sk - 1) * p.ks_s + hh * 8;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {  // (the queries from memory too: their registers are needed here)
        x = M::run(__builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(kp + ks * 16)), __builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(qp + ks * 16)), x);
      }
      const uint32_t sees = static_cast<uint32_t>((range_bits(its.x, its.y, t0) | range_bits(its.z, its.w, t0)) >> (32 * (i & 1))) >> (4 * hh);
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int away = k0 + key_of(e) + 4 * hh - at;
        float bias = 0.f;
        if constexpr (BIAS == 1) bias = -slope * fabsf(static_cast<float>(away));
        if constexpr (BIAS == 2) bias = table[clampi(away, -p.radius, p.radius) + p.radius + kPad];
        x[e] = (sees >> key_of(e)) & 1 ? (CAP ? p.cap.of_any(x[e]) : x[e]) + bias : -INFINITY;
        mx = fmaxf(mx, x[e]);
      }
      const float m_new = fmaxf(m_run, fmaxf(mx, swapped(mx))), m_safe = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_safe) * c);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = fabsf(o[dt][e]) < INFINITY ? o[dt][e] * alpha : o[dt][e];
      u32x4_v weights[2], ones[2];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f((x[e] - m_safe) * c), p1 = __builtin_amdgcn_exp2f((x[e + 1] - m_safe) * c);
        l_run += p0 + p1;
        weights[e >> 3][(e & 7) >> 1] = M::pack2(p0, p1);
        ones[e >> 3][(e & 7) >> 1] = M::pack2((sees >> key_of(e)) & 1 ? 1.f : 0.f, (sees >> key_of(e + 1)) & 1 ? 1.f : 0.f);
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          uint32_t v[8];
          bool others = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = min(k0 + g * 16 + (j >> 2) * 8 + 4 * hh + (j & 3), p.Sk - 1);
            v[j] = *reinterpret_cast<const uint16_t*>(vbase + key * p.vs_s + dt * 32 + l32);
            others |= not_finite<T>(v[j]);
          }
          u32x4_v clean;
#pragma unroll
          for (int j = 0; j < 8; j += 2) clean[j >> 1] = (not_finite<T>(v[j]) ? 0u : v[j]) | (not_finite<T>(v[j + 1]) ? 0u : v[j + 1] << 16);
          o[dt] = M::run(__builtin_bit_cast(frag, clean), __builtin_bit_cast(frag, weights[g]), o[dt]);
          if (!__any(others)) continue;
          const auto kind = [](uint32_t u) { return !not_finite<T>(u) ? 0.f : is_nan<T>(u) ? 4096.f : (u & 0x8000u) ? 64.f : 1.f; };
          u32x4_v kinds;
          f32x16_v found;
#pragma unroll
          for (int j = 0; j < 8; j += 2) kinds[j >> 1] = M::pack2(kind(v[j]), kind(v[j + 1]));
#pragma unroll
          for (int e = 0; e < 16; ++e) found[e] = 0.f;
          found = M::run(__builtin_bit_cast(frag, kinds), __builtin_bit_cast(frag, ones[g]), found);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int n = static_cast<int>(found[e]);
            if (n >= 4096) o[dt][e] = NAN;
            if (n & 63) o[dt][e] += INFINITY;
            if (n & 4032) o[dt][e] -= INFINITY;
          }
        }
    }
    l_tot = l_run + swapped(l_run);
    store(mine && ((bad >> l32) & 1) != 0);
  }
}

// Joins the chunks' sums, a wavefront for each row: o = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c, m = max_c m_c. Lane c has chunk c's
// maximum and sum; the features' loads go out eight at a time.
constexpr int kMaxChunks = 32;
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_ruled_merge_kernel(const RuledParams p) {
  constexpr int EPL = D / 64;
  static_assert(kMaxChunks <= 64, "a lane for each chunk");
  const int lane = threadIdx.x & 63;
  const int64_t gr = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (gr >= static_cast<int64_t>(p.units) * p.Sq) return;
  const int unit = static_cast<int>(gr / p.Sq), row = static_cast<int>(gr - static_cast<int64_t>(unit) * p.Sq);
  const int64_t first = (static_cast<int64_t>(unit) * p.n_qblocks + row / p.bm) * p.chunks;
  const float* const ml = p.ws + static_cast<int64_t>(p.units) * p.n_qblocks * p.chunks * p.bm * D;
  const float* const po = p.ws + (first * p.bm + row % p.bm) * D + lane * EPL;
  const int mine = lane < p.chunks ? lane : 0;
  const float2 own = *reinterpret_cast<const float2*>(ml + ((first + mine) * p.bm + row % p.bm) * 2);
  const float mc = lane < p.chunks ? own.x : -INFINITY;
  float m = mc;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
  const float w = __builtin_amdgcn_exp2f((mc - (m == -INFINITY ? 0.f : m)) * p.unit), l = wave_sum(lane < p.chunks ? w * own.y : 0.f);
  float acc[EPL] = {};
  for (int c0 = 0; c0 < p.chunks; c0 += 8) {
    float x[8][EPL];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < EPL; ++e) x[i][e] = c0 + i < p.chunks ? po[static_cast<int64_t>(c0 + i) * p.bm * D + e] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), (c0 + i) & 63));
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[e] = fmaf(wi, x[i][e], acc[e]);
    }
  }
  T* const op = static_cast<T*>(p.o) + unit / p.H * p.os_b + unit % p.H * p.os_h + row * p.os_s + lane * EPL;
#pragma unroll
  for (int e = 0; e < EPL; ++e) op[e] = from_float<T>(l == 0.f ? 0.f : acc[e] / l);
}

// How a call is cut.
// Two wavefronts share 32 queries (KH = 1) where query blocks of 128 would leave compute units without any, or, under a causal order, are so
// few that the longest of them decide: a tile then takes a wavefront alone on its SIMD 0.83 us, 1.1 otherwise, and there are twice as many
// blocks, but each of them reads all its keys. us, KH = 2 / 1, blocks of 128 in brackets, of 128 features if not said otherwise:
//   causal      S=512 H=8 [32] 14.5 / 12.3    S=512 H=32 of 64 [128] 11.8 / 9.9    S=1024 H=24 [192] 25.0 / 22.0    S=2048 H=32 of 64 [512] 37.6 / 31.3
//               S=4096 H=16 [512] 93.5 / 85.9    S=8192 H=8 [512] 176 / 159    S=3000 H=24 [576] 75.3 / 79.0    S=4096 H=24 of 64 [768] 75.9 / 79.3
//   all keys    S=512 H=8 [32] 14.0 / 12.1    S=512 H=32 of 64 [128] 11.6 / 9.9    S=1024 H=24 [192] 25.4 / 25.8    B=3 S=300 H=24 [216] 11.7 / 12.9
//               S=2048 H=32 [512] 72 / 86    S=1024 H=64 of 64 [512] 27.5 / 29.6
//   documents   (ragged, whose workgroups end at different times) S=1024 H=24 [192] 25.1 / 22.9, causal 23.0 / 20.0    S=1024 H=64 [512] 32.7 / 43.5
//               of 64 features: S=1024 H=64 [512] with a table 28.1 / 27.3, causal 20.7 / 18.8    8 in S=2048 H=32 causal [512] 25.0 / 20.4
//               S=1500 H=64 causal [768] 29.5 / 26.6    10 in S=4000 H=48 causal [1536] 46.0 / 47.6    23 in S=12007 H=32 causal [3008] 100 / 107
// Where a call still has fewer workgroups than the GPU has room for, its tiles are cut into chunks, as many as cost least: the join is a launch
// of 3 us and its sums' way to memory and back, 8 bytes a feature.
// With slopes, a launch that reads all keys once gives the bound that far tiles are left out by (behind a cap too, which bounds scores by itself but does
// not say whether keys are numbers). us, without / with it, causal, slopes from 2^(-8/H) to 2^-8, and the same with a cap of 30: 2048 tokens, 24 heads of
// 128, 46.7 / 51.3, 53.4 / 57.0; 4096, 24, 116 / 116, 139 / 139; 4096, 16 of 64, 64.4 / 67.3, 81.5 / 84.2; 6144, 32 on 8 of 128, 260 / 217, 348 / 271;
// 8192, 32 on 8, 436 / 339, 579 / 427; 16384, 16, 796 / 571, 1064 / 735. In a window, which leaves far tiles out by itself: 8192, 32 on 8, windows of 512,
// 1024, 2048 and 4096, 103 / 111, 150 / 149, 230 / 209, 352 / 285; 16384, 16, windows of 2048 and 4096, 260 / 275, 414 / 358; 8192 of 64 features, 16, both ways,
// 2048 and 4096, 162 / 167, 259 / 222.
struct RuledPlan { int halves, chunks; bool norms; };
static RuledPlan ruled_plan(int B, int Sq, int Sk, int H, int D, const odit_attn_rules& r) {
  const int docs = r.docs, window = r.window, causal = r.causal;
  const auto blocks = [&](int bm) { return static_cast<int64_t>((Sq + bm - 1) / bm) * H * B; };
  const int64_t few = docs > 0 ? (D == 128 ? 256 : 768) : causal ? 512 : 128;
  // (slopes, and every query has a key at its own place)
  RuledPlan plan{blocks(128) <= few ? 1 : 2, 1, r.slopes != nullptr && docs == 0 && Sk >= Sq && Sq >= 1024 && Sk >= 6144 && (window == 0 || window >= Sk / 4)};
  const int64_t mine = blocks(64 * plan.halves), room = D == 128 ? 512 : 768;  // (1024 at halves of 64 features: 500 rows of 3000 keys 31.1 us, so 29.7)
  int64_t keys = docs > 0 ? 2 * (Sk / docs) + 64 : Sk;  // that a query block may see, about
  if (window > 0) {
    const int64_t most = (causal ? 1ll : 2ll) * window + 128;
    keys = most < keys ? most : keys;
  }
  const double tiles = static_cast<double>(keys) / 64, each = plan.halves == 1 ? 0.83 : 1.1, join = static_cast<double>(B) * H * Sq * D * 8 / 4e6;
  double cost = each * tiles;
  for (int n = 2; n <= kMaxChunks && n * mine <= room && n <= tiles; ++n) {
    const double t = each * tiles / n + 3.0 + n * join;
    if (t < cost) { cost = t; plan.chunks = n; }
  }
  return plan;
}

static size_t ruled_norms_bytes(const RuledPlan& plan, int B, int H) {  // (as if each head had keys of its own)
  return plan.norms ? static_cast<size_t>(B) * H * kNormParts * sizeof(float) : 0;
}
static size_t ruled_workspace_bytes(const RuledPlan& plan, int B, int Sq, int H, int D) {
  const int bm = 64 * plan.halves;
  return ruled_norms_bytes(plan, B, H) + (plan.chunks > 1 ? static_cast<size_t>((Sq + bm - 1) / bm) * H * B * plan.chunks * bm * (D + 2) * sizeof(float) : 0);
}

template <typename T, int D, int KH>
static int launch_ruled(RuledParams& p, bool cap, int bias, hipStream_t stream) {
  p.bm = 64 * KH;
  p.n_qblocks = (p.Sq + p.bm - 1) / p.bm;
  p.units = p.H * p.B;
  p.group = p.H / p.Hkv;
  const int64_t total = static_cast<int64_t>(p.n_qblocks) * p.H * p.B * p.chunks;
  ODIT_CHECK_ARG(total < (1ll << 24), "odit_attn_ruled: grid of %lld workgroups is too large", static_cast<long long>(total));
  p.by_blocks = quotient(p.n_qblocks * p.units);
  p.by_units = quotient(bias != 1 && p.units % kNumXcd == 0 ? p.units / kNumXcd : p.units);
  p.by_heads = quotient(p.H);
  p.by_group = quotient(p.group);
  const size_t lds = bias == 2 ? (2 * p.radius + 1 + 2 * kTablePad) * sizeof(float) : 0;
  if (p.norms != nullptr) {
    const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv * kNormParts;
    ODIT_CHECK_ARG(heads < (1ll << 24), "odit_attn_ruled: grid of %lld workgroups is too large", static_cast<long long>(heads));
    hipLaunchKernelGGL((attn_ruled_norms_kernel<T, D>), dim3(heads), dim3(256), 0, stream, p, const_cast<float*>(p.norms));
  }
#define ODIT_RULED_GO(C, X) hipLaunchKernelGGL((attn_ruled_kernel<T, D, C, X, KH>), dim3(total), dim3(256), lds, stream, p)
  if (cap) {
    if (bias == 0) ODIT_RULED_GO(true, 0); else if (bias == 1) ODIT_RULED_GO(true, 1); else ODIT_RULED_GO(true, 2);
  } else {
    if (bias == 0) ODIT_RULED_GO(false, 0); else if (bias == 1) ODIT_RULED_GO(false, 1); else ODIT_RULED_GO(false, 2);
  }
#undef ODIT_RULED_GO
  if (p.chunks > 1) {
    const int64_t rows = static_cast<int64_t>(p.units) * p.Sq;
    hipLaunchKernelGGL((attn_ruled_merge_kernel<T, D>), dim3((rows + 3) / 4), dim3(256), 0, stream, p);
  }
  return check_launch("odit_attn_ruled");
}
template <typename T, int D>
static int launch_ruled(RuledParams& p, const RuledPlan& plan, bool cap, int bias, hipStream_t stream) {
  return plan.halves == 1 ? launch_ruled<T, D, 1>(p, cap, bias, stream) : launch_ruled<T, D, 2>(p, cap, bias, stream);
}

}  // namespace odit

extern "C" size_t odit_attn_ruled_workspace_bytes(int B, int Sq, int Sk, int H, int D, const odit_attn_rules* rules) {
  using namespace odit;
  if (B <= 0 || Sq <= 0 || Sk <= 0 || H <= 0 || D <= 0 || rules == nullptr) return 0;
  return ruled_workspace_bytes(ruled_plan(B, Sq, Sk, H, D, *rules), B, Sq, H, D);
}

extern "C" int odit_attn_ruled(const void* q, const void* k, const void* v, void* o, int B, int Sq, int Sk, int H, int Hkv, int D,
                               const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                               const int64_t o_strides[3], float scale, const odit_attn_rules* rules, int dtype, void* workspace,
                               size_t workspace_bytes, void* stream) {
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
  ODIT_CHECK_ARG(scale >= kMinScale && scale <= kMaxScale, "odit_attn_ruled: softmax scale %g outside [%g, %g]", scale, kMinScale, kMaxScale);
  ODIT_CHECK_ARG(r.window >= 0 && r.window <= kMost, "odit_attn_ruled: window=%d outside [0, %d]", r.window, kMost);
  ODIT_CHECK_ARG(r.docs >= 0 && (r.docs == 0 || (r.q_starts && r.k_starts)), "odit_attn_ruled: documents need q_starts and k_starts");
  ODIT_CHECK_ARG(r.cap == 0.f || (r.cap >= kMinScale && r.cap <= kMaxCap), "odit_attn_ruled: cap=%g is neither 0 nor in [%g, %g]", r.cap, kMinScale, kMaxCap);
  ODIT_CHECK_ARG(r.slopes == nullptr || r.distance == nullptr, "odit_attn_ruled: slopes and a table exclude each other");
  ODIT_CHECK_ARG(r.distance == nullptr || (r.radius >= 0 && r.radius <= kMaxRadius), "odit_attn_ruled: radius=%d outside [0, %d]", r.radius,
                 kMaxRadius);
  ODIT_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o), "odit_attn_ruled: q/k/v/o must be 16-byte aligned");
  ODIT_CHECK_ARG(aligned16(workspace), "odit_attn_ruled: the workspace must be 16-byte aligned");
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
  p.bias_scale = 1.f / scale;
  p.unit = r.cap > 0.f ? 1.f : p.scale_log2;
  // (without scratch, or with less than that takes, a query block's tiles stay in one piece and all are visited)
  RuledPlan plan = ruled_plan(B, Sq, Sk, H, D, r);
  if (workspace == nullptr || workspace_bytes < ruled_workspace_bytes(plan, B, Sq, H, D)) {
    plan.chunks = 1;
    plan.norms = false;
  }
  p.chunks = plan.chunks;
  p.norms = plan.norms ? static_cast<float*>(workspace) : nullptr;
  p.ws = static_cast<float*>(workspace) + ruled_norms_bytes(plan, B, H) / sizeof(float);
  p.cap = make_cap(r.cap, scale);
  const int bias = r.slopes != nullptr ? 1 : r.distance != nullptr ? 2 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODIT_BF16) return D == 128 ? launch_ruled<bf16_t, 128>(p, plan, r.cap > 0.f, bias, st) : launch_ruled<bf16_t, 64>(p, plan, r.cap > 0.f, bias, st);
  return D == 128 ? launch_ruled<f16_t, 128>(p, plan, r.cap > 0.f, bias, st) : launch_ruled<f16_t, 64>(p, plan, r.cap > 0.f, bias, st);
}

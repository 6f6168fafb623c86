// Attention of one new token per sequence over a paged cache of keys and values.
//
//   o_h = sum_j p_j v_j / sum_j p_j,  p_j = exp2(x_j - m),  x_j in attn_rules.h; j over the last `window` of the sequence's `length` keys,
//   the query being the last of them. Key j lies in row j % page of cache page table[j / page].
//
// Bound by memory: the keys and values are read once, for all query heads of their group together. The group's heads (up to 16; more take
// another workgroup) are the columns of 16 x 16 products, S^T = K Q^T and O^T = V^T P^T, so that the arithmetic costs the
// same for one head as for 16 and stays far below the loads. A lane then owns one head and the same keys in both products: P stays in registers.
//
// The sequences' keys are cut into chunks, a workgroup each; a chunk's tiles of 16 keys go round its 4 wavefronts. A wavefront has two stages
// of LDS of its own and fills one, 16 bytes a lane straight from global memory, while it computes the other: no barrier in the loop. The page
// numbers of the chunk wait in LDS, so nothing else is loaded there but, of a table of biases, those of keys within its radius: the wait for them
// is one for the tile on its way too (32 sequences, 24 heads of 64, window of 1024: 36.4 us without a table, 37.7 with a radius of 128, 44.5 with
// 1024). (Tiles of 32 keys leave room for one workgroup of head size 128 on a compute unit, and nothing runs while it begins and ends: 8 sequences
// of 4096 keys 37 to 51 us, so 31.) The wavefronts' sums are joined in LDS, the chunks' by the last workgroup of a sequence to be done, or by a
// second launch.
//
// Rows behind a sequence's last key are never read, as a page may hold anything there: the tile's rest is the last key again, with no
// weight and values of zero.
#include <type_traits>

#include "attn_rules.h"
#include "quotient.h"

namespace odit {

typedef short s16x4_p __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4_p __attribute__((ext_vector_type(4)));
template <typename T> struct Mma16;
template <> struct Mma16<bf16_t> {
  using frag = bf16x8_v;
  static __device__ __forceinline__ f32x4_v run(frag a, frag b, f32x4_v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4_v half(s16x4_p a, s16x4_p b, f32x4_v c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
};
template <> struct Mma16<f16_t> {
  using frag = f16x8_v;
  static __device__ __forceinline__ f32x4_v run(frag a, frag b, f32x4_v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4_v half(s16x4_p a, s16x4_p b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_p, a), __builtin_bit_cast(f16x4_p, b), c, 0, 0, 0);
  }
};

typedef __attribute__((address_space(3))) s16x4_p* lds_s16x4_pp;
typedef __attribute__((address_space(3))) void* lds_void_pp;

struct PagedParams {
  const void *q, *k, *v;
  void* o;
  const int *table, *lengths;
  const float *slopes, *distance;
  int B, H, Hkv, pages, page, max_pages, window, radius;
  Quotient by_page;
  int64_t qs_b, qs_h, kc_p, kc_r, kc_h, vc_p, vc_r, vc_h, ts, os_b, os_h;
  float scale_log2;
  float unit;  // from what scores are kept in to units of log2: scale log2(e), or 1 where a cap or a bias has made them that
  Cap cap;
  int group, head_blocks, units;  // units: key heads' blocks of up to 16 query heads, of one sequence
  int wanted, room;               // chunks of all sequences, about, and the most keys of one
  bool whole;                     // no sequence has more than one
  float* ws;  // per chunk and unit: [heads of a block][D] sums, then [heads of a block] (maximum in units of scores, sum)
  unsigned* tickets;  // a word for each sequence and unit, zero between launches (nullptr: the join is a launch of its own)
};

constexpr int kPagedWaves = 4, kPagedTile = 16, kPagedEntries = 1024, kPagedStep = kPagedWaves * kPagedTile;
constexpr int kPagedLeast = 2;  // steps of a chunk: with one, a sequence of 1000 keys takes 9.7 us, with two 8.4
constexpr int kPagedWhole = 256;  // keys up to which a sequence is one chunk: the join takes as long as twice 128 keys
constexpr int kPagedWanted = 512;  // workgroups: two to a compute unit at head size 128 (us, 448 / 512 / 640 / 768: 4 sequences of 100000 to 131072 keys
                                   // 345 / 335 / 366 / 362, 8 of 4096 33 / 31 / 35 / 36, one of 32768 37 / 36 / 41 / 41; head size 64 the same)
constexpr int kPagedJoin = 12;  // chunks whose parts are loaded at once (at head size 64 16 wavefronts share a compute unit's registers)
// keys of a sequence of this length that its query sees: [first, end)
__device__ __forceinline__ void paged_range(const PagedParams& p, int length, int* first, int* end) {
  const int64_t most = static_cast<int64_t>(p.max_pages) * p.page;
  int n = p.pages > 0 ? length : 0;
  if (n > most) n = static_cast<int>(most);
  if (n < 0) n = 0;
  *end = n;
  *first = p.window > 0 && n > p.window ? n - p.window : 0;
}

// the wavefront's sum in every lane, and the sum of the lanes up to this one
__device__ __forceinline__ int wave_sum_int(int v) {
  const auto moved = [](int x, auto ctrl) { return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xf, 0xf, false); };
  v += moved(v, std::integral_constant<int, 0xB1>());
  v += moved(v, std::integral_constant<int, 0x4E>());
  v += moved(v, std::integral_constant<int, 0x141>());
  v += moved(v, std::integral_constant<int, 0x140>());
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48);
}
__device__ __forceinline__ int wave_scan_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr by 1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast of lane 15 to the second and fourth 16, of lane 31 to the upper half
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// How the sequences are cut, from their lengths, which the host does not know: into chunks of one size, whole steps of the workgroup, about
// `wanted` in all (what runs at once), and no more than that where the sequences are few, as one chunk more would then have the others' time
// again. Cut by the longest that the table has room for instead, into 2048: 8 sequences of 4096 keys 38 us where this takes 31, 48 of 17 to
// 8192 67 and 62; and what is short in a wide table would run on few compute units.
// Workgroups [0, B) have the sequences' first chunks, those behind them the further ones, sequence by sequence: where many sequences are
// short, next to nobody has to count what lies ahead (numbered sequence by sequence: 4096 sequences of 16 to 64 keys 1500 us, so 300; 1000 of
// 16 to 300 keys 190 and 136). Every wavefront works it out by itself.
struct PagedPlace { int b, part, parts, before, chunk, length; };  // before: chunks of the sequences ahead
// keys that sequence b's query sees
__device__ __forceinline__ int paged_keys(const PagedParams& p, int b, int* length) {
  *length = b < p.B ? p.lengths[b] : 0;
  int first, end;
  paged_range(p, *length, &first, &end);
  return end - first;
}
// a sequence's chunks past the first
__device__ __forceinline__ int paged_more(int keys, int chunk) {
  return keys <= kPagedWhole ? 0 : static_cast<int>(static_cast<uint32_t>(keys - 1) / static_cast<uint32_t>(chunk));
}
// The place of chunk `index` among 64 sequences from b0 on, whose keys and lengths the lanes hold; *before: chunks past the first of the
// sequences ahead of them. True if it is there; otherwise *before includes these 64.
__device__ __forceinline__ bool paged_among(const PagedParams& p, int index, int b0, int keys, int length, int* before, PagedPlace* at) {
  const int more = paged_more(keys, at->chunk), upto = wave_scan_int(more);  // of this sequence and those ahead of it among the 64
  const int past = index - p.B;  // (below 0: a first chunk, of sequence `index`)
  const int l = __popcll(__ballot(past < 0 ? b0 + static_cast<int>(threadIdx.x & 63) < index : *before + upto <= past));
  if (l == 64) {
    *before += __builtin_amdgcn_readlane(upto, 63);
    return false;
  }
  const int own = __builtin_amdgcn_readlane(more, l), ahead = *before + __builtin_amdgcn_readlane(upto, l) - own;
  at->b = b0 + l;
  at->before = at->b + ahead;
  at->parts = 1 + own;
  at->part = past < 0 ? 0 : 1 + past - ahead;
  at->length = __builtin_amdgcn_readlane(length, l);
  return true;
}
__device__ __forceinline__ PagedPlace paged_place(const PagedParams& p, int index) {
  const int lane = threadIdx.x & 63;
  PagedPlace at{p.B, 0, 1, 0, 0, 0};  // (b == B: behind the last chunk)
  int length, before = 0;
  const int mine = paged_keys(p, lane, &length);
  if (p.B <= 64) {
    // (in steps, so that the sum of 64 stays in 32 bits)
    const int steps = wave_sum_int((mine + kPagedStep - 1) / kPagedStep);
    int each = max(kPagedLeast, (steps + p.wanted - 1) / p.wanted);
    if (4 * p.B <= p.wanted) {
      for (int i = 0; i < 3; ++i) {
        const int made = p.B + wave_sum_int(paged_more(mine, each * kPagedStep));
        if (made <= p.wanted) break;
        each = static_cast<int>(static_cast<int64_t>(each) * made / p.wanted) + 1;
      }
    }
    at.chunk = min(each, p.room / kPagedStep) * kPagedStep;
    paged_among(p, index, 0, mine, length, &before, &at);
    return at;
  }
  int other;
  if (p.whole) {
    at.b = index;
    at.length = p.lengths[index];
    return at;
  }
  int64_t sum = mine;
  for (int b0 = 64; b0 < p.B; b0 += 512) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += paged_keys(p, b0 + i * 64 + lane, &other);
  }
  double total = static_cast<double>(sum);  // (exact: below 2^53)
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) total += __shfl_xor(total, s, 64);
  const double each = ceil(total / (static_cast<double>(p.wanted) * kPagedStep));
  at.chunk = static_cast<int>(each < kPagedLeast ? kPagedLeast : each > p.room / kPagedStep ? p.room / kPagedStep : each) * kPagedStep;
  at.chunk = max(__builtin_amdgcn_readfirstlane(at.chunk), kPagedStep);
  if (index < p.B && paged_more(paged_keys(p, index, &other), at.chunk) == 0) {
    at.b = index;
    at.length = other;
    return at;
  }
  for (int b0 = 0; b0 < p.B; b0 += 512) {  // 512 sequences at once where the place is none of theirs
    int more = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) more += paged_more(paged_keys(p, b0 + i * 64 + lane, &other), at.chunk);
    const int all = wave_sum_int(more);
    if (index < p.B ? b0 + 512 <= index : before + all <= index - p.B) {
      before += all;
      continue;
    }
    for (int i = 0; i < 512; i += 64) {
      const int keys = paged_keys(p, b0 + i + lane, &length);
      if (paged_among(p, index, b0 + i, keys, length, &before, &at)) return at;
    }
  }
  return at;
}

// 16 bytes per lane from the lane's own address to LDS bytes lds + 16 * lane
__device__ __forceinline__ void load_lds16_at(uint32_t lds, const void* from) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(from) : "memory", "m0");
#pragma clang diagnostic pop
#endif
}

// pairs of floats that workgroups of one launch hand to each other: past the caches of their XCD, both ways
__device__ __forceinline__ void put_pair(float* at, float x0, float x1) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(at), static_cast<unsigned long long>(__float_as_uint(x1)) << 32 | __float_as_uint(x0),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_pair(const float* at) {
  const unsigned long long x = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float(static_cast<uint32_t>(x)), __uint_as_float(static_cast<uint32_t>(x >> 32)));
}

// A sequence's chunks joined, features d and d + 1 of head hd: o = sum_c a_c o_c / sum_c a_c l_c with a_c = 2^((m_c - m) unit), m = max_c m_c, in the chunks'
// order. kPagedJoin chunks' loads are on their way at once. part0: the first chunk's part, `step` floats ahead of the next one's.
template <typename T, int D>
__device__ __forceinline__ uint32_t join_parts(const float* part0, int64_t step, int most, int hd, int d, int parts, float unit) {
  float m = -INFINITY, l = 0.f, x0 = 0.f, x1 = 0.f;
  const uint32_t at_ml = most * D + 2 * hd, at_x = hd * D + d;
  for (int c0 = 0; c0 < parts; c0 += kPagedJoin) {
    float2 ml[kPagedJoin], x[kPagedJoin];
#pragma unroll
    for (int c = 0; c < kPagedJoin; ++c) {
      if (c0 + c < parts) {
        const float* const part = part0 + (c0 + c) * step;
        ml[c] = get_pair(part + at_ml);
        x[c] = get_pair(part + at_x);
      }
    }
    float m_new = m;
#pragma unroll
    for (int c = 0; c < kPagedJoin; ++c)
      if (c0 + c < parts) m_new = fmaxf(m_new, ml[c].x);
    const float m_safe = m_new == -INFINITY ? 0.f : m_new, a0 = __builtin_amdgcn_exp2f((m - m_safe) * unit);
    m = m_new;
    l *= a0; x0 *= a0; x1 *= a0;
#pragma unroll
    for (int c = 0; c < kPagedJoin; ++c) {
      if (c0 + c < parts) {
        const float a = __builtin_amdgcn_exp2f((ml[c].x - m_safe) * unit);
        l = fmaf(a, ml[c].y, l);
        x0 = fmaf(a, x[c].x, x0);
        x1 = fmaf(a, x[c].y, x1);
      }
    }
  }
  return l == 0.f ? 0u : Mma<T>::pack2(x0 / l, x1 / l);
}

template <typename T, int D, bool CAP, int BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 2))) void attn_paged_kernel(const PagedParams p) {
  using M = Mma16<T>;
  using frag = typename M::frag;
  constexpr int NW = kPagedWaves, BN = kPagedTile;
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPI = 64 / CPR, TILEB = BN * ROWB, IPT = BN / RPI;
  constexpr int KS = D / 32, DT = D / 16;
  static_assert(BN == 16, "a tile is one product's rows");
  __shared__ __attribute__((aligned(1024))) char lds[NW * 4 * TILEB];  // of each wavefront: K0 V0 K1 V1
  __shared__ int entries[kPagedEntries];
  __shared__ int outside[NW];  // whether a wavefront found page numbers that are none of the cache's

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int unit = blockIdx.x % p.units;
  const PagedPlace at = paged_place(p, blockIdx.x / p.units);
  if (at.b >= p.B) return;
  const int hb = unit % p.head_blocks, hkv = unit / p.head_blocks, b = at.b;
  const int h0 = hkv * p.group + hb * 16, heads = min(16, p.group - hb * 16);
  const int h = h0 + min(l16, heads - 1);  // this lane's head
  const auto page_of = [&](int key) { return p.by_page(key); };

  int first, n;
  paged_range(p, at.length, &first, &n);
  const int parts = at.parts, begin = first + at.part * at.chunk, end = parts == 1 ? n : min(n, begin + at.chunk), pg0 = page_of(begin);
  bool bad = false;
  if (end > begin) {
    const int npg = page_of(end - 1) - pg0 + 1;
    for (int i = tid; i < npg; i += NW * 64) {
      int e = p.table[b * p.ts + pg0 + i];
      if (e < 0 || e >= p.pages) { e = -1; bad = true; }
      entries[i] = e;
    }
  }
  const T* const qrow = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h;
  frag qf[KS];
#pragma unroll
  for (int st = 0; st < KS; ++st) qf[st] = __builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(qrow + g * 8 + st * 32));
  const float slope = BIAS == 1 ? in_units(p.slopes[h], kLog2e) : 0.f;
  const float* const dist = BIAS == 2 ? p.distance + static_cast<int64_t>(h) * (2 * p.radius + 1) + p.radius : nullptr;  // [away]
  const float far = BIAS == 2 ? in_units(dist[-p.radius], kLog2e) : 0.f;
  {
    const bool any = __any(bad);
    if (lane == 0) outside[wave] = any;
  }
  __syncthreads();
  const bool invalid = (outside[0] | outside[1] | outside[2] | outside[3]) != 0;

  const int tiles = (max(end - begin, 0) + BN - 1) / BN, mine = tiles > wave ? (tiles - wave + NW - 1) / NW : 0;
  const T* const kbase = static_cast<const T*>(p.k) + hkv * p.kc_h;
  const T* const vbase = static_cast<const T*>(p.v) + hkv * p.vc_h;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_pp)lds)) + wave * 4 * TILEB;
  char* const own = lds + wave * 4 * TILEB;
  // Lane l of the load's instruction j fills the 16 bytes of row RPI j + l / CPR at chunk l % CPR; which chunk of the key or value that
  // is, is swizzled by the row, so that the reads below touch all banks: K rows of a fragment by row (row / 2 at head size 64, where two
  // rows share the banks), V rows of a transposed read by pairs of chunks.
  auto load_tile = [&](int i) {
    const int k0 = begin + (wave + i * NW) * BN;
    const uint32_t to = lds0 + (i & 1) * 2 * TILEB;
#pragma unroll
    for (int j = 0; j < IPT; ++j) {
      const int r = RPI * j + lane / CPR, pc = lane % CPR;
      const int fk = D == 128 ? r % 16 : (r / 2) % 8, fv = D == 128 ? 2 * (r % 8) : 2 * (r / 2 % 4);
      const int key = min(k0 + r, end - 1);
      const int pg = page_of(key), e = entries[pg - pg0], at = key - pg * p.page;
      // (a key whose page is none of the cache's has no weight; some memory has to stand in for it)
      const T* const kr = e >= 0 ? kbase + e * p.kc_p + at * p.kc_r : qrow;
      const T* const vr = e >= 0 ? vbase + e * p.vc_p + at * p.vc_r : qrow;
      load_lds16_at(to + j * 1024, kr + ((pc ^ fk) % CPR) * 8);
      load_lds16_at(to + TILEB + j * 1024, vr + ((pc ^ fv) % CPR) * 8);
    }
  };

  f32x4_v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4_v{0.f, 0.f, 0.f, 0.f};
  constexpr bool MADE = CAP || BIAS != 0;
  const float c = MADE ? 1.f : p.scale_log2;
  float m_run = -INFINITY, l_run = 0.f, m_off = 0.f;  // m_off: m_run, or 0 while there is none
  const int k_lane = l16 * ROWB + (((g ^ (D == 128 ? l16 : l16 / 2)) % CPR) << 4);
  const int vkey = 4 * g + (l16 >> 2), vf = D == 128 ? 2 * (vkey % 8) : 2 * (vkey / 2 % 4);
  const int v_lane = vkey * ROWB + ((((l16 & 3) >> 1) ^ vf) << 4) + ((l16 & 1) << 3);

  const auto counts = [&](int key) { return key < end && (!invalid || entries[page_of(key) - pg0] >= 0); };

  // what was loaded above is here: a wait for it inside the loop would also be one for the tiles on their way
  __builtin_amdgcn_s_waitcnt(0);
#pragma unroll
  for (int st = 0; st < KS; ++st) asm volatile("" : "+v"(qf[st]));
  if (mine > 0) load_tile(0);
  for (int i = 0; i < mine; ++i) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage that is filled next has been read
    if (i + 1 < mine) {
      load_tile(i + 1);
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * IPT) : "memory");  // all but the loads of the tile just asked for
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const char* const kb = own + (i & 1) * 2 * TILEB;
    const char* const vb = kb + TILEB;
    const int k0 = begin + (wave + i * NW) * BN;
    const bool rest = k0 + BN > end || invalid;
    f32x4_v s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < KS; ++st) s = M::run(__builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(kb + (k_lane ^ (st * 64)))), qf[st], s);
    if (rest) {  // what stands in for keys that are none: values of zero, whatever the memory holds (0 times infinity is NaN)
#pragma unroll
      for (int j = 0; j < IPT; ++j) {
        const int key = k0 + RPI * j + lane / CPR;
        if (!counts(key)) *reinterpret_cast<u32x4_v*>(own + ((i & 1) * 2 + 1) * TILEB + j * 1024 + lane * 16) = u32x4_v{0, 0, 0, 0};
      }
      asm volatile("" ::: "memory");
    }
    const bool near = BIAS == 2 && k0 + BN - 1 - (n - 1) > -p.radius;  // some key has a bias of its own
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = k0 + g * 4 + e;
      float x = s[e];
      if constexpr (MADE) x = CAP ? p.cap.of_any(x) : x * p.scale_log2;
      if constexpr (BIAS == 1) x = fmaf(-slope, static_cast<float>(n - 1 - key), x);
      if constexpr (BIAS == 2) {
        if (near) x += in_units(dist[max(min(key, n - 1) - (n - 1), -p.radius)], kLog2e);
        else x += far;
      }
      if (rest) x = counts(key) ? x : -INFINITY;
      s[e] = x;
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 4; ++e) mx = __builtin_elementwise_maximum(mx, s[e]);
    if (__any((mx - m_run) * c > 8.f)) {  // (as in attn_fwd.hip: the maximum moves only where it is left behind by a factor of 2^8)
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m_run, mx), m_safe = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_safe) * c);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][e] *= alpha;
      m_run = m_new;
      m_off = m_safe;
    }
    u32x2_v pb;  // (differences first: with the maximum times c, rounded, in one fma, an exponent of zero comes out above 128 for scores past 2^31)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f((s[e] - m_off) * c), p1 = __builtin_amdgcn_exp2f((s[e + 1] - m_off) * c);
      l_run += p0 + p1;
      pb[e / 2] = Mma<T>::pack2(p0, p1);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const s16x4_p v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_pp)(vb + (v_lane ^ (dt * 32))));
      o[dt] = M::half(v, __builtin_bit_cast(s16x4_p, pb), o[dt]);
    }
  }

  // ---- the wavefronts' sums joined: [wave][head][D + 4] sums and [wave][head] (maximum in units of scores, sum) ----
  constexpr int OP = D + 4;
  float* const jo = reinterpret_cast<float*>(lds);
  float2* const jm = reinterpret_cast<float2*>(lds + NW * 16 * OP * 4);
  static_assert(NW * 16 * (OP * 4 + 8) <= static_cast<int>(sizeof(lds)), "the join fits the tiles' memory");
  float l_tot = l_run + __shfl_xor(l_run, 16, 64);
  l_tot += __shfl_xor(l_tot, 32, 64);
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_v*>(jo + (wave * 16 + l16) * OP + dt * 16 + g * 4) = o[dt];
  if (g == 0) jm[wave * 16 + l16] = make_float2(m_run, l_tot);
  __syncthreads();
  // what the call's chunks leave is written past the caches of this XCD, as another workgroup's may read it
  const int most = min(16, p.group);
  const int64_t step = static_cast<int64_t>(p.units) * most * (D + 2);
  float* const part0 = p.ws + at.before * step + static_cast<int64_t>(unit) * most * (D + 2);
  for (int i = tid; i < heads * (D / 2); i += NW * 64) {
    const int hd = i / (D / 2), d = i % (D / 2) * 2;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, jm[w * 16 + hd].x);
    const float m_safe = m == -INFINITY ? 0.f : m;
    float l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = __builtin_amdgcn_exp2f((jm[w * 16 + hd].x - m_safe) * c);
      l = fmaf(a, jm[w * 16 + hd].y, l);
      x0 = fmaf(a, jo[(w * 16 + hd) * OP + d], x0);
      x1 = fmaf(a, jo[(w * 16 + hd) * OP + d + 1], x1);
    }
    if (parts == 1) {
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.os_b + (h0 + hd) * p.os_h + d) = l == 0.f ? 0u : Mma<T>::pack2(x0 / l, x1 / l);
    } else {
      float* const part = part0 + at.part * step;
      put_pair(part + hd * D + d, x0, x1);
      if (d == 0) put_pair(part + most * D + 2 * hd, m, l);
    }
  }
  if (parts == 1 || p.tickets == nullptr) return;
  // The last of the sequence's workgroups to be done joins them, in their order, and puts the word back to zero.
  __shared__ int is_last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's part is where the others see it
  __syncthreads();
  if (tid == 0) {
    const unsigned before = __hip_atomic_fetch_add(p.tickets + b * p.units + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = before == static_cast<unsigned>(parts - 1);
    if (is_last) __hip_atomic_store(p.tickets + b * p.units + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;
  for (int i = tid; i < heads * (D / 2); i += NW * 64) {
    const int hd = i / (D / 2), d = i % (D / 2) * 2;
    *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.os_b + (h0 + hd) * p.os_h + d) = join_parts<T, D>(part0, step, most, hd, d, parts, p.unit);
  }
}

// the join as a launch of its own: a wavefront (or its first half) for each sequence and head
template <typename T, int D>
__global__ __launch_bounds__(64) void attn_paged_join_kernel(const PagedParams p) {
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, d = threadIdx.x * 2;
  const PagedPlace at = paged_place(p, b);
  if (at.parts <= 1 || d >= D) return;  // (one chunk's workgroup has written the result)
  const int most = min(16, p.group), unit = h / p.group * p.head_blocks + h % p.group / 16, hd = h % p.group % 16;
  const int64_t step = static_cast<int64_t>(p.units) * most * (D + 2);
  *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.os_b + h * p.os_h + d) =
      join_parts<T, D>(p.ws + at.before * step + static_cast<int64_t>(unit) * most * (D + 2), step, most, hd, d, at.parts, p.unit);
}

// The most chunks that any lengths can make, and what the kernels work them out from. Where a chunk's page numbers have to fit kPagedEntries
// it may have to be smaller than wanted.
struct PagedPlan { int wanted, room; int64_t chunks; };
static PagedPlan paged_plan(int B, int units, int64_t most_keys, int page) {
  PagedPlan plan;
  plan.wanted = kPagedWanted / units < 1 ? 1 : kPagedWanted / units;
  int64_t room = static_cast<int64_t>(kPagedEntries - 1) * page / kPagedStep * kPagedStep;  // (a chunk may begin inside a page)
  if (room > 1 << 29) room = 1 << 29;
  plan.room = static_cast<int>(room < kPagedStep ? kPagedStep : room);
  // (each sequence's last chunk may be a part of one)
  const int64_t by_room = (B * most_keys + plan.room - 1) / plan.room;
  plan.chunks = B + (most_keys <= kPagedWhole ? 0 : by_room > plan.wanted ? by_room : plan.wanted);
  return plan;
}

static int64_t paged_most_keys(int64_t max_pages, int page, int window) {
  const int64_t most = max_pages * page;
  return window > 0 && window < most ? window : most;
}

template <typename T, int D>
static int launch_paged(const PagedParams& p, int64_t chunks, bool cap, int bias, hipStream_t stream) {
  const int64_t grid = p.units * chunks;
  ODIT_CHECK_ARG(grid < (1ll << 24), "odit_attn_paged: grid of %lld workgroups is too large", static_cast<long long>(grid));
#define ODIT_PAGED_GO(C, X) hipLaunchKernelGGL((attn_paged_kernel<T, D, C, X>), dim3(grid), dim3(256), 0, stream, p)
  if (cap) {
    if (bias == 0) ODIT_PAGED_GO(true, 0); else if (bias == 1) ODIT_PAGED_GO(true, 1); else ODIT_PAGED_GO(true, 2);
  } else {
    if (bias == 0) ODIT_PAGED_GO(false, 0); else if (bias == 1) ODIT_PAGED_GO(false, 1); else ODIT_PAGED_GO(false, 2);
  }
#undef ODIT_PAGED_GO
  if (chunks > p.B && p.tickets == nullptr) hipLaunchKernelGGL((attn_paged_join_kernel<T, D>), dim3(p.B * p.H), dim3(64), 0, stream, p);
  return check_launch("odit_attn_paged");
}

static int paged_head_blocks(int H, int Hkv) { return (H / Hkv + 15) / 16; }

}  // namespace odit

extern "C" size_t odit_attn_paged_workspace_bytes(int B, int H, int Hkv, int D, int max_pages, int page_size, int window) {
  using namespace odit;
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0 || max_pages <= 0 || page_size <= 0) return 0;
  const int units = Hkv * paged_head_blocks(H, Hkv), heads = H / Hkv < 16 ? H / Hkv : 16;
  const PagedPlan plan = paged_plan(B, units, paged_most_keys(max_pages, page_size, window), page_size);
  return plan.chunks > B ? static_cast<size_t>(plan.chunks) * units * heads * (D + 2) * sizeof(float) : 0;
}

extern "C" int odit_attn_paged(const void* q, const void* key_cache, const void* value_cache, const int* table, const int* lengths, void* o,
                               int B, int H, int Hkv, int D, int pages, int page_size, int max_pages, const int64_t q_strides[2],
                               const int64_t key_cache_strides[3], const int64_t value_cache_strides[3], int64_t table_stride,
                               const int64_t o_strides[2], float scale, const odit_attn_rules* rules, int dtype, void* workspace,
                               size_t workspace_bytes, unsigned* tickets, size_t n_tickets, void* stream) {
  using namespace odit;
  ODIT_CHECK_ARG(rules != nullptr, "odit_attn_paged: null rules");
  const odit_attn_rules& r = *rules;
  if (dtype != ODIT_BF16 && dtype != ODIT_F16) {
    set_error("odit_attn_paged: dtype code %d unsupported (bf16 and fp16 only)", dtype);
    return ODIT_ENOTSUP;
  }
  if (D != 64 && D != 128) {
    set_error("odit_attn_paged: head size %d unsupported (64 and 128 only)", D);
    return ODIT_ENOTSUP;
  }
  constexpr int kMost = 1 << 30;
  ODIT_CHECK_ARG(q_strides && key_cache_strides && value_cache_strides && o_strides, "odit_attn_paged: null strides");
  ODIT_CHECK_ARG(B >= 0 && H > 0 && Hkv > 0 && pages >= 0 && max_pages >= 0 && page_size > 0, "odit_attn_paged: bad shape");
  ODIT_CHECK_ARG(H % Hkv == 0, "odit_attn_paged: H=%d is not a multiple of Hkv=%d", H, Hkv);
  ODIT_CHECK_ARG(static_cast<int64_t>(B) * H < (1ll << 26), "odit_attn_paged: %d sequences of %d heads are too many", B, H);
  ODIT_CHECK_ARG(static_cast<int64_t>(max_pages) * page_size <= kMost, "odit_attn_paged: %d pages of %d keys are more than %d keys",
                 max_pages, page_size, kMost);
  ODIT_CHECK_ARG(scale >= kMinScale && scale <= kMaxScale, "odit_attn_paged: softmax scale %g outside [%g, %g]", scale, kMinScale, kMaxScale);
  ODIT_CHECK_ARG(r.window >= 0 && r.window <= kMost, "odit_attn_paged: window=%d outside [0, %d]", r.window, kMost);
  ODIT_CHECK_ARG(r.docs == 0 && r.prefix == nullptr, "odit_attn_paged: documents and prefixes are for whole prompts");
  ODIT_CHECK_ARG(r.cap == 0.f || (r.cap >= kMinScale && r.cap <= kMaxCap), "odit_attn_paged: cap=%g is neither 0 nor in [%g, %g]", r.cap, kMinScale, kMaxCap);
  ODIT_CHECK_ARG(r.slopes == nullptr || r.distance == nullptr, "odit_attn_paged: slopes and a table exclude each other");
  ODIT_CHECK_ARG(r.distance == nullptr || (r.radius >= 0 && r.radius <= kMaxRadius), "odit_attn_paged: radius=%d outside [0, %d]", r.radius,
                 kMaxRadius);
  ODIT_CHECK_ARG(aligned16(q) && aligned16(key_cache) && aligned16(value_cache) && aligned16(o), "odit_attn_paged: tensors must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    ODIT_CHECK_ARG(key_cache_strides[i] % 8 == 0 && value_cache_strides[i] % 8 == 0 && (i == 2 || (q_strides[i] % 8 == 0 && o_strides[i] % 8 == 0)),
                   "odit_attn_paged: strides must be multiples of 8 elements");
  if (B == 0) return ODIT_OK;
  ODIT_CHECK_ARG(q && o && lengths && (max_pages == 0 || table) && (pages == 0 || (key_cache && value_cache)),
                 "odit_attn_paged: tensors must not be null");
  const size_t need = odit_attn_paged_workspace_bytes(B, H, Hkv, D, max_pages, page_size, r.window);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
    set_error("odit_attn_paged: workspace of %zu bytes, needs %zu aligned to 16", workspace_bytes, need);
    return ODIT_EWORKSPACE;
  }
  PagedParams p;
  p.q = q; p.k = key_cache; p.v = value_cache; p.o = o; p.table = table; p.lengths = lengths; p.slopes = r.slopes; p.distance = r.distance;
  p.B = B; p.H = H; p.Hkv = Hkv; p.pages = pages; p.page = page_size; p.max_pages = max_pages; p.window = r.window; p.radius = r.radius;
  p.by_page = quotient(page_size);
  p.qs_b = q_strides[0]; p.qs_h = q_strides[1]; p.os_b = o_strides[0]; p.os_h = o_strides[1]; p.ts = table_stride;
  p.kc_p = key_cache_strides[0]; p.kc_r = key_cache_strides[1]; p.kc_h = key_cache_strides[2];
  p.vc_p = value_cache_strides[0]; p.vc_r = value_cache_strides[1]; p.vc_h = value_cache_strides[2];
  p.scale_log2 = scale * kLog2e;
  p.unit = r.cap > 0.f || r.slopes != nullptr || r.distance != nullptr ? 1.f : p.scale_log2;
  p.cap = make_cap(r.cap, scale);
  p.group = H / Hkv; p.head_blocks = paged_head_blocks(H, Hkv);
  p.units = Hkv * p.head_blocks;
  const PagedPlan plan = paged_plan(B, p.units, paged_most_keys(max_pages, page_size, r.window), page_size);
  p.wanted = plan.wanted; p.room = plan.room;
  p.whole = plan.chunks == B;
  p.ws = static_cast<float*>(workspace);
  p.tickets = tickets != nullptr && n_tickets >= static_cast<size_t>(B) * p.units ? tickets : nullptr;
  const int bias = r.slopes != nullptr ? 1 : r.distance != nullptr ? 2 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODIT_BF16) return D == 128 ? launch_paged<bf16_t, 128>(p, plan.chunks, r.cap > 0.f, bias, st) : launch_paged<bf16_t, 64>(p, plan.chunks, r.cap > 0.f, bias, st);
  return D == 128 ? launch_paged<f16_t, 128>(p, plan.chunks, r.cap > 0.f, bias, st) : launch_paged<f16_t, 64>(p, plan.chunks, r.cap > 0.f, bias, st);
}

// Attention of one new token per sequence over a paged cache of keys and values.
//
//   o_h = sum_j p_j v_j / sum_j p_j,  p_j = exp2(x_j - m),  x_j in attn_rules.h; j over the last `window` of the sequence's `length` keys,
//   the query being the last of them. Key j lies in row j % page of cache page table[j / page].
//
// Bound by memory: the keys and values are read once, for all query heads of their group together. The group's heads (up to 16; more take
// another workgroup) are the columns of v_mfma_f32_16x16x32 in both products, S^T = K Q^T and O^T = V^T P^T, so that the arithmetic costs the
// same for one head as for 16 and stays far below the loads. A lane then owns one head and the same keys in both products: P stays in registers.
//
// A sequence's keys are cut into chunks, a workgroup each; a chunk's tiles of 32 keys go round its 4 wavefronts. A wavefront has two stages
// of LDS of its own and fills one, 16 bytes a lane straight from global memory, while it computes the other: no barrier in the loop. The page
// numbers of the chunk wait in LDS, so nothing else is loaded there. The wavefronts' sums are joined in LDS; the chunks' by a second launch.
//
// Rows behind a sequence's last key are never read, as a page may hold anything there: the tile's rest is the last key again, with no
// weight and values of zero.
#include "attn_rules.h"

namespace odit {

template <typename T> struct Mma16;
template <> struct Mma16<bf16_t> {
  using frag = bf16x8_v;
  static __device__ __forceinline__ f32x4_v run(frag a, frag b, f32x4_v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma16<f16_t> {
  using frag = f16x8_v;
  static __device__ __forceinline__ f32x4_v run(frag a, frag b, f32x4_v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

typedef short s16x4_p __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_p* lds_s16x4_pp;
typedef __attribute__((address_space(3))) void* lds_void_pp;

struct PagedParams {
  const void *q, *k, *v;
  void* o;
  const int *table, *lengths;
  const float *slopes, *distance;
  int B, H, Hkv, pages, page, max_pages, window, radius;
  uint32_t page_mul;  // key / page = key * page_mul >> page_shift
  int page_shift;
  int64_t qs_b, qs_h, kc_p, kc_r, kc_h, vc_p, vc_r, vc_h, ts, os_b, os_h;
  float scale_log2;
  Cap cap;
  int group, head_blocks, units, splits, chunk;
  float* ws;  // per unit and split: [heads of a block][D] sums, then [heads of a block] (maximum, sum)
  unsigned* tickets;  // a word for each unit, zero between launches (nullptr: the join is a launch of its own)
};

// The join by the last workgroup costs it a trip to memory behind the others (1 us) where a launch of its own costs 2.6 us and 3 of the
// host's; it holds all chunks' parts at once, so it is for up to kPagedTickets of them.
constexpr int kPagedTickets = 16;
constexpr int kPagedWaves = 4, kPagedTile = 32, kPagedEntries = 1024;
// keys of a sequence of this length that its query sees: [first, end)
__device__ __forceinline__ void paged_range(const PagedParams& p, int length, int* first, int* end) {
  const int64_t most = static_cast<int64_t>(p.max_pages) * p.page;
  int n = p.pages > 0 ? length : 0;
  if (n > most) n = static_cast<int>(most);
  if (n < 0) n = 0;
  *end = n;
  *first = p.window > 0 && n > p.window ? n - p.window : 0;
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

// Up to kPagedTickets chunks' sums joined, features d and d + 1 of head hd: o = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c, m = max_c m_c.
// All loads are ahead of their first use.
template <typename T, int D>
__device__ __forceinline__ uint32_t join_few(const float* part0, int most, int hd, int d, int parts) {
  float2 ml[kPagedTickets], x[kPagedTickets];
#pragma unroll
  for (int c = 0; c < kPagedTickets; ++c) {
    if (c < parts) {
      const float* const part = part0 + c * most * (D + 2);
      ml[c] = get_pair(part + most * D + 2 * hd);
      x[c] = get_pair(part + hd * D + d);
    }
  }
  float m = -INFINITY, l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
  for (int c = 0; c < kPagedTickets; ++c)
    if (c < parts) m = fmaxf(m, ml[c].x);
  const float m_safe = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int c = 0; c < kPagedTickets; ++c) {
    if (c < parts) {
      const float a = __builtin_amdgcn_exp2f(ml[c].x - m_safe);
      l = fmaf(a, ml[c].y, l);
      x0 = fmaf(a, x[c].x, x0);
      x1 = fmaf(a, x[c].y, x1);
    }
  }
  return l == 0.f ? 0u : Mma<T>::pack2(x0 / l, x1 / l);
}

template <typename T, int D, bool CAP, int BIAS>
__global__ __launch_bounds__(256) void attn_paged_kernel(const PagedParams p) {
  using M = Mma16<T>;
  using frag = typename M::frag;
  constexpr int NW = kPagedWaves, BN = kPagedTile;
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPI = 64 / CPR, TILEB = BN * ROWB, IPT = BN / RPI;
  constexpr int KS = D / 32, DT = D / 16;
  __shared__ __attribute__((aligned(1024))) char lds[NW * 4 * TILEB];  // of each wavefront: K0 V0 K1 V1
  __shared__ int entries[kPagedEntries];
  __shared__ int outside[NW];  // whether a wavefront found page numbers that are none of the cache's

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int unit = blockIdx.x % p.units, split = blockIdx.x / p.units;
  const int hb = unit % p.head_blocks, hkv = unit / p.head_blocks % p.Hkv, b = unit / p.head_blocks / p.Hkv;
  const int h0 = hkv * p.group + hb * 16, heads = min(16, p.group - hb * 16);
  const int h = h0 + min(l16, heads - 1);  // this lane's head
  const auto page_of = [&](int key) { return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(key)) * p.page_mul >> p.page_shift); };

  // Without a window a chunk's place does not depend on the sequence's length: its page numbers are on their way while that is (one trip to
  // memory of four in a call of one short sequence)
  const int length = p.lengths[b];
  int first = 0, n = p.max_pages * p.page;  // (up to 2^30)
  if (p.window > 0) paged_range(p, length, &first, &n);
  const int begin = first + split * p.chunk;
  const int pg0 = page_of(begin);
  int bad = 0x7fffffff;  // the first of this thread's page numbers that is none
  if (n > begin) {
    const int npg = page_of(min(n, begin + p.chunk) - 1) - pg0 + 1;
    for (int i = tid; i < npg; i += NW * 64) {
      int e = p.table[b * p.ts + pg0 + i];
      if (e < 0 || e >= p.pages) { e = -1; bad = min(bad, i); }
      entries[i] = e;
    }
  }
  const T* const qrow = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h;
  frag qf[KS];
#pragma unroll
  for (int st = 0; st < KS; ++st) qf[st] = __builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(qrow + g * 8 + st * 32));
  const float slope = BIAS == 1 ? p.slopes[h] * kLog2e : 0.f;
  const float* const dist = BIAS == 2 ? p.distance + static_cast<int64_t>(h) * (2 * p.radius + 1) + p.radius : nullptr;  // [away]
  const float far = BIAS == 2 ? dist[-p.radius] * kLog2e : 0.f;
  if (p.window == 0) paged_range(p, length, &first, &n);
  const int parts = max(1, (n - first + p.chunk - 1) / p.chunk);  // of this sequence; an empty one has one, too
  if (split >= parts) return;
  const int end = min(n, begin + p.chunk);
  {
    const bool any = __any(end > begin && bad <= page_of(end - 1) - pg0);  // (pages behind the sequence's last key may be anything)
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
  float m_run = -INFINITY, l_run = 0.f, mc = 0.f;
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
      if constexpr (IPT == 8) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const char* const kb = own + (i & 1) * 2 * TILEB;
    const char* const vb = kb + TILEB;
    const int k0 = begin + (wave + i * NW) * BN;
    const bool rest = k0 + BN > end || invalid;
    f32x4_v s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int st = 0; st < KS; ++st)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        s[kt] = M::run(__builtin_bit_cast(frag, *reinterpret_cast<const u32x4_v*>(kb + kt * 16 * ROWB + (k_lane ^ (st * 64)))), qf[st], s[kt]);
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
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + kt * 16 + g * 4 + e;
        float x = s[kt][e];
        if constexpr (MADE) x = CAP ? p.cap(x) : x * p.scale_log2;
        if constexpr (BIAS == 1) x = fmaf(-slope, static_cast<float>(n - 1 - key), x);
        if constexpr (BIAS == 2) {
          if (near) x = fmaf(dist[max(min(key, n - 1) - (n - 1), -p.radius)], kLog2e, x);
          else x += far;
        }
        if (rest) {
          x = counts(key) ? x : -INFINITY;
        }
        s[kt][e] = x;
      }
    float mx = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = __builtin_elementwise_maximum(mx, s[kt][e]);
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
      mc = m_safe * c;
    }
    u32x4_v pb;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt][e], c, -mc)), p1 = __builtin_amdgcn_exp2f(fmaf(s[kt][e + 1], c, -mc));
        l_run += p0 + p1;
        pb[kt * 2 + e / 2] = Mma<T>::pack2(p0, p1);
      }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const char* const vp = vb + (v_lane ^ (dt * 32));
      const s16x4_p lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_pp)(vp));
      const s16x4_p hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_pp)(vp + 16 * ROWB));
      o[dt] = M::run(__builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), __builtin_bit_cast(frag, pb), o[dt]);
    }
  }

  // ---- the wavefronts' sums joined: [wave][head][D + 4] sums and [wave][head] (maximum in units of log2, sum) ----
  constexpr int OP = D + 4;
  float* const jo = reinterpret_cast<float*>(lds);
  float2* const jm = reinterpret_cast<float2*>(lds + NW * 16 * OP * 4);
  static_assert(NW * 16 * (OP * 4 + 8) <= static_cast<int>(sizeof(lds)), "the join fits the tiles' memory");
  float l_tot = l_run + __shfl_xor(l_run, 16, 64);
  l_tot += __shfl_xor(l_tot, 32, 64);
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_v*>(jo + (wave * 16 + l16) * OP + dt * 16 + g * 4) = o[dt];
  if (g == 0) jm[wave * 16 + l16] = make_float2(m_run * c, l_tot);
  __syncthreads();
  // what the call's chunks leave is written past the caches of this XCD, as another workgroup's may read it
  const int most = min(16, p.group);
  float* const part0 = p.ws + static_cast<int64_t>(unit) * p.splits * most * (D + 2);
  for (int i = tid; i < heads * (D / 2); i += NW * 64) {
    const int hd = i / (D / 2), d = i % (D / 2) * 2;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, jm[w * 16 + hd].x);
    const float m_safe = m == -INFINITY ? 0.f : m;
    float l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = __builtin_amdgcn_exp2f(jm[w * 16 + hd].x - m_safe);
      l = fmaf(a, jm[w * 16 + hd].y, l);
      x0 = fmaf(a, jo[(w * 16 + hd) * OP + d], x0);
      x1 = fmaf(a, jo[(w * 16 + hd) * OP + d + 1], x1);
    }
    if (parts == 1) {
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.os_b + (h0 + hd) * p.os_h + d) = l == 0.f ? 0u : Mma<T>::pack2(x0 / l, x1 / l);
    } else {
      float* const part = part0 + split * most * (D + 2);
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
    const unsigned before = __hip_atomic_fetch_add(p.tickets + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = before == static_cast<unsigned>(parts - 1);
    if (is_last) __hip_atomic_store(p.tickets + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;
  for (int i = tid; i < heads * (D / 2); i += NW * 64) {
    const int hd = i / (D / 2), d = i % (D / 2) * 2;
    *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.os_b + (h0 + hd) * p.os_h + d) = join_few<T, D>(part0, most, hd, d, parts);
  }
}

// one workgroup a head of a sequence: its wavefronts go round the chunks' sums
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_paged_merge_kernel(const PagedParams p) {
  constexpr int EPL = D / 64;
  __shared__ float jo[4][D], jml[4][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H;
  const int hkv = h / p.group, hb = h % p.group / 16, hd = h % p.group % 16;
  const int64_t unit = (static_cast<int64_t>(b) * p.Hkv + hkv) * p.head_blocks + hb;
  int first, n;
  paged_range(p, p.lengths[b], &first, &n);
  const int parts = (n - first + p.chunk - 1) / p.chunk, most = min(16, p.group);
  if (parts <= 1) return;  // (written by its only workgroup)
  if (parts <= kPagedTickets) {
    const int d = threadIdx.x * 2;
    if (d < D)
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.os_b + h * p.os_h + d) = join_few<T, D>(p.ws + unit * p.splits * most * (D + 2), most, hd, d, parts);
    return;
  }
  float m = -INFINITY, l = 0.f, x[EPL] = {};
  for (int i = wave; i < parts; i += 4) {
    const float* const part = p.ws + (unit * p.splits + i) * most * (D + 2);
    const float pm = part[most * D + 2 * hd], pl = part[most * D + 2 * hd + 1];
    const float m_new = fmaxf(m, pm), m_safe = m_new == -INFINITY ? 0.f : m_new;
    const float a = __builtin_amdgcn_exp2f(m - m_safe), w = __builtin_amdgcn_exp2f(pm - m_safe);
    m = m_new;
    l = fmaf(l, a, w * pl);
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = fmaf(x[e], a, w * part[hd * D + lane * EPL + e]);
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e) jo[wave][lane * EPL + e] = x[e];
  if (lane == 0) { jml[wave][0] = m; jml[wave][1] = l; }
  __syncthreads();
  if (threadIdx.x < D) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, jml[w][0]);
    const float m_safe = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = __builtin_amdgcn_exp2f(jml[w][0] - m_safe);
      ll = fmaf(a, jml[w][1], ll);
      y = fmaf(a, jo[w][threadIdx.x], y);
    }
    static_cast<T*>(p.o)[b * p.os_b + h * p.os_h + threadIdx.x] = from_float<T>(ll == 0.f ? 0.f : y / ll);
  }
}

// How the keys of a call are cut: the host knows the longest that a sequence can be, not how long each is. Chunks are of whole tiles for
// each wavefront, small enough that the call has some workgroups for every compute unit, and their page numbers fit kPagedEntries.
struct PagedPlan { int chunk, splits; };
static PagedPlan paged_plan(int64_t units, int64_t most_keys, int page) {
  constexpr int64_t kStep = kPagedWaves * kPagedTile;
  int64_t chunk = (most_keys * units + 2047) / 2048;
  chunk = (chunk + kStep - 1) / kStep * kStep;
  const int64_t room = static_cast<int64_t>(kPagedEntries - 1) * page / kStep * kStep;  // (a chunk may begin inside a page)
  if (chunk > room) chunk = room;
  if (chunk < kStep) chunk = kStep;
  const int64_t splits = (most_keys + chunk - 1) / chunk;
  return {static_cast<int>(chunk), static_cast<int>(splits < 1 ? 1 : splits)};
}

static int64_t paged_most_keys(int64_t max_pages, int page, int window) {
  const int64_t most = max_pages * page;
  return window > 0 && window < most ? window : most;
}

template <typename T, int D>
static int launch_paged(const PagedParams& p, bool cap, int bias, hipStream_t stream) {
  const int64_t grid = static_cast<int64_t>(p.units) * p.splits;
  ODIT_CHECK_ARG(grid <= 0x7fffffffll, "odit_attn_paged: grid of %lld workgroups is too large", static_cast<long long>(grid));
#define ODIT_PAGED_GO(C, X) hipLaunchKernelGGL((attn_paged_kernel<T, D, C, X>), dim3(grid), dim3(256), 0, stream, p)
  if (cap) {
    if (bias == 0) ODIT_PAGED_GO(true, 0); else if (bias == 1) ODIT_PAGED_GO(true, 1); else ODIT_PAGED_GO(true, 2);
  } else {
    if (bias == 0) ODIT_PAGED_GO(false, 0); else if (bias == 1) ODIT_PAGED_GO(false, 1); else ODIT_PAGED_GO(false, 2);
  }
#undef ODIT_PAGED_GO
  if (p.splits > 1 && p.tickets == nullptr) hipLaunchKernelGGL((attn_paged_merge_kernel<T, D>), dim3(p.B * p.H), dim3(256), 0, stream, p);
  return check_launch("odit_attn_paged");
}

static int paged_head_blocks(int H, int Hkv) { return (H / Hkv + 15) / 16; }

}  // namespace odit

extern "C" size_t odit_attn_paged_workspace_bytes(int B, int H, int Hkv, int D, int max_pages, int page_size, int window) {
  using namespace odit;
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0 || max_pages <= 0 || page_size <= 0) return 0;
  const int64_t units = static_cast<int64_t>(B) * Hkv * paged_head_blocks(H, Hkv);
  const PagedPlan plan = paged_plan(units, paged_most_keys(max_pages, page_size, window), page_size);
  if (plan.splits == 1) return 0;
  const int heads = H / Hkv < 16 ? H / Hkv : 16;
  return static_cast<size_t>(units) * plan.splits * heads * (D + 2) * sizeof(float);
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
  ODIT_CHECK_ARG(static_cast<int64_t>(B) * H <= 0x7fffffffll, "odit_attn_paged: %d sequences of %d heads are too many", B, H);
  ODIT_CHECK_ARG(static_cast<int64_t>(max_pages) * page_size <= kMost, "odit_attn_paged: %d pages of %d keys are more than %d keys",
                 max_pages, page_size, kMost);
  ODIT_CHECK_ARG(scale > 0.f, "odit_attn_paged: softmax scale must be positive (got %g)", scale);
  ODIT_CHECK_ARG(r.window >= 0 && r.window <= kMost, "odit_attn_paged: window=%d outside [0, %d]", r.window, kMost);
  ODIT_CHECK_ARG(r.docs == 0 && r.prefix == nullptr, "odit_attn_paged: documents and prefixes are for whole prompts");
  ODIT_CHECK_ARG(r.cap >= 0.f && r.cap <= kMaxCap, "odit_attn_paged: cap=%g outside [0, %g]", r.cap, kMaxCap);
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
  p.page_shift = 31;  // (rounded up: exact for keys below 2^31)
  while ((1ll << (p.page_shift - 31)) < page_size) ++p.page_shift;
  p.page_mul = static_cast<uint32_t>(((1ull << p.page_shift) + page_size - 1) / page_size);
  p.qs_b = q_strides[0]; p.qs_h = q_strides[1]; p.os_b = o_strides[0]; p.os_h = o_strides[1]; p.ts = table_stride;
  p.kc_p = key_cache_strides[0]; p.kc_r = key_cache_strides[1]; p.kc_h = key_cache_strides[2];
  p.vc_p = value_cache_strides[0]; p.vc_r = value_cache_strides[1]; p.vc_h = value_cache_strides[2];
  p.scale_log2 = scale * kLog2e;
  p.cap = make_cap(r.cap, scale);
  p.group = H / Hkv; p.head_blocks = paged_head_blocks(H, Hkv);
  const int64_t units = static_cast<int64_t>(B) * Hkv * p.head_blocks;
  p.units = static_cast<int>(units);
  const PagedPlan plan = paged_plan(units, paged_most_keys(max_pages, page_size, r.window), page_size);
  p.chunk = plan.chunk; p.splits = plan.splits;
  p.ws = static_cast<float*>(workspace);
  p.tickets = p.splits <= kPagedTickets && tickets != nullptr && n_tickets >= static_cast<size_t>(units) ? tickets : nullptr;
  const int bias = r.slopes != nullptr ? 1 : r.distance != nullptr ? 2 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODIT_BF16) return D == 128 ? launch_paged<bf16_t, 128>(p, r.cap > 0.f, bias, st) : launch_paged<bf16_t, 64>(p, r.cap > 0.f, bias, st);
  return D == 128 ? launch_paged<f16_t, 128>(p, r.cap > 0.f, bias, st) : launch_paged<f16_t, 64>(p, r.cap > 0.f, bias, st);
}

// Exact attention of one new token per sequence over a page pool: o = sum_t softmax(scale q.k_t) v_t over all (or the last
// `window`) tokens of the sequence.
//
// Work is a row of rounds: for every sequence, for every unit of it (a KV head and a tile of its query heads), ROUND keys at a
// time.  The host does not know the lengths, so every CTA adds them up itself and takes its share of the row, as many rounds
// as any other, whatever the lengths are.  A unit that lies in one CTA's share is finished there; the parts of one that does not go
// to scratch (numerators, maximum, denominator) and the merge kernel joins them in order.
#include "common.cuh"

namespace hipattn {
namespace {

constexpr int kSMs = 148;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;

using Params = hipattn_paged_decode_params_t;

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? __ldg((const long long*)p + i) : (int64_t)__ldg((const int*)p + i);
}

// sequence of entry b: its row of the table and the positions [lo, hi) it attends
struct Sequence {
  int64_t row;
  int lo, hi;
};
__device__ __forceinline__ Sequence sequence_of(const Params& p, int b, bool report) {
  Sequence s{0, 0, 0};
  s.row = p.rows ? load_index(p.rows, p.rows_is_i64, b) : b;
  if (s.row < 0 || s.row >= p.n_rows) {
    if (report && s.row >= p.n_rows) atomicOr(p.status, HIPATTN_STATUS_SEQUENCE);
    s.row = 0;
    return s;
  }
  const int64_t n = load_index(p.k.cache_seq_lens, p.k.seq_lens_is_i64, s.row);
  const int64_t most = min((int64_t)p.k.table_width * p.k.page_size, (int64_t)0x7fff0000);
  if (report && n > most) atomicOr(p.status, HIPATTN_STATUS_TOKEN_RANGE);
  s.hi = (int)max((int64_t)0, min(n, most));
  s.lo = p.window > 0 ? max(0, s.hi - p.window) : 0;
  return s;
}
// rounds of a unit; an empty sequence has one, which writes its zeros
__device__ __forceinline__ int rounds_of(const Sequence& s, int round) { return max(1, (s.hi - s.lo + round - 1) / round); }

// Sum of rounds over all sequences (`total`) and over those before sequence b (`before`), for the merge kernel; all threads.
template <int THREADS>
__device__ __forceinline__ void sum_rounds(const Params& p, int b, int round, int64_t* s_sum, int64_t& total, int64_t& before) {
  int64_t t = 0, f = 0;
  for (int i = threadIdx.x; i < p.B; i += THREADS) {
    const int r = rounds_of(sequence_of(p, i, false), round);
    t += r;
    if (i < b) f += r;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    t += __shfl_xor_sync(0xffffffffu, t, o);
    f += __shfl_xor_sync(0xffffffffu, f, o);
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[(threadIdx.x >> 5) * 2] = t;
    s_sum[(threadIdx.x >> 5) * 2 + 1] = f;
  }
  __syncthreads();
  total = before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    total += s_sum[w * 2];
    before += s_sum[w * 2 + 1];
  }
}

__device__ __forceinline__ int64_t share_of(int64_t total, int ctas, int least) {
  const int64_t s = (total + ctas - 1) / ctas;
  return s < least ? least : s;
}

template <int DT>
__device__ __forceinline__ void widen16(const uint4& w, float* out) {
  if constexpr (DT == HIPATTN_F32) {
    out[0] = __uint_as_float(w.x); out[1] = __uint_as_float(w.y); out[2] = __uint_as_float(w.z); out[3] = __uint_as_float(w.w);
  } else {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == HIPATTN_BF16) {
        out[2 * i] = __uint_as_float(v[i] << 16);
        out[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
        out[2 * i] = f.x;
        out[2 * i + 1] = f.y;
      }
    }
  }
}
// sixteen bytes of a cache row as floats
template <int DT, bool F8>
__device__ __forceinline__ void widen_row(const uint4& w, float* out) {
  if constexpr (F8) {
    widen16<HIPATTN_F16>(widen_fp8_e5m2<HIPATTN_F16>(make_uint2(w.x, w.y)), out);
    widen16<HIPATTN_F16>(widen_fp8_e5m2<HIPATTN_F16>(make_uint2(w.z, w.w)), out + 8);
  } else {
    widen16<DT>(w, out);
  }
}

// element e of the output row of head h, from the joined maximum (base 2), numerator and denominator
template <int DT>
__device__ __forceinline__ void finish(const Params& p, int b, int h, int e, float M, float num, float den) {
  // (a denominator of exactly zero: nothing was attended.  NaN and infinite logits stay visible.)
  const bool none = den == 0.f;
  reinterpret_cast<typename Elem<DT>::type*>(p.out)[(int64_t)b * p.o_stride_b + (int64_t)h * p.o_stride_h + e] = Elem<DT>::from_f32(none ? 0.f : num / den);
  if (e == 0 && p.lse_out) p.lse_out[(int64_t)b * p.H + h] = none ? -INFINITY : (M > -INFINITY ? M : 0.f) + log2f(den);
}

// Geometry of the kernel: RB = bytes of a row of DP elements, KEYS = keys a warp takes at once, STAGES = depth of its ring
template <int DT, bool F8, int DP>
struct Geo {
  static constexpr int EB = F8 ? 1 : Elem<DT>::bytes;
  static constexpr int RB = DP * EB;
  static constexpr int VEC = 16 / EB;
  static constexpr int NPC = RB / 16;                         // pieces of a row
  static constexpr int KEYS = 4096 / RB > 32 ? 32 : 4096 / RB;
  static constexpr int LPK = 32 / KEYS;                       // lanes of a key in the logits
  static constexpr int STAGES = 3;
  static constexpr int ROUND = KEYS * kWarps;
  static constexpr int STAGE_BYTES = 2 * KEYS * RB;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES * kWarps;
  static constexpr int PPL = NPC > 32 ? NPC / 32 : 1;         // pieces of a V row that a lane owns
  static constexpr int KP = NPC < 32 ? 32 / NPC : 1;          // V rows that a warp reads at once
};

// Byte offset of piece `pc` of row `key`: the lanes of a quarter warp, LPK to a row, reach eight different bank groups.
template <int RB, int LPK>
__device__ __forceinline__ int place(int key, int pc) {
  return key * RB + ((pc ^ ((key * LPK) & 7 & (RB / 16 - 1))) << 4);
}

// GT: query heads of a unit.  One warp: KEYS keys at a time from a ring of its own, its own running maximum, sum and output.
template <int DT, bool F8, int DP, int GT>
__global__ void __launch_bounds__(kThreads, 1) paged_decode_kernel(const Params p, int tiles, int split, int least) {
  using G = Geo<DT, F8, DP>;
  using T = typename Elem<DT>::type;
  constexpr int KEYS = G::KEYS, NPC = G::NPC, LPK = G::LPK, VEC = G::VEC, MS = DP + 2;
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* ring = smem + (threadIdx.x >> 5) * (G::STAGES * G::STAGE_BYTES);
  float* s_merge = reinterpret_cast<float*>(smem);                   // [kWarps][GT][MS], over the rings when they are empty
  float* s_q = reinterpret_cast<float*>(smem + G::RING_BYTES);       // [GT][DP]
  __shared__ int64_t s_scan[kWarps];
  __shared__ int64_t s_found[2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = p.H / p.HKV, units = p.HKV * tiles;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // (the merge waits for the whole of this grid)

  // ---- this CTA's share of the rounds ----
  int b = 0;
  int64_t first = 0, last = 0, unit_at = 0;     // [first, last): what is left of the share; where sequence b begins in the row
  if (split) {
    int64_t total = 0, base = 0;
    for (int pass = 0; pass < 2; ++pass) {
      // pass 0: the total; pass 1: the sequence that the share begins in.  (One sequence per thread: the second pass reads
      // nothing again.)
      const int64_t share = pass ? share_of(total * units, gridDim.x, least) : 0;
      first = share * blockIdx.x;
      if (pass && first >= total * units) return;
      base = 0;
      for (int c = 0; c < p.B; c += kThreads) {
        const int i = c + tid;
        int64_t x = i < p.B ? rounds_of(sequence_of(p, i, false), G::ROUND) : 0, sum = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        if (lane == 31) s_scan[warp] = sum;
        __syncthreads();
        int64_t all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) sum += s_scan[w];
          all += s_scan[w];
        }
        if (pass) {
          const int64_t end = (base + sum) * units;
          if (first < end && first >= end - x * units) {
            s_found[0] = i;
            s_found[1] = end - x * units;
          }
        }
        base += all;
        __syncthreads();
      }
      total = base;
      if (pass) last = min(first + share, total * units);
    }
    b = (int)s_found[0];
    unit_at = s_found[1];
  } else {
    b = blockIdx.x / units;
  }
  const int64_t share_first = first;

  const int page_size = p.k.page_size;
  const int page_shift = (page_size & (page_size - 1)) == 0 ? 31 - __clz(page_size) : -1;
  const int npc = p.D * G::EB / 16;         // pieces of a row that exist
  const float cap = p.logit_softcap, scale = p.sm_scale;

  for (;;) {
    const Sequence seq = sequence_of(p, b, tid == 0);
    const int rounds = rounds_of(seq, G::ROUND);
    int u0 = 0, r0 = 0;
    if (split) {
      u0 = (int)((first - unit_at) / rounds);
      r0 = (int)((first - unit_at) % rounds);
    } else {
      u0 = blockIdx.x % units;
    }
    const int r1 = split ? (int)min((int64_t)rounds, r0 + (last - first)) : rounds;
    const int hkv = u0 / tiles, tile = u0 % tiles, h0 = hkv * heads + tile * GT, live_heads = min(GT, heads - tile * GT);

    // ---- the unit's queries ----
    __syncthreads();
    for (int i = tid; i < GT * DP; i += kThreads) {
      const int g = i / DP, e = i % DP;
      float x = 0.f;
      if (g < live_heads && e < p.D) x = Elem<DT>::to_f32(reinterpret_cast<const T*>(p.q)[(int64_t)b * p.q_stride_b + (int64_t)(h0 + g) * p.q_stride_h + e]);
      s_q[i] = x;
    }
    __syncthreads();

    float m_run[GT], l_run[GT], acc[GT][G::PPL][VEC];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      m_run[g] = -INFINITY;
      l_run[g] = 0.f;
#pragma unroll
      for (int i = 0; i < G::PPL; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[g][i][e] = 0.f;
    }
    const char* kb = (const char*)p.k.cache + (int64_t)hkv * p.k.stride_ch * G::EB;
    const char* vb = (const char*)p.v.cache + (int64_t)hkv * p.v.stride_ch * G::EB;

    // positions of round r: seq.lo + r * ROUND + warp * KEYS ..; lane `key` resolves a key's page one round ahead
    int64_t page = 0;
    auto fetch_page = [&](int r) {
      const int t = seq.lo + r * G::ROUND + warp * KEYS + lane;
      page = 0;
      if (r < r1 && lane < KEYS && t < seq.hi)
        page = load_index(p.k.block_table, p.k.table_is_i64, seq.row * p.k.table_stride_b + (page_shift >= 0 ? t >> page_shift : t / page_size));
    };
    auto copy = [&](int r, int slot) {
      const int t0 = seq.lo + r * G::ROUND + warp * KEYS;
      if (page < 0 || page >= p.k.n_pages) {
        atomicOr(p.status, HIPATTN_STATUS_PAGE_RANGE);
        page = 0;
      }
      const int t = t0 + lane, off = page_shift >= 0 ? t & (page_size - 1) : t % page_size;
      const uint32_t ks = (uint32_t)__cvta_generic_to_shared(ring + slot * G::STAGE_BYTES), vs = ks + KEYS * G::RB;
#pragma unroll
      for (int i = 0; i < KEYS * NPC / 32; ++i) {
        const int idx = i * 32 + lane, key = idx / NPC, pc = idx % NPC;
        const int pg = __shfl_sync(0xffffffffu, (int)page, key), of = __shfl_sync(0xffffffffu, off, key);
        const bool live = r < r1 && t0 + key < seq.hi && pc < npc;
        const int64_t ko = live ? ((int64_t)pg * p.k.stride_page + (int64_t)of * p.k.stride_off) * G::EB + pc * 16 : 0;
        const int64_t vo = live ? ((int64_t)pg * p.v.stride_page + (int64_t)of * p.v.stride_off) * G::EB + pc * 16 : 0;
        cp_async16_zfill(ks + place<G::RB, LPK>(key, pc), kb + ko, live);
        cp_async16_zfill(vs + place<G::RB, LPK>(key, pc), vb + vo, live);
      }
    };
    fetch_page(r0);
#pragma unroll
    for (int i = 0; i < G::STAGES - 1; ++i) {
      copy(r0 + i, i);
      cp_async_commit();
      fetch_page(r0 + i + 1);
    }
    int slot = 0;
    for (int r = r0; r < r1; ++r) {
      cp_async_wait<G::STAGES - 2>();
      __syncwarp();
      const unsigned char* ks = ring + slot * G::STAGE_BYTES;
      const unsigned char* vs = ks + KEYS * G::RB;
      // ---- logits: LPK lanes to a key ----
      const int key = lane / LPK, sub = lane % LPK;
      float s[GT];
#pragma unroll
      for (int g = 0; g < GT; ++g) s[g] = 0.f;
#pragma unroll 4
      for (int j = 0; j < NPC / LPK; ++j) {
        const int pc = j * LPK + sub;
        float kv[VEC];
        widen_row<DT, F8>(*reinterpret_cast<const uint4*>(ks + place<G::RB, LPK>(key, pc)), kv);
#pragma unroll
        for (int g = 0; g < GT; ++g)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[g] = fmaf(s_q[g * DP + pc * VEC + e], kv[e], s[g]);
      }
      const bool in = seq.lo + r * G::ROUND + warp * KEYS + key < seq.hi;
      float pr[GT];
#pragma unroll
      for (int g = 0; g < GT; ++g) {
#pragma unroll
        for (int o = LPK >> 1; o > 0; o >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
        s[g] *= scale;
        if (cap > 0.f) s[g] = tanhf(s[g] / cap) * cap;
        s[g] = in ? s[g] * kLog2e : -INFINITY;
        float mx = s[g];
#pragma unroll
        for (int o = 16; o >= LPK; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m_new = fmaxf(m_run[g], mx), base = m_new > -INFINITY ? m_new : 0.f;
        const float alpha = exp2f(m_run[g] - base);
        pr[g] = exp2f(s[g] - base);
        l_run[g] = l_run[g] * alpha + (sub == 0 ? pr[g] : 0.f);
        m_run[g] = m_new;
#pragma unroll
        for (int i = 0; i < G::PPL; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[g][i][e] *= alpha;
      }
      // ---- o += p V: a lane owns pieces of the row ----
#pragma unroll
      for (int k0 = 0; k0 < KEYS; k0 += G::KP) {
        const int k = k0 + (G::KP > 1 ? lane / NPC : 0);
#pragma unroll
        for (int i = 0; i < G::PPL; ++i) {
          float vv[VEC];
          widen_row<DT, F8>(*reinterpret_cast<const uint4*>(vs + place<G::RB, LPK>(k, lane % NPC + i * 32)), vv);
#pragma unroll
          for (int g = 0; g < GT; ++g) {
            const float x = __shfl_sync(0xffffffffu, pr[g], k * LPK);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[g][i][e] = fmaf(x, vv[e], acc[g][i][e]);
          }
        }
      }
      __syncwarp();
      copy(r + G::STAGES - 1, slot == 0 ? G::STAGES - 1 : slot - 1);
      cp_async_commit();
      fetch_page(r + G::STAGES);
      slot = slot + 1 == G::STAGES ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- join the warps ----
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l_run[g] += __shfl_xor_sync(0xffffffffu, l_run[g], o);
#pragma unroll
      for (int i = 0; i < G::PPL; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#pragma unroll
          for (int o = NPC; o < 32; o <<= 1) acc[g][i][e] += __shfl_xor_sync(0xffffffffu, acc[g][i][e], o);
          if (lane < NPC) s_merge[(warp * GT + g) * MS + (lane % NPC + i * 32) * VEC + e] = acc[g][i][e];
        }
      if (lane == 0) {
        s_merge[(warp * GT + g) * MS + DP] = m_run[g];
        s_merge[(warp * GT + g) * MS + DP + 1] = l_run[g];
      }
    }
    __syncthreads();
    const bool whole = r0 == 0 && r1 == rounds;
    float* part = reinterpret_cast<float*>(p.scratch) + ((int64_t)blockIdx.x * 2 + (first == share_first ? 0 : 1)) * GT * MS;
    for (int i = tid; i < live_heads * p.D; i += kThreads) {
      const int g = i / p.D, e = i % p.D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_merge[(w * GT + g) * MS + DP]);
      const float base = M > -INFINITY ? M : 0.f;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2f(s_merge[(w * GT + g) * MS + DP] - base);
        num += f * s_merge[(w * GT + g) * MS + e];
        den += f * s_merge[(w * GT + g) * MS + DP + 1];
      }
      if (whole) {
        finish<DT>(p, b, h0 + g, e, M, num, den);
      } else {
        part[g * MS + e] = num;
        if (e == 0) {
          part[g * MS + DP] = M;
          part[g * MS + DP + 1] = den;
        }
      }
    }
    if (!split) return;
    first += r1 - r0;
    if (first >= last) return;
    if (first == unit_at + (int64_t)rounds * units) {
      unit_at = first;
      ++b;
    }
  }
}

// Joins the parts of a unit that lies in several shares, in their order.  One CTA per sequence and unit.
template <int DT, int DP, int GT>
__global__ void __launch_bounds__(128) paged_decode_merge_kernel(const Params p, int tiles, int ctas, int round, int least) {
  constexpr int MS = DP + 2;
  __shared__ int64_t s_sum[8];
  const int heads = p.H / p.HKV, units = p.HKV * tiles;
  const int b = blockIdx.x / units, u = blockIdx.x % units;
  const int rounds = rounds_of(sequence_of(p, b, false), round);
  int64_t total, before;
  sum_rounds<128>(p, b, round, s_sum, total, before);
  const int64_t share = share_of(total * units, ctas, least), begin = before * units + (int64_t)u * rounds;
  const int c0 = (int)(begin / share), c1 = (int)((begin + rounds - 1) / share);
  asm volatile("griddepcontrol.wait;\n" ::: "memory");   // (every CTA: what follows on the stream waits for this grid alone)
  if (c0 == c1) return;
  const int tile = u % tiles, h0 = u / tiles * heads + tile * GT, live_heads = min(GT, heads - tile * GT);
  const int first_slot = begin == c0 * share ? 0 : 1;
  const float* parts = reinterpret_cast<const float*>(p.scratch);
  for (int i = threadIdx.x; i < live_heads * p.D; i += 128) {
    const int g = i / p.D, e = i % p.D;
    float M = -INFINITY, num = 0.f, den = 0.f;
    for (int c = c0; c <= c1; ++c) M = fmaxf(M, parts[(((int64_t)c * 2 + (c == c0 ? first_slot : 0)) * GT + g) * MS + DP]);
    const float base = M > -INFINITY ? M : 0.f;
    for (int c = c0; c <= c1; ++c) {
      const float* part = parts + (((int64_t)c * 2 + (c == c0 ? first_slot : 0)) * GT + g) * MS;
      const float f = exp2f(part[DP] - base);
      num += f * part[e];
      den += f * part[DP + 1];
    }
    finish<DT>(p, b, h0 + g, e, M, num, den);
  }
}

// How a call is laid out: head tiles, CTAs, whether units are cut
struct Layout {
  int gt, tiles, split, least;
  int64_t ctas;
};
constexpr int kLeastRounds = 2;   // rounds of a share

int padded_dim(int D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }

template <int DT, bool F8, int DP>
Layout layout_of(const Params& p) {
  Layout l;
  const int heads = p.H / p.HKV;
  l.gt = heads <= 4 ? 4 : 8;
  l.tiles = cdiv(heads, l.gt);
  const int64_t units = (int64_t)p.B * p.HKV * l.tiles;
  int64_t most = (int64_t)p.k.table_width * p.k.page_size;
  if (p.window > 0 && p.window < most) most = p.window;
  l.least = kLeastRounds;
  l.split = most > (int64_t)l.least * Geo<DT, F8, DP>::ROUND;
  l.ctas = l.split ? kSMs : units;
  return l;
}
template <int DP>
int64_t scratch_bytes(const Layout& l) { return l.split ? l.ctas * 2 * l.gt * (DP + 2) * (int64_t)sizeof(float) : 0; }

template <int DT, bool F8, int DP, int GT>
int launch_gt(const Params& p, const Layout& l, cudaStream_t stream) {
  using G = Geo<DT, F8, DP>;
  constexpr size_t smem = G::RING_BYTES + sizeof(float) * GT * DP;
  static_assert(sizeof(float) * kWarps * GT * (DP + 2) <= G::RING_BYTES, "the join of the warps lies over the rings");
  HIPATTN_REQUIRE(l.ctas < 0x7fffffffLL, HIPATTN_ERR_INVALID, "paged_decode: grid of %lld blocks", (long long)l.ctas);
  auto kern = paged_decode_kernel<DT, F8, DP, GT>;
  HIPATTN_CUDA_OK(allow_smem((const void*)kern, smem));
  kern<<<(unsigned)l.ctas, kThreads, smem, stream>>>(p, l.tiles, l.split, l.least);
  int rc = check_launch("paged_decode_kernel");
  if (rc || !l.split) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.HKV * l.tiles));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  HIPATTN_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<DT, DP, GT>, p, l.tiles, (int)l.ctas, (int)G::ROUND, l.least));
  return check_launch("paged_decode_merge_kernel");
}

// `stream` null with `bytes`: only the scratch of the call
template <int DT, bool F8, int DP>
int launch_dp(const Params& p, cudaStream_t stream, int64_t* bytes) {
  const Layout l = layout_of<DT, F8, DP>(p);
  const int64_t need = scratch_bytes<DP>(l);
  if (bytes) {
    *bytes = need;
    return HIPATTN_OK;
  }
  HIPATTN_REQUIRE(need == 0 || (p.scratch && p.scratch_bytes >= need && (uintptr_t)p.scratch % 16 == 0), HIPATTN_ERR_INVALID,
                  "paged_decode: %lld bytes of scratch are needed (16-byte aligned), %lld were given", (long long)need, (long long)p.scratch_bytes);
  return l.gt == 4 ? launch_gt<DT, F8, DP, 4>(p, l, stream) : launch_gt<DT, F8, DP, 8>(p, l, stream);
}
template <int DT, bool F8>
int launch_type(const Params& p, cudaStream_t stream, int64_t* bytes) {
  switch (padded_dim(p.D)) {
    case 64: return launch_dp<DT, F8, 64>(p, stream, bytes);
    case 128: return launch_dp<DT, F8, 128>(p, stream, bytes);
    default: return launch_dp<DT, F8, 256>(p, stream, bytes);
  }
}
int launch(const Params& p, cudaStream_t stream, int64_t* bytes) {
  if (p.dtype == HIPATTN_F32) return launch_type<HIPATTN_F32, false>(p, stream, bytes);
  if (p.dtype == HIPATTN_BF16) return p.k.fp8_e5m2 ? launch_type<HIPATTN_BF16, true>(p, stream, bytes) : launch_type<HIPATTN_BF16, false>(p, stream, bytes);
  return p.k.fp8_e5m2 ? launch_type<HIPATTN_F16, true>(p, stream, bytes) : launch_type<HIPATTN_F16, false>(p, stream, bytes);
}

int validate(const Params* p) {
  HIPATTN_REQUIRE(p != nullptr, HIPATTN_ERR_INVALID, "paged_decode: params are null");
  HIPATTN_REQUIRE(p->B > 0 && p->H > 0 && p->HKV > 0 && p->H % p->HKV == 0 && p->D > 0 && p->n_rows > 0, HIPATTN_ERR_INVALID,
                  "paged_decode: bad shape B=%d H=%d HKV=%d D=%d rows=%d", p->B, p->H, p->HKV, p->D, p->n_rows);
  HIPATTN_REQUIRE(p->dtype == HIPATTN_F32 || p->dtype == HIPATTN_F16 || p->dtype == HIPATTN_BF16, HIPATTN_ERR_INVALID, "paged_decode: unknown dtype %d", p->dtype);
  HIPATTN_REQUIRE(p->D <= 256, HIPATTN_ERR_UNSUPPORTED, "paged_decode: head dimension %d is larger than 256", p->D);
  HIPATTN_REQUIRE(p->k.cache && p->v.cache, HIPATTN_ERR_INVALID, "paged_decode: k and v must be page pools");
  HIPATTN_REQUIRE(p->k.n_pages == p->v.n_pages && p->k.page_size == p->v.page_size && p->k.fp8_e5m2 == p->v.fp8_e5m2 && p->k.n_pages <= 0x7fffffffLL,
                  HIPATTN_ERR_INVALID, "paged_decode: k and v must be pools of the same pages and type");
  HIPATTN_REQUIRE(p->rows || p->n_rows >= p->B, HIPATTN_ERR_INVALID, "paged_decode: %d entries, but a table of %d rows", p->B, p->n_rows);
  HIPATTN_REQUIRE(p->window >= 0, HIPATTN_ERR_INVALID, "paged_decode: window %d is negative", p->window);
  HIPATTN_REQUIRE(p->logit_softcap >= 0.f && p->sm_scale == p->sm_scale, HIPATTN_ERR_INVALID, "paged_decode: bad scale or soft-cap");
  const int eb = p->dtype == HIPATTN_F32 ? 4 : 2;
  int rc = validate_tokens(p->k, eb, p->D, "k");
  if (rc) return rc;
  rc = validate_tokens(p->v, eb, p->D, "v");
  if (rc) return rc;
  if (p->k.fp8_e5m2) {
    HIPATTN_REQUIRE(p->D % 16 == 0 && p->k.stride_page % 16 == 0 && p->k.stride_off % 16 == 0 && p->k.stride_ch % 16 == 0 &&
                        p->v.stride_page % 16 == 0 && p->v.stride_off % 16 == 0 && p->v.stride_ch % 16 == 0,
                    HIPATTN_ERR_UNSUPPORTED, "paged_decode: fp8 rows must be a multiple of 16 bytes and start on 16-byte boundaries");
  }
  return HIPATTN_OK;
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" int64_t hipattn_paged_decode_scratch(const hipattn_paged_decode_params_t* p) {
  if (validate(p) != HIPATTN_OK) return 0;
  int64_t bytes = 0;
  hipattn::launch(*p, nullptr, &bytes);
  return bytes;
}

extern "C" int hipattn_paged_decode(const hipattn_paged_decode_params_t* p, void* stream) {
  const int rc = validate(p);
  if (rc) return rc;
  HIPATTN_REQUIRE(p->q && p->out && p->status, HIPATTN_ERR_INVALID, "paged_decode: q, out and status are required");
  return hipattn::launch(*p, (cudaStream_t)stream, nullptr);
}

// Exact attention of one new token per sequence over a page pool: o = sum_t softmax(scale q.k_t) v_t over all (or the last
// `window`) tokens of the sequence.  Bound: HBM (every attended K and V row is read once, 4 D flop a head and key).
//
// Work is a row of rounds: for every sequence, for every unit of it (a KV head and a tile of its query heads), ROUND keys at a
// time.  The host does not know the lengths, so every CTA adds them up itself and takes its share of the row, as many rounds
// as any other, whatever the lengths are.  A unit that lies in one CTA's share is finished there; the parts of one that does not go
// to scratch (numerators, the base of their weights, denominator) and the merge kernel joins them in order.
//
// A warp takes KEYS keys at a time from a ring of its own in shared memory, filled with 16-byte asynchronous copies, and keeps
// its own running maximum, sum and output: nothing in the loop waits for another warp.  paged_decode_mma_kernel: 16-bit and fp8
// rows; paged_decode_fma_kernel: fp32.
//
// Measured: one sequence of 1048571 tokens, bf16, 8 KV heads of dimension 128 (4.3 GB) 620 us, 6.9 TB/s; 32 sequences of up to 16384
// tokens (1.18 GB) 180 us, 6.5 TB/s; 12 fp8 sequences in pages of one token, soft-capped (0.56 GB) 109 to 115 us by box, 4.9 to 5.1 TB/s; one
// fp16 sequence of 389 tokens, 16 heads over 4 of dimension 64, 5.1 to 5.4 us.
#include <cfloat>
#include <type_traits>

#include "in_turn.cuh"
#include "mma_common.cuh"

namespace hipattn {
namespace {

constexpr int kSMs = 148;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;

using Params = hipattn_paged_decode_params_t;

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? __ldcg((const long long*)p + i) : (int64_t)__ldcg((const int*)p + i);
}

// sequence of entry b: its row of the table and the positions [lo, hi) it attends
struct Sequence {
  int64_t row;
  bool there;     // the row is in the table (else it is read as row 0, and empty)
  int lo, hi;
};
__device__ __forceinline__ Sequence row_of(const Params& p, int b, bool report) {
  Sequence s{0, true, 0, 0};
  s.row = p.rows ? load_index(p.rows, p.rows_is_i64, b) : b;
  if (s.row < 0 || s.row >= p.n_rows) {
    if (report && s.row >= p.n_rows) atomicOr(p.status, HIPATTN_STATUS_SEQUENCE);
    s.row = 0;
    s.there = false;
  }
  return s;
}
__device__ __forceinline__ void read_length(const Params& p, Sequence& s, bool report) {
  const int64_t n = load_index(p.k.cache_seq_lens, p.k.seq_lens_is_i64, s.row);
  const int64_t most = min((int64_t)p.k.table_width * p.k.page_size, (int64_t)0x7fff0000);
  if (!s.there) return;
  if (report && n > most) atomicOr(p.status, HIPATTN_STATUS_TOKEN_RANGE);
  s.hi = (int)max((int64_t)0, min(n, most));
  s.lo = p.window > 0 ? max(0, s.hi - p.window) : 0;
}
__device__ __forceinline__ Sequence sequence_of(const Params& p, int b) {
  Sequence s = row_of(p, b, false);
  read_length(p, s, false);
  return s;
}
// rounds of a unit; an empty sequence has one, which writes its zeros
__device__ __forceinline__ int rounds_of(const Sequence& s, int round) { return max(1, (s.hi - s.lo + round - 1) / round); }

// Sum of rounds (and `extra` each) over all sequences (`total`) and over those before sequence b (`before`), for the merge kernel; all threads.
template <int THREADS>
__device__ __forceinline__ void sum_rounds(const Params& p, int b, int round, int extra, int64_t* s_sum, int64_t& total, int64_t& before) {
  int64_t t = 0, f = 0;
  for (int i = threadIdx.x; i < p.B; i += THREADS) {
    const int r = rounds_of(sequence_of(p, i), round) + extra;
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

// a / b of numbers that are not negative: in 32 bits wherever they fit (a division of 64 bits is a hundred instructions)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int64_t share_of(int64_t total, int ctas, int least) {
  const int64_t s = quotient(total + ctas - 1, ctas);
  return s < least ? least : s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// A product q.k as a logit to base 2: scale log2 e x, or with a soft-cap log2 e cap tanh(scale x / cap), in one of two forms.
// Short: tanh(y) = 1 - 2 / (e^2y + 1), off by a few 2^-24 of the cap, in five instructions.  For 16-bit products and caps up to kShortCap, where that
// is below 2^-16, what the two 16-bit terms of a weight keep.
// Else (fp32 products, larger caps): tanhf, off by a few 2^-24 of the logit itself, and the plain logit where the cap changes less than 2^-25 of it, so
// that a cap far above the logits changes nothing.  Kernels of their own: 12 fp8 sequences with a cap of 30 115 us in the short form, 124 in this one, and
// with both in one kernel others lose 4 % to it that have no cap at all.  fp32, 16 sequences of up to 16384 tokens: 222 us
// without a cap, 224 with one; 243 and 246 with both in one kernel in the short form.
constexpr float kShortCap = 64.f;
struct Logit {
  float k, cap;      // cap 0: none, else log2 e cap.  k = log2 e scale, short form 2 log2 e scale / cap.  k is positive: queries are multiplied by `sign` before
  __device__ __forceinline__ Logit(const Params& p, float scale, bool is_short) {
    // (never zero nor infinite: the zero of a scale of zero, which the queries carry, and of an empty product has to stay one.  A tiny scale over a
    // head's power of two may come out as zero.)
    const float size = fmaxf(fabsf(scale), FLT_TRUE_MIN);
    cap = fminf(p.logit_softcap * kLog2e, FLT_MAX);
    k = fminf(kLog2e * size, FLT_MAX);
    if (p.logit_softcap > 0.f && is_short) k = fminf(2.f * kLog2e * size / p.logit_softcap, FLT_MAX);
  }
  __device__ __forceinline__ float capped_short(float x) const {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(ex2(x * k) + 1.f));
    return fmaf(-2.f * cap, r, cap);
  }
  __device__ __forceinline__ float per_cap() const { return fminf(k / cap, FLT_MAX); }     // scale / cap
  __device__ __forceinline__ float capped(float x, float per_cap) const {
    const float y = x * per_cap;
    return fabsf(y) < 0x1p-12f ? x * k : cap * tanhf(y);
  }
  __device__ static __forceinline__ float sign(const Params& p) { return p.sm_scale > 0.f ? 1.f : (p.sm_scale < 0.f ? -1.f : 0.f); }
};

// How a call is laid out.  split: every CTA takes a share of the row of rounds.  Else a unit is a CTA's, or a cluster's.
struct Plan {
  int tiles, split, least, cluster;   // head tiles of a KV head; rounds that a share has at least
  int extra;                          // rounds that beginning and ending a unit counts for in a share
  int vector_out;                     // output rows begin where four elements can be stored at once
};

// Columns 4 v .. 4 v + 3 of the output row of head h, from the joined base of the weights, numerators and denominator
template <int DT>
__device__ __forceinline__ void finish(const Params& p, const Plan& plan, int b, int h, int v, float M, const float4& num, float den) {
  using T = typename Elem<DT>::type;
  // (a denominator of exactly zero: nothing was attended.  NaN and infinite logits stay visible.)
  const bool none = den == 0.f;
  const float r = none ? 0.f : 1.f / den;
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.o_stride_b + (int64_t)h * p.o_stride_h + v * 4;
  const float x[4] = {none ? 0.f : num.x * r, none ? 0.f : num.y * r, none ? 0.f : num.z * r, none ? 0.f : num.w * r};
  if (plan.vector_out) {
    if constexpr (DT == HIPATTN_F32) *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = Elem<DT>::from_f32(x[e]);
  }
  if (v == 0 && p.lse_out) p.lse_out[(int64_t)b * p.H + h] = none ? -INFINITY : (M > -INFINITY ? M : 0.f) + log2f(den);
}

// Geometry of the kernels: RB = bytes of a row of DP elements, KEYS = keys a warp takes at once, STAGES = depth of its ring
template <int DT, bool F8, int DP>
struct Geo {
  static constexpr int EB = F8 ? 1 : Elem<DT>::bytes;
  static constexpr int RB = DP * EB;
  static constexpr int NPC = RB / 16;                         // pieces of a row
  static constexpr int KEYS = DT == HIPATTN_F32 ? 4096 / RB : (RB <= 128 ? 32 : 16);
  static constexpr int STAGES = 3;
  static constexpr int ROUND = KEYS * kWarps;
  static constexpr int STAGE_BYTES = 2 * KEYS * RB;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES * kWarps;
  static constexpr int CTAS = RB == 64 ? 3 : 200 * 1024 / RING_BYTES;        // per multiprocessor: 3, 2 or 1
};
template <int DP>
struct FmaGeo : Geo<HIPATTN_F32, false, DP> {
  using B = Geo<HIPATTN_F32, false, DP>;
  static constexpr int LPK = 32 / B::KEYS;                          // lanes of a key in the logits
  static constexpr int PPL = B::NPC > 32 ? B::NPC / 32 : 1;         // pieces of a V row that a lane owns
  static constexpr int KP = B::NPC < 32 ? 32 / B::NPC : 1;          // V rows that a warp reads at once
};

// A CTA's share of the row of rounds
struct Share {
  int64_t first, last, unit_at;   // [first, last): what is left of it; where sequence b begins in the row
  int b;
};
// false: the share is empty.  All threads.
__device__ __forceinline__ bool find_share(const Params& p, int units, int round, const Plan& plan, Share& sh) {
  __shared__ int64_t s_scan[2][kWarps];
  __shared__ int64_t s_found[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int64_t total = 0, x = 0, sum = 0;
  // rounds (and extra) of sequence c + tid (x) and of those of [c, c + tid] (sum); the sum over the CTA is returned
  auto scan = [&](int c, int turn) {
    const int i = c + tid;
    x = sum = i < p.B ? rounds_of(sequence_of(p, i), round) + plan.extra : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) s_scan[turn & 1][warp] = sum;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) sum += s_scan[turn & 1][w];
      all += s_scan[turn & 1][w];
    }
    return all;
  };
  int turn = 0;
  for (int c = 0; c < p.B; c += kThreads) total += scan(c, turn++);
  const int64_t share = share_of(total * units, gridDim.x, plan.least);
  sh.first = share * blockIdx.x;
  sh.last = min(sh.first + share, total * units);
  if (sh.first >= sh.last) return false;
  int64_t base = 0;
  for (int c = 0; c < p.B; c += kThreads) {
    const int64_t all = p.B > kThreads ? scan(c, turn++) : total;   // (one sequence to a thread: it is in its registers)
    const int64_t end = (base + sum) * units;
    if (sh.first < end && sh.first >= end - x * units) {
      s_found[0] = c + tid;
      s_found[1] = end - x * units;
    }
    base += all;
  }
  __syncthreads();
  sh.b = (int)s_found[0];
  sh.unit_at = s_found[1];
  return true;
}

// What a CTA works on next: rounds [r0, r1) of one unit, `step` keys apart, round 0 beginning at key `lo`.  The CTAs of a cluster take
// its rounds in turn.
struct Segment {
  Sequence seq;
  int rounds, r0, r1, lo, step, hkv, h0, live_heads, used;      // used: what it takes of the share
};
__device__ __forceinline__ void set_unit(const Params& p, Segment& g, int u, int tiles, int gt) {
  const int heads = p.H / p.HKV, tile = u % tiles;
  g.hkv = u / tiles;
  g.h0 = g.hkv * heads + tile * gt;
  g.live_heads = min(gt, heads - tile * gt);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, int rank) {   // the same shared-memory address in CTA `rank` of the cluster
  uint32_t a;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// The share moves on behind a segment; false: that was the last
__device__ __forceinline__ bool next_segment(const Segment& g, Share& sh, int units, const Plan& plan) {
  sh.first += g.used;
  if (sh.first >= sh.last) return false;
  if (sh.first == sh.unit_at + (int64_t)(g.rounds + plan.extra) * units) {
    sh.unit_at = sh.first;
    ++sh.b;
  }
  return true;
}

// The segment's result from the warps' parts, s_merge [kWarps][GT][DP + 4]: to the output, to scratch, or (a cluster) to s_cta [GT][DP + 4],
// which the CTAs of the cluster read together: as many lanes as there are CTAs to four columns, each finishing some of them.  Returns
// whether more is to come.
template <int DT, int DP, int GT>
__device__ __forceinline__ bool end_segment(const Params& p, const Segment& g, Share& sh, int64_t share_first, int units, const Plan& plan, const float* s_merge,
                                            float* s_cta) {
  constexpr int MS = DP + 4, V = DP / 4;
  const bool whole = plan.split ? g.r0 == 0 && g.r1 == g.rounds : plan.cluster == 1;
  float* part = s_cta;
  if (plan.split) part = reinterpret_cast<float*>(p.scratch) + ((int64_t)blockIdx.x * 2 + (sh.first == share_first ? 0 : 1)) * GT * MS;
#pragma unroll
  for (int i0 = 0; i0 < GT * V; i0 += kThreads) {
    const int i = i0 + threadIdx.x, h = i / V, v = i % V;
    if (h >= g.live_heads || v * 4 >= p.D) continue;
    float m[kWarps], M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      m[w] = s_merge[(w * GT + h) * MS + DP];
      M = fmaxf(M, m[w]);
    }
    const float base = M > -INFINITY ? M : 0.f;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(m[w] - base);
      const float4 x = *reinterpret_cast<const float4*>(s_merge + (w * GT + h) * MS + v * 4);
      num.x += f * x.x;
      num.y += f * x.y;
      num.z += f * x.z;
      num.w += f * x.w;
      den += f * s_merge[(w * GT + h) * MS + DP + 1];
    }
    if (whole) {
      finish<DT>(p, plan, sh.b, g.h0 + h, v, M, num, den);
    } else {
      *reinterpret_cast<float4*>(part + h * MS + v * 4) = num;
      if (v == 0) *reinterpret_cast<float4*>(part + h * MS + DP) = make_float4(M, den, 0.f, 0.f);
    }
  }
  if (plan.cluster > 1) {
    const int rank = blockIdx.x % plan.cluster;
    int lanes = 2;
    while (lanes < plan.cluster) lanes *= 2;
    const int sub = threadIdx.x % lanes, groups = kThreads / lanes, live_v = (p.D + 3) / 4, outputs = g.live_heads * live_v;
    cluster_arrive();
    cluster_wait();
    const uint32_t own = (uint32_t)__cvta_generic_to_shared(s_cta);
    for (int o0 = rank * groups; o0 < outputs; o0 += plan.cluster * groups) {
      const int o = o0 + threadIdx.x / lanes, h = o / live_v, v = o - h * live_v;
      float4 num = make_float4(0.f, 0.f, 0.f, 0.f), ml = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      if (o < outputs && sub < plan.cluster) {
        num = ld_cluster4(own + (uint32_t)(h * MS + v * 4) * 4, sub);
        ml = ld_cluster4(own + (uint32_t)(h * MS + DP) * 4, sub);
      }
      float M = ml.x;
      for (int s = lanes >> 1; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
      const float f = ex2(ml.x - (M > -INFINITY ? M : 0.f));
      float den = f * ml.y;
      num.x *= f;
      num.y *= f;
      num.z *= f;
      num.w *= f;
      for (int s = lanes >> 1; s > 0; s >>= 1) {
        den += __shfl_xor_sync(0xffffffffu, den, s);
        num.x += __shfl_xor_sync(0xffffffffu, num.x, s);
        num.y += __shfl_xor_sync(0xffffffffu, num.y, s);
        num.z += __shfl_xor_sync(0xffffffffu, num.z, s);
        num.w += __shfl_xor_sync(0xffffffffu, num.w, s);
      }
      if (o < outputs && sub == 0) finish<DT>(p, plan, sh.b, g.h0 + h, v, M, num, den);
    }
    cluster_arrive();
    cluster_wait();   // no CTA leaves while another reads its shared memory
  }
  return plan.split && next_segment(g, sh, units, plan);
}

__device__ __forceinline__ void cp_async16(uint32_t smem_addr, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_addr), "l"(gmem));
}
// A table entry as it lies: its low word, and the high word of an int64.
struct Entry {
  uint32_t lo = 0, hi = 0;
};
// Where piece `pc` of row `key` of a tile lies: rows of RB bytes, their pieces turned by Kind::turn(key), which is an xor of its bits
template <int RB, class Kind>
struct Place {
  __device__ static __forceinline__ constexpr int at(int key, int pc) { return key * RB + ((pc ^ Kind::turn(key)) << 4); }
};
// Asynchronous copies of a warp's keys into its ring; a row that is not attended is sixteen zero bytes a piece (what lies there may be
// anything, NaN too).  Lane `key` has a key's table entry fetched two rounds before its rows, into shared memory: a register that a load is
// to fill stalls the warp when it is as much as moved (pages of one token, 1.1 GB of rows: 206 us with entries in registers, 192 so).
template <class G, class At>
struct Feeder {
  const Params& p;
  Segment g;
  const char *kb, *vb;            // the KV head's rows
  const char *k_piece, *v_piece;  // and this lane's piece of them
  uint32_t lane_at;               // where this lane's piece of a stage's first rows lies
  const char* table;              // the sequence's row of the table
  uint32_t ring, entries;         // shared-memory addresses: [STAGES] stages, [4][KEYS] entries
  int page_size, page_shift, warp, lane, npc, most;
  bool wide;                      // int64 entries
  bool same, fast;                // K and V pools are laid out alike; and rows have all DP columns and begin within 64 GB of the pool's beginning
  Entry e0, e1;                   // of the segment's first two rounds

  // Finds the segment: its sequence, unit and rounds.  `early` is called as soon as the unit is known.  The loads do not wait for one another
  // where they need not: the first table entries and what `early` loads are on their way when the length is asked for (not for shares,
  // whose unit follows from the lengths; entries of a window follow from the length too).
  template <class Early>
  __device__ __forceinline__ Feeder(const Params& p_, const Share& sh, const Plan& plan, int units, int gt, int warp_, int lane_, const unsigned char* ring_,
                                    const unsigned char* entries_, Early early)
      : p(p_), warp(warp_), lane(lane_) {
    g.seq = row_of(p, sh.b, threadIdx.x == 0);
    page_size = p.k.page_size;
    page_shift = (page_size & (page_size - 1)) == 0 ? 31 - __clz(page_size) : -1;
    most = (int)min((int64_t)p.k.table_width * page_size, (int64_t)0x7fff0000);
    wide = p.k.table_is_i64 != 0;
    table = (const char*)p.k.block_table + g.seq.row * p.k.table_stride_b * (wide ? 8 : 4);
    const int rank = blockIdx.x % plan.cluster;
    g.step = G::ROUND * plan.cluster;
    g.lo = rank * G::ROUND;
    g.r0 = 0;
    const bool ahead = !plan.split && p.window == 0;
    if (ahead) {
      e0 = load_entry(0);
      e1 = load_entry(1);
    }
    if (!plan.split) {
      set_unit(p, g, blockIdx.x / plan.cluster % units, plan.tiles, gt);
      early(g);
    }
    read_length(p, g.seq, threadIdx.x == 0);
    g.rounds = rounds_of(g.seq, G::ROUND);
    g.lo += g.seq.lo;
    if (plan.split) {
      const int size = g.rounds + plan.extra;      // of a unit: what it takes to begin it, then its rounds
      const int64_t from = sh.first - sh.unit_at, u = quotient(from, size);
      set_unit(p, g, (int)u, plan.tiles, gt);
      early(g);
      const int begin = (int)(from - u * size), end = (int)min((int64_t)size, begin + (sh.last - sh.first));
      g.used = end - begin;
      g.r0 = max(0, begin - plan.extra);
      g.r1 = max(0, end - plan.extra);
    } else {
      g.r1 = max(0, (g.rounds - rank + plan.cluster - 1) / plan.cluster);
    }
    if (!ahead) {
      e0 = load_entry(g.r0);
      e1 = load_entry(g.r0 + 1);
    }
    ring = (uint32_t)__cvta_generic_to_shared(ring_);
    entries = (uint32_t)__cvta_generic_to_shared(entries_) + (uint32_t)lane * 8;
    npc = p.D * G::EB / 16;
    kb = (const char*)p.k.cache + (int64_t)g.hkv * p.k.stride_ch * G::EB;
    vb = (const char*)p.v.cache + (int64_t)g.hkv * p.v.stride_ch * G::EB;
    k_piece = kb + lane % G::NPC * 16;
    v_piece = vb + lane % G::NPC * 16;
    lane_at = At::at(G::NPC < 32 ? lane / G::NPC : 0, lane % G::NPC);
    same = p.k.stride_page == p.v.stride_page && p.k.stride_off == p.v.stride_off;
    fast = same && npc == G::NPC && (p.k.n_pages * p.k.stride_page + page_size * p.k.stride_off) * G::EB < (int64_t)1 << 36;
  }
  // first key of this warp in round r
  __device__ __forceinline__ int key_at(int r) const { return g.lo + r * g.step + warp * G::KEYS; }
  // The entry of this lane's key in round r.  (Any entry of the table may be read, those behind the sequence's pages are not used.)
  __device__ __forceinline__ const char* entry_at(int r) const {
    const int t = key_at(r) + lane;
    if (lane >= G::KEYS || t >= most) return nullptr;
    return table + (int64_t)(page_shift >= 0 ? t >> page_shift : t / page_size) * (wide ? 8 : 4);
  }
  __device__ __forceinline__ Entry load_entry(int r) const {
    Entry e;
    if (const char* at = entry_at(r)) {
      e.lo = __ldcg((const uint32_t*)at);
      if (wide) e.hi = __ldcg((const uint32_t*)at + 1);
    }
    return e;
  }
  __device__ __forceinline__ void fetch_entry(int r) const {
    if (const char* at = entry_at(r)) {
      const uint32_t to = entries + (uint32_t)(r & 3) * (G::KEYS * 8);
      if (wide) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to), "l"(at));
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to), "l"(at));
    }
  }
  __device__ __forceinline__ Entry fetched_entry(int r) const {
    Entry e;
    if (lane < G::KEYS) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(e.lo), "=r"(e.hi) : "r"(entries + (uint32_t)(r & 3) * (G::KEYS * 8)) : "memory");
    return e;
  }
  __device__ __forceinline__ void copy(int r, int slot, const Entry& e) const {
    if (r >= g.r1) return;
    const int t0 = key_at(r), live_keys = g.seq.hi - t0;
    uint32_t page = e.lo;
    if (page >= (uint32_t)p.k.n_pages || (wide && e.hi != 0)) {
      if (lane < min(live_keys, G::KEYS)) atomicOr(p.status, HIPATTN_STATUS_PAGE_RANGE);
      page = 0;
    }
    const int t = t0 + lane, off = page_shift >= 0 ? t & (page_size - 1) : t % page_size;
    const uint32_t ks = ring + (uint32_t)slot * G::STAGE_BYTES;
    if (fast && live_keys >= G::KEYS) {      // most rounds: no row to leave out, offsets in units of 16 bytes
      const uint32_t at = page * (uint32_t)(p.k.stride_page * G::EB / 16) + (uint32_t)off * (uint32_t)(p.k.stride_off * G::EB / 16);
#pragma unroll
      for (int i = 0; i < G::KEYS * G::NPC / 32; ++i) {
        // lane's row and piece of the first copy; those of copy i are `first` rows further
        constexpr int ROWS = G::NPC < 32 ? 32 / G::NPC : 1;
        const int first = G::NPC > 32 ? i / (G::NPC / 32) : i * ROWS, pc0 = G::NPC > 32 ? i % (G::NPC / 32) * 32 : 0;
        const uint64_t row = (uint64_t)__shfl_sync(0xffffffffu, at, first + (G::NPC < 32 ? lane / G::NPC : 0)) * 16 + pc0 * 16;
        const uint32_t to = ((ks + lane_at) ^ (At::turn(first) << 4)) + first * G::RB + pc0 * 16;
        cp_async16(to, k_piece + row);
        cp_async16(to + G::KEYS * G::RB, v_piece + row);
      }
      return;
    }
    const int64_t ko = ((int64_t)page * p.k.stride_page + (int64_t)off * p.k.stride_off) * G::EB;
    const int64_t vo = same ? ko : ((int64_t)page * p.v.stride_page + (int64_t)off * p.v.stride_off) * G::EB;
#pragma unroll
    for (int i = 0; i < G::KEYS * G::NPC / 32; ++i) {
      const int idx = i * 32 + lane, key = idx / G::NPC, pc = idx % G::NPC;
      const int64_t k0 = __shfl_sync(0xffffffffu, ko, key);
      const int64_t v0 = same ? k0 : __shfl_sync(0xffffffffu, vo, key);
      // (a key that is not attended has the address of a row of page 0, which is not read)
      const bool live = key < live_keys && pc < npc;
      const int piece = pc < npc ? pc * 16 : 0;
      const uint32_t to = ks + At::at(key, pc);
      cp_async16_zfill(to, kb + piece + k0, live);
      cp_async16_zfill(to + G::KEYS * G::RB, vb + piece + v0, live);
    }
  }
  // the first two rounds of a segment on their way, and the entries of the two after them
  __device__ __forceinline__ void begin() const {
    static_assert(G::STAGES == 3, "two rounds of rows in flight, entries for two more");
    fetch_entry(g.r0 + 2);
    fetch_entry(g.r0 + 3);
    copy(g.r0, 0, e0);
    cp_async_commit();
    copy(g.r0 + 1, 1, e1);
    cp_async_commit();
  }
  // Round r, in place `slot` of the ring, has arrived (all of the warp are done with the round before it): round r + 2 takes the place of that one.
  __device__ __forceinline__ void next(int r, int slot) const {
    copy(r + 2, slot == 0 ? 2 : slot - 1, fetched_entry(r + 2));
    fetch_entry(r + 4);
    cp_async_commit();
  }
};

// ---------------------------------------------------------------------------------------------------
// 16-bit and fp8 rows: mma.sync m16n8k16, the GT (8 or 16) query heads of a unit are the rows of the tile.
//
// S = Q K^T: ldmatrix gives the B operand from K rows as they lie; its columns 2 t, 2 t + 1 of a row are the A operand's of
// O += P V, whose B operand is ldmatrix.trans of V rows.  fp8 (e5m2) rows are kept as bytes up to the registers, where an
// element becomes the half-precision number whose upper byte it is: for K the four bytes that a lane gets are four
// consecutive elements, so the contraction runs in that order and Q's fragments are laid out alike; for V a lane gets
// two columns of two keys, the even columns of a block make one product and the odd ones another.  With fp8 rows all products
// are in half precision; bfloat16 queries are brought to its range by a power of two per head (exact down to 2^-39 of the
// head's largest element, below what the sum keeps).
//
// The weights go in two 16-bit terms, the rounded weight and what the rounding left.  Half-precision weights are scaled by 2^14
// (largest: 16384), so that a weight of 2^-28 of the largest is still a normal number: many small weights add up.  Of eight heads the
// second terms are the rows 8 to 15 of the tile, with sums of their own, and cost nothing; of sixteen they are a second product.
// The second term may be zero or negative, which an infinite value turns into NaN: eight heads leave it out where the first sum is
// not finite; of sixteen a warp that finds NaN in its output goes through its keys once more and leaves the second term out of those sums
// (the others come out as they were: a value that is not finite costs its neighbours nothing).
// ---------------------------------------------------------------------------------------------------
// the halves of two packed 16-bit elements
template <int MT>
__device__ __forceinline__ float lower(uint32_t w) {
  return MT == HIPATTN_BF16 ? __uint_as_float(w << 16) : __low2float(*reinterpret_cast<const __half2*>(&w));
}
template <int MT>
__device__ __forceinline__ float upper(uint32_t w) {
  return MT == HIPATTN_BF16 ? __uint_as_float(w & 0xffff0000u) : __high2float(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ void ldsm_x4_at(uint32_t* r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm_x4_t_at(uint32_t* r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}

template <int RB>
struct MmaPlace : Place<RB, MmaPlace<RB>> {   // the eight rows that ldmatrix reads at once lie in eight different groups of banks
  __device__ static __forceinline__ constexpr int turn(int key) { return RB >= 128 ? key & 7 : (key >> 1) & (RB / 16 - 1); }
};

template <int DT, bool F8, int DP, int GT, bool LONG_CAP>
__global__ void __launch_bounds__(kThreads, Geo<DT, F8, DP>::CTAS) paged_decode_mma_kernel(const Params p, const Plan plan) {
  using G = Geo<DT, F8, DP>;
  using P = MmaPlace<G::RB>;
  using T = typename Elem<DT>::type;
  constexpr int MT = F8 ? HIPATTN_F16 : DT;          // type of the products
  constexpr int AHEAD = DP == 256 ? 0 : (G::NPC / 2 < 4 ? G::NPC / 2 : 4);      // loads of values before the weights are made
  constexpr int KEYS = G::KEYS, MS = DP + 4, KS = DP / 16, NT = DP / 8, AR = GT / 4;   // AR: registers of an A fragment that are not padding
  constexpr float kShift = MT == HIPATTN_F16 ? 14.f : 0.f;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, jq = lane & 3;
  unsigned char* ring = smem + warp * (G::STAGES * G::STAGE_BYTES);
  float* s_merge = reinterpret_cast<float*>(smem);                       // over the rings when they are empty
  uint32_t* s_q = reinterpret_cast<uint32_t*>(smem + G::RING_BYTES);     // [KS][32][AR]: A fragments
  const unsigned char* entries = smem + G::RING_BYTES + 2 * GT * DP + warp * (4 * KEYS * 8);
  __shared__ uint32_t s_nan[GT == 16 ? NT / 8 * kThreads : 1];           // [NT / 8][kThreads]: a bit for a sum that the first pass left NaN
  __shared__ float s_up[16];                                             // power of two that a head's queries were multiplied by
  const int units = p.HKV * plan.tiles;
  in_turn();

  Share sh{0, 0, 0, (int)(blockIdx.x / plan.cluster / units)};
  if (plan.split && !find_share(p, units, G::ROUND, plan, sh)) return;
  const int64_t share_first = sh.first;
  // rows and pieces of ldmatrix: 16-bit K eight keys by two pieces twice, fp8 K a piece of all keys or two of sixteen, V sixteen keys by two
  const uint32_t k_lane = F8 ? (KEYS == 32 ? P::at(lane, 0) : P::at(lane & 15, lane >> 4)) : P::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
  const uint32_t v_lane = KEYS * G::RB + P::at(lane & 15, lane >> 4);

  const bool pairs = ((uintptr_t)p.q | (uintptr_t)(p.q_stride_b * 2) | (uintptr_t)(p.q_stride_h * 2)) % 4 == 0;    // two elements in one load

  for (bool more = true; more;) {
    __syncthreads();
    // ---- the segment, and its queries: register r of lane l of a fragment is row l / 4 (+ 8), elements 2 (l % 4) .. (+ 8) of a step; with
    // fp8 rows 4 (l % 4) .. (+ 2) ----
    uint32_t qw[KS * 32 * AR / kThreads];
    auto row_and_element = [&](int j, int& row, int& e) {
      const int i = j * kThreads + tid, r = i % AR, l = i / AR % 32, ks = i / AR / 32, second = GT == 16 ? r >> 1 : r;
      row = (l >> 2) + (GT == 16 && (r & 1) ? 8 : 0);
      e = ks * 16 + (F8 ? (l & 3) * 4 + second * 2 : (l & 3) * 2 + second * 8);
    };
    const T* q = nullptr;
    auto load_queries = [&](const Segment& g) {
      q = reinterpret_cast<const T*>(p.q) + (int64_t)sh.b * p.q_stride_b + (int64_t)g.h0 * p.q_stride_h;
#pragma unroll
      for (int j = 0; j < KS * 32 * AR / kThreads; ++j) {
        int row, e;
        row_and_element(j, row, e);
        qw[j] = 0u;
        if (row < g.live_heads && e < p.D) {
          const T* at = q + (int64_t)row * p.q_stride_h + e;
          if (pairs) qw[j] = __ldcg(reinterpret_cast<const uint32_t*>(at));
          else qw[j] = (uint32_t)*reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + 1) << 16;
        }
      }
    };
    const Feeder<G, P> feed(p, sh, plan, units, GT, warp, lane, ring, entries, load_queries);
    const Segment& g = feed.g;
    if (plan.split && g.r0 == g.r1) {      // (the share has no round of the unit, only its beginning)
      more = next_segment(g, sh, units, plan);
      continue;
    }
    feed.begin();
    if constexpr (F8 && DT == HIPATTN_BF16) {
      for (int h = warp; h < GT; h += kWarps) {
        float mx = 0.f;
        if (h < g.live_heads)
          for (int e = lane; e < p.D; e += 32) mx = fmaxf(mx, fabsf(Elem<DT>::to_f32(q[(int64_t)h * p.q_stride_h + e])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        // 2^k with mx 2^k in [2^14, 2^15); k at most 126, so that 2^-k is a normal number too
        int e = 0;
        if (mx > 0.f && mx < INFINITY) frexpf(mx, &e);
        if (lane == 0) s_up[h] = mx > 0.f && mx < INFINITY ? exp2f((float)min(15 - e, 126)) : 1.f;
      }
      __syncthreads();
    }
    const float sign = Logit::sign(p);
#pragma unroll
    for (int j = 0; j < KS * 32 * AR / kThreads; ++j) {
      int row, e;
      row_and_element(j, row, e);
      float up = sign;
      if constexpr (F8 && DT == HIPATTN_BF16) up *= s_up[row];
      s_q[j * kThreads + tid] = pack2<MT>(lower<DT>(qw[j]) * up, upper<DT>(qw[j]) * up);
    }
    __syncthreads();
    const Logit logit0(p, F8 && DT == HIPATTN_BF16 ? p.sm_scale / s_up[gr] : p.sm_scale, !LONG_CAP);
    const Logit logit1(p, F8 && DT == HIPATTN_BF16 && GT == 16 ? p.sm_scale / s_up[gr + 8] : p.sm_scale, !LONG_CAP);

    // b_run: what the logits are lowered by before they become weights, the running maximum less kShift.  It is this base that a round keeps or
    // moves, so that sums of rounds with one maximum stay as they are: the factor to them has to be exactly 1 there (from the maxima, with
    // the shift subtracted again, it is off by up to 2^-16 for logits near -256, in every round alike: 3e-3 of the output after 1024 rounds).
    float o[NT][4], b_run[GT / 8], l_run[GT / 8];
    // all rounds.  TWO: with both terms of the weights, else with the second one only where s_nan has no bit
    auto pass = [&](auto both) {
      constexpr bool TWO = decltype(both)::value;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < GT / 8; ++i) { b_run[i] = -INFINITY; l_run[i] = 0.f; }
      int slot = 0;
      for (int r = g.r0; r < g.r1; ++r) {
        cp_async_wait<1>();
        __syncwarp();
        // this lane's row and first piece in K and in V; piece j further is the address xor 16 j (a row begins on a multiple of its size)
        const uint32_t ks = feed.ring + slot * G::STAGE_BYTES + k_lane, vs = feed.ring + slot * G::STAGE_BYTES + v_lane;
        // ---- S = Q K^T ----
        [[maybe_unused]] uint32_t kept[4];
        float s[KEYS / 8][4], s2[2][4];      // (sixteen keys: odd steps have sums of their own, four chains of products in all)
#pragma unroll
        for (int i = 0; i < KEYS / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) s2[i][0] = s2[i][1] = s2[i][2] = s2[i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t a[4] = {0u, 0u, 0u, 0u};
          if constexpr (GT == 16) {
            const uint4 w = reinterpret_cast<const uint4*>(s_q)[k * 32 + lane];
            a[0] = w.x; a[1] = w.y; a[2] = w.z; a[3] = w.w;
          } else {
            const uint2 w = reinterpret_cast<const uint2*>(s_q)[k * 32 + lane];
            a[0] = w.x; a[2] = w.y;
          }
          if constexpr (F8) {
            uint32_t b[4];
            if constexpr (KEYS == 32) {
              ldsm_x4_at(b, ks ^ (k << 4));
            } else {                                   // two pieces of 16 keys
              if ((k & 1) == 0) ldsm_x4_at(kept, ks ^ (k << 4));
              b[0] = kept[(k & 1) * 2];
              b[1] = kept[(k & 1) * 2 + 1];
            }
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) mma16816<MT>(KEYS == 16 && (k & 1) ? s2[n & 1] : s[n], a, __byte_perm(b[n], 0, 0x1404), __byte_perm(b[n], 0, 0x3424));
          } else {
#pragma unroll
            for (int n = 0; n < KEYS / 8; n += 2) {
              uint32_t b[4];
              ldsm_x4_at(b, (ks ^ (k << 5)) + n * 8 * G::RB);
              mma16816<MT>(KEYS == 16 && (k & 1) ? s2[0] : s[n], a, b[0], b[1]);
              mma16816<MT>(KEYS == 16 && (k & 1) ? s2[1] : s[n + 1], a, b[2], b[3]);
            }
          }
        }
        if constexpr (KEYS == 16) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < GT / 4; ++e) s[n][e] += s2[n][e];
        }
        // the first values on their way while the weights are made
        uint32_t vf[AHEAD > 0 ? AHEAD : 1][4];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ldsm_x4_t_at(vf[i], vs ^ (i << 5));
        // ---- online softmax ----
        const int t0 = feed.key_at(r) + 2 * jq;
        const bool tail = feed.key_at(r) + KEYS > g.seq.hi;
        uint32_t pa[KEYS / 16][4], pl[KEYS / 16][4];     // A fragments; of eight heads pa alone, the second terms in its rows 8 to 15
        bool moved = false;
        float alpha[GT / 8];
#pragma unroll
        for (int i = 0; i < GT / 8; ++i) {
          const Logit& logit = i ? logit1 : logit0;
          float k = logit.k;      // logits are s k
          if (logit.cap > 0.f) {
            const float per_cap = LONG_CAP ? logit.per_cap() : 0.f;
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) s[n][2 * i + e] = LONG_CAP ? logit.capped(s[n][2 * i + e], per_cap) : logit.capped_short(s[n][2 * i + e]);
            k = 1.f;
          }
          if (tail) {
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (t0 + n * 8 + e >= g.seq.hi) s[n][2 * i + e] = -INFINITY;
          }
          float mx = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
          for (int n = 1; n < KEYS / 8; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          float b_new = fmaxf(b_run[i], fmaf(mx, k, -kShift));
          if (fabsf(b_new) >= 0x1p24f) {      // neighbours are two and more apart there: a logit that is not rounded itself may lie far above the largest one
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) s[n][2 * i + e] = __fmul_rn(s[n][2 * i + e], k);
            b_new = fmaxf(b_run[i], __fmul_rn(mx, k));
            k = 1.f;
          }
          const float base = b_new > -INFINITY ? b_new : 0.f;
          alpha[i] = ex2(b_run[i] - base);
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < KEYS / 8; ++n) {
            const float x = ex2(fmaf(s[n][2 * i], k, -base)), y = ex2(fmaf(s[n][2 * i + 1], k, -base));
            sum += x + y;
            const uint32_t hi = pack2<MT>(x, y), lo = pack2<MT>(x - lower<MT>(hi), y - upper<MT>(hi));
            pa[n / 2][(n & 1) * 2 + i] = hi;
            if constexpr (GT == 8) pa[n / 2][(n & 1) * 2 + 1] = lo;
            else pl[n / 2][(n & 1) * 2 + i] = lo;
          }
          l_run[i] = l_run[i] * alpha[i] + sum;      // (this lane's keys; the four lanes of a row are added up at the end)
          b_run[i] = b_new;
          moved |= alpha[i] != 1.f;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= alpha[GT == 16 ? e >> 1 : 0];
        }
        feed.next(r, slot);
        // ---- O += P V ----
        auto product = [&](int n, int c, uint32_t b0, uint32_t b1) {
          mma16816<MT>(o[n], pa[c], b0, b1);
          if constexpr (GT == 16 && TWO) {
            mma16816<MT>(o[n], pl[c], b0, b1);
          } else if constexpr (GT == 16) {
            const float one[4] = {o[n][0], o[n][1], o[n][2], o[n][3]};
            mma16816<MT>(o[n], pl[c], b0, b1);
            const uint32_t nan = *(volatile uint32_t*)&s_nan[n / 8 * kThreads + tid] >> (n % 8 * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (nan >> e & 1u) o[n][e] = one[e];
          }
        };
#pragma unroll
        for (int c = 0; c < KEYS / 16; ++c) {
#pragma unroll
          for (int pc = 0; pc < G::NPC; pc += 2) {
            uint32_t b[4];
            if (c == 0 && pc / 2 < AHEAD) {
#pragma unroll
              for (int e = 0; e < 4; ++e) b[e] = vf[pc / 2 < AHEAD ? pc / 2 : 0][e];
            } else {
              ldsm_x4_t_at(b, (vs ^ (pc << 4)) + c * 16 * G::RB);
            }
            if constexpr (F8) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                product((pc + h) * 2, c, __byte_perm(b[2 * h], 0, 0x2404), __byte_perm(b[2 * h + 1], 0, 0x2404));
                product((pc + h) * 2 + 1, c, __byte_perm(b[2 * h], 0, 0x3414), __byte_perm(b[2 * h + 1], 0, 0x3414));
              }
            } else {
              product(pc, c, b[0], b[1]);
              product(pc + 1, c, b[2], b[3]);
            }
          }
        }
        slot = slot == 2 ? 0 : slot + 1;
      }
      cp_async_wait<0>();
    };
    pass(std::true_type());
    if constexpr (GT == 8) {
      // the terms together; where the first is infinite or NaN the second says nothing (zero times infinity)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (fabsf(o[n][e]) < INFINITY) o[n][e] += o[n][e + 2];
    } else {
      uint32_t any = 0;
#pragma unroll
      for (int w = 0; w < NT / 8; ++w) {
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) nan |= o[w * 8 + i / 4][i % 4] != o[w * 8 + i / 4][i % 4] ? 1u << i : 0u;
        s_nan[w * kThreads + tid] = nan;
        any |= nan;
      }
      if (__any_sync(0xffffffffu, any != 0)) {
        __syncwarp();      // (all of the warp are done with the last rows)
        feed.begin();
        pass(std::false_type());
      }
    }
    __syncthreads();

    // ---- the warps' parts ----
#pragma unroll
    for (int i = 0; i < GT / 8; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      float* dst = s_merge + (warp * GT + gr + i * 8) * MS;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) dst[F8 ? (n >> 1) * 16 + (2 * jq + e) * 2 + (n & 1) : n * 8 + 2 * jq + e] = o[n][2 * i + e];
      if (jq == 0) {
        dst[DP] = b_run[i];
        dst[DP + 1] = l_run[i];
      }
    }
    __syncthreads();
    more = end_segment<DT, DP, GT>(p, g, sh, share_first, units, plan, s_merge, s_merge + kWarps * GT * MS);
  }
}

// ---------------------------------------------------------------------------------------------------
// fp32: FMA.  LPK lanes to a key for the logits, a lane owns columns of the output.
// ---------------------------------------------------------------------------------------------------
template <int RB, int LPK>
struct FmaPlace : Place<RB, FmaPlace<RB, LPK>> {   // the lanes of a quarter warp, LPK to a row, reach eight different groups of banks
  __device__ static __forceinline__ constexpr int turn(int key) { return (key * LPK) & 7; }
};

template <int DP, int GT, bool CAP>
__global__ void __launch_bounds__(kThreads, FmaGeo<DP>::CTAS) paged_decode_fma_kernel(const Params p, const Plan plan) {
  using G = FmaGeo<DP>;
  using P = FmaPlace<G::RB, G::LPK>;
  constexpr int KEYS = G::KEYS, NPC = G::NPC, LPK = G::LPK, MS = DP + 4;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* ring = smem + warp * (G::STAGES * G::STAGE_BYTES);
  float* s_merge = reinterpret_cast<float*>(smem);                   // over the rings when they are empty
  float* s_q = reinterpret_cast<float*>(smem + G::RING_BYTES);       // [GT][DP]
  const unsigned char* entries = smem + G::RING_BYTES + 4 * GT * DP + warp * (4 * KEYS * 8);
  const int units = p.HKV * plan.tiles;
  in_turn();

  Share sh{0, 0, 0, (int)(blockIdx.x / plan.cluster / units)};
  if (plan.split && !find_share(p, units, G::ROUND, plan, sh)) return;
  const int64_t share_first = sh.first;
  const Logit logit(p, p.sm_scale, false);
  const float per_cap = CAP ? logit.per_cap() : 0.f;

  for (bool more = true; more;) {
    __syncthreads();
    float qw[GT * DP / kThreads];
    auto load_queries = [&](const Segment& g) {
#pragma unroll
      for (int j = 0; j < GT * DP / kThreads; ++j) {
        const int h = (j * kThreads + tid) / DP, e = (j * kThreads + tid) % DP;
        qw[j] = 0.f;
        if (h < g.live_heads && e < p.D) qw[j] = reinterpret_cast<const float*>(p.q)[(int64_t)sh.b * p.q_stride_b + (int64_t)(g.h0 + h) * p.q_stride_h + e];
      }
    };
    const Feeder<G, P> feed(p, sh, plan, units, GT, warp, lane, ring, entries, load_queries);
    const Segment& g = feed.g;
    if (plan.split && g.r0 == g.r1) {      // (the share has no round of the unit, only its beginning)
      more = next_segment(g, sh, units, plan);
      continue;
    }
    feed.begin();
#pragma unroll
    for (int j = 0; j < GT * DP / kThreads; ++j) s_q[j * kThreads + tid] = qw[j] * Logit::sign(p);
    __syncthreads();

    float m_run[GT], l_run[GT], acc[GT][G::PPL][4];
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      m_run[h] = -INFINITY;
      l_run[h] = 0.f;
#pragma unroll
      for (int i = 0; i < G::PPL; ++i) acc[h][i][0] = acc[h][i][1] = acc[h][i][2] = acc[h][i][3] = 0.f;
    }
    int slot = 0;
    for (int r = g.r0; r < g.r1; ++r) {
      cp_async_wait<1>();
      __syncwarp();
      feed.next(r, slot);
      const unsigned char* ks = ring + slot * G::STAGE_BYTES;
      const unsigned char* vs = ks + KEYS * G::RB;
      // ---- logits ----
      const int key = lane / LPK, sub = lane % LPK;
      float s[GT];
#pragma unroll
      for (int h = 0; h < GT; ++h) s[h] = 0.f;
#pragma unroll 4
      for (int j = 0; j < NPC / LPK; ++j) {
        const int pc = j * LPK + sub;
        const float4 kv = *reinterpret_cast<const float4*>(ks + P::at(key, pc));
#pragma unroll
        for (int h = 0; h < GT; ++h) {
          const float4 qv = reinterpret_cast<const float4*>(s_q + h * DP)[pc];
          s[h] = fmaf(qv.w, kv.w, fmaf(qv.z, kv.z, fmaf(qv.y, kv.y, fmaf(qv.x, kv.x, s[h]))));
        }
      }
      const bool in = feed.key_at(r) + key < g.seq.hi;
      float pr[GT];
#pragma unroll
      for (int h = 0; h < GT; ++h)
#pragma unroll
        for (int o = LPK >> 1; o > 0; o >>= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], o);
      if constexpr (CAP) {       // a key's lanes take a head each (every lane all heads: a tenth of the kernel's time)
#pragma unroll
        for (int h0 = 0; h0 < GT; h0 += LPK) {
          float mine = s[h0];
#pragma unroll
          for (int j = 1; j < LPK && h0 + j < GT; ++j) mine = sub == j ? s[h0 + j] : mine;
          mine = logit.capped(mine, per_cap);
#pragma unroll
          for (int j = 0; j < LPK && h0 + j < GT; ++j) s[h0 + j] = __shfl_sync(0xffffffffu, mine, (lane & ~(LPK - 1)) + j);
        }
      }
#pragma unroll
      for (int h = 0; h < GT; ++h) {
        s[h] = in ? (CAP ? s[h] : s[h] * logit.k) : -INFINITY;
        float mx = s[h];
#pragma unroll
        for (int o = 16; o >= LPK; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m_new = fmaxf(m_run[h], mx), base = m_new > -INFINITY ? m_new : 0.f;
        const float alpha = ex2(m_run[h] - base);
        pr[h] = ex2(s[h] - base);
        l_run[h] = l_run[h] * alpha + (sub == 0 ? pr[h] : 0.f);
        m_run[h] = m_new;
#pragma unroll
        for (int i = 0; i < G::PPL; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[h][i][e] *= alpha;
      }
      // ---- o += p V ----
#pragma unroll
      for (int k0 = 0; k0 < KEYS; k0 += G::KP) {
        const int k = k0 + (G::KP > 1 ? lane / NPC : 0);
#pragma unroll
        for (int i = 0; i < G::PPL; ++i) {
          const float4 vv = *reinterpret_cast<const float4*>(vs + P::at(k, lane % NPC + i * 32));
#pragma unroll
          for (int h = 0; h < GT; ++h) {
            const float x = __shfl_sync(0xffffffffu, pr[h], k * LPK);
            acc[h][i][0] = fmaf(x, vv.x, acc[h][i][0]);
            acc[h][i][1] = fmaf(x, vv.y, acc[h][i][1]);
            acc[h][i][2] = fmaf(x, vv.z, acc[h][i][2]);
            acc[h][i][3] = fmaf(x, vv.w, acc[h][i][3]);
          }
        }
      }
      slot = slot == 2 ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- the warps' parts ----
#pragma unroll
    for (int h = 0; h < GT; ++h) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], o);
#pragma unroll
      for (int i = 0; i < G::PPL; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int o = NPC; o < 32; o <<= 1) acc[h][i][e] += __shfl_xor_sync(0xffffffffu, acc[h][i][e], o);
          if (lane < NPC) s_merge[(warp * GT + h) * MS + (lane % NPC + i * 32) * 4 + e] = acc[h][i][e];
        }
      if (lane == 0) {
        s_merge[(warp * GT + h) * MS + DP] = m_run[h];
        s_merge[(warp * GT + h) * MS + DP + 1] = l_run[h];
      }
    }
    __syncthreads();
    more = end_segment<HIPATTN_F32, DP, GT>(p, g, sh, share_first, units, plan, s_merge, s_merge + kWarps * GT * MS);
  }
}

// Joins the parts of a unit that lies in several shares, in their order.  One CTA per sequence, unit and `hb` of its heads; the
// warps of a head (all eight of them for a single head) take the parts in turn and meet in shared memory.
constexpr int kMergeWarps = 8;
template <int DT, int DP, int GT>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_decode_merge_kernel(const Params p, const Plan plan, int ctas, int round, int hb) {
  constexpr int PS = DP + 4, V = DP / 4, VL = V > 32 ? V / 32 : 1;       // float4s of a row, and of a lane
  __shared__ int64_t s_sum[2 * kMergeWarps];
  __shared__ __align__(16) float s_num[kMergeWarps][DP];
  const int tiles = plan.tiles, heads = p.H / p.HKV, units = p.HKV * tiles, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / units, u = blockIdx.x % units;
  const int rounds = rounds_of(sequence_of(p, b), round);
  int64_t total, before;
  sum_rounds<kMergeWarps * 32>(p, b, round, plan.extra, s_sum, total, before);
  const int64_t share = share_of(total * units, ctas, plan.least), begin = before * units + (int64_t)u * (rounds + plan.extra);
  const int c0 = (int)quotient(begin + plan.extra, share), c1 = (int)quotient(begin + plan.extra + rounds - 1, share);
  in_turn();    // (the lengths do not change under the launch before)
  if (c0 == c1) return;
  const int tile = u % tiles, h0 = u / tiles * heads + tile * GT, live_heads = min(GT, heads - tile * GT);
  const float* parts = reinterpret_cast<const float*>(p.scratch) + ((int64_t)c0 * 2 + (begin <= c0 * share ? 0 : 1)) * GT * PS;   // of share c0
  const float* later = reinterpret_cast<const float*>(p.scratch);                                                               // of share c: c * 2 * GT * PS
  const int per_head = hb < kMergeWarps ? kMergeWarps / hb : 1;           // warps of a head
  for (int i0 = 0; i0 < hb; i0 += kMergeWarps / per_head) {
    const int h = blockIdx.y * hb + i0 + warp / per_head, sub = warp % per_head;
    const bool live = h < live_heads && h < (int)(blockIdx.y + 1) * hb;
    float M = -INFINITY, den = 0.f;
    float4 num[VL];
#pragma unroll
    for (int j = 0; j < VL; ++j) num[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
      auto row = [&](int c) { return (c == c0 ? parts : later + (int64_t)c * 2 * GT * PS) + h * PS; };
      for (int c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, __ldcg(row(c) + DP));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      const float base = M > -INFINITY ? M : 0.f;
      for (int c = c0 + lane; c <= c1; c += 32) den += ex2(__ldcg(row(c) + DP) - base) * __ldcg(row(c) + DP + 1);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
#pragma unroll 4
      for (int c = c0 + sub; c <= c1; c += per_head) {
        const float f = ex2(__ldcg(row(c) + DP) - base);
#pragma unroll
        for (int j = 0; j < VL; ++j) {
          if (V < 32 && lane >= V) continue;
          const float4 x = __ldcg(reinterpret_cast<const float4*>(row(c)) + lane + j * 32);
          num[j].x += f * x.x;
          num[j].y += f * x.y;
          num[j].z += f * x.z;
          num[j].w += f * x.w;
        }
      }
#pragma unroll
      for (int j = 0; j < VL; ++j)
        if (V >= 32 || lane < V) *reinterpret_cast<float4*>(&s_num[warp][(lane + j * 32) * 4]) = num[j];
    }
    __syncthreads();
    if (live) {
      for (int v = sub * 32 + lane; v * 4 < p.D; v += per_head * 32) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = warp - sub; w < warp - sub + per_head; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(&s_num[w][v * 4]);
          x.x += y.x;
          x.y += y.y;
          x.z += y.z;
          x.w += y.w;
        }
        finish<DT>(p, plan, b, h0 + h, v, M, x, den);
      }
    }
    __syncthreads();
  }
}

// The layout's bounds, in rounds.  Measured in bf16 with 32 heads over 8, D 128 (rounds of 64 keys), device times in us.
//
// A share has two rounds at least (one round instead: a sequence of 389 tokens behind a wide table 12.0 -> 9.3, one of 100 7.3 -> 9.0, one of 1000
// 10.2 -> 11.4, the rest the same).
constexpr int kLeastRounds = 2;
// Beginning and ending a unit takes as long as some four rounds (2.5 us); without them in the shares' sizes a CTA that got a dozen short or
// empty sequences ended last by far (64 sequences of up to 1000 tokens behind a wide table: 45 without, 34 so; 12 of up to 8000 44.8 and 43.8).  Few units
// are cut as small as they may be (4 sequences of 2000 behind a wide table: 14.1 so, 15.4 with beginnings counted; 4 of up to 20000 43.1 and 41.7).
constexpr int kUnitRounds = 4;
constexpr int kManyUnits = 64;
// CTAs of a cluster (beyond eight: allowed per kernel).  With eight at most: one sequence of 8000 16.6, 13.9 so; of 1000 6.7, 7.1 so.
constexpr int kMaxCluster = 16;
// Rounds of a CTA of a cluster.  Longer units gain less from the second launch that a cluster does without than they lose where lengths differ (one
// sequence of 30000, no others beside it: 35.2 in shares, 33.4 with up to 32 rounds); with up to eight, 4 of 5000 21.5, 16.3 so.
constexpr int kClusterRounds = 16;
// Rounds of a unit that is a CTA's.  With up to 64: 40 sequences of 3000 (47 rounds) 106, in shares 83, of up to 3000 59 and 53; 64 of 2000 (32 rounds) 85 and 91,
// of up to 2000 58 and 55.  With up to 12: 32 of 800 (13 rounds) 18.8 so, 24 in shares, of up to 800 16.4 and 19.9; 20 of up to 1500 25.6 and 19.6.
constexpr int kWholeRounds = 24;

int padded_dim(int D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }

template <int DT, bool F8, int DP, int GT, bool LONG_CAP>
struct Kernel {
  using G = Geo<DT, F8, DP>;
  static constexpr size_t smem = G::RING_BYTES + (DT == HIPATTN_F32 ? sizeof(float) : sizeof(uint16_t)) * GT * DP + kWarps * 4 * G::KEYS * 8;
  static_assert(sizeof(float) * (kWarps + 1) * GT * (DP + 4) <= G::RING_BYTES, "the join of the warps lies over the rings");
  static void (*kern())(const Params, const Plan) {
    if constexpr (DT == HIPATTN_F32) return paged_decode_fma_kernel<DP, GT, LONG_CAP>;
    else return paged_decode_mma_kernel<DT, F8, DP, GT, LONG_CAP>;
  }
  // How the call is laid out, and its CTAs.  Reads shapes and what the device holds.
  static Plan plan(const Params& p, int64_t* ctas) {
    Plan l;
    l.tiles = cdiv(p.H / p.HKV, GT);
    l.split = 0;
    l.cluster = 1;
    constexpr int EB = Elem<DT>::bytes;
    l.vector_out = ((uintptr_t)p.out | (uintptr_t)(p.o_stride_b * EB) | (uintptr_t)(p.o_stride_h * EB)) % (4 * EB) == 0;
    const int64_t units = (int64_t)p.B * p.HKV * l.tiles;
    l.extra = units >= kManyUnits ? kUnitRounds : 0;
    l.least = kLeastRounds + l.extra;
    int64_t most = (int64_t)p.k.table_width * p.k.page_size;
    if (p.window > 0 && p.window < most) most = p.window;
    const int64_t rounds = (most + G::ROUND - 1) / G::ROUND;      // a unit has at most
    // Few units that cannot be long: a cluster to each, joined in shared memory without a second launch
    int64_t c = (int64_t)kSMs * G::CTAS / units;
    if (c > kMaxCluster) c = kMaxCluster;
    if (c > rounds) c = rounds;
    if (c > 1 && rounds <= c * kClusterRounds && allow_smem((const void*)kern(), smem) == cudaSuccess) {
      while (c > 1 && resident_clusters((const void*)kern(), (int)c, kThreads, smem) < units) --c;
      if (c > 1 && rounds <= c * kClusterRounds) l.cluster = (int)c;
    }
    if (l.cluster == 1) l.split = rounds > kWholeRounds;
    *ctas = l.split ? kSMs * G::CTAS : units * l.cluster;
    return l;
  }
  static int64_t scratch(const Plan& l, int64_t ctas) { return l.split ? ctas * 2 * GT * (DP + 4) * (int64_t)sizeof(float) : 0; }

  static int launch(const Params& p, cudaStream_t stream, int64_t* bytes) {
    int64_t ctas;
    const Plan l = plan(p, &ctas);
    const int64_t need = scratch(l, ctas);
    if (bytes) {      // only what the call needs
      *bytes = need;
      return HIPATTN_OK;
    }
    HIPATTN_REQUIRE(need == 0 || (p.scratch && p.scratch_bytes >= need && (uintptr_t)p.scratch % 16 == 0), HIPATTN_ERR_INVALID,
                    "paged_decode: %lld bytes of scratch are needed (16-byte aligned), %lld were given", (long long)need, (long long)p.scratch_bytes);
    const int64_t units = (int64_t)p.B * p.HKV * l.tiles;
    HIPATTN_REQUIRE(ctas < 0x7fffffffLL && units < 0x7fffffffLL, HIPATTN_ERR_INVALID, "paged_decode: grid of %lld blocks", (long long)ctas);
    HIPATTN_CUDA_OK(allow_smem((const void*)kern(), smem));
    InTurn main(ctas, kThreads, smem, stream, l.cluster);
    HIPATTN_CUDA_OK(cudaLaunchKernelEx(&main.cfg, kern(), p, l));
    const int rc = check_launch("paged_decode_kernel");
    if (rc || !l.split) return rc;
    // few units have many parts each: one CTA per head then
    const int hb = units < kSMs ? 1 : GT, heads = p.H / p.HKV;
    InTurn merge(units, kMergeWarps * 32, 0, stream);
    merge.cfg.gridDim.y = (unsigned)cdiv(heads < GT ? heads : GT, hb);
    HIPATTN_CUDA_OK(cudaLaunchKernelEx(&merge.cfg, paged_decode_merge_kernel<DT, DP, GT>, p, l, (int)ctas, (int)G::ROUND, hb));
    return check_launch("paged_decode_merge_kernel");
  }
};

// `bytes`: only the scratch of the call
template <int DT, bool F8, int DP, bool LONG_CAP>
int launch_heads(const Params& p, cudaStream_t stream, int64_t* bytes) {
  constexpr int SMALL = DT == HIPATTN_F32 ? 4 : 8;
  return p.H / p.HKV <= SMALL ? Kernel<DT, F8, DP, SMALL, LONG_CAP>::launch(p, stream, bytes) : Kernel<DT, F8, DP, SMALL * 2, LONG_CAP>::launch(p, stream, bytes);
}
template <int DT, bool F8, int DP>
int launch_dim(const Params& p, cudaStream_t stream, int64_t* bytes) {
  if (p.logit_softcap > (DT == HIPATTN_F32 ? 0.f : kShortCap)) return launch_heads<DT, F8, DP, true>(p, stream, bytes);
  return launch_heads<DT, F8, DP, false>(p, stream, bytes);
}
template <int DT, bool F8>
int launch_type(const Params& p, cudaStream_t stream, int64_t* bytes) {
  switch (padded_dim(p.D)) {
    case 64: return launch_dim<DT, F8, 64>(p, stream, bytes);
    case 128: return launch_dim<DT, F8, 128>(p, stream, bytes);
    default: return launch_dim<DT, F8, 256>(p, stream, bytes);
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
  HIPATTN_REQUIRE(p->logit_softcap >= 0.f && p->logit_softcap < INFINITY && fabsf(p->sm_scale) < INFINITY, HIPATTN_ERR_INVALID,
                  "paged_decode: scale %g and soft-cap %g must be finite, the cap not negative", p->sm_scale, p->logit_softcap);
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

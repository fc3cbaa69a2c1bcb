// Next tokens from logits: temperature, top-k, top-p and min-p, by inversion from one given uniform number a row.
// Bound by HBM and by 64-bit arithmetic alike: every logit is read once and takes one exponential.
//
// m = max x, e_i = exp((x_i - m) / temperature); order: x descending, index ascending.
//   S1 = the first top_k,  S2 = the shortest prefix of S1 with mass >= top_p * mass(S1),  S3 = {i in S2 : e_i >= min_p}
//   token = the first i by index with  sum_{j <= i, j in S3} e_j > u * mass(S3)
// A token next to a border of its interval, or a set next to its cut, must not depend on rounding: exponentials
// and sums are 64-bit (fp64 fma runs at the rate of fp32 here). Sets are prefixes of the order, so each is a cut
// (a value, and how many of its ties by index), found by radix selection over integer keys; masses in its histograms are
// integers of 2^-s, whose sums do not depend on the order of the atomics.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int SEG = 1024;            // logits of one wave in the first pass
constexpr int SEG_LANE = SEG / 64;   // per lane
constexpr int SUBS = 16;             // maxima kept of a segment where top-k asks for them, one per four lanes
constexpr int64_t MAX_SEGS = 4096;   // vocabularies up to 4 Mi
constexpr int LIST = 4096;           // candidates held in LDS
constexpr double LOG2E = 1.4426950408889634;

// Logit types: VEC elements of 16 bytes, loaded from any element (unaligned access is enabled on gfx950).
struct F32 {
  typedef float S;
  typedef f32x4 Vec __attribute__((aligned(4)));
  static constexpr int VEC = 4, LOW = 0;  // LOW: bits of an fp32 key that are the same for all values of the type
  static DEVI void widen(const f32x4& v, float* o) { o[0] = v[0]; o[1] = v[1]; o[2] = v[2]; o[3] = v[3]; }
  static DEVI float one(float v) { return v; }
};
struct BF16 {
  typedef u16 S;
  typedef u32x4 Vec __attribute__((aligned(2)));
  static constexpr int VEC = 8, LOW = 16;
  static DEVI void widen(const u32x4& v, float* o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __builtin_bit_cast(float, v[i] << 16);
      o[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xffff0000u);
    }
  }
  static DEVI float one(u16 v) { return bf16_bits_to_f32(v); }
};
struct FP16 {
  typedef _Float16 S;
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  typedef f16x8 Vec __attribute__((aligned(2)));
  static constexpr int VEC = 8, LOW = 13;
  static DEVI void widen(const f16x8& v, float* o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)v[i];
  }
  static DEVI float one(_Float16 v) { return (float)v; }
};

// Fixed-size view of a call, by value to every kernel. *_rows: one entry a row, or null for the scalar.
struct Call {
  const void* logits;
  int64_t ld;
  int V, segs;
  const void* uniforms;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const void* top_k_rows;
  double temperature, top_p, min_p;
  int64_t top_k;
  int wide_uniforms, wide_top_k, subs, fixed_bits;
  int64_t* tokens;
  float *logprobs, *full_logprobs;
  uint32_t* kept;
  int64_t kept_ld;
  // workspace, for the rows of one launch
  float* seg_max;
  double* seg_sum;
  float* sub_max;
  float* cut;      // [rows]: kept are logits above it,
  int* cut_index;  // and those equal to it up to this index
};

// A row's settings. top_k: V where there is no limit; top1: the first of the order alone.
struct Settings {
  double c;  // log2(e) / temperature
  double top_p, min_p;
  int64_t top_k;
  bool top1, greedy, bad;
};
DEVI Settings settings_of(const Call& a, int64_t row) {
  Settings s;
  const double tau = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  s.top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  s.min_p = a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p;
  s.top_k = a.top_k_rows == nullptr ? a.top_k
            : a.wide_top_k          ? ((const int64_t*)a.top_k_rows)[row]
                                    : (int64_t)((const int32_t*)a.top_k_rows)[row];
  if (s.top_k <= 0 || s.top_k > a.V) s.top_k = a.V;
  s.bad = tau != tau || s.top_p != s.top_p || s.min_p != s.min_p;
  s.greedy = tau <= 0.;
  s.top1 = s.greedy || s.top_k == 1 || s.top_p <= 0.;
  s.min_p = fmin(s.min_p, 1.);
  s.c = s.greedy ? LOG2E : fmin(LOG2E / tau, 1e300);  // (finite: the largest logit has weight 1 at any temperature)
  return s;
}

// 2^t for t <= 0. 2^f = 1 + f q(f) on [-1/2, 1/2], q interpolated at the Chebyshev nodes (relative error of 2^f 2.2e-12;
// exactly 1 at 0): a token is drawn wrongly if its uniform number falls that close to a border, which at 150,000
// tokens of equal weight happens to one row in 10^6. Results below 2^-1000 are taken as that.
DEVI double exp2_low(double t) {
  t = fmax(t, -1000.);
  constexpr double MAGIC = 6755399441055744.;  // 1.5 * 2^52: the sum's low bits are the nearest integer
  const double s = t + MAGIC, f = t - (s - MAGIC);
  double q = 0x1.63b2d7960e61cp-20;
  q = fma(q, f, 0x1.00c0e4e159a42p-16);
  q = fma(q, f, 0x1.4308c7183e3d5p-13);
  q = fma(q, f, 0x1.5d87759835031p-10);
  q = fma(q, f, 0x1.3b2ab70ad255fp-7);
  q = fma(q, f, 0x1.c6b08da70cce4p-5);
  q = fma(q, f, 0x1.ebfbdff82a734p-3);
  q = fma(q, f, 0x1.62e42fef9cc69p-1);
  const double r = fma(q, f, 1.);
  int2 b = __builtin_bit_cast(int2, r);
  b.y += __builtin_bit_cast(int2, s).x << 20;
  return __builtin_bit_cast(double, b);
}
// The same, and 0 from 2^-1000 down (also for a NaN, which -inf times a rate of 0 is).
DEVI double weight_of(float x, double m, double c) {
  const double t = ((double)x - m) * c;
  return t > -1000. ? exp2_low(t) : 0.;
}

// Integers in the order of the floats; -0 and +0 are the same.
DEVI uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
DEVI float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// Element g * VEC + j of a lane is logit base + (g * 64 + lane) * VEC + j; behind the row: -inf.
template <class E, bool NT = false>
DEVI void load_seg(const typename E::S* row, int base, int V, int lane, float (&x)[SEG_LANE]) {
  constexpr int VEC = E::VEC, G = SEG_LANE / VEC;
  if (base + SEG <= V) {
    typename E::Vec v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const auto* const at = (const typename E::Vec*)(row + base + (g * 64 + lane) * VEC);
      v[g] = NT ? __builtin_nontemporal_load(at) : *at;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) E::widen(v[g], x + g * VEC);
  } else {
#pragma unroll
    for (int i = 0; i < SEG_LANE; ++i) {
      const int at = base + ((i / VEC) * 64 + lane) * VEC + i % VEC;
      x[i] = at < V ? E::one(row[at]) : neg_inf();
    }
  }
}

// First pass, a wave per segment: its largest logit and the mass relative to that.
template <class E, bool NT>
__global__ __launch_bounds__(256) void sample_segments_kernel(Call a, unsigned units, int64_t row0) {
  const unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int lane = threadIdx.x & 63;
  const unsigned r = unit / (unsigned)a.segs;
  const int seg = (int)(unit - r * (unsigned)a.segs);
  const int64_t row = row0 + r;
  float x[SEG_LANE];
  load_seg<E, NT>((const typename E::S*)a.logits + row * a.ld, seg * SEG, a.V, lane, x);
  const Settings s = settings_of(a, row);
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < SEG_LANE; ++i) mx = stat_max(mx, x[i]);  // a NaN stays
  if (a.subs) {
    float q = stat_max(mx, dpp_move<0xb1>(mx, mx));  // quad_perm [1,0,3,2]
    q = stat_max(q, dpp_move<0x4e>(q, q));           // quad_perm [2,3,0,1]
    if ((lane & 3) == 0) a.sub_max[(int64_t)unit * SUBS + (lane >> 2)] = q;
  }
  mx = wave_stat_max(mx);
  double sum = 0.;
  if (mx > neg_inf()) {  // (rows with a NaN or +inf come out bad whatever their sums are)
    const double m = mx;
#pragma unroll
    for (int i = 0; i < SEG_LANE; ++i) sum += exp2_low(((double)x[i] - m) * s.c);
    sum = wave_sum(sum);
  }
  if (lane == 0) {
    a.seg_max[unit] = mx;
    a.seg_sum[unit] = sum;
  }
}

template <int WAVES, class T>
struct BlockScan {
  T part[WAVES];
  // Exclusive prefix of the threads' values (in thread order, the same for every run) and their total.
  DEVI T exclusive(T v, T& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T incl = wave_inclusive_scan(v, T(0), [](T x, T y) { return x + y; });
    __syncthreads();  // an earlier scan's readers
    if (lane == 63) part[w] = incl;
    __syncthreads();
    T base = T(0), all = T(0);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      if (i == w) base = all;
      all += part[i];
    }
    total = all;
    return base + wave_shift_up(incl, T(0));
  }
};

struct Picked {
  int index;    // -1: no element with a weight
  bool inside;  // the target lies in it (else: the last with a weight)
};
// The first element in index order whose running sum (from `base`) passes `target`, by one wave.
template <class E>
DEVI Picked wave_pick(const double (&w)[SEG_LANE], int seg_base, double base, double target, int lane) {
  constexpr int VEC = E::VEC, G = SEG_LANE / VEC;
  int last = -1;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    double s = 0.;
    int mine = -1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      s += w[g * VEC + j];
      if (w[g * VEC + j] > 0.) mine = seg_base + (g * 64 + lane) * VEC + j;
    }
    const double incl = wave_inclusive_scan(s, 0., [](double x, double y) { return x + y; });
    const unsigned long long cross = __builtin_amdgcn_ballot_w64(s > 0. && base + incl > target);
    if (cross != 0) {
      const int at = __builtin_ctzll(cross);
      double cum = base + wave_shift_up(incl, 0.);
      int found = mine;  // rounding may leave it to the lane's last
      bool open = true;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        cum += w[g * VEC + j];
        if (open && w[g * VEC + j] > 0. && cum > target) {
          found = seg_base + (g * 64 + lane) * VEC + j;
          open = false;
        }
      }
      return {__builtin_amdgcn_readlane(found, at), true};
    }
    const unsigned long long any = __builtin_amdgcn_ballot_w64(mine >= 0);
    if (any != 0) last = __builtin_amdgcn_readlane(mine, 63 - __builtin_clzll(any));
    base += lane_value(incl, 63);
  }
  return {last, false};
}

// Positions of flagged elements (bit g * VEC + j of `flags`) in index order: starts[g] of a lane's first in group g,
// counted from `base`. Returns the wave's number of them.
template <class E>
DEVI int order_in_wave(unsigned flags, int base, int (&starts)[SEG_LANE / E::VEC]) {
  constexpr int VEC = E::VEC, G = SEG_LANE / VEC;
  int at = base;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int n = __popc((flags >> (g * VEC)) & ((1u << VEC) - 1));
    const int incl = wave_inclusive_scan(n, 0, [](int x, int y) { return x + y; });
    starts[g] = at + incl - n;
    at += lane_value(incl, 63);
  }
  return at - base;
}

// A row's cut and its token, one workgroup a row.
template <int THREADS>
struct RowShared {
  static constexpr int WAVES = THREADS / 64;
  BlockScan<WAVES, double> scan_f64;
  BlockScan<WAVES, int> scan_int;
  unsigned long long mass[256];
  uint32_t count[256];
  union {
    struct {
      uint32_t key[LIST];
      int index[LIST];
    } list;
    struct {
      double mass[MAX_SEGS];
      int ties[MAX_SEGS];
    } seg;
  };
  unsigned short active[MAX_SEGS];
  unsigned long long above;
  int bin, ties, first, last, wave_count[WAVES];
  uint32_t low_key;
  int cut_index;
  float xmax[WAVES];
  double target;
};

template <class E, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_rows_kernel(Call a, int64_t row0) {
  constexpr int VEC = E::VEC, G = SEG_LANE / VEC, WAVES = THREADS / 64, LOW = E::LOW;
  __shared__ RowShared<THREADS> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned r = blockIdx.x;
  const int64_t row = row0 + r;
  const typename E::S* x_row = (const typename E::S*)a.logits + row * a.ld;
  const float* seg_max = a.seg_max + (int64_t)r * a.segs;
  const double* seg_sum = a.seg_sum + (int64_t)r * a.segs;
  const Settings s = settings_of(a, row);
  double u = a.wide_uniforms ? ((const double*)a.uniforms)[row] : (double)((const float*)a.uniforms)[row];
  u = fmin(fmax(u, 0.), 1.);

  const int per = (a.segs + THREADS - 1) / THREADS;  // segments of a thread, in order
  const int seg_begin = min(tid * per, a.segs), seg_end = min(seg_begin + per, a.segs);
  float mx = neg_inf();
  for (int i = seg_begin; i < seg_end; ++i) mx = stat_max(mx, seg_max[i]);
  mx = wave_stat_max(mx);
  if (lane == 0) sh.xmax[wave] = mx;
  if (tid == 0) {
    sh.first = 0x7fffffff;
    sh.last = -1;
    sh.low_key = 0xffffffffu;
    sh.cut_index = -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) mx = stat_max(mx, sh.xmax[i]);
  if (s.bad || !(mx < pos_inf()) || !(mx > neg_inf())) {  // NaN, +inf, or nothing but -inf
    if (tid == 0) {
      a.tokens[row] = -1;
      a.logprobs[row] = a.full_logprobs[row] = __builtin_nanf("");
      a.cut[r] = pos_inf();
      a.cut_index[r] = -1;
    }
    return;
  }
  const double m = mx;
  double own = 0.;
  for (int i = seg_begin; i < seg_end; ++i) own += seg_sum[i] * weight_of(seg_max[i], m, s.c);
  double all_mass;
  const double before = sh.scan_f64.exclusive(own, all_mass);

  // Results, by thread 0. z: the mass of the kept set.
  auto finish = [&](int token, double z, float cut, int cut_index) {
    const double d = ((double)E::one(x_row[token]) - m) * s.c;
    constexpr double LN2 = 0.6931471805599453;
    a.tokens[row] = token;
    a.logprobs[row] = (float)(s.top1 ? 0. : fma(d, LN2, -log(z)));
    a.full_logprobs[row] = (float)(s.greedy ? 0. : fma(d, LN2, -log(all_mass)));
    a.cut[r] = cut;
    a.cut_index[r] = cut_index;
  };

  if (s.top1) {  // the lowest index of the largest logit
    for (int i = seg_begin; i < seg_end; ++i)
      if (seg_max[i] == mx) {
        atomicMin(&sh.first, i);
        break;
      }
    __syncthreads();
    if (wave == 0) {
      const int seg = sh.first;
      float x[SEG_LANE];
      load_seg<E>(x_row, seg * SEG, a.V, lane, x);
      int at = 0x7fffffff;
#pragma unroll
      for (int i = SEG_LANE - 1; i >= 0; --i)
        if (x[i] == mx) at = seg * SEG + ((i / VEC) * 64 + lane) * VEC + i % VEC;
      at = wave_reduce(at, [](int p, int q) { return p < q ? p : q; });
      if (lane == 0) finish(at, 1., mx, at);
    }
    return;
  }

  const bool use_k = s.top_k < a.V, use_p = s.top_p < 1., use_min = s.min_p > 0.;
  if (!use_k && !use_p && !use_min) {  // the whole distribution: only the segment with the target is read again
    const double target = u * all_mass;
    double cum = before;
    for (int i = seg_begin; i < seg_end; ++i) {
      const double w = seg_sum[i] * weight_of(seg_max[i], m, s.c);
      if (w > 0.) {
        if (cum + w > target) {
          atomicMin(&sh.first, i);
          break;
        }
        atomicMax(&sh.last, i);
      }
      cum += w;
    }
    __syncthreads();
    const int seg = sh.first != 0x7fffffff ? sh.first : sh.last;
    if (seg >= seg_begin && seg < seg_end) {
      double c2 = before;
      for (int i = seg_begin; i < seg; ++i) c2 += seg_sum[i] * weight_of(seg_max[i], m, s.c);
      sh.target = c2;
    }
    __syncthreads();
    if (wave == 0) {
      float x[SEG_LANE];
      double w[SEG_LANE];
      load_seg<E>(x_row, seg * SEG, a.V, lane, x);
#pragma unroll
      for (int i = 0; i < SEG_LANE; ++i) w[i] = weight_of(x[i], m, s.c);
      const Picked p = wave_pick<E>(w, seg * SEG, sh.target, target, lane);
      if (lane == 0) finish(p.index, all_mass, neg_inf(), -1);
    }
    return;
  }

  // ---- a lower bound on the kept logits, so that few candidates are looked at ----
  // clears the counts, then `add` fills them; the descending bin in which the running count reaches `want`
  auto select_bin = [&](int64_t want) {
    __syncthreads();
    if (wave == 0) {
      uint32_t c[4];
      int n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) n += (int)(c[i] = sh.count[255 - 4 * lane - i]);
      const int incl = wave_inclusive_scan(n, 0, [](int x, int y) { return x + y; });
      if (incl - n < want && incl >= want) {
        int cum = incl - n;
        bool open = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (open && cum + (int)c[i] >= want) {
            sh.bin = 255 - 4 * lane - i;
            sh.above = (unsigned long long)cum;
            sh.ties = (int)c[i];
            open = false;
          }
          cum += (int)c[i];
        }
      }
    }
    __syncthreads();
  };
  auto clear_bins = [&] {
    __syncthreads();
    for (int i = tid; i < 256; i += THREADS) {
      sh.count[i] = 0;
      sh.mass[i] = 0;
    }
    __syncthreads();
  };
  const uint32_t top_key = key_of(mx);
  double bound = -1.7e308;
  // No token lighter than this is in S2: all those together weigh less than (1 - top_p) of the mass.
  if (use_p && !use_k) bound = fmax(bound, m + log2((1. - s.top_p) * all_mass / a.V) / s.c);
  if (use_min && !(use_k && use_p)) bound = fmax(bound, m + log2(s.min_p) / s.c);  // (else S1's whole mass is needed)
  bound -= 1e-6 * fabs(bound) + 1e-6 / s.c;
  float low = bound > -3.4e38 ? (float)bound : -3.402823466e38f;
  if (use_k && a.subs && s.top_k <= (int64_t)a.segs * SUBS) {
    // top_k maxima of disjoint parts of the row are that many logits: the top_k-th largest of the row is no lower than
    // theirs. Its upper 16 bits are enough.
    const float* subs = a.sub_max + (int64_t)r * a.segs * SUBS;
    const int n = a.segs * SUBS;
    uint32_t prefix = 0;
    int64_t want = s.top_k;
#pragma unroll
    for (int shift = 24; shift >= 16; shift -= 8) {
      clear_bins();
      for (int i = tid; i < n; i += THREADS) {
        const uint32_t key = key_of(subs[i]);
        if (shift == 24 || (key >> 24) == (prefix >> 24)) atomicAdd(&sh.count[(key >> shift) & 255], 1u);
      }
      select_bin(want);
      prefix |= (uint32_t)sh.bin << shift;
      want -= (int64_t)sh.above;
    }
    const float lowest = value_of(prefix);
    if (lowest > low) low = lowest;  // (not where it is a NaN's pattern, below that of -inf)
  }

  // ---- the segments and the logits that reach it, in index order ----
  int mine = 0;
  for (int i = seg_begin; i < seg_end; ++i) mine += seg_max[i] >= low;
  int n_active;
  int at = sh.scan_int.exclusive(mine, n_active);
  for (int i = seg_begin; i < seg_end; ++i)
    if (seg_max[i] >= low) sh.active[at++] = (unsigned short)i;
  __syncthreads();
  int n_cand = 0;
  for (int i0 = 0; i0 < n_active; i0 += WAVES) {
    float x[SEG_LANE];
    unsigned flags = 0;
    int base = 0;
    if (i0 + wave < n_active) {
      base = (int)sh.active[i0 + wave] * SEG;
      load_seg<E>(x_row, base, a.V, lane, x);
#pragma unroll
      for (int i = 0; i < SEG_LANE; ++i) flags |= (x[i] >= low ? 1u : 0u) << i;
    }
    int starts[G];
    const int n = order_in_wave<E>(flags, 0, starts);
    if (lane == 0) sh.wave_count[wave] = n;
    __syncthreads();
    int to = n_cand;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) to = n_cand;
      n_cand += sh.wave_count[w];
    }
    if (flags != 0) {
#pragma unroll
      for (int i = 0; i < SEG_LANE; ++i) {
        if (flags >> i & 1) {
          const int p = to + starts[i / VEC] + __popc((flags >> (i / VEC * VEC)) & ((1u << (i % VEC)) - 1));
          if (p < LIST) {
            sh.list.key[p] = key_of(x[i]);
            sh.list.index[p] = base + ((i / VEC) * 64 + lane) * VEC + i % VEC;
          }
        }
      }
    }
    __syncthreads();
  }
  const bool listed = n_cand <= LIST;

  // f(key) of every candidate, in any order
  auto each = [&](auto f) {
    if (listed) {
      for (int i = tid; i < n_cand; i += THREADS) f(sh.list.key[i]);
    } else {
      for (int i = wave; i < n_active; i += WAVES) {
        float x[SEG_LANE];
        load_seg<E>(x_row, (int)sh.active[i] * SEG, a.V, lane, x);
#pragma unroll
        for (int j = 0; j < SEG_LANE; ++j)
          if (x[j] >= low) f(key_of(x[j]));
      }
    }
  };
  // Bits in which the candidates' keys can differ, downwards from `top_bits`.
  const uint32_t low_key = key_of(low);
  const int top_bits = low_key == top_key ? 0 : 32 - __builtin_clz(low_key ^ top_key);
  auto whole_key = [&](uint32_t prefix) {  // the type's own lowest bits: 0, or of negative values 1
    return prefix | ((prefix >> 31) ? 0u : (1u << LOW) - 1);
  };

  // ---- top-k: the key of the last logit of S1 and how many of its ties are in ----
  uint32_t cut_key = 0;
  int take = 0x7fffffff;
  unsigned long long tied_out = 0;  // mass of the ties of cut_key that are not in S1
  const bool cut_k = use_k && n_cand > s.top_k;
  const double unit = (double)(1ull << a.fixed_bits);
  auto fixed_mass = [&](uint32_t key) {  // 2^52 plus it has it in the low bits, rounded
    const double w = fma(weight_of(value_of(key), m, s.c), unit, 4503599627370496.);
    return __builtin_bit_cast(unsigned long long, w) & 0xfffffffffffffull;
  };
  if (cut_k) {
    uint32_t mask = top_bits == 32 ? 0 : ~0u << top_bits, prefix = top_key & mask;
    int64_t want = s.top_k;
    int ties = n_cand;
    for (int bits = top_bits; bits > LOW;) {
      const int shift = max(bits - 8, LOW);
      clear_bins();
      each([&](uint32_t key) {
        if ((key & mask) == prefix) atomicAdd(&sh.count[(key >> shift) & ((1u << (bits - shift)) - 1)], 1u);
      });
      select_bin(want);
      prefix |= (uint32_t)sh.bin << shift;
      mask = ~0u << shift;
      want -= (int64_t)sh.above;
      ties = sh.ties;
      bits = shift;
    }
    cut_key = whole_key(prefix);
    take = (int)want;
    tied_out = (unsigned long long)(ties - take) * fixed_mass(cut_key);
  }

  // ---- top-p inside S1 ----
  if (use_p) {
    uint32_t mask = top_bits == 32 ? 0 : ~0u << top_bits, prefix = top_key & mask;
    unsigned long long want = 0;
    bool found = true;
    int bits = top_bits;
    bool first = true;
    do {
      const int shift = max(bits - 8, LOW);
      const uint32_t field = (1u << (max(bits, shift) - shift)) - 1;
      clear_bins();
      each([&](uint32_t key) {
        if ((key & mask) == prefix && key >= cut_key) atomicAdd(&sh.mass[(key >> shift) & field], fixed_mass(key));
      });
      __syncthreads();
      if (wave == 0) {
        unsigned long long c[4], n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += c[i] = sh.mass[255 - 4 * lane - i];
        const unsigned long long incl =
            wave_inclusive_scan(n, 0ull, [](unsigned long long x, unsigned long long y) { return x + y; });
        if (first) {  // in S2: what has less than top_p of S1's mass in front of it
          const double z1 = use_k ? (double)(lane_value(incl, 63) - tied_out) : all_mass * unit;
          want = (unsigned long long)ceil(s.top_p * z1);
          if (want == 0) want = 1;
        }
        if (lane == 0) sh.bin = -1;
        if (incl - n < want && incl >= want) {
          unsigned long long cum = incl - n;
          bool open = true;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (open && cum + c[i] >= want) {
              sh.bin = 255 - 4 * lane - i;
              sh.above = want - cum;
              open = false;
            }
            cum += c[i];
          }
        }
      }
      __syncthreads();
      first = false;
      if (sh.bin < 0) {  // less mass than that among the candidates: all of them stay
        found = false;
        break;
      }
      prefix |= (uint32_t)sh.bin << shift;
      mask = ~0u << shift;
      want = sh.above;
      bits = shift;
    } while (bits > LOW);
    if (found) {
      const uint32_t key = whole_key(prefix);
      const unsigned long long w = fixed_mass(key);
      const int ties = w == 0 ? 0x7fffffff : (int)min((want + w - 1) / w, 0x7fffffffull);
      take = key == cut_key ? min(take, ties) : ties;
      cut_key = key;
    }
  }

  // ---- the token, in index order; and the cut of the kept set ----
  // kept: key > cut_key, or among the first `take` of its ties; and heavy enough
  if (listed) {
    constexpr int PER = LIST / THREADS;
    const int i0 = tid * PER;
    double w[PER];
    int tied = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) tied += i0 + i < n_cand && sh.list.key[i0 + i] == cut_key;
    int all_tied;
    int rank = sh.scan_int.exclusive(tied, all_tied);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      w[i] = 0.;
      if (i0 + i < n_cand) {
        const uint32_t key = sh.list.key[i0 + i];
        const bool in = key > cut_key || (key == cut_key && rank < take);
        rank += key == cut_key;
        const double e = weight_of(value_of(key), m, s.c);
        if (in && e >= s.min_p) {
          w[i] = e;
          sum += e;
          atomicMin(&sh.low_key, key);
        }
      }
    }
    double z;
    double cum = sh.scan_f64.exclusive(sum, z);
    const double target = u * z;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cum += w[i];
      if (w[i] > 0.) {
        if (cum > target) atomicMin(&sh.first, i0 + i);
        atomicMax(&sh.last, i0 + i);
      }
    }
    const uint32_t lowest = sh.low_key;
    rank -= tied;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i0 + i < n_cand && sh.list.key[i0 + i] == lowest) {
        if (lowest != cut_key || rank < take) atomicMax(&sh.cut_index, sh.list.index[i0 + i]);
        rank += lowest == cut_key;
      }
    __syncthreads();
    if (tid == 0)
      finish(sh.list.index[sh.first != 0x7fffffff ? sh.first : sh.last], z, value_of(lowest), sh.cut_index);
    return;
  }
  // Too many for the list: once over the segments for their ties, once for their masses, the token's once more.
  // (`list` is not read any more, `seg` takes its place.)
  __syncthreads();
  for (int i = wave; i < n_active; i += WAVES) {
    float x[SEG_LANE];
    load_seg<E>(x_row, (int)sh.active[i] * SEG, a.V, lane, x);
    int n = 0;
#pragma unroll
    for (int j = 0; j < SEG_LANE; ++j) n += x[j] >= low && key_of(x[j]) == cut_key;
    n = wave_sum(n);
    if (lane == 0) sh.seg.ties[i] = n;
  }
  __syncthreads();
  const int act_per = (n_active + THREADS - 1) / THREADS;
  const int act_begin = min(tid * act_per, n_active), act_end = min(act_begin + act_per, n_active);
  {
    int n = 0, total;
    for (int i = act_begin; i < act_end; ++i) n += sh.seg.ties[i];
    int cum = sh.scan_int.exclusive(n, total);
    for (int i = act_begin; i < act_end; ++i) {
      const int own_ties = sh.seg.ties[i];
      sh.seg.ties[i] = cum;
      cum += own_ties;
    }
  }
  __syncthreads();
  // weights of the kept logits of active segment i; the lowest key among them and its last index
  auto kept_weights = [&](int i, double (&w)[SEG_LANE], float (&x)[SEG_LANE]) {
    load_seg<E>(x_row, (int)sh.active[i] * SEG, a.V, lane, x);
    unsigned tied = 0;
#pragma unroll
    for (int j = 0; j < SEG_LANE; ++j) tied |= (x[j] >= low && key_of(x[j]) == cut_key ? 1u : 0u) << j;
    int starts[G];
    order_in_wave<E>(tied, sh.seg.ties[i], starts);
#pragma unroll
    for (int j = 0; j < SEG_LANE; ++j) {
      const uint32_t key = key_of(x[j]);
      const int rank = starts[j / VEC] + __popc((tied >> (j / VEC * VEC)) & ((1u << (j % VEC)) - 1));
      const bool in = x[j] >= low && (key > cut_key || (key == cut_key && rank < take));
      const double e = weight_of(x[j], m, s.c);
      const bool keep = in && e >= s.min_p;
      w[j] = keep ? e : 0.;
      if (!keep) x[j] = pos_inf();
    }
  };
  for (int i = wave; i < n_active; i += WAVES) {
    double w[SEG_LANE], sum = 0.;
    float x[SEG_LANE];
    kept_weights(i, w, x);
    float lowest = x[0];
#pragma unroll
    for (int j = 0; j < SEG_LANE; ++j) {
      sum += w[j];
      lowest = fminf(lowest, x[j]);
    }
    sum = wave_sum(sum);
    lowest = wave_min(lowest);
    if (lane == 0) {
      sh.seg.mass[i] = sum;
      if (lowest < pos_inf()) atomicMin(&sh.low_key, key_of(lowest));
    }
  }
  __syncthreads();
  double own_mass = 0.;
  for (int i = act_begin; i < act_end; ++i) own_mass += sh.seg.mass[i];
  double z;
  const double front = sh.scan_f64.exclusive(own_mass, z);
  const double target = u * z;
  double cum = front;
  for (int i = act_begin; i < act_end; ++i) {
    const double w = sh.seg.mass[i];
    if (w > 0.) {
      if (cum + w > target) {
        atomicMin(&sh.first, i);
        break;
      }
      atomicMax(&sh.last, i);
    }
    cum += w;
  }
  __syncthreads();
  const int chosen = sh.first != 0x7fffffff ? sh.first : sh.last;
  if (chosen >= act_begin && chosen < act_end) {
    double c2 = front;
    for (int i = act_begin; i < chosen; ++i) c2 += sh.seg.mass[i];
    sh.target = c2;
  }
  const float lowest = value_of(sh.low_key);
  if (a.kept != nullptr) {  // its last index among the kept
    for (int i = wave; i < n_active; i += WAVES) {
      double w[SEG_LANE];
      float x[SEG_LANE];
      kept_weights(i, w, x);
      int last = -1;
#pragma unroll
      for (int j = 0; j < SEG_LANE; ++j)
        if (x[j] == lowest) last = (int)sh.active[i] * SEG + ((j / VEC) * 64 + lane) * VEC + j % VEC;
      last = wave_reduce(last, [](int p, int q) { return p > q ? p : q; });
      if (lane == 0 && last >= 0) atomicMax(&sh.cut_index, last);
    }
  }
  __syncthreads();
  if (wave == 0) {
    double w[SEG_LANE];
    float x[SEG_LANE];
    kept_weights(chosen, w, x);
    const Picked p = wave_pick<E>(w, (int)sh.active[chosen] * SEG, sh.target, target, lane);
    if (lane == 0) finish(p.index, z, lowest, sh.cut_index);
  }
}

// The kept sets as bits, a wave per segment (32 words); segments below the cut are not read.
template <class E>
__global__ __launch_bounds__(256) void sample_kept_kernel(Call a, unsigned units, int64_t row0) {
  const unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  constexpr int VEC = E::VEC;
  const int lane = threadIdx.x & 63;
  const unsigned r = unit / (unsigned)a.segs;
  const int seg = (int)(unit - r * (unsigned)a.segs), base = seg * SEG;
  const float cut = a.cut[r];
  const int cut_index = a.cut_index[r];
  unsigned flags = 0;  // bit g * VEC + j
  if (a.seg_max[unit] >= cut) {
    float x[SEG_LANE];
    load_seg<E>((const typename E::S*)a.logits + (row0 + r) * a.ld, base, a.V, lane, x);
#pragma unroll
    for (int i = 0; i < SEG_LANE; ++i) {
      const int at = base + ((i / VEC) * 64 + lane) * VEC + i % VEC;
      flags |= (x[i] > cut || (x[i] == cut && at <= cut_index) ? 1u : 0u) << i;
    }
  }
  // word w of the segment: logits [32 w, 32 w + 32), of 32 / VEC lanes of group w * 32 / (64 * VEC)
  uint32_t word = 0;
  const int first = lane * 32 % (64 * VEC) / VEC, group = lane * 32 / (64 * VEC);
#pragma unroll
  for (int i = 0; i < 32 / VEC; ++i) {
    const uint32_t part = (uint32_t)__shfl((int)flags, (first + i) & 63, 64) >> (group * VEC & 31);
    word |= (part & ((1u << VEC) - 1)) << (i * VEC);
  }
  const int at = seg * (SEG / 32) + lane;
  if (lane < SEG / 32 && at < (a.V + 31) / 32) a.kept[(row0 + r) * a.kept_ld + at] = word;
}

// Rows of one set of launches: bounds the workspace and the number of blocks.
int64_t rows_per_launch(int64_t rows, int64_t segs) {
  return std::min(rows, std::max<int64_t>((int64_t)(1 << 22) / segs, 1));
}
struct Layout {
  int64_t rows, seg_max, seg_sum, sub_max, cut, cut_index, bytes;
  Layout(int64_t n, int64_t V) {
    const int64_t segs = ceil_div_i64(V, SEG);
    rows = rows_per_launch(n, segs);
    int64_t at = 0;
    auto take = [&](int64_t bytes_) {
      const int64_t p = at;
      at += round_up_i64(bytes_, 256);
      return p;
    };
    seg_sum = take(rows * segs * 8);
    seg_max = take(rows * segs * 4);
    sub_max = take(rows * segs * SUBS * 4);
    cut = take(rows * 4);
    cut_index = take(rows * 4);
    bytes = at;
  }
};

template <class E>
int launch_sample(Call a, int64_t n, const Layout& l, hipStream_t stream) {
  for (int64_t row0 = 0; row0 < n; row0 += l.rows) {
    const int64_t rows = std::min(l.rows, n - row0);
    const unsigned units = (unsigned)(rows * a.segs), blocks = (units + 3) / 4;
    hipLaunchKernelGGL((sample_segments_kernel<E, false>), dim3(blocks), dim3(256), 0, stream, a, units, row0);
    hipLaunchKernelGGL((sample_rows_kernel<E, 1024>), dim3((unsigned)rows), dim3(1024), 0, stream, a, row0);
    if (a.kept != nullptr)
      hipLaunchKernelGGL((sample_kept_kernel<E>), dim3(blocks), dim3(256), 0, stream, a, units, row0);
    AREAL_CHECK_LAUNCH();
  }
  return AREAL_OK;
}

}  // namespace

extern "C" {

size_t areal_sample_tokens_workspace_bytes(int64_t N, int64_t V) {
  if (N <= 0 || V <= 0 || V > MAX_SEGS * SEG) return 0;
  return (size_t)Layout(N, V).bytes;
}

int areal_sample_tokens(const void* logits, int dtype, int64_t ld, int64_t N, int64_t V, const void* uniforms,
                        int uniforms_fp64, double temperature, const float* temperature_rows, int64_t top_k,
                        const void* top_k_rows, int top_k_int64, double top_p, const float* top_p_rows, double min_p,
                        const float* min_p_rows, int64_t* tokens, float* logprobs, float* full_logprobs,
                        uint32_t* kept, int64_t kept_ld, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
  if (N < 0 || V <= 0 || ld < V || (kept != nullptr && kept_ld < ceil_div_i64(V, 32))) return AREAL_ERR_BAD_ARG;
  if ((temperature_rows == nullptr && !(temperature >= 0.)) || (top_p_rows == nullptr && !(top_p >= 0.)) ||
      (min_p_rows == nullptr && !(min_p >= 0.)))
    return AREAL_ERR_BAD_ARG;
  if (N == 0) return AREAL_OK;
  if (!logits || !uniforms || !tokens || !logprobs || !full_logprobs) return AREAL_ERR_BAD_ARG;
  if (V > MAX_SEGS * SEG) return AREAL_ERR_UNSUPPORTED;
  const Layout l(N, V);
  if (workspace == nullptr || workspace_bytes < (size_t)l.bytes) return AREAL_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return AREAL_ERR_ALIGNMENT;
  char* const ws = (char*)workspace;
  Call a{};
  a.logits = logits; a.ld = ld; a.V = (int)V; a.segs = (int)ceil_div_i64(V, SEG);
  a.uniforms = uniforms; a.wide_uniforms = uniforms_fp64 != 0;
  a.temperature = temperature; a.temperature_rows = temperature_rows;
  a.top_k = top_k; a.top_k_rows = top_k_rows; a.wide_top_k = top_k_int64 != 0;
  a.top_p = top_p; a.top_p_rows = top_p_rows; a.min_p = min_p; a.min_p_rows = min_p_rows;
  a.subs = top_k_rows != nullptr || (top_k > 1 && top_k < V);
  a.fixed_bits = 0;
  while ((1ll << (62 - a.fixed_bits - 1)) >= V && a.fixed_bits < 51) ++a.fixed_bits;  // V weights of at most 1 stay below 2^62
  a.tokens = tokens; a.logprobs = logprobs; a.full_logprobs = full_logprobs; a.kept = kept; a.kept_ld = kept_ld;
  a.seg_sum = (double*)(ws + l.seg_sum); a.seg_max = (float*)(ws + l.seg_max); a.sub_max = (float*)(ws + l.sub_max);
  a.cut = (float*)(ws + l.cut); a.cut_index = (int*)(ws + l.cut_index);
  if (dtype == 0) return launch_sample<F32>(a, N, l, stream);
  if (dtype == 1) return launch_sample<BF16>(a, N, l, stream);
  if (dtype == 2) return launch_sample<FP16>(a, N, l, stream);
  return AREAL_ERR_BAD_ARG;
}

}  // extern "C"

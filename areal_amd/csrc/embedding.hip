// Rows of the [V, H] weight for token ids, times a scale, and the weight's gradient. Bound by HBM: the forward copies
// T rows, the gradient reads T rows and writes V (or adds to the rows that occur).
//
//   out[t] = scale * weight[ids[t]]            (an id outside [0, V): zeros)
//   dweight[v] = scale * sum_{t : ids[t] = v} grad[t]   (none for ids outside [0, V) and for padding_idx)
//
// The gradient sums in fp32 in token order, the same in every run: no atomics on sums. One launch sorts the tokens by
// id, each workgroup those of a range of ids; the next adds the rows of 32 consecutive places of that order (so a
// frequent token is spread over the chip), writes ids that lie within, and clears the rows of the others; the last
// joins ids that go over the end of such a run.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace {

template <typename T> DEVI float widen1(T v);
template <> DEVI float widen1(float v) { return v; }
template <> DEVI float widen1(u16 v) { return bf16_bits_to_f32(v); }
template <> DEVI float widen1(_Float16 v) { return (float)v; }
template <typename T> DEVI T narrow1(float v);
template <> DEVI float narrow1(float v) { return v; }
template <> DEVI u16 narrow1(float v) { return f32_to_bf16_bits(v); }
// The product in front is rounded to fp32 first, as for the other types: the mixed-precision fma that the compiler
// makes of product and conversion rounds once, and makes +0 of -0.
template <> DEVI _Float16 narrow1(float v) {
  asm("" : "+v"(v));
  return (_Float16)v;
}

// VEC elements (8, aligned to 16 bytes, or 1).
template <typename T, int VEC> struct Pack { T v[VEC]; };
template <typename T, int VEC>
DEVI void load_pack(const T* p, Pack<T, VEC>& o) {
  if constexpr (VEC == 1) {
    o.v[0] = *p;
  } else {
    constexpr int N = sizeof(T) * VEC / 16;
    u32x4 raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = ((const u32x4*)p)[i];
    __builtin_memcpy(&o, raw, sizeof(o));
  }
}
template <typename T, int VEC>
DEVI void store_pack(T* p, const Pack<T, VEC>& o) {
  if constexpr (VEC == 1) {
    *p = o.v[0];
  } else {
    constexpr int N = sizeof(T) * VEC / 16;
    u32x4 raw[N];
    __builtin_memcpy(raw, &o, sizeof(o));
#pragma unroll
    for (int i = 0; i < N; ++i) ((u32x4*)p)[i] = raw[i];
  }
}

// Loads that run ahead of their use have no condition: behind the row's or the list's end they repeat its first or last
// piece. (Behind a branch each, the compiler waits for the one before: the 32 rows of embedding_sum_kernel one by one, 127
// us for 32768 x 4096 bf16 that take 60.)

// A wave takes ROW_PACKS packs per lane of one row: all loads before the first store.
constexpr int ROW_PACKS = 4;
template <typename W, typename O, int VEC>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const W* __restrict__ weight, int64_t ldw,
                                                            const int64_t* __restrict__ ids, unsigned units,
                                                            unsigned parts, int V, int H, float scale,
                                                            O* __restrict__ out) {
  const unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const unsigned t = unit / parts, part = unit - t * parts;
  const int lane = threadIdx.x & 63, begin = (int)part * (64 * VEC * ROW_PACKS) + lane * VEC;
  const int64_t id = ids[t];
  const bool in = id >= 0 && id < V;
  const W* const src = weight + (in ? id : 0) * ldw;
  O* const dst = out + (int64_t)t * H;
  Pack<W, VEC> x[ROW_PACKS];
#pragma unroll
  for (int i = 0; i < ROW_PACKS; ++i) {
    const int at = begin + i * 64 * VEC;
    load_pack<W, VEC>(src + (at < H ? at : 0), x[i]);
  }
#pragma unroll
  for (int i = 0; i < ROW_PACKS; ++i) {
    const int at = begin + i * 64 * VEC;
    if (at < H) {
      Pack<O, VEC> y;
#pragma unroll
      for (int j = 0; j < VEC; ++j) y.v[j] = narrow1<O>(in ? widen1<W>(x[i].v[j]) * scale : 0.f);
      store_pack<O, VEC>(dst + at, y);
    }
  }
}

// ---- the order of the tokens by id ----
constexpr int SORT_WAVES = 16;
constexpr int RANGE_BITS = 10;
constexpr int RANGE_MAX = 768;  // ids of a workgroup: 16 waves' counts of them take 48 KB of LDS
constexpr int SORT_UNROLL = 8;

// order[start[v] .. start[v + 1]): the tokens of id v, ascending. A workgroup reads all ids twice (from the L2 of its
// XCD) and places those of its range; how many tokens have lower ids, it counts on the way. A wave takes one run of
// tokens, so that places follow from the counts of the waves before it.
__global__ __launch_bounds__(64 * SORT_WAVES) void embedding_order_kernel(const int64_t* __restrict__ ids, int T, int V,
                                                                          int range, int64_t padding_idx,
                                                                          int* __restrict__ start,
                                                                          int* __restrict__ order) {
  extern __shared__ int counts[];  // [SORT_WAVES][range]
  __shared__ int part[SORT_WAVES], below_of[SORT_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t lo = (int64_t)blockIdx.x * range;
  const int n = (int)min((int64_t)range, V - lo);
  for (int i = tid; i < SORT_WAVES * range; i += 64 * SORT_WAVES) counts[i] = 0;
  __syncthreads();
  int* const own = counts + wave * range;
  // an odd number of 512-byte steps: with runs of 16 KB all waves of all workgroups read the same channel of an L2
  const int run = (int)(((int64_t)T + SORT_WAVES * 64 - 1) / (SORT_WAVES * 64) | 1) * 64;
  const int64_t t0 = min((int64_t)wave * run, (int64_t)T), t1 = min(t0 + run, (int64_t)T);
  // f(token, id - lo as an unsigned number): below n for ids of the range, above -lo for lower ones; SORT_UNROLL x 64
  // tokens at a time. (NONE, of ids that count nowhere, is neither: V is at most 2^31 - 2.)
  constexpr uint32_t NONE = 0xffffffffu;
  const uint32_t padding = padding_idx < 0 ? NONE : (uint32_t)padding_idx;
  auto sweep = [&](auto f) {
    for (int64_t t = t0; t < t1; t += SORT_UNROLL * 64) {
      uint2 raw[SORT_UNROLL];
#pragma unroll
      for (int i = 0; i < SORT_UNROLL; ++i) {
        const int64_t at = t + i * 64 + lane;
        raw[i] = at < t1 ? ((const uint2*)ids)[at] : make_uint2(NONE, NONE);
      }
#pragma unroll
      for (int i = 0; i < SORT_UNROLL; ++i) {
        const uint32_t id = raw[i].y == 0 && raw[i].x < (uint32_t)V && raw[i].x != padding ? raw[i].x : NONE;
        f((int)(t + i * 64 + lane), id);
      }
    }
  };
  int below = 0;
  sweep([&](int, uint32_t id) {
    below += id < (uint32_t)lo;
    if (id - (uint32_t)lo < (uint32_t)n) atomicAdd(&own[id - (uint32_t)lo], 1);
  });
  below = wave_sum(below);
  if (lane == 0) below_of[wave] = below;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) base += below_of[w];
  // thread v: id lo + v (range <= threads)
  int total = 0;
  if (tid < n)
    for (int w = 0; w < SORT_WAVES; ++w) total += counts[w * range + tid];
  const int incl = wave_inclusive_scan(total, 0, [](int x, int y) { return x + y; });
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int at = base + incl - total;
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) at += w < wave ? part[w] : 0;
  if (tid < n) {
    start[lo + tid] = at;
    if (lo + tid == V - 1) start[V] = at + total;
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int c = counts[w * range + tid];
      counts[w * range + tid] = at;
      at += c;
    }
  }
  __syncthreads();
  volatile int* const places = own;  // of this wave alone from here on
  sweep([&](int t, uint32_t id) {
    const uint32_t rel = id - (uint32_t)lo;
    const bool in = rel < (uint32_t)n;
    const unsigned long long all = __builtin_amdgcn_ballot_w64(in);
    if (all == 0) return;
    // the lanes with this lane's id: those that agree with it in every bit (a hot range has a dozen ids among 64 tokens,
    // one id at a time took 37 us of 85 at 32 Ki tokens)
    unsigned long long same = all;
#pragma unroll
    for (int bit = 0; bit < RANGE_BITS; ++bit) {
      const unsigned long long set = __builtin_amdgcn_ballot_w64(rel >> bit & 1);
      same &= rel >> bit & 1 ? set : ~set;
    }
    if (in) {
      const int to = places[rel], before = __popcll(same & ((1ull << lane) - 1));
      order[to + before] = t;
      if (before == 0) places[rel] = to + __popcll(same);
    }
  });
}

// ---- the sums ----
constexpr int RUN = 32;      // places of the order that a wave adds
constexpr int ROWS_AHEAD = 8;
constexpr int FILL_ROWS = 16;  // rows of dweight that a wave looks at to clear

struct Sums {
  const int64_t* ids;
  const int *start, *order;
  float* partial;  // [runs][2][H]: of an id that began before the run; of one that began in it and goes on
  int T, V, H;
  int* over;       // [runs]: the id that begins in the run and goes on behind it, or -1
  unsigned runs, slabs, sum_blocks;
  float scale;
};

// Writes or (ADD) adds a row's piece.
template <typename D, int VEC, bool ADD>
DEVI void put_row(D* p, const float (&acc)[VEC], float scale) {
  Pack<D, VEC> y;
  if (ADD) load_pack<D, VEC>(p, y);
#pragma unroll
  for (int j = 0; j < VEC; ++j) y.v[j] = narrow1<D>(ADD ? fmaf(acc[j], scale, widen1<D>(y.v[j])) : acc[j] * scale);
  store_pack<D, VEC>(p, y);
}

template <typename G, typename D, int VEC, bool ADD>
__global__ __launch_bounds__(256) void embedding_sum_kernel(Sums a, const G* __restrict__ grad, D* __restrict__ dweight) {
  const int lane = threadIdx.x & 63;
  const unsigned wave = threadIdx.x >> 6;
  if (blockIdx.x >= a.sum_blocks) {  // clear the rows of ids that do not occur
    const int64_t v0 = ((int64_t)(blockIdx.x - a.sum_blocks) * 4 + wave) * FILL_ROWS;
    if (v0 >= a.V) return;
    const int n = (int)min((int64_t)FILL_ROWS, a.V - v0);
    const bool empty = lane < n && a.start[v0 + lane] == a.start[v0 + lane + 1];
    unsigned long long left = __builtin_amdgcn_ballot_w64(empty);
    while (left != 0) {
      D* const row = dweight + (v0 + __builtin_ctzll(left)) * a.H;
      constexpr int STEP = VEC == 1 ? 1 : 16 / sizeof(D);  // (whole lines of 16-byte stores, whatever the type)
      for (int at = lane * STEP; at < a.H; at += 64 * STEP) {
        if constexpr (VEC == 1) row[at] = narrow1<D>(0.f);
        else *(u32x4*)(row + at) = u32x4{};
      }
      left &= left - 1;
    }
    return;
  }
  const unsigned unit = blockIdx.x * 4 + wave;
  if (unit >= a.runs * a.slabs) return;
  const unsigned run = unit / a.slabs, slab = unit - run * a.slabs;
  const int p0 = (int)run * RUN, valid = a.start[a.V];
  if (p0 >= valid) return;
  const int n = min(RUN, valid - p0);
  const int column = (int)slab * 64 * VEC + lane * VEC;
  const bool inside = column < a.H;
  const G* const grad_column = grad + (inside ? column : 0);
  // place i of the run: lane i
  int token = 0, id = -1, first = 0, end = 0;
  if (lane < n) {
    token = a.order[p0 + lane];
    id = (int)a.ids[token];
    first = a.start[id];
    end = a.start[id + 1];
  }
  if (slab == 0 && lane == n - 1) a.over[run] = first >= p0 && end > p0 + RUN ? id : -1;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  for (int i0 = 0; i0 < n; i0 += ROWS_AHEAD) {
    Pack<G, VEC> g[ROWS_AHEAD];
#pragma unroll
    for (int i = 0; i < ROWS_AHEAD; ++i) {
      const int t = __builtin_amdgcn_readlane(token, min(i0 + i, n - 1));
      load_pack<G, VEC>(grad_column + (int64_t)t * a.H, g[i]);
    }
#pragma unroll
    for (int i = 0; i < ROWS_AHEAD; ++i) {
      if (i0 + i < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += widen1<G>(g[i].v[j]);
        const int last = __builtin_amdgcn_readlane(end, i0 + i), p = p0 + i0 + i;
        if (p + 1 == last || i0 + i + 1 == n) {  // the id ends here, or the run does
          const int from = __builtin_amdgcn_readlane(first, i0 + i);
          if (inside) {
            if (from >= p0 && p + 1 == last) {
              const int v = __builtin_amdgcn_readlane(id, i0 + i);
              put_row<D, VEC, ADD>(dweight + (int64_t)v * a.H + column, acc, a.scale);
            } else {
              Pack<float, VEC> y;
#pragma unroll
              for (int j = 0; j < VEC; ++j) y.v[j] = acc[j];
              store_pack<float, VEC>(a.partial + ((int64_t)run * 2 + (from >= p0 ? 1 : 0)) * a.H + column, y);
            }
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        }
      }
    }
  }
}

// Ids that go over the end of the run they begin in: one workgroup joins the pieces of one, 64 * VEC columns at a time,
// a wave a stretch of them.
constexpr int JOIN_WAVES = 4;
template <typename D, int VEC, bool ADD>
__global__ __launch_bounds__(64 * JOIN_WAVES) void embedding_join_kernel(Sums a, D* __restrict__ dweight) {
  __shared__ float sums[JOIN_WAVES][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned run = blockIdx.x / a.slabs, slab = blockIdx.x - run * a.slabs;
  const int next = ((int)run + 1) * RUN, valid = a.start[a.V], id = a.over[run];
  if (next >= valid || id < 0) return;  // (over is written up to the last run with a token)
  const int end = a.start[id + 1];
  const int column = (int)slab * 64 * VEC + lane * VEC;
  const bool inside = column < a.H;
  // pieces: slot 1 of this run, then slot 0 of the `more` runs after it
  const int more = (end - 1) / RUN - (int)run, pieces = more + 1;
  const int per = (pieces + JOIN_WAVES - 1) / JOIN_WAVES;
  const int begin = min(wave * per, pieces), stop = min(begin + per, pieces);
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  const float* const partial = a.partial + (inside ? column : 0);
  for (int i0 = begin; i0 < stop; i0 += ROWS_AHEAD) {
    Pack<float, VEC> g[ROWS_AHEAD];
#pragma unroll
    for (int i = 0; i < ROWS_AHEAD; ++i) {
      const int piece = min(i0 + i, stop - 1);
      load_pack<float, VEC>(partial + (((int64_t)run + piece) * 2 + (piece == 0 ? 1 : 0)) * a.H, g[i]);
    }
#pragma unroll
    for (int i = 0; i < ROWS_AHEAD; ++i)
      if (i0 + i < stop) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += g[i].v[j];
      }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sums[wave][j * 64 + lane] = acc[j];
  __syncthreads();
  if (wave == 0 && inside) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      for (int w = 1; w < JOIN_WAVES; ++w) acc[j] += sums[w][j * 64 + lane];
    put_row<D, VEC, ADD>(dweight + (int64_t)id * a.H + column, acc, a.scale);
  }
}

template <class F>
int with_type(int dtype, F f) {
  if (dtype == 0) return f(float{});
  if (dtype == 1) return f(u16{});
  if (dtype == 2) return f(_Float16{});
  return AREAL_ERR_BAD_ARG;
}
// whole 16-byte steps: sizes and pitches are multiples of 8 elements, addresses of 16 bytes
bool packed8(int64_t H, int64_t ld, const void* p, const void* q) {
  return H % 8 == 0 && ld % 8 == 0 && aligned_to(p, 16) && aligned_to(q, 16);
}
constexpr int64_t MAX_THREADS = (int64_t)1 << 32;

struct BwdLayout {
  int64_t runs, start, order, over, partial, bytes;
  BwdLayout(int64_t T, int64_t H, int64_t V) {
    runs = ceil_div_i64(T, RUN);
    start = 0;
    order = round_up_i64((V + 1) * 4, 256);
    over = order + round_up_i64(T * 4, 256);
    partial = over + round_up_i64(runs * 4, 256);
    bytes = partial + runs * 2 * H * 4;
  }
};

}  // namespace

extern "C" {

int areal_embedding_fwd(const void* weight, int weight_dtype, int64_t ldw, const int64_t* ids, int64_t T, int64_t H,
                        int64_t V, float scale, void* out, int out_dtype, hipStream_t stream) {
  if (T < 0 || H <= 0 || V <= 0 || ldw < H) return AREAL_ERR_BAD_ARG;
  if (weight_dtype < 0 || weight_dtype > 2 || out_dtype < 0 || out_dtype > 2) return AREAL_ERR_BAD_ARG;
  if (T == 0) return AREAL_OK;
  if (!weight || !ids || !out) return AREAL_ERR_BAD_ARG;
  if (T > INT32_MAX || V > INT32_MAX || H > INT32_MAX / 2) return AREAL_ERR_UNSUPPORTED;
  return with_type(weight_dtype, [&](auto w) {
    return with_type(out_dtype, [&](auto o) {
      using W = decltype(w);
      using O = decltype(o);
      auto launch = [&](auto vec) -> int {
        constexpr int VEC = decltype(vec)::value;
        const int64_t parts = ceil_div_i64(H, 64 * VEC * ROW_PACKS), units = T * parts;
        if (units * 64 >= MAX_THREADS) return AREAL_ERR_UNSUPPORTED;
        hipLaunchKernelGGL((embedding_fwd_kernel<W, O, VEC>), dim3((unsigned)ceil_div_i64(units, 4)), dim3(256), 0,
                           stream, (const W*)weight, ldw, ids, (unsigned)units, (unsigned)parts, (int)V, (int)H, scale,
                           (O*)out);
        AREAL_CHECK_LAUNCH();
        return AREAL_OK;
      };
      return packed8(H, ldw, weight, out) ? launch(std::integral_constant<int, 8>{})
                                          : launch(std::integral_constant<int, 1>{});
    });
  });
}

size_t areal_embedding_bwd_workspace_bytes(int64_t T, int64_t H, int64_t V) {
  if (T < 0 || H <= 0 || V <= 0) return 0;
  return (size_t)BwdLayout(T, H, V).bytes;
}

int areal_embedding_bwd(const void* grad, int grad_dtype, const int64_t* ids, int64_t T, int64_t H, int64_t V,
                        float scale, int64_t padding_idx, void* dweight, int dweight_dtype, int accumulate,
                        void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (T < 0 || H <= 0 || V <= 0 || !dweight) return AREAL_ERR_BAD_ARG;
  if (grad_dtype < 0 || grad_dtype > 2 || dweight_dtype < 0 || dweight_dtype > 2) return AREAL_ERR_BAD_ARG;
  if (accumulate && dweight_dtype != 0) return AREAL_ERR_UNSUPPORTED;
  if (T > 0 && (!grad || !ids)) return AREAL_ERR_BAD_ARG;
  if (T == 0 && accumulate) return AREAL_OK;
  if (T > INT32_MAX - 64 || V > INT32_MAX - 1 || H > INT32_MAX / 2) return AREAL_ERR_UNSUPPORTED;
  const BwdLayout l(T, H, V);
  if (workspace == nullptr || workspace_bytes < (size_t)l.bytes) return AREAL_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return AREAL_ERR_ALIGNMENT;
  char* const ws = (char*)workspace;
  return with_type(grad_dtype, [&](auto g) {
    return with_type(dweight_dtype, [&](auto d) {
      using G = decltype(g);
      using D = decltype(d);
      auto launch = [&](auto vec) -> int {
        constexpr int VEC = decltype(vec)::value;
        Sums a{};
        a.ids = ids;
        a.start = (int*)(ws + l.start);
        a.order = (int*)(ws + l.order);
        a.partial = (float*)(ws + l.partial);
        a.T = (int)T; a.V = (int)V; a.H = (int)H; a.scale = scale;
        const int64_t slabs = ceil_div_i64(H, 64 * VEC), sum_blocks = ceil_div_i64(l.runs * slabs, 4);
        const int64_t range = std::min<int64_t>(ceil_div_i64(V, 256), RANGE_MAX);
        const int64_t ranges = ceil_div_i64(V, range);
        const int64_t fill_blocks = accumulate ? 0 : ceil_div_i64(V, 4 * FILL_ROWS);
        if ((sum_blocks + fill_blocks) * 256 >= MAX_THREADS || l.runs * slabs * 64 * JOIN_WAVES >= MAX_THREADS ||
            ranges * 64 * SORT_WAVES >= MAX_THREADS)
          return AREAL_ERR_UNSUPPORTED;
        a.over = (int*)(ws + l.over);
        a.runs = (unsigned)l.runs; a.slabs = (unsigned)slabs; a.sum_blocks = (unsigned)sum_blocks;
        hipLaunchKernelGGL(embedding_order_kernel, dim3((unsigned)ranges), dim3(64 * SORT_WAVES),
                           (size_t)range * SORT_WAVES * 4, stream, ids, (int)T, (int)V, (int)range, padding_idx,
                           (int*)(ws + l.start), (int*)(ws + l.order));
        AREAL_CHECK_LAUNCH();
        auto sums = [&](auto add) {
          constexpr bool ADD = decltype(add)::value;
          if (sum_blocks + fill_blocks > 0)
            hipLaunchKernelGGL((embedding_sum_kernel<G, D, VEC, ADD>), dim3((unsigned)(sum_blocks + fill_blocks)),
                               dim3(256), 0, stream, a, (const G*)grad, (D*)dweight);
          if (l.runs > 1)
            hipLaunchKernelGGL((embedding_join_kernel<D, VEC, ADD>), dim3((unsigned)(l.runs * slabs)),
                               dim3(64 * JOIN_WAVES), 0, stream, a, (D*)dweight);
        };
        if constexpr (std::is_same<D, float>::value) {
          if (accumulate)
            sums(std::true_type{});
          else
            sums(std::false_type{});
        } else {
          sums(std::false_type{});
        }
        AREAL_CHECK_LAUNCH();
        return AREAL_OK;
      };
      return packed8(H, 8, grad, dweight) ? launch(std::integral_constant<int, 8>{})
                                          : launch(std::integral_constant<int, 1>{});
    });
  });
}

}  // extern "C"

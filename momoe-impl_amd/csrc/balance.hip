// Load-balancing loss of a router with its counts, and its gradient.
//
// Over the Ng routed of N experts p = softmax(l) per token; for each group of S tokens (a sequence, or all of them) with T
// tokens that count and c_i of them at expert i, P = sum_i c_i over the routed ones,
//   loss_g = Ng / (T P) * sum_i c_i * sum_tokens p_i,      loss = mean of loss_g over the groups with P > 0,
//   d loss / d l_j = Ng / (T P groups) * p_j * (c_j - sum_i c_i p_i)      (the counts are constants).
// A group's softmax is passed over once forward, for the column sums of p, and once backward; nothing of size
// [tokens, experts] is kept between the two.
//
// A token's columns lie in LPT consecutive lanes, eight in each, so that a wavefront works on 64 / LPT tokens at a time, a
// lane's columns are 16 bytes (bf16) and a lane's share of the column sums stays in its registers for all its tokens.  (One
// wavefront a token, as in the router, costs ten times the instructions for 64 experts: its reductions take as many
// steps for two elements a lane as for sixteen.)
//
// Bound by launches up to some ten thousand tokens, then by the reads of the mask, four bytes an element.  Pieces, their sum, gradient:
// 8, 6, 6 us for 8192 x 128 bf16 logits, 15, 6, 9 us for 65536 x 64 (25 MB forward, 16 backward: 1.7 and 1.8 TB/s).
// The column sums of a workgroup's tokens go to the workspace and one workgroup adds them in a fixed order: the same bits each time.
// (Atomics count tokens only, whole numbers in LDS.)
#include "lanes.hpp"

namespace momoe {
namespace {

typedef _Float16 f16;
constexpr int kColsPerLane = 8;
constexpr int kMaxExperts = 64 * kColsPerLane;
constexpr int kThreadsFwd = 256, kWavesFwd = kThreadsFwd / 64;
constexpr int kThreadsSum = 1024;

struct BalanceArgs {
  const void* logits;
  int64_t ld;
  const int32_t* mask;
  int64_t sn, sm;
  const uint8_t* valid;  // [M], or NULL: all tokens count
  int S, G, N, Ng;
  int C, TB;             // a group is cut into C pieces of TB tokens, a workgroup each
  float* part_p;         // [G * C][N] column sums of p
  int32_t* part_c;       // [G * C][N] tokens at each expert
  int32_t* part_t;       // [G * C] tokens that count
  float* group_p;        // [G][N]
  float* group_loss;     // [G]
  int64_t* counts;       // [G][N]
  int64_t* kept;         // the same once more, or NULL
  float* info;           // [0]: 1 / groups with pairs (0: there are none), [1 + g]: Ng / (T P) (0: none)
  float* loss;
};

// Eight consecutive columns of a token, from `j0` on; those past the routed ones are -inf.  VEC: N and the pitch are multiples of
// eight and the rows on 16-byte boundaries.
template <class T, bool VEC>
struct Columns {
  alignas(16) T raw[kColsPerLane];
  __device__ __forceinline__ void load(const T* row, int j0, int N) {
    if constexpr (VEC) {
      struct alignas(16) Vec { T v[16 / sizeof(T)]; };
      const Vec* p = (const Vec*)(row + (j0 < N ? j0 : 0));
#pragma unroll
      for (int i = 0; i < (int)(kColsPerLane * sizeof(T) / 16); ++i) *(Vec*)(raw + i * (16 / sizeof(T))) = p[i];
    } else {
#pragma unroll
      for (int i = 0; i < kColsPerLane; ++i) raw[i] = row[min(j0 + i, N - 1)];
    }
  }
  // softmax over the Ng routed columns in the LPT lanes of the token
  template <int LPT>
  __device__ __forceinline__ void softmax(int j0, int Ng, float (&p)[kColsPerLane]) const {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kColsPerLane; ++i) {
      p[i] = j0 + i < Ng ? (float)raw[i] : -INFINITY;
      top = fmaxf(top, p[i]);
    }
    top = max_over_lanes<LPT>(top);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kColsPerLane; ++i) {
      p[i] = j0 + i < Ng ? expf(p[i] - top) : 0.0f;
      sum += p[i];
    }
    const float scale = 1.0f / sum_over_lanes<LPT>(sum);
#pragma unroll
    for (int i = 0; i < kColsPerLane; ++i) p[i] *= scale;
  }
};

__device__ __forceinline__ void store_count(const BalanceArgs& p, int64_t at, int64_t count) {
  p.counts[at] = count;
  if (p.kept != nullptr) p.kept[at] = count;
}

// The sum of one value a thread over the workgroup, in every thread; `room` holds a value per wavefront
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* room) {
  v = sum_over_lanes<64>(v);
  __syncthreads();  // (the room may still be read from the last sum)
  if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += room[w];
  return v;
}

// Column sums and counts of one piece of a group.  C == 1: the piece is all of it, and its loss follows at once.
template <class T, int LPT, bool VEC>
__global__ __launch_bounds__(kThreadsFwd) void balance_piece_kernel(BalanceArgs p) {
  constexpr int TPW = 64 / LPT, AHEAD = 4;
  __shared__ float sum_of[kWavesFwd][LPT * kColsPerLane];
  __shared__ int count_of[kMaxExperts];
  __shared__ int tokens_of;
  __shared__ float room[kWavesFwd];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int g = blockIdx.x / p.C, t0 = (blockIdx.x - g * p.C) * p.TB, t1 = min(p.S, t0 + p.TB);
  const int64_t m0 = (int64_t)g * p.S;
  for (int j = threadIdx.x; j < p.N; j += kThreadsFwd) count_of[j] = 0;
  if (threadIdx.x == 0) tokens_of = 0;
  __syncthreads();

  // p summed over the tokens, in chains of 256 at the most and then the chains: over some thousand equal terms the roundings of one
  // chain go one way
  constexpr int STEP = kWavesFwd * TPW * AHEAD, CHAIN = 256 / AHEAD * STEP;
  const int j0 = (lane % LPT) * kColsPerLane;
  float sum[kColsPerLane];
#pragma unroll
  for (int i = 0; i < kColsPerLane; ++i) sum[i] = 0.0f;
  for (int from = t0; from < t1; from += CHAIN) {
    float part[kColsPerLane];
#pragma unroll
    for (int i = 0; i < kColsPerLane; ++i) part[i] = 0.0f;
    for (int base = from + wave * TPW; base < min(t1, from + CHAIN); base += STEP) {
      Columns<T, VEC> col[AHEAD];
      bool on[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int t = base + a * kWavesFwd * TPW + lane / LPT;
        const int64_t m = m0 + min(t, t1 - 1);
        col[a].load((const T*)p.logits + m * p.ld, j0, p.N);
        on[a] = t < t1 && (p.valid == nullptr || p.valid[m] != 0);
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        float pr[kColsPerLane];
        col[a].template softmax<LPT>(j0, p.Ng, pr);
        // (a token that does not count may hold anything, NaN too)
#pragma unroll
        for (int i = 0; i < kColsPerLane; ++i) part[i] += on[a] ? pr[i] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kColsPerLane; ++i) sum[i] += part[i];
  }
#pragma unroll
  for (int i = 0; i < kColsPerLane; ++i) {
    const float all = sum_over_strides<LPT>(sum[i]);
    if (lane < LPT) sum_of[wave][j0 + i] = all;
  }

  // tokens at each expert
  if (p.sm == 1) {  // [N, M]: lanes along the tokens, an expert's 64 flags in one ballot
    constexpr int EXPERTS = 8;
    for (int t = t0; t < t1; t += 64) {
      const int64_t m = m0 + min(t + lane, t1 - 1);
      const uint64_t on = __ballot(t + lane < t1 && (p.valid == nullptr || p.valid[m] != 0));
      if (wave == 0 && lane == 0) tokens_of += __popcll(on);
      for (int jb = wave * EXPERTS; jb < p.N; jb += kWavesFwd * EXPERTS) {
        int v[EXPERTS];
#pragma unroll
        for (int e = 0; e < EXPERTS; ++e) v[e] = p.mask[(int64_t)min(jb + e, p.N - 1) * p.sn + m];
#pragma unroll
        for (int e = 0; e < EXPERTS; ++e) {
          const int here = __popcll(__ballot(v[e] != 0) & on);
          if (lane == e && jb + e < p.N) count_of[jb + e] += here;  // (an expert is this wavefront's alone)
        }
      }
    }
  } else {  // any other strides: lanes along the experts
    for (int t = t0 + wave; t < t1; t += kWavesFwd) {
      const int64_t m = m0 + t;
      if (p.valid != nullptr && p.valid[m] == 0) continue;  // wave-uniform
      if (lane == 0) atomicAdd(&tokens_of, 1);
      for (int j = lane; j < p.N; j += 64)
        if (p.mask[j * p.sn + m * p.sm] != 0) atomicAdd(&count_of[j], 1);
    }
  }
  __syncthreads();

  const auto sum_at = [&](int j) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWavesFwd; ++w) v += sum_of[w][j];
    return v;
  };
  if (p.C > 1) {
    for (int j = threadIdx.x; j < p.N; j += kThreadsFwd) {
      p.part_p[(int64_t)blockIdx.x * p.N + j] = sum_at(j);
      p.part_c[(int64_t)blockIdx.x * p.N + j] = count_of[j];
    }
    if (threadIdx.x == 0) p.part_t[blockIdx.x] = tokens_of;
    return;
  }
  float pairs = 0.0f, dot = 0.0f;
  for (int j = threadIdx.x; j < p.N; j += kThreadsFwd) {
    store_count(p, (int64_t)g * p.N + j, count_of[j]);
    if (j < p.Ng) {
      pairs += (float)count_of[j];
      dot += (float)count_of[j] * sum_at(j);
    }
  }
  pairs = block_sum<kThreadsFwd>(pairs, room);
  dot = block_sum<kThreadsFwd>(dot, room);
  if (threadIdx.x == 0) {
    const float scale = pairs > 0.0f ? (float)p.Ng / ((float)tokens_of * pairs) : 0.0f;
    const float loss = pairs > 0.0f ? scale * dot : 0.0f;
    p.info[1 + g] = scale;
    if (p.G == 1) {
      p.info[0] = pairs > 0.0f ? 1.0f : 0.0f;
      *p.loss = loss;
    } else {
      p.group_loss[g] = loss;
    }
  }
}

// One workgroup: the pieces of every group, then the groups.
__global__ __launch_bounds__(kThreadsSum) void balance_sum_kernel(BalanceArgs p) {
  __shared__ float room[kThreadsSum / 64];
  __shared__ float some_p[kThreadsSum];
  __shared__ int some_c[kThreadsSum];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  if (p.C > 1) {
    // (group, expert) pairs in `items` threads, the pieces of each in `slices` of them
    const int64_t all = (int64_t)p.G * p.N;
    int items = kThreadsSum;
    while (items / 2 >= all && kThreadsSum / items < p.C) items /= 2;
    const int slices = kThreadsSum / items, item = tid % items, slice = tid / items;
    for (int64_t base = 0; base < all; base += items) {
      const int64_t q = base + item;
      float sum = 0.0f;
      int count = 0;
      if (q < all) {
        constexpr int AHEAD = 8;
        const int64_t at = q / p.N * p.C * p.N + q % p.N;
        for (int c0 = slice; c0 < p.C; c0 += AHEAD * slices) {
          float v[AHEAD];
          int n[AHEAD];
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            const int64_t c = min(c0 + a * slices, p.C - 1);
            v[a] = p.part_p[at + c * p.N];
            n[a] = p.part_c[at + c * p.N];
          }
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            sum += c0 + a * slices < p.C ? v[a] : 0.0f;
            count += c0 + a * slices < p.C ? n[a] : 0;
          }
        }
      }
      some_p[tid] = sum;
      some_c[tid] = count;
      __syncthreads();
      if (slice == 0 && q < all) {
        for (int s = 1; s < slices; ++s) {
          sum += some_p[s * items + item];
          count += some_c[s * items + item];
        }
        p.group_p[q] = sum;
        store_count(p, q, count);
      }
      __syncthreads();
    }
    for (int g = wave; g < p.G; g += kThreadsSum / 64) {
      float tokens = 0.0f, pairs = 0.0f, dot = 0.0f;
      for (int c = lane; c < p.C; c += 64) tokens += (float)p.part_t[(int64_t)g * p.C + c];
      for (int j = lane; j < p.Ng; j += 64) {
        const float c = (float)p.counts[(int64_t)g * p.N + j];
        pairs += c;
        dot += c * p.group_p[(int64_t)g * p.N + j];
      }
      tokens = sum_over_lanes<64>(tokens);
      pairs = sum_over_lanes<64>(pairs);
      dot = sum_over_lanes<64>(dot);
      if (lane == 0) {
        const float scale = pairs > 0.0f ? (float)p.Ng / (tokens * pairs) : 0.0f;
        p.info[1 + g] = scale;
        p.group_loss[g] = pairs > 0.0f ? scale * dot : 0.0f;
      }
    }
    __syncthreads();
  }
  float loss = 0.0f, groups = 0.0f;
  for (int64_t g = tid; g < p.G; g += kThreadsSum) {
    loss += p.group_loss[g];
    groups += p.info[1 + g] != 0.0f ? 1.0f : 0.0f;
  }
  loss = block_sum<kThreadsSum>(loss, room);
  groups = block_sum<kThreadsSum>(groups, room);
  if (tid == 0) {
    p.info[0] = groups > 0.0f ? 1.0f / groups : 0.0f;
    *p.loss = groups > 0.0f ? loss / groups : 0.0f;
  }
}

struct BalanceBwdArgs {
  const void* logits;
  int64_t ld;
  const uint8_t* valid;
  const int64_t* counts;
  const float* info;
  const float* g_loss;
  const void* add;  // of the gradient's type, or NULL; may be the gradient itself
  void* out;        // [M][N]
  int S, G, N, Ng, C, TB;
};

template <class T, class U, int LPT, bool VEC>
__global__ __launch_bounds__(kThreadsFwd) void balance_bwd_kernel(BalanceBwdArgs p) {
  constexpr int TPW = 64 / LPT, AHEAD = 2;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int g = blockIdx.x / p.C, t0 = (blockIdx.x - g * p.C) * p.TB, t1 = min(p.S, t0 + p.TB);
  const int64_t m0 = (int64_t)g * p.S;
  const int j0 = (lane % LPT) * kColsPerLane;
  const float per_group = p.info[1 + g], weight = *p.g_loss * p.info[0] * per_group;
  const bool any = per_group != 0.0f;
  int64_t count[kColsPerLane];
#pragma unroll
  for (int i = 0; i < kColsPerLane; ++i) count[i] = p.counts[(int64_t)g * p.N + min(j0 + i, p.Ng - 1)];
  float c[kColsPerLane];
  for (int base = t0 + wave * TPW; base < t1; base += kWavesFwd * TPW * AHEAD) {
    Columns<T, VEC> col[AHEAD];
    Columns<U, VEC> add[AHEAD];
    bool on[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int t = base + a * kWavesFwd * TPW + lane / LPT;
      const int64_t m = m0 + min(t, t1 - 1);
      col[a].load((const T*)p.logits + m * p.ld, j0, p.N);
      if (p.add != nullptr) add[a].load((const U*)p.add + m * p.N, j0, p.N);
      on[a] = any && (p.valid == nullptr || p.valid[m] != 0);
    }
    if (base == t0 + wave * TPW) {  // (behind the first tokens' requests)
      // Counts from their mean on: the p add up to one, so that all may be less by the same, and of an even load nothing but the
      // differences is left of them.
      float all = 0.0f;
#pragma unroll
      for (int i = 0; i < kColsPerLane; ++i) all += j0 + i < p.Ng ? (float)count[i] : 0.0f;
      const int64_t mean = (int64_t)(sum_over_lanes<LPT>(all) / (float)p.Ng);
#pragma unroll
      for (int i = 0; i < kColsPerLane; ++i) c[i] = j0 + i < p.Ng ? (float)(count[i] - mean) : 0.0f;
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int t = base + a * kWavesFwd * TPW + lane / LPT;
      float pr[kColsPerLane], inner = 0.0f;
      col[a].template softmax<LPT>(j0, p.Ng, pr);
#pragma unroll
      for (int i = 0; i < kColsPerLane; ++i) inner += c[i] * pr[i];
      inner = sum_over_lanes<LPT>(inner);
      alignas(16) U out[kColsPerLane];
#pragma unroll
      for (int i = 0; i < kColsPerLane; ++i) {
        // (columns past the routed ones hold p = c = 0: their gradient is zero unless the token is NaN)
        float v = on[a] && j0 + i < p.Ng ? weight * (pr[i] * (c[i] - inner)) : 0.0f;
        if (p.add != nullptr) v += (float)add[a].raw[i];
        out[i] = (U)v;
      }
      if (t >= t1) continue;
      U* const row = (U*)p.out + (m0 + t) * p.N;
      if constexpr (VEC) {
        struct alignas(16) Vec { U v[16 / sizeof(U)]; };
        if (j0 < p.N)
#pragma unroll
          for (int i = 0; i < (int)(kColsPerLane * sizeof(U) / 16); ++i) ((Vec*)(row + j0))[i] = *(Vec*)(out + i * (16 / sizeof(U)));
      } else {
#pragma unroll
        for (int i = 0; i < kColsPerLane; ++i)
          if (j0 + i < p.N) row[j0 + i] = out[i];
      }
    }
  }
}

// How a launch cuts its groups: pieces of 16 tokens at the least, and as many as give a workgroup to each CU.
struct Plan {
  int64_t C, TB;
};
Plan plan_of(int64_t G, int64_t S, int64_t wanted, int64_t least) {
  const int64_t pieces = std::max<int64_t>(1, std::min(cdiv64(wanted, G), cdiv64(S, least)));
  const int64_t tb = cdiv64(cdiv64(S, pieces), 16) * 16;
  return {cdiv64(S, tb), tb};
}
// Forward: one piece a group, whose workgroup gives the group's loss, for up to 256 tokens in all (with one group one launch), and of
// more than 64 groups as long as these are short: what the sum of the pieces takes grows with the groups, what it saves with their
// tokens.  In a graph, us, one piece a group | pieces, of 64 experts: 65 groups of 256 tokens 15 | 19, of 512 25 | 21, of 4096 183 | 71;
// 128 of 512 26 | 31, of 1024 49 | 45, of 4096 185 | 115; 200 of 1024 52 | 62, of 4096 211 | 158; 255 of 1024 52 | 70, of 4096 211 | 174;
// of 512 experts: 65 of 256 95 | 92, of 512 186 | 120; 128 of 512 187 | 209, of 1024 413 | 336; 255 of 1024 429 | 495, of 4096 1646 | 1270.
Plan fwd_plan(int64_t G, int64_t S) {
  return G * S <= 256 || (G > 64 && S <= 7 * G) ? Plan{1, S} : plan_of(G, S, 256, 16);
}

int check_balance(int64_t G, int64_t S, int64_t N, int64_t Ks, int64_t ld) {
  if (G <= 0 || S <= 0 || N <= 0 || Ks < 0 || Ks >= N || ld < N) return MOMOE_ERR_BAD_ARG;
  return N > kMaxExperts || G > (1ll << 30) || S > (1ll << 30) || G * S > (1ll << 30) ? MOMOE_ERR_UNSUPPORTED : MOMOE_OK;
}
bool type_ok(int t) { return t == MOMOE_TYPE_BF16 || t == MOMOE_TYPE_F32 || t == MOMOE_TYPE_F16; }
int64_t type_bytes(int t) { return t == MOMOE_TYPE_F32 ? 4 : 2; }
int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }

template <class F>
void with_type(int type, F f) {
  if (type == MOMOE_TYPE_BF16) f(bf16{});
  else if (type == MOMOE_TYPE_F32) f(float{});
  else f(f16{});
}
template <class F>
void with_width(int64_t N, F f) {
  if (N <= 32) f(std::integral_constant<int, 4>{});
  else if (N <= 64) f(std::integral_constant<int, 8>{});
  else if (N <= 128) f(std::integral_constant<int, 16>{});
  else if (N <= 256) f(std::integral_constant<int, 32>{});
  else f(std::integral_constant<int, 64>{});
}

}  // namespace
}  // namespace momoe

using namespace momoe;

extern "C" int64_t momoe_balance_workspace_bytes(int64_t G, int64_t S, int64_t N) {
  if (check_balance(G, S, N, 0, N) != MOMOE_OK) return -1;
  const Plan plan = fwd_plan(G, S);
  if (plan.C == 1) return up16(4 * G);
  return up16(4 * G) + up16(4 * G * N) + 2 * up16(4 * G * plan.C * N) + up16(4 * G * plan.C);
}

extern "C" int momoe_balance_fwd(const void* logits, int logits_type, int64_t ld, const int32_t* mask_NM, int64_t stride_n,
                                 int64_t stride_m, const uint8_t* valid_M, int64_t G, int64_t S, int64_t N, int64_t Ks,
                                 float* loss, int64_t* counts_GN, float* info, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  return momoe_balance_fwd_kept(logits, logits_type, ld, mask_NM, stride_n, stride_m, valid_M, G, S, N, Ks, loss, counts_GN, nullptr,
                                info, workspace, workspace_bytes, stream);
}

extern "C" int momoe_balance_fwd_kept(const void* logits, int logits_type, int64_t ld, const int32_t* mask_NM, int64_t stride_n,
                                      int64_t stride_m, const uint8_t* valid_M, int64_t G, int64_t S, int64_t N, int64_t Ks,
                                      float* loss, int64_t* counts_GN, int64_t* kept_GN, float* info, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  if (!logits || !mask_NM || !loss || !counts_GN || !info || !workspace || !type_ok(logits_type)) return MOMOE_ERR_BAD_ARG;
  const int status = check_balance(G, S, N, Ks, ld);
  if (status != MOMOE_OK) return status;
  if (workspace_bytes < momoe_balance_workspace_bytes(G, S, N) || ((uintptr_t)workspace & 15)) return MOMOE_ERR_BAD_ARG;
  const Plan plan = fwd_plan(G, S);
  BalanceArgs a{logits, ld, mask_NM, stride_n, stride_m, valid_M, (int)S, (int)G, (int)N, (int)(N - Ks), (int)plan.C, (int)plan.TB};
  a.counts = counts_GN;
  a.kept = kept_GN;
  a.info = info;
  a.loss = loss;
  char* at = (char*)workspace;
  const auto take = [&](int64_t bytes) { char* const p = at; at += up16(bytes); return p; };
  a.group_loss = (float*)take(4 * G);
  if (plan.C > 1) {
    a.group_p = (float*)take(4 * G * N);
    a.part_p = (float*)take(4 * G * plan.C * N);
    a.part_c = (int32_t*)take(4 * G * plan.C * N);
    a.part_t = (int32_t*)take(4 * G * plan.C);
  }
  const bool vec = N % 8 == 0 && ld % 8 == 0 && ((uintptr_t)logits & 15) == 0;
  hipStream_t st = (hipStream_t)stream;
  with_type(logits_type, [&](auto type) {
    with_width(N, [&](auto lanes) {
      using T = decltype(type);
      constexpr int LPT = decltype(lanes)::value;
      auto kernel = vec ? balance_piece_kernel<T, LPT, true> : balance_piece_kernel<T, LPT, false>;
      kernel<<<(unsigned)(G * plan.C), kThreadsFwd, 0, st>>>(a);
    });
  });
  const int launched = launch_status();
  if (launched != MOMOE_OK || (G == 1 && plan.C == 1)) return launched;
  balance_sum_kernel<<<1, kThreadsSum, 0, st>>>(a);
  return launch_status();
}

extern "C" int momoe_balance_bwd(const void* logits, int logits_type, int64_t ld, const uint8_t* valid_M, const int64_t* counts_GN,
                                 const float* info, const float* G_loss, const void* add_MN, void* Glogits_MN, int grad_type,
                                 int64_t G, int64_t S, int64_t N, int64_t Ks, void* stream) {
  if (!logits || !counts_GN || !info || !G_loss || !Glogits_MN || !type_ok(logits_type) || !type_ok(grad_type))
    return MOMOE_ERR_BAD_ARG;
  if (grad_type != logits_type && grad_type != MOMOE_TYPE_BF16) return MOMOE_ERR_UNSUPPORTED;
  const int status = check_balance(G, S, N, Ks, ld);
  if (status != MOMOE_OK) return status;
  const Plan plan = plan_of(G, S, 1024, 16);
  if (G * plan.C >= (1ll << 31)) return MOMOE_ERR_UNSUPPORTED;
  const BalanceBwdArgs a{logits, ld, valid_M, counts_GN, info, G_loss, add_MN, Glogits_MN, (int)S, (int)G, (int)N, (int)(N - Ks),
                         (int)plan.C, (int)plan.TB};
  const bool vec = N % 8 == 0 && ld % 8 == 0 && (((uintptr_t)logits | (uintptr_t)add_MN | (uintptr_t)Glogits_MN) & 15) == 0;
  with_type(logits_type, [&](auto type) {
    with_width(N, [&](auto lanes) {
      using T = decltype(type);
      constexpr int LPT = decltype(lanes)::value;
      auto same = vec ? balance_bwd_kernel<T, T, LPT, true> : balance_bwd_kernel<T, T, LPT, false>;
      auto to_bf16 = vec ? balance_bwd_kernel<T, bf16, LPT, true> : balance_bwd_kernel<T, bf16, LPT, false>;
      (grad_type == logits_type ? same : to_bf16)<<<(unsigned)(G * plan.C), kThreadsFwd, 0, (hipStream_t)stream>>>(a);
    });
  });
  return launch_status();
}

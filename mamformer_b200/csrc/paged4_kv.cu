// The paged 4-bit cache (paged4.cuh) besides appending and attention: reading values back, and eviction by received weight.
//
// Eviction keeps, for each sequence of more than `budget` tokens and each KV head by itself, the last `recent` tokens and of
// the others the budget - recent of largest mass, ties to the lower slot, and moves them, in order, to slots 0 .. budget - 1.
//
// select: a cluster of CTAs per (sequence, head) finds the least kept mass by radix: four times 8 bits of the weights' order
// as whole numbers, each pass a histogram in shared memory that the cluster's CTAs add up through distributed shared
// memory.  Weights lie in few bins of their leading bits, so the lanes of a warp count
// apart.  A thread holds the 16 slots of a block, in order, so a scan of the threads' counts gives each kept slot its place.
// move: a warp gathers the tokens of two blocks and writes them whole.  To other pages in one pass; in place through a
// packed copy, since the kept tokens' places overlap.
//
// 64 sequences of 4096 slots cut to 2048, 8 heads of 128: 82 us to other pages, 132 in place (every byte twice).  The choice is
// 18 us (bound by instructions and the four passes' barriers: 59% of the issue slots, 8 MB read), the move 63 (DRAM 69%:
// 243 MB read for 155, a token's parameters and weight are parts of a 32-byte sector).  One sequence of 131,000 slots, cut to
// 32,000: 41 us and 52, of which the choice is 22, on 64 CTAs.  300,000 slots, whose weights no longer fit in registers and
// are read in every pass: 79 us.
#include "paged4.cuh"

#include <cooperative_groups.h>

namespace mamf {
namespace kv4 {

using namespace paged4;
namespace cg = cooperative_groups;

__device__ int g_err = 0;
__device__ __forceinline__ void record(int code) { atomicCAS(&g_err, 0, code); }

// ---- read ------------------------------------------------------------------------------------------
constexpr int NR = 256;

template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    Vec16<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.v[j] = from_f<T>(f[i * N + j]);
    st16(p + i * N, v);
  }
}
// 8 dims of a word of codes
__device__ __forceinline__ void values8(uint32_t w, uint32_t params, const Base& base, float* f) {
  uint32_t h[4];
  decode(w, levels_of(params, base), base, h);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
    f[e] = v.x;
    f[e + 4] = v.y;
  }
}

// TPT lanes per token, of every gridDim.y-th head: 8 dims of each half of keys and values a lane.
template <typename T, int HD>
__global__ void __launch_bounds__(NR) read_kernel(const Cache4 c, T* __restrict__ k, T* __restrict__ v) {
  constexpr int TPT = HD / 16, J = HD / 32;
  if (blockIdx.x + blockIdx.y == 0)
    for (int b = threadIdx.x; b < c.B; b += NR)
      if (!in_order(c, b)) record(ERR_LENGTH);
  const int sub = threadIdx.x % TPT, d = sub * 8;
  const int64_t item = ((int64_t)blockIdx.x * NR + threadIdx.x) / TPT;
  if (item >= c.T) return;
  const int t = (int)item, b = sequence_of(c.cu, c.B, t);
  int slot = 0, pg = -1;
  if (b >= 0) {
    const int t0 = c.cu[b], n = c.cu[b + 1] - t0, len = c.lens[b];
    slot = len - n + (t - t0);
    if (in_order(c, b) && t >= t0 && t - t0 < n && len >= 0) {
      if (slot >= 0) {                                // a sequence of fewer tokens than were asked for: zeros in front
        const int j = slot >> c.shift;
        pg = j < c.W ? c.table[(int64_t)b * c.W + j] : -1;
        if (pg < 0 || pg >= c.P) { pg = -1; if (sub == 0) record(ERR_PAGE); }
      }
    } else if (sub == 0) {
      record(ERR_LENGTH);
    }
  }
  for (int g = blockIdx.y; g < c.G; g += gridDim.y) {
    float f[32] = {};
    if (pg >= 0) {
      const uint8_t* blk = block_of<HD>(c, pg, g, slot);
      const int row = slot & 15;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint8_t* at = blk + x * HALF<HD>;
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(at + row * (HD / 2) + sub * 4);
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(at + row * (HD / 2) + HD / 4 + sub * 4);
        const uint32_t params = *reinterpret_cast<const uint32_t*>(at + PARAMS<HD> + (row * (J / 2) + sub % (J / 2)) * 4);
        values8(w0, params, c.base, f + 16 * x);
        values8(w1, params, c.base, f + 16 * x + 8);
      }
    }
    const int64_t to = ((int64_t)t * c.G + g) * HD + d;
    store8(k + to, f);
    store8(k + to + HD / 2, f + 8);
    store8(v + to, f + 16);
    store8(v + to + HD / 2, f + 24);
  }
}

// ---- eviction: which slots -------------------------------------------------------------------------
constexpr int KPT = 16, BINS = 256;                  // slots of a thread, bins of a pass
constexpr int MOST = 8;                               // CTAs of a cluster

struct Evict {
  Cache4 c;
  const int* out_table;
  int* kept;                                          // (B, G, budget)
  int* lens_out;                                      // (B)
  uint8_t* packed;                                    // in place: the kept tokens on their way
  int out_W, budget, recent;
  int most;                                           // tokens that a sequence can keep: budget, or what the table has room for
};

// The order of floats as that of whole numbers, -0 as 0, and any NaN above infinity: the sum makes the positive one of it
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums of (a, b) over the threads before this one, and over all.
template <int NS>
__device__ __forceinline__ int2 scan2(int2 v, int2& total, int2* sm) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) { x.x += a; x.y += b; }
  }
  if (lane == 31) sm[w] = x;
  __syncthreads();
  // the warps' totals, a lane each
  const int2 t = lane < NS / 32 ? sm[lane] : make_int2(0, 0);
  total = make_int2(__reduce_add_sync(0xffffffffu, t.x), __reduce_add_sync(0xffffffffu, t.y));
  const int2 before = make_int2(__reduce_add_sync(0xffffffffu, lane < w ? t.x : 0), __reduce_add_sync(0xffffffffu, lane < w ? t.y : 0));
  __syncthreads();
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// NS threads, C CTAs of a cluster for each (sequence, head).
template <int NS, int C>
__global__ void __launch_bounds__(NS) select_kernel(const __grid_constant__ Evict p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = C == 1 ? 0 : (int)cluster.block_rank();
  auto everybody = [&]() { if (C == 1) __syncthreads(); else cluster.sync(); };
  // lanes count by themselves, or every eighth together where there are few keys to count and the sums cost more
  constexpr int L = NS == 1024 ? 32 : 8;
  __shared__ int hist[BINS * (L + 1)];
  __shared__ int sums[2][BINS];                       // of the lanes; the passes take turns
  __shared__ int2 sm[32], mine[2];
  __shared__ int s_bin[2], s_above[2];
  asm volatile("griddepcontrol.launch_dependents;");  // the move waits for this grid's end by itself
  const Cache4& c = p.c;
  const int g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int len = cached_length(c, c.lens[b]), K = p.budget;
  int* kept = p.kept + ((int64_t)b * c.G + g) * K;
  if (g == 0 && rank == 0 && tid == 0) {
    p.lens_out[b] = min(len, K);
    if (len != c.lens[b]) record(ERR_LENGTH);
  }
  if (len <= K) {                                     // the cluster's CTAs agree on this: nobody waits
    for (int i = rank * NS + tid; i < K; i += C * NS) kept[i] = i < len ? i : -1;
    return;
  }
  const int old = len - p.recent;                     // the slots that compete for `want` places
  int want = K - p.recent;
  // batch i of this CTA: slots (i C + rank) NS KPT + tid KPT ..
  const int batches = (int)(((int64_t)old + (int64_t)C * NS * KPT - 1) / ((int64_t)C * NS * KPT));
  uint32_t key[KPT];
  auto first_of = [&](int i) { return (int64_t)(i * C + rank) * (NS * KPT) + tid * KPT; };
  auto load = [&](int i) {
    const int64_t s0 = first_of(i);
    int pg = -1;
    if (s0 < old) {
      pg = c.table[(int64_t)b * c.W + (s0 >> c.shift)];
      if (pg < 0 || pg >= c.P) { pg = -1; record(ERR_PAGE); }
    }
    const float* m = c.mass + (((int64_t)pg * c.G + g) << c.shift) + (s0 & (c.page - 1));
#pragma unroll
    for (int e = 0; e < KPT; e += 4) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (pg >= 0) v = *reinterpret_cast<const float4*>(m + e);
      key[e] = order_of(v.x);
      key[e + 1] = order_of(v.y);
      key[e + 2] = order_of(v.z);
      key[e + 3] = order_of(v.w);
    }
  };
  load(0);
  for (int i = tid; i < BINS * (L + 1); i += NS) hist[i] = 0;
  __syncthreads();
  uint32_t at = 0;                                    // the bits of the least kept weight found so far
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass, turn = pass & 1;
    const uint32_t above = pass == 0 ? 0u : 0xFFFFFFFFu << (shift + 8);      // bits that are settled
    if (want > 0)
#pragma unroll 1
      for (int i = 0; i < batches; ++i) {
        if (batches > 1) load(i);
        const int64_t s0 = first_of(i);
#pragma unroll
        for (int e = 0; e < KPT; ++e)
          if (s0 + e < old && (key[e] & above) == at) atomicAdd(&hist[(key[e] >> shift & (BINS - 1)) * (L + 1) + tid % L], 1);
      }
    __syncthreads();
    const int bin = BINS - 1 - tid;                   // from the top, a bin per thread
    int n = 0;
    if (tid < BINS) {
#pragma unroll
      for (int k = 0; k < L; ++k) {
        n += hist[bin * (L + 1) + k];
        hist[bin * (L + 1) + k] = 0;                  // for the next pass
      }
      if (C > 1) sums[turn][bin] = n;
    }
    if (C > 1) {
      cluster.sync();                                 // the pass before the last has been read by all, too
      if (tid < BINS) {
        int part[C];
#pragma unroll
        for (int r = 0; r < C; ++r) part[r] = *cluster.map_shared_rank(&sums[turn][bin], r);
        n = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) n += part[r];
      }
    }
    int2 total;
    const int before = scan2<NS>(make_int2(n, 0), total, sm).x;
    if (before < want && want <= before + n) { s_bin[turn] = bin; s_above[turn] = before; }
    if (want == 0 && tid == 0) { s_bin[turn] = BINS - 1; s_above[turn] = 0; }      // no place: nothing is as heavy
    __syncthreads();
    at |= (uint32_t)s_bin[turn] << shift;
    want -= s_above[turn];
  }
  // `want` of those as heavy as `at` are kept, the lowest slots, and all heavier ones
  int2 done = make_int2(0, 0);                        // heavier, and as heavy, in slots before the batch
#pragma unroll 1
  for (int i = 0; i < batches; ++i) {
    if (batches > 1) load(i);
    const int64_t s0 = first_of(i);
    int2 v = make_int2(0, 0), total;
#pragma unroll
    for (int e = 0; e < KPT; ++e)
      if (s0 + e < old) { v.x += key[e] > at; v.y += key[e] == at; }
    int2 x = scan2<NS>(v, total, sm);
    int2 batch = total;
    if (C > 1) {
      if (tid == 0) mine[i & 1] = total;              // the batches take turns
      cluster.sync();
      batch = make_int2(0, 0);
#pragma unroll
      for (int r = 0; r < C; ++r) {
        const int2 o = *cluster.map_shared_rank(&mine[i & 1], r);
        if (r < rank) { x.x += o.x; x.y += o.y; }
        batch.x += o.x;
        batch.y += o.y;
      }
    }
    x.x += done.x;
    x.y += done.y;
    done.x += batch.x;
    done.y += batch.y;
#pragma unroll
    for (int e = 0; e < KPT; ++e)
      if (s0 + e < old) {
        const bool heavier = key[e] > at, same = key[e] == at;
        if (heavier || (same && x.y < want)) kept[x.x + min(x.y, want)] = (int)(s0 + e);
        x.x += heavier;
        x.y += same;
      }
  }
  for (int i = rank * NS + tid; i < p.recent; i += C * NS) kept[K - p.recent + i] = old + i;
  everybody();                                        // nobody leaves while its shared memory is read
}

template <int NS, int C> void launch_select(const Evict& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)C, (unsigned)p.c.G, (unsigned)p.c.B);
  cfg.blockDim = dim3(NS);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, select_kernel<NS, C>, p));
}

// ---- eviction: the move ----------------------------------------------------------------------------
constexpr int NM = 128, PAIR = 2;                                    // threads, blocks that a warp moves at once
template <int HD> constexpr int PACKED = BLOCK<HD> + 64;             // a packed block: its tokens, their masses

enum Mode { DIRECT, PACK, UNPACK };

// A warp fills blocks of the kept tokens' places: lanes 4 t .. 4 t + 3 take the codes of tokens t and t + 8, 16 bytes a lane
// of keys and of values (8 of 64 dims), lanes t and t + 16 the parameters of token t, lane t its mass.  What is written is
// whole blocks.
template <int HD> struct Piece {
  uint4 code[2][2];
  uint2 param;
  float mass;
};
template <int HD>
__device__ __forceinline__ void copy_codes(uint4& to, const uint8_t* from) {
  if (HD == 128) to = *reinterpret_cast<const uint4*>(from);
  else *reinterpret_cast<uint2*>(&to) = *reinterpret_cast<const uint2*>(from);
}
template <int HD>
__device__ __forceinline__ void copy_codes(uint8_t* to, const uint4& from) {
  if (HD == 128) *reinterpret_cast<uint4*>(to) = from;
  else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(&from);
}

template <int HD, int MODE>
__global__ void __launch_bounds__(NM) move_kernel(const __grid_constant__ Evict p) {
  const Cache4& c = p.c;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = blockIdx.y, b = blockIdx.z, q = lane & 3;
  const int blocks = (p.most + 15) >> 4;
  const int first = (blockIdx.x * (NM / 32) + w) * PAIR;
  if (first >= blocks) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int* kept = p.kept + ((int64_t)b * c.G + g) * p.budget;
  const int* table = c.table + (int64_t)b * c.W;
  const int* to = p.out_table + (int64_t)b * p.out_W;
  int src[PAIR], page[PAIR];                          // of token lane & 15: its slot and that one's page
  uint8_t* dst[PAIR];
  float* dst_mass[PAIR];
#pragma unroll
  for (int u = 0; u < PAIR; ++u) {
    const int r = (first + u) * 16 + (lane & 15);
    src[u] = r < p.budget ? kept[r] : -1;
    // in place, blocks whose tokens stay are left alone, by both passes
    if (MODE != DIRECT && __all_sync(0xffffffffu, src[u] < 0 || src[u] == r)) src[u] = -1;
  }
#pragma unroll
  for (int u = 0; u < PAIR; ++u) {
    const int r0 = (first + u) * 16;
    page[u] = 0;
    dst[u] = nullptr;
    if (__all_sync(0xffffffffu, src[u] < 0)) continue;
    if (src[u] >= 0) page[u] = table[src[u] >> c.shift];
    if (MODE == PACK) {
      dst[u] = p.packed + (((int64_t)b * c.G + g) * blocks + first + u) * PACKED<HD>;
      dst_mass[u] = reinterpret_cast<float*>(dst[u] + BLOCK<HD>);
      continue;
    }
    const int pg = to[r0 >> c.shift];
    if (pg >= 0 && pg < c.P) {
      dst[u] = block_of<HD>(c, pg, g, r0);
      dst_mass[u] = c.mass + (((int64_t)pg * c.G + g) << c.shift) + (r0 & (c.page - 1));
    } else if (lane == 0) {
      record(ERR_PAGE);
    }
  }
  Piece<HD> x[PAIR];
#pragma unroll
  for (int u = 0; u < PAIR; ++u) {
    if (!dst[u]) continue;
    // no page: nothing comes of the token, also not out of the packed copy, where its place was never written
    if (src[u] >= 0 && (page[u] < 0 || page[u] >= c.P)) { src[u] = -1; record(ERR_PAGE); }
    const uint8_t* packed = MODE == UNPACK ? p.packed + (((int64_t)b * c.G + g) * blocks + first + u) * PACKED<HD> : nullptr;
    // where the token's block is, and its row of it
    const int64_t mine = MODE == UNPACK ? 0 : src[u] >= 0 ? block_of<HD>(c, page[u], g, src[u]) - c.blocks : -1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = (lane >> 2) + 8 * h, s = __shfl_sync(0xffffffffu, src[u], t);
      const int64_t off = __shfl_sync(0xffffffffu, mine, t);
      if (s < 0) continue;
      const uint8_t* blk = MODE == UNPACK ? packed : c.blocks + off;
      const int row = MODE == UNPACK ? t : s & 15;
      copy_codes<HD>(x[u].code[h][0], blk + row * (HD / 2) + q * (HD / 8));
      copy_codes<HD>(x[u].code[h][1], blk + HALF<HD> + row * (HD / 2) + q * (HD / 8));
    }
    if (src[u] >= 0) {
      const uint8_t* blk = MODE == UNPACK ? packed : c.blocks + mine;
      const int row = MODE == UNPACK ? lane & 15 : src[u] & 15;
      const uint8_t* at = blk + (lane >> 4) * HALF<HD> + PARAMS<HD> + row * (HD / 16);
      if (HD == 128) x[u].param = *reinterpret_cast<const uint2*>(at);
      else x[u].param.x = *reinterpret_cast<const uint32_t*>(at);
      if (lane < 16) x[u].mass = MODE == UNPACK ? reinterpret_cast<const float*>(packed + BLOCK<HD>)[row]
                                                : c.mass[(((int64_t)page[u] * c.G + g) << c.shift) + (src[u] & (c.page - 1))];
    }
  }
#pragma unroll
  for (int u = 0; u < PAIR; ++u) {
    if (!dst[u]) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = (lane >> 2) + 8 * h;
      if (__shfl_sync(0xffffffffu, src[u], t) < 0) continue;
      copy_codes<HD>(dst[u] + t * (HD / 2) + q * (HD / 8), x[u].code[h][0]);
      copy_codes<HD>(dst[u] + HALF<HD> + t * (HD / 2) + q * (HD / 8), x[u].code[h][1]);
    }
    if (src[u] >= 0) {
      uint8_t* at = dst[u] + (lane >> 4) * HALF<HD> + PARAMS<HD> + (lane & 15) * (HD / 16);
      if (HD == 128) *reinterpret_cast<uint2*>(at) = x[u].param;
      else *reinterpret_cast<uint32_t*>(at) = x[u].param.x;
      if (lane < 16) dst_mass[u][lane] = x[u].mass;
    }
  }
}

template <int HD, int MODE> void launch_move(const Evict& p) {
  const int per = NM / 32 * PAIR * 16;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.most + per - 1) / per), (unsigned)p.c.G, (unsigned)p.c.B);
  cfg.blockDim = dim3(NM);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = MODE == UNPACK ? 0 : 1;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, move_kernel<HD, MODE>, p));
}
template <int HD> void move_kept(Evict& p, bool in_place) {
  if (!in_place) { launch_move<HD, DIRECT>(p); return; }
  const int64_t blocks = (int64_t)p.c.B * p.c.G * ((p.most + 15) / 16);
  const at::Tensor ws = at::empty({blocks * PACKED<HD>}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA));
  p.packed = ws.data_ptr<uint8_t>();
  launch_move<HD, PACK>(p);
  launch_move<HD, UNPACK>(p);
}

}  // namespace kv4

// Values of the last cu[b + 1] - cu[b] tokens of each sequence: k, v (T, G, hd).
std::vector<at::Tensor> kv4_read(at::Tensor blocks, at::Tensor table, at::Tensor cu, at::Tensor lens, int64_t T, at::ScalarType dtype) {
  using namespace kv4;
  TORCH_CHECK(blocks.is_cuda() && blocks.dim() == 4, "kv_read: blocks (P, G, page / 16, 18 hd) on a GPU");
  c10::cuda::CUDAGuard guard(blocks.device());
  TORCH_CHECK(T >= 0, "kv_read: tokens must not be negative");
  const int64_t hd = blocks.size(3) / 18;
  const Cache4 c = check_cache4("kv_read", blocks, c10::nullopt, table, &cu, lens, T, hd);
  const auto opts = blocks.options().dtype(dtype);
  std::vector<at::Tensor> out{at::empty({T, c.G, hd}, opts), at::empty({T, c.G, hd}, opts)};
  if (T == 0) return out;
  if (c.B == 0) { out[0].zero_(); out[1].zero_(); return out; }
  const int64_t units = (T * (hd / 16) + NR - 1) / NR;
  TORCH_CHECK(units < (1LL << 31), "kv_read: sizes");
  const dim3 grid((unsigned)units, (unsigned)std::max<int64_t>(1, std::min<int64_t>(c.G, 8LL * num_sms() / units)));
  MAMF_DISPATCH_FLOAT_BF16(dtype, "kv_read", [&] {
    auto* k = (scalar_t*)out[0].data_ptr();
    auto* v = (scalar_t*)out[1].data_ptr();
    if (hd == 128) read_kernel<scalar_t, 128><<<grid, NR, 0, stream()>>>(c, k, v);
    else read_kernel<scalar_t, 64><<<grid, NR, 0, stream()>>>(c, k, v);
  });
  MAMF_LAUNCH_CHECK();
  return out;
}

// Moves the kept tokens (out_table: to its pages; none: in place).  Returns the kept slots (B, G, budget), -1 for none, and
// the new lengths.
std::vector<at::Tensor> kv4_evict(at::Tensor blocks, at::Tensor mass, at::Tensor table, at::Tensor lens, int64_t budget,
                                  int64_t recent, c10::optional<at::Tensor> out_table) {
  using namespace kv4;
  TORCH_CHECK(blocks.is_cuda() && blocks.dim() == 4, "kv_evict: blocks (P, G, page / 16, 18 hd) on a GPU");
  c10::cuda::CUDAGuard guard(blocks.device());
  const int64_t hd = blocks.size(3) / 18;
  Evict p{};
  p.c = check_cache4("kv_evict", blocks, mass, table, nullptr, lens, 0, hd);
  TORCH_CHECK(aligned16(p.c.mass), "kv_evict: 16-byte aligned mass");
  TORCH_CHECK(budget >= 1 && recent >= 0 && recent <= budget && budget < (1LL << 30), "kv_evict: 0 <= recent <= budget and budget >= 1, got ",
              recent, " and ", budget);
  const at::Tensor& to = out_table.has_value() ? *out_table : table;
  TORCH_CHECK(to.is_cuda() && to.device() == blocks.device() && to.is_contiguous() && to.scalar_type() == at::kInt && to.dim() == 2 &&
              to.size(0) == p.c.B, "kv_evict: a contiguous int32 out_table with a row for each sequence");
  const int64_t most = std::min<int64_t>(budget, (int64_t)p.c.W * p.c.page);      // tokens that a sequence can keep
  TORCH_CHECK(to.size(1) * p.c.page >= most, "kv_evict: out_table has room for ", to.size(1) * p.c.page, " of ", most, " tokens");
  TORCH_CHECK(p.c.B < 65536, "kv_evict: at most 65535 sequences");
  at::Tensor kept = at::empty({p.c.B, p.c.G, budget}, table.options()), lens_out = at::empty({p.c.B}, table.options());
  if (p.c.B == 0) return {kept, lens_out};
  p.out_table = to.data_ptr<int>();
  p.out_W = (int)to.size(1);
  p.kept = kept.data_ptr<int>();
  p.lens_out = lens_out.data_ptr<int>();
  p.budget = (int)budget;
  p.recent = (int)recent;
  p.most = (int)std::max<int64_t>(1, most);
  // As many threads and CTAs per (sequence, head) as the longest sequence that the table has room for has blocks (the host does
  // not know the lengths).  us to cut one sequence of 8 heads to half: 4096 slots on 256 threads 13.6, on 512 14.7; 8192 on
  // 256 22.9, on 512 16.7, on two CTAs 18.8; 16384 on one CTA 27.4, on two 19.2, on four 20.8; 32768 on two 37.4, on four 22.9;
  // 65536 on four 47.5, on eight 31.9; 131072 on eight 68.8, with 1024 threads each 58.6.  Sequences far shorter than the table
  // pay for its width: 64 of 4096 slots take 22 us on 256 threads, 52 on two CTAs, 204 on eight.
  const int64_t threads = (int64_t)p.c.W * p.c.page / KPT;
  if (threads <= 256) launch_select<256, 1>(p);
  else if (threads <= 512) launch_select<512, 1>(p);
  else if (threads <= 1024) launch_select<512, 2>(p);
  else if (threads <= 2048) launch_select<512, 4>(p);
  else if (threads <= 4096) launch_select<512, 8>(p);
  else launch_select<1024, 8>(p);
  const bool in_place = to.data_ptr() == table.data_ptr();
  if (hd == 128) move_kept<128>(p, in_place); else move_kept<64>(p, in_place);
  return {kept, lens_out};
}

int64_t kv4_error(bool clear) { return paged::take_code(kv4::g_err, clear); }

}  // namespace mamf

// Training operators around the model: the embedding lookup and its gradient,
// and the next-byte loss with its gradients.  (The recurrence between them is
// in train_scan.hip.)
#include <algorithm>

#include "train_kernels.h"

namespace boa {

namespace {

__device__ __forceinline__ float4 raw_f4(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}

// V consecutive elements of a row: 16 bytes (V = 4 fp32, 8 bf16) or one element
template <int V>
__device__ __forceinline__ void ld_vec(const float* p, float (&v)[V]) {
  if constexpr (V == 4) {
    const float4 t = raw_f4(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
    v[0] = *p;
  }
}
template <int V>
__device__ __forceinline__ void ld_vec(const uint16_t* p, float (&v)[V]) {
  if constexpr (V == 8) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = u2f(w[i] << 16);
      v[2 * i + 1] = u2f(w[i] & 0xFFFF0000u);
    }
  } else {
    v[0] = bf16_to_f32(*p);
  }
}
template <int V>
__device__ __forceinline__ void st_vec(float* p, const float (&v)[V]) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}
template <int V>
__device__ __forceinline__ void st_vec(uint16_t* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *p = f32_to_bf16(v[0]);
  }
}

// ... past the caches (stream): rows that the L2s cannot hold until they are
// read (embedding of 261,000 bf16 rows of 256, 133 MB: 38 us through them, 29
// past them; loss with 533 MB of gradients: 173, 167)
template <typename T, int V>
__device__ __forceinline__ void st_rows(T* p, const float (&v)[V], bool stream) {
  if constexpr (sizeof(T) * V == 16) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    if (stream) {
      u4 w;
      if constexpr (V == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f2u(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
      }
      __builtin_nontemporal_store(w, reinterpret_cast<u4*>(p));
      return;
    }
  }
  st_vec<V>(p, v);
}
constexpr size_t CACHED_BYTES = (size_t)32 << 20;  // the eight L2s

// whether rows of `width` elements can be moved 16 bytes at a time (element by
// element the embedding of 521,000 bf16 rows of 256 takes 150 us and not 44, the
// gradient of as many 108 and not 84, of fp32 rows of 64 57 and not 36)
bool rows16(const void* d, int64_t lane, int64_t row, int width, int size) {
  const int v = 16 / size;
  return ((uintptr_t)d & 15) == 0 && lane % v == 0 && row % v == 0 && width % v == 0;
}

// -------------------------------------------------------------- embedding
// out[r] = scale table[tok[r]], one rounding.  Bound by the writes of the
// rows: the 256 table rows stay in the L2s.  A block takes whole rows, about
// 256 U vectors of 16 bytes, U a thread, whose bytes, table rows and stores
// are each under way together: 250 x 2085 ragged bf16 rows of 256 (133 MB
// within the lengths) in 27 us, 5 TB/s.  inv = ceil(2^32 / vectors a row) divides the
// block's vectors by a multiplication; a row's lane and position follow from
// the block's first row's.
template <typename T, int V, int U>
__global__ __launch_bounds__(256) void embed_kernel(const EmbedArgs a, uint32_t rows,
                                                    uint32_t block_rows, uint32_t inv, bool stream) {
  const uint32_t vpr = a.width / V, len = a.q.T;
  for (uint64_t b0 = (uint64_t)blockIdx.x * block_rows; b0 < rows;
       b0 += (uint64_t)gridDim.x * block_rows) {
    const uint32_t r0 = (uint32_t)b0, l0 = r0 / len, t0 = r0 - l0 * len;
    const uint32_t n = min(block_rows, rows - r0) * vpr;
    uint32_t l[U], t[U], col[U], byte[U];
    bool ok[U];
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = threadIdx.x + 256 * u, k = vpr == 1 ? i : __umulhi(i, inv);
      col[u] = (i - k * vpr) * V;
      l[u] = l0;
      t[u] = t0 + k;
      if (t[u] >= len) {
        if (block_rows <= len) {
          l[u] += 1;
          t[u] -= len;
        } else {
          const uint32_t d = t[u] / len;
          l[u] += d;
          t[u] -= d * len;
        }
      }
      ok[u] = i < n;
      if (!ok[u]) l[u] = t[u] = 0;
    }
    // no branch lies between loads (each would wait for those before it): what
    // takes no part reads the table's first byte as its token
#pragma unroll
    for (int u = 0; u < U; ++u) ok[u] = ok[u] && (int)t[u] < seq_len(a.q, l[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      byte[u] = *(ok[u] ? a.tok + l[u] * a.tok_lane + t[u] : (const uint8_t*)a.table);
#pragma unroll
    for (int u = 0; u < U; ++u)
      ld_vec<V>((const T*)a.table + byte[u] * (uint32_t)a.width + col[u], v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ok[u]) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[u][j] *= a.scale;
        st_rows<T, V>((T*)a.out.d + l[u] * a.out.lane + t[u] * a.out.row + col[u], v[u], stream);
      }
  }
}

// ----------------------------------------------------- embedding gradient
// dtable[v] = scale sum of dout's rows whose token is v, in fp32 and in an
// order that the sizes, lengths and tokens decide (no atomics: a call repeated
// gives the same bits; other tokens elsewhere may change a byte's last bits).  A block sorts the tokens of
// `chunk` rows by a stable counting sort in LDS.  Then its groups of G lanes
// take equal parts of the sorted rows and sum run by run, so a byte that fills
// most rows is spread over all groups like any other.  Runs that cross a
// group's border leave their later pieces in LDS, and the group they start in
// adds them in order.  One partial row per byte that occurs in the chunk goes
// to the workspace; the second kernel sums a byte's partials over the chunks.
// dout is read once; the partials are at most 256 / chunk of it.  A chunk is
// batches of 64 rows from all over the sequences, so that blocks come by as
// many rows within their lanes' lengths.
// Bound by dout's bytes; 1000 x 521 ragged fp32 rows of 256, most bytes zero
// (267 MB within the lengths): 88 us with consecutive rows and 512 threads, 81
// with batches, 75 with 1024 threads (3.6 TB/s; the sort and the runs of single
// rows, which one wave of a block gets all of, are the rest).
constexpr int EG_THREADS = 1024, EG_WAVES = EG_THREADS / 64, EG_MAX_CHUNK = 2048;

// Rows a block sorts: at least a block a CU, then as many as there can be, for
// few partials (twice the blocks of half the rows: as fast at 521,000 rows, and
// the second kernel takes 11 us and not 7).
int embed_grad_chunk(int64_t rows) {
  int chunk = 64;
  while (chunk < EG_MAX_CHUNK && rows > (int64_t)chunk * 256) chunk *= 2;
  return chunk;
}

struct EgPlan {
  int chunk, chunks, slots;
};
EgPlan embed_grad_plan(int64_t rows) {
  EgPlan p;
  p.chunk = embed_grad_chunk(rows);
  p.chunks = (int)((rows + p.chunk - 1) / p.chunk);
  p.slots = std::min(p.chunk, 256);
  return p;
}

// lanes that share a row of n vectors
int group_lanes(int n) {
  int g = 1;
  while (g < 64 && g < n) g *= 2;
  return g;
}

template <typename T, int V, int NV>
__global__ __launch_bounds__(EG_THREADS) void embed_grad_kernel(
    const EmbedGradArgs a, uint32_t rows, int chunk, int chunks, int slots, int G,
    float* __restrict__ part, uint16_t* __restrict__ slot_map) {
  __shared__ uint32_t hist[EG_WAVES][256];
  __shared__ uint64_t list[EG_MAX_CHUNK];  // dout offset, the byte in the top 8 bits
  __shared__ uint16_t start[257], slot[256];
  __shared__ uint32_t wave_tot[4];
  __shared__ float head[V * NV][EG_THREADS];
  const int tid = threadIdx.x, w = tid >> 6, ln = tid & 63;
  const uint32_t c = blockIdx.x;

  // each wave ranks its own consecutive batches of 64 rows among equal bytes
  for (int i = tid; i < EG_WAVES * 256; i += EG_THREADS) (&hist[0][0])[i] = 0;
  __syncthreads();
  constexpr int MB = EG_MAX_CHUNK / EG_THREADS;
  const int batches = (chunk / 64 + EG_WAVES - 1) / EG_WAVES;
  uint64_t key[MB];
  uint32_t rank[MB];
  bool valid[MB];
  volatile uint32_t* my_hist = hist[w];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const uint32_t b = w * batches + i;
    const uint64_t r64 = ((uint64_t)b * chunks + c) * 64 + ln;
    const uint32_t r = (uint32_t)r64;
    valid[i] = false;
    key[i] = 0;
    rank[i] = 0;
    if (i < batches && b < (uint32_t)chunk / 64 && r64 < rows) {
      const uint32_t l = r / (uint32_t)a.q.T, t = r - l * a.q.T;
      if ((int)t < seq_len(a.q, l)) {
        valid[i] = true;
        key[i] = ((uint64_t)a.tok[l * a.tok_lane + t] << 56) |
                 (uint64_t)(l * a.dout.lane + t * a.dout.row);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    if (i < batches) {
      const uint32_t byte = (uint32_t)(key[i] >> 56);
      uint64_t same = __builtin_amdgcn_ballot_w64(valid[i]);
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const bool on = (byte >> bit) & 1;
        const uint64_t bal = __builtin_amdgcn_ballot_w64(on);
        same &= on ? bal : ~bal;
      }
      const uint32_t before = __popcll(same & ((1ull << ln) - 1));
      const uint32_t base = my_hist[byte];
      rank[i] = base + before;
      if (valid[i] && before == 0) my_hist[byte] = base + __popcll(same);
    }
  }
  __syncthreads();
  // exclusive prefix over bytes of (rows, bytes that occur), then over waves
  uint32_t mine = 0, incl = 0;
  if (tid < 256) {
#pragma unroll
    for (int k = 0; k < EG_WAVES; ++k) mine += hist[k][tid];
    mine |= mine ? 0x10000u : 0;
    incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t up = __shfl_up(incl, off, 64);
      if (ln >= off) incl += up;
    }
    if (ln == 63) wave_tot[w] = incl;
  }
  __syncthreads();
  if (tid < 256) {
    for (int k = 0; k < w; ++k) incl += wave_tot[k];
    const uint32_t excl = incl - mine;
    uint32_t at = excl & 0xFFFF;
    start[tid] = (uint16_t)at;
    slot[tid] = mine ? (uint16_t)(excl >> 16) : 0xFFFF;
    if (tid == 255) start[256] = (uint16_t)(incl & 0xFFFF);
    if (slot_map) slot_map[(size_t)tid * chunks + c] = slot[tid];
#pragma unroll
    for (int k = 0; k < EG_WAVES; ++k) {
      const uint32_t n = hist[k][tid];
      hist[k][tid] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MB; ++i)
    if (valid[i]) list[hist[w][key[i] >> 56] + rank[i]] = key[i];
  __syncthreads();

  const int n = start[256], groups = EG_THREADS / G, g = tid / G, gl = tid % G;
  const int per = (n + groups - 1) / groups;
  const int p0 = min(n, g * per), p1 = min(n, p0 + per);
  const T* dout = (const T*)a.dout.d;
  float acc[V * NV];
#pragma unroll
  for (int j = 0; j < V * NV; ++j) acc[j] = 0.0f;
  int cur = p0 < p1 ? (int)(list[p0] >> 56) : 0;
  // where the run's sum goes: bytes that occur have consecutive slots, in order
  const bool partial = slot_map != nullptr;
  const float scale = partial ? 1.0f : a.scale;
  float* dst = partial ? part + ((size_t)c * slots + slot[cur]) * a.width
                       : a.dtable + (size_t)cur * a.width;
  auto store = [&](float* to) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * G + gl) * V;
      if (col < a.width) {
        if constexpr (V > 1) {  // width is a multiple of V, and so of four
#pragma unroll
          for (int j = 0; j < V; j += 4)
            *reinterpret_cast<f4_any*>(to + col + j) =
                f4_any{acc[k * V + j] * scale, acc[k * V + j + 1] * scale,
                       acc[k * V + j + 2] * scale, acc[k * V + j + 3] * scale};
        } else {
          to[col] = acc[k] * scale;
        }
      }
    }
  };
  bool begun = p0 < p1 && start[cur] < p0;  // the run began in an earlier group
  auto flush = [&]() {                      // the run ends here
    if (begun) {
#pragma unroll
      for (int j = 0; j < V * NV; ++j) head[j][tid] = acc[j];
      begun = false;
    } else {
      store(dst);
    }
  };
  // U rows are summed while the next U are on their way
  constexpr int U = V * NV <= 4 ? 8 : V > 1 ? 4 : 2;
  float v[2][U][NV][V];
  int byte[2][U];
  auto fetch = [&](int p, int h) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t e = list[min(p + k, p1 - 1)];
      byte[h][k] = (int)(e >> 56);
      const T* src = dout + (e & 0x00FFFFFFFFFFFFFFull);
#pragma unroll
      for (int m = 0; m < NV; ++m) {
        // without a branch, which would wait for the loads before it: lanes past
        // the width read its last vector
        ld_vec<V>(src + min((m * G + gl) * V, a.width - V), v[h][k][m]);
      }
    }
  };
  auto add = [&](int p, int h) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (p + k < p1) {
        if (byte[h][k] != cur) {
          flush();
          dst += (size_t)(partial ? 1 : byte[h][k] - cur) * a.width;
          cur = byte[h][k];
#pragma unroll
          for (int j = 0; j < V * NV; ++j) acc[j] = 0.0f;
        }
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[m * V + j] += v[h][k][m][j];
      }
    }
  };
  if (p0 < p1) fetch(p0, 0);
  for (int p = p0; p < p1; p += 2 * U) {
    if (p + U < p1) fetch(p + U, 1);
    add(p, 0);
    if (p + 2 * U < p1) fetch(p + 2 * U, 0);
    if (p + U < p1) add(p + U, 1);
  }
  const int end = start[cur + 1];
  const bool goes_on = p0 < p1 && !begun && end > p1;
  if (p0 < p1 && !goes_on) flush();
  __syncthreads();
  // a run that starts here and goes on: its later pieces are the next groups' heads
  if (goes_on) {
    for (int h = g + 1; h < groups && h * per < end; ++h)
#pragma unroll
      for (int j = 0; j < V * NV; ++j) acc[j] += head[j][h * G + gl];
    store(dst);
  }
  if (!partial)  // the only chunk: bytes that do not occur have no gradient
    for (int i = tid; i < 256 * a.width; i += EG_THREADS)
      if (slot[i / a.width] == 0xFFFF) a.dtable[i] = 0.0f;
}

// a byte's partial rows summed over the chunks: the slots of up to 1024 chunks
// come to LDS at once, groups of G lanes take every groups-th chunk, and the
// groups' sums are added in order
constexpr int EG_SLOTS = 1024;
template <int V>
__global__ __launch_bounds__(EG_THREADS) void embed_grad_sum_kernel(
    const float* __restrict__ part, const uint16_t* __restrict__ slot_map, int chunks, int slots,
    int width, int G, float scale, float* __restrict__ dtable) {
  __shared__ float sums[V][EG_THREADS];
  __shared__ uint16_t map[EG_SLOTS];
  const int byte = blockIdx.x, tid = threadIdx.x, g = tid / G, gl = tid % G, groups = EG_THREADS / G;
  const int col = (blockIdx.y * G + gl) * V;
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.0f;
  for (int c0 = 0; c0 < chunks; c0 += EG_SLOTS) {
    const int n = min(EG_SLOTS, chunks - c0);
    __syncthreads();
    for (int i = tid; i < EG_SLOTS; i += EG_THREADS)
      map[i] = i < n ? slot_map[(size_t)byte * chunks + c0 + i] : 0xFFFF;
    __syncthreads();
    if (col < width) {
      constexpr int U = 8;
      for (int c = g; c < n; c += U * groups) {
        float v[U][V];
        bool on[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int cc = c + k * groups;
          const uint32_t s = cc < n ? map[cc] : 0xFFFF;
          on[k] = s != 0xFFFF;  // else the first partial row is read, and not added
          ld_vec<V>(part + (on[k] ? ((size_t)(c0 + cc) * slots + s) * width : 0) + col, v[k]);
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += on[k] ? v[k][j] : 0.0f;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sums[j][tid] = acc[j];
  __syncthreads();
  if (g == 0 && col < width) {
    for (int h = 1; h < groups; ++h)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += sums[j][h * G + gl];
#pragma unroll
    for (int j = 0; j < V; ++j) dtable[(size_t)byte * width + col + j] = acc[j] * scale;
  }
}

// ---------------------------------------------------------- next-byte loss
// loss = log sum_j e^{x_j} - x_target, dx = scale (softmax - onehot).  A row
// belongs to 16 lanes, 16 logits each, so a wave works on four rows at once:
// the maximum and the sum take four steps within a DPP row, the logarithm and
// the reciprocal serve four rows, and the next four rows are on their way
// meanwhile.  Each logit is read once and its gradient written once: bound by
// those bytes (1000 x 521 fp32 rows: 5.1 TB/s, as fast as a copy).  The largest
// logit's own term (1) stays out of the sum: rest = sum of the others, loss =
// log1p(rest) + (max - x_target), so a byte predicted with near certainty keeps
// its small loss and gradient, which 1 + rest would round away.
constexpr int LOSS_THREADS = 512, LOSS_WAVES = LOSS_THREADS / 64, LOSS_U = 4;

// blocks: four rows at a time for each wave, at most two blocks a CU (521,000
// rows, one, two and three blocks a CU: bf16 149, 131, 133 us; fp32 192, 209,
// 218, but with ragged lanes 188, 168 with one and two); few rows stay in one,
// which needs no second launch (72 rows: 8.8 us, 11.8 in two blocks)
int loss_blocks(int64_t rows) {
  return rows <= 128 ? 1 : (int)std::min<int64_t>(512, (rows + 63) / 64);
}

// sum and maximum over the 16 lanes of a DPP row, in all of them
__device__ __forceinline__ float row_sum(float x) {
  x = dpp_add<DPP_XOR1>(x);
  x = dpp_add<DPP_XOR2>(x);
  x = dpp_add<DPP_HALF_MIRROR>(x);
  return dpp_add<DPP_MIRROR>(x);
}
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, dpp_move<DPP_XOR1>(x));
  x = fmaxf(x, dpp_move<DPP_XOR2>(x));
  x = fmaxf(x, dpp_move<DPP_HALF_MIRROR>(x));
  return fmaxf(x, dpp_move<DPP_MIRROR>(x));
}

// VEC: rows aligned for 16-byte accesses (521,000 rows: fp32 209 us, bf16 131;
// element by element 213 and 140).  A lane's logits are V neighbours (16 bytes)
// of every 16 V.
template <typename T, bool VEC>
__global__ __launch_bounds__(LOSS_THREADS) void loss_kernel(const LossArgs a, uint32_t rows,
                                                            bool stream,
                                                            float* __restrict__ part_bias,
                                                            double* __restrict__ part_total) {
  constexpr int V = 16 / sizeof(T), K = 16 / V;
  __shared__ float sm[LOSS_WAVES][256];
  __shared__ double st[LOSS_WAVES];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = threadIdx.x & 63;
  const int i = ln & 15;
  const uint32_t waves = gridDim.x * LOSS_WAVES, me = blockIdx.x * LOSS_WAVES + w;
  T* dx = (T*)a.dlogits.d;
  float bias[16], db[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    bias[j] = a.bias ? a.bias[16 * V * (j / V) + V * i + j % V] : 0.0f;
    db[j] = 0.0f;
  }
  // the four rows of a group: this lane's row, its raw logits and target
  struct Group {
    bool in, live;
    uint32_t l, t;
    int tgt;
    uint32_t raw[K][4];
  };
  auto fetch = [&](uint64_t g, Group& r) {
    const uint64_t row = g * LOSS_U + (ln >> 4);
    r.in = row < rows;
    const uint32_t rr = r.in ? (uint32_t)row : 0;
    r.l = rr / (uint32_t)a.q.T;
    r.t = rr - r.l * a.q.T;
    r.live = r.in && (int)r.t < seq_len(a.q, r.l);
    r.tgt = 0;
    if (r.live) {
      r.tgt = a.tgt[r.l * a.tgt_lane + r.t];
      const T* p = (const T*)a.logits.d + r.l * a.logits.lane + r.t * a.logits.row + V * i;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if constexpr (VEC) {
          const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * V * k);
          r.raw[k][0] = v.x; r.raw[k][1] = v.y; r.raw[k][2] = v.z; r.raw[k][3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4)
              r.raw[k][j] = f2u(p[16 * V * k + j]);
            else
              r.raw[k][j] = (uint32_t)p[16 * V * k + 2 * j] | (uint32_t)p[16 * V * k + 2 * j + 1] << 16;
          }
        }
      }
    }
  };
  double total = 0.0;
  Group nx;
  if ((uint64_t)me * LOSS_U < rows) fetch(me, nx);
  for (uint64_t g = me; g * LOSS_U < rows; g += waves) {
    const Group c = nx;
    float e[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if constexpr (sizeof(T) == 4) e[j] = u2f(c.raw[j / V][j % V]);
      else e[j] = u2f(j % 2 ? c.raw[j / V][j % V / 2] & 0xFFFF0000u : c.raw[j / V][j % V / 2] << 16);
      e[j] += bias[j];
    }
    if ((g + waves) * LOSS_U < rows) fetch(g + waves, nx);
    float m = e[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) m = fmaxf(m, e[j]);
    m = row_max(m);
    const bool none = m == -__builtin_huge_valf();  // nothing is allowed
    m = none ? 0.0f : m;
    // the target's place among this lane's logits, or none
    const int at = (c.tgt / V) % 16 == i ? c.tgt / (16 * V) * V + c.tgt % V : -1;
    float pick = 0.0f, rest = 0.0f, tops = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float d = e[j] - m;
      pick = at == j ? d : pick;
      e[j] = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
      rest += d == 0.0f ? 0.0f : e[j];
      tops += d == 0.0f ? 1.0f : 0.0f;
    }
    const float dt = row_sum(pick);  // x_target - max
    rest = row_sum(rest) + (row_sum(tops) - 1.0f);
    // log1p(rest): what 1 + rest loses is put back
    const float sum = 1.0f + rest, lost = rest - (sum - 1.0f), inv_sum = __builtin_amdgcn_rcpf(sum);
    float loss = __builtin_fmaf(__builtin_amdgcn_logf(sum), 0.69314718055994530942f,
                                lost * inv_sum) - dt;
    loss = none ? __builtin_huge_valf() + rest : loss;  // a NaN beside -inf stays one
    // (rest - rest: 0, or that NaN, which every byte's gradient then is)
    const float inv = !c.live ? 0.0f : none ? rest - rest : a.scale * inv_sum;
    const float gt = (dt == 0.0f ? -rest : __builtin_amdgcn_exp2f(dt * 1.44269504088896340736f) - sum) * inv;
    float gr[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      gr[j] = at == j ? gt : e[j] * inv;
      gr[j] = c.live ? gr[j] : 0.0f;  // what was not read may be anything
      db[j] += gr[j];
    }
    if (c.live && i == 0) {
      total += (double)loss;
      a.loss[c.l * (int64_t)a.q.T + c.t] = loss;
    }
    if (dx && c.in) {
      T* p = dx + c.l * a.dlogits.lane + c.t * a.dlogits.row + V * i;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = gr[k * V + j];
        if constexpr (VEC) {
          st_rows<T, V>(p + 16 * V * k, v, stream);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) stv(p + 16 * V * k + j, v[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float x = fold16(db[j], db[j]), s = fold32(x, x);
    if (ln < 16) sm[w][16 * V * (j / V) + V * i + j % V] = s;
  }
  total += __shfl_xor(total, 16, 64);
  total += __shfl_xor(total, 32, 64);
  if (ln == 0) st[w] = total;
  __syncthreads();
  const int tid = threadIdx.x;
  if (tid < 256) {
    float s = sm[0][tid];
#pragma unroll
    for (int k = 1; k < LOSS_WAVES; ++k) s += sm[k][tid];
    if (gridDim.x == 1) {
      if (a.dbias) a.dbias[tid] = s;
    } else {
      part_bias[(size_t)blockIdx.x * 256 + tid] = s;
    }
  }
  if (tid == 0) {
    double s = st[0];
    for (int k = 1; k < LOSS_WAVES; ++k) s += st[k];
    if (gridDim.x == 1) {
      if (a.total) *a.total = (float)s;
    } else {
      part_total[blockIdx.x] = s;
    }
  }
}

// the blocks' sums: blocks 0 .. 15 take 16 columns of dbias each, block 16 the total
__global__ __launch_bounds__(256) void loss_sum_kernel(const float* __restrict__ part_bias,
                                                       const double* __restrict__ part_total,
                                                       int n, float* dbias, float* total) {
  __shared__ float sm[16][16];
  __shared__ double st[256];
  const int tid = threadIdx.x;
  if (blockIdx.x < 16) {
    if (!dbias) return;
    const int col = tid & 15, g = tid >> 4;
    float s = 0.0f;
#pragma unroll 8
    for (int k = g; k < n; k += 16) s += part_bias[(size_t)k * 256 + blockIdx.x * 16 + col];
    sm[g][col] = s;
    __syncthreads();
    if (g == 0) {
      for (int k = 1; k < 16; ++k) s += sm[k][col];
      dbias[blockIdx.x * 16 + col] = s;
    }
  } else {
    if (!total) return;
    double s = 0.0;
    for (int k = tid; k < n; k += 256) s += part_total[k];
    st[tid] = s;
    __syncthreads();
    for (int off = 128; off > 0; off >>= 1) {
      if (tid < off) st[tid] += st[tid + off];
      __syncthreads();
    }
    if (tid == 0) *total = (float)st[0];
  }
}

}  // namespace

hipError_t launch_embed(const EmbedArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const int size = a.bf16 ? 2 : 4;
  const bool vec = rows16(a.out.d, a.out.lane, a.out.row, a.width, size) &&
                   ((uintptr_t)a.table & 15) == 0;
  const uint32_t vpr = vec ? a.width * size / 16 : a.width;
  // a block's threads take 4 vectors each; with fewer than two such blocks a CU,
  // one (64 rows of 64 fp32: the kernel 2.3 us, 3.4 with four; 521,000 ragged bf16
  // rows of 256: 36 us with one, 29 with four)
  const int u = (uint64_t)rows * vpr >= 512ull * 1024 ? 4 : 1;
  const uint32_t block_rows = std::max<uint32_t>(1, 256 * u / vpr);
  const uint32_t blocks = (rows + block_rows - 1) / block_rows;
  const uint32_t inv = (uint32_t)(((1ull << 32) + vpr - 1) / vpr);
  const dim3 grid(std::min(MAX_BLOCKS, blocks));
  const bool stream = (size_t)rows * a.width * size > CACHED_BYTES;
#define BOA_EMBED(Tv, Vv)                                                                      \
  if (block_rows * vpr > 256)                                                                  \
    BOA_LAUNCH((embed_kernel<Tv, Vv, 4>), grid, dim3(256), 0, s, a, rows, block_rows, inv,     \
               stream);                                                                        \
  else                                                                                         \
    BOA_LAUNCH((embed_kernel<Tv, Vv, 1>), grid, dim3(256), 0, s, a, rows, block_rows, inv,     \
               stream)
  if (a.bf16) {
    if (vec) { BOA_EMBED(uint16_t, 8); }
    else { BOA_EMBED(uint16_t, 1); }
  } else {
    if (vec) { BOA_EMBED(float, 4); }
    else { BOA_EMBED(float, 1); }
  }
#undef BOA_EMBED
  return hipGetLastError();
}

// workspace: the partial rows, then the map of a byte's slot in each chunk
static size_t eg_part_bytes(const EgPlan& p, int width) {
  return ((size_t)p.chunks * p.slots * width * 4 + 255) / 256 * 256;
}
size_t embed_grad_work(int64_t rows, int width) {
  const EgPlan p = embed_grad_plan(rows);
  return p.chunks == 1 ? 0 : eg_part_bytes(p, width) + (size_t)256 * p.chunks * 2;
}

hipError_t launch_embed_grad(const EmbedGradArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const EgPlan p = embed_grad_plan(rows);
  const int size = a.bf16 ? 2 : 4;
  const bool vec = rows16(a.dout.d, a.dout.lane, a.dout.row, a.width, size);
  const int V = vec ? 16 / size : 1, vpr = a.width / V, G = group_lanes(vpr);
  float* part = p.chunks == 1 ? nullptr : (float*)a.work;
  uint16_t* map =
      p.chunks == 1 ? nullptr : (uint16_t*)((char*)a.work + eg_part_bytes(p, a.width));
#define BOA_EG(Tv, Vv, NVv)                                                                     \
  BOA_LAUNCH((embed_grad_kernel<Tv, Vv, NVv>), dim3(p.chunks), dim3(EG_THREADS), 0, s, a, rows, \
             p.chunk, p.chunks, p.slots, G, part, map)
  if (a.bf16) {
    if (vec) BOA_EG(uint16_t, 8, 1);
    else BOA_EG(uint16_t, 1, 8);
  } else {
    if (!vec) BOA_EG(float, 1, 8);
    else if (vpr <= 64) BOA_EG(float, 4, 1);
    else BOA_EG(float, 4, 2);
  }
#undef BOA_EG
  if (map) {
    const int V2 = a.width % 4 == 0 ? 4 : 1, G2 = group_lanes(a.width / V2);
    const dim3 grid(256, (a.width / V2 + G2 - 1) / G2);
    if (V2 == 4)
      BOA_LAUNCH(embed_grad_sum_kernel<4>, grid, dim3(EG_THREADS), 0, s, part, map, p.chunks,
                 p.slots, a.width, G2, a.scale, a.dtable);
    else
      BOA_LAUNCH(embed_grad_sum_kernel<1>, grid, dim3(EG_THREADS), 0, s, part, map, p.chunks,
                 p.slots, a.width, G2, a.scale, a.dtable);
  }
  return hipGetLastError();
}

size_t loss_work(int64_t rows) {
  const int n = loss_blocks(rows);
  return n == 1 ? 0 : (size_t)n * (256 * 4 + 8);
}

hipError_t launch_loss(const LossArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const int n = loss_blocks(rows), v = a.bf16 ? 8 : 4;
  auto fits = [&](const void* d, int64_t lane, int64_t row) {
    return ((uintptr_t)d & 15) == 0 && lane % v == 0 && row % v == 0;
  };
  const bool vec = fits(a.logits.d, a.logits.lane, a.logits.row) &&
                   (!a.dlogits.d || fits(a.dlogits.d, a.dlogits.lane, a.dlogits.row));
  const bool stream = (size_t)rows * 256 * (a.bf16 ? 2 : 4) > CACHED_BYTES;
  // doubles first: the workspace is 8-byte aligned
  double* pt = (double*)a.work;
  float* pb = n == 1 ? nullptr : (float*)(pt + n);
#define BOA_LOSS(Tv, VECv) \
  BOA_LAUNCH((loss_kernel<Tv, VECv>), dim3(n), dim3(LOSS_THREADS), 0, s, a, rows, stream, pb, \
             pt)
  if (a.bf16) {
    if (vec) BOA_LOSS(uint16_t, true);
    else BOA_LOSS(uint16_t, false);
  } else {
    if (vec) BOA_LOSS(float, true);
    else BOA_LOSS(float, false);
  }
#undef BOA_LOSS
  if (n > 1 && (a.dbias || a.total))
    BOA_LAUNCH(loss_sum_kernel, dim3(17), dim3(256), 0, s, pb, pt, n, a.dbias, a.total);
  return hipGetLastError();
}

}  // namespace boa

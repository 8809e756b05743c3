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
      w[i] = (uint32_t)f32_to_bf16(v[2 * i]) | ((uint32_t)f32_to_bf16(v[2 * i + 1]) << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *p = f32_to_bf16(v[0]);
  }
}

// whether rows of `width` elements can be moved 16 bytes at a time
bool rows16(const void* d, int64_t lane, int64_t row, int width, int size) {
  const int v = 16 / size;
  return ((uintptr_t)d & 15) == 0 && lane % v == 0 && row % v == 0 && width % v == 0;
}

// -------------------------------------------------------------- embedding
// out[r] = scale table[tok[r]], one rounding.  Bound by the writes of the
// rows: the 256 table rows stay in the L2s.  A thread moves 16 bytes a step,
// `steps` of them, over per_block consecutive vectors of the output.
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_kernel(const EmbedArgs a, uint32_t rows,
                                                    uint32_t block_rows) {
  const uint32_t vpr = a.width / V;
  for (uint64_t r0 = (uint64_t)blockIdx.x * block_rows; r0 < rows;
       r0 += (uint64_t)gridDim.x * block_rows) {
    const uint32_t n = (uint32_t)min((uint64_t)block_rows, rows - r0) * vpr;
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
      const uint32_t k = i / vpr, col = (i - k * vpr) * V, r = (uint32_t)r0 + k;
      const uint32_t l = r / (uint32_t)a.q.T, t = r - l * a.q.T;
      if ((int)t >= seq_len(a.q, l)) continue;
      const uint32_t byte = a.tok[l * a.tok_lane + t];
      float v[V];
      ld_vec<V>((const T*)a.table + (size_t)byte * a.width + col, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= a.scale;
      st_vec<V>((T*)a.out.d + l * a.out.lane + t * a.out.row + col, v);
    }
  }
}

// ----------------------------------------------------- embedding gradient
// dtable[v] = scale sum of dout's rows whose token is v, in fp32 and in an
// order that only the sizes decide (no atomics).  A block sorts the tokens of
// `chunk` rows (a stable counting sort in LDS), then its groups of G lanes
// take equal parts of the sorted rows and sum run by run, so a byte that
// fills most rows is spread over all groups like any other.  Runs that cross
// a group's border leave their pieces in LDS, and the group they start in
// joins them in order.  One partial row per byte that occurs in the chunk
// goes to the workspace; the second kernel sums a byte's partials over the
// chunks.  dout is read once; the partials are at most 256 / chunk of it.
constexpr int EG_THREADS = 512, EG_WAVES = EG_THREADS / 64, EG_MAX_CHUNK = 2048;

// rows a block sorts: enough blocks for every CU, few partials
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
  __shared__ float head[V * NV][EG_THREADS], tail[V * NV][EG_THREADS];
  const int tid = threadIdx.x, w = tid >> 6, ln = tid & 63;
  const uint32_t c = blockIdx.x, r0 = c * (uint32_t)chunk;

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
    valid[i] = false;
    key[i] = 0;
    rank[i] = 0;
    if (i < batches) {
      const int b = w * batches + i;
      const uint32_t lr = b * 64 + ln, r = r0 + lr;
      uint32_t byte = 0;
      if (lr < (uint32_t)chunk && r < rows) {
        const uint32_t l = r / (uint32_t)a.q.T, t = r - l * a.q.T;
        if ((int)t < seq_len(a.q, l)) {
          valid[i] = true;
          byte = a.tok[l * a.tok_lane + t];
          key[i] = ((uint64_t)byte << 56) | (uint64_t)(l * a.dout.lane + t * a.dout.row);
        }
      }
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
  auto store = [&](int byte, const float (&acc)[V * NV]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * G + gl) * V;
      if (col < a.width) {
        float v[V];
        float* dst;
        if (slot_map) {
          dst = part + ((size_t)c * slots + slot[byte]) * a.width + col;
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = acc[k * V + j];
        } else {
          dst = a.dtable + (size_t)byte * a.width + col;
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = acc[k * V + j] * a.scale;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) dst[j] = v[j];
      }
    }
  };
  float acc[V * NV];
#pragma unroll
  for (int j = 0; j < V * NV; ++j) acc[j] = 0.0f;
  int cur = p0 < p1 ? (int)(list[p0] >> 56) : 0;
  auto flush = [&](int byte) {  // the run of `byte` ends here, or the group's part does
    if (start[byte] < p0) {
#pragma unroll
      for (int j = 0; j < V * NV; ++j) head[j][tid] = acc[j];
    } else if (start[byte + 1] > p1) {
#pragma unroll
      for (int j = 0; j < V * NV; ++j) tail[j][tid] = acc[j];
    } else {
      store(byte, acc);
    }
  };
  constexpr int U = 4;  // rows in flight
  for (int p = p0; p < p1; p += U) {
    float v[U][NV][V];
    int byte[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t e = list[min(p + k, p1 - 1)];
      byte[k] = (int)(e >> 56);
      const T* src = dout + (e & 0x00FFFFFFFFFFFFFFull);
#pragma unroll
      for (int m = 0; m < NV; ++m) {
        const int col = (m * G + gl) * V;
        if (col < a.width) ld_vec<V>(src + col, v[k][m]);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (p + k < p1) {
        if (byte[k] != cur) {
          flush(cur);
          cur = byte[k];
#pragma unroll
          for (int j = 0; j < V * NV; ++j) acc[j] = 0.0f;
        }
#pragma unroll
        for (int m = 0; m < NV; ++m)
          if ((m * G + gl) * V < a.width)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[m * V + j] += v[k][m][j];
      }
    }
  }
  if (p0 < p1) flush(cur);
  __syncthreads();
  // a run that starts here and goes on: its later pieces are the next groups' heads
  if (p0 < p1 && start[cur] >= p0 && start[cur + 1] > p1) {
#pragma unroll
    for (int j = 0; j < V * NV; ++j) acc[j] = tail[j][tid];
    const int end = start[cur + 1];
    for (int h = g + 1; h < groups && h * per < end; ++h)
#pragma unroll
      for (int j = 0; j < V * NV; ++j) acc[j] += head[j][h * G + gl];
    store(cur, acc);
  }
  if (!slot_map)  // the only chunk: bytes that do not occur have no gradient
    for (int i = tid; i < 256 * a.width; i += EG_THREADS)
      if (slot[i / a.width] == 0xFFFF) a.dtable[i] = 0.0f;
}

// a byte's partial rows summed over the chunks: groups of G lanes take every
// groups-th chunk, then the groups' sums are added in order
template <int V>
__global__ __launch_bounds__(EG_THREADS) void embed_grad_sum_kernel(
    const float* __restrict__ part, const uint16_t* __restrict__ slot_map, int chunks, int slots,
    int width, int G, float scale, float* __restrict__ dtable) {
  __shared__ float sums[V][EG_THREADS];
  const int byte = blockIdx.x, tid = threadIdx.x, g = tid / G, gl = tid % G, groups = EG_THREADS / G;
  const int col = (blockIdx.y * G + gl) * V;
  const uint16_t* map = slot_map + (size_t)byte * chunks;
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.0f;
  if (col < width) {
    constexpr int U = 8;
    for (int c = g; c < chunks; c += U * groups) {
      float v[U][V];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int cc = c + k * groups;
        const uint32_t s = cc < chunks ? map[cc] : 0xFFFF;
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = 0.0f;
        if (s != 0xFFFF) ld_vec<V>(part + ((size_t)cc * slots + s) * width + col, v[k]);
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[k][j];
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
// loss = log sum_j e^{x_j} - x_target, dx = scale (softmax - onehot).  A wave
// holds a row, four logits a lane, so each logit is read once and its
// gradient written once: bound by those bytes.  The largest logit's own term
// (1) stays out of the sum: rest = sum of the others, loss = log1p(rest) +
// (max - x_target), so a byte predicted with near certainty keeps its small
// loss and gradient, which 1 + rest would round away.
constexpr int LOSS_THREADS = 512, LOSS_WAVES = LOSS_THREADS / 64, LOSS_U = 4;

// blocks: four rows at a time for each wave, at most two blocks a CU
int loss_blocks(int64_t rows) {
  return (int)std::min<int64_t>(512, (rows + 63) / 64);
}

__device__ __forceinline__ void ld_row4(const float* p, float (&v)[4]) {
  const float4 t = raw_f4(p);
  v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ void ld_row4(const uint16_t* p, float (&v)[4]) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  v[0] = u2f(t.x << 16); v[1] = u2f(t.x & 0xFFFF0000u);
  v[2] = u2f(t.y << 16); v[3] = u2f(t.y & 0xFFFF0000u);
}
__device__ __forceinline__ void st_row4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void st_row4(uint16_t* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) =
      make_uint2((uint32_t)f32_to_bf16(v[0]) | ((uint32_t)f32_to_bf16(v[1]) << 16),
                 (uint32_t)f32_to_bf16(v[2]) | ((uint32_t)f32_to_bf16(v[3]) << 16));
}

// log(1 + x), x >= 0: log(y) x / (y - 1) with y = 1 + x rounded corrects y's rounding
__device__ __forceinline__ float log1p_pos(float x) {
  const float y = 1.0f + x, d = y - 1.0f;
  const float r = d > 0.0f ? log_core(y) * (x / d) : x;
  return y < __builtin_huge_valf() ? r : y;  // inf and NaN
}

// VEC: rows aligned for a lane's four logits at once
template <typename T, bool VEC>
__global__ __launch_bounds__(LOSS_THREADS) void loss_kernel(const LossArgs a, uint32_t rows,
                                                            float* __restrict__ part_bias,
                                                            double* __restrict__ part_total) {
  __shared__ float sm[LOSS_WAVES][256];
  __shared__ double st[LOSS_WAVES];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = threadIdx.x & 63;
  const uint32_t waves = gridDim.x * LOSS_WAVES, me = blockIdx.x * LOSS_WAVES + w;
  const T* in = (const T*)a.logits.d;
  T* dx = (T*)a.dlogits.d;
  float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f}, db[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.bias)
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[j] = a.bias[4 * ln + j];
  double total = 0.0;
  for (uint64_t g = me; g * LOSS_U < rows; g += waves) {
    float x[LOSS_U][4];
    uint32_t l[LOSS_U], t[LOSS_U];
    bool in_rows[LOSS_U], live[LOSS_U];
#pragma unroll
    for (int k = 0; k < LOSS_U; ++k) {
      const uint64_t r = g * LOSS_U + k;
      in_rows[k] = r < rows;
      const uint32_t rr = in_rows[k] ? (uint32_t)r : 0;
      l[k] = rr / (uint32_t)a.q.T;
      t[k] = rr - l[k] * a.q.T;
      live[k] = in_rows[k] && (int)t[k] < seq_len(a.q, l[k]);
      if (live[k]) {
        const T* p = in + l[k] * a.logits.lane + t[k] * a.logits.row + 4 * ln;
        if constexpr (VEC) {
          ld_row4(p, x[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[k][j] = ldv(p + j);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < LOSS_U; ++k) {
      if (!in_rows[k]) continue;
      float gr[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (live[k]) {
        const int tgt = a.tgt[l[k] * a.tgt_lane + t[k]];
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = x[k][j] + bias[j];
        const float m = wave_max(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])));
        // the value at the target, and the place of the first largest logit
        const int tj = tgt & 3, tl = tgt >> 2;
        const float pick = tj == 0 ? e[0] : tj == 1 ? e[1] : tj == 2 ? e[2] : e[3];
        const float xt = u2f(__builtin_amdgcn_readlane(f2u(pick), tl));
        const int mj = e[0] == m ? 0 : e[1] == m ? 1 : e[2] == m ? 2 : e[3] == m ? 3 : 4;
        const uint64_t has = __builtin_amdgcn_ballot_w64(mj < 4);
        const int ml = has ? __builtin_ctzll(has) : -1;
        const int top = ml < 0 ? -1 : 4 * ml + __builtin_amdgcn_readlane(mj, ml);
        float rest = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          e[j] = __builtin_amdgcn_exp2f((e[j] - m) * 1.44269504088896340736f);
          rest += 4 * ln + j == top ? 0.0f : e[j];
        }
        rest = wave_sum(rest);
        float loss;
        if (m == -__builtin_huge_valf()) {  // nothing is allowed: no gradient
          loss = __builtin_huge_valf();
        } else {
          loss = log1p_pos(rest) + (m - xt);
          const float sum = 1.0f + rest, inv = a.scale / sum;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            gr[j] = e[j] * inv;
            if (4 * ln + j == tgt) gr[j] = tgt == top ? -(rest * inv) : (e[j] - sum) * inv;
            db[j] += gr[j];
          }
        }
        total += (double)loss;
        if (ln == 0) a.loss[l[k] * (int64_t)a.q.T + t[k]] = loss;
      }
      if (dx) {
        T* p = dx + l[k] * a.dlogits.lane + t[k] * a.dlogits.row + 4 * ln;
        if constexpr (VEC) {
          st_row4(p, gr);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) stv(p + j, gr[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) sm[w][4 * ln + j] = db[j];
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
  // a block's threads take 8 vectors each; with fewer than two blocks a CU, one
  const uint64_t vecs = (uint64_t)rows * vpr;
  const uint32_t per = vecs >= 512ull * 2048 ? 2048 : 256;
  const uint32_t block_rows = std::max<uint32_t>(1, per / vpr);
  const dim3 grid(std::min<uint32_t>(MAX_BLOCKS, (rows + block_rows - 1) / block_rows));
  if (a.bf16) {
    if (vec) BOA_LAUNCH((embed_kernel<uint16_t, 8>), grid, dim3(256), 0, s, a, rows, block_rows);
    else BOA_LAUNCH((embed_kernel<uint16_t, 1>), grid, dim3(256), 0, s, a, rows, block_rows);
  } else {
    if (vec) BOA_LAUNCH((embed_kernel<float, 4>), grid, dim3(256), 0, s, a, rows, block_rows);
    else BOA_LAUNCH((embed_kernel<float, 1>), grid, dim3(256), 0, s, a, rows, block_rows);
  }
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
  const int n = loss_blocks(rows), al = a.bf16 ? 8 : 16;
  auto fits = [&](const void* d, int64_t lane, int64_t row) {
    return ((uintptr_t)d & (al - 1)) == 0 && lane % 4 == 0 && row % 4 == 0;
  };
  const bool vec = fits(a.logits.d, a.logits.lane, a.logits.row) &&
                   (!a.dlogits.d || fits(a.dlogits.d, a.dlogits.lane, a.dlogits.row));
  // doubles first: the workspace is 8-byte aligned
  double* pt = (double*)a.work;
  float* pb = n == 1 ? nullptr : (float*)(pt + n);
#define BOA_LOSS(Tv, VECv) \
  BOA_LAUNCH((loss_kernel<Tv, VECv>), dim3(n), dim3(LOSS_THREADS), 0, s, a, rows, pb, pt)
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

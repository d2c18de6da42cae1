// Attention over a paged 8-bit key / value cache (csrc/cache.cu describes the cache).
//
// For query j of request i (n_i queries, L_i tokens in the cache, these queries' own among them), head h of
// key / value head h / G, with ks, vs the scales of the page a token lies in:
//   o = sum_t p_t vs_t V_t / sum_t p_t,   p_t = exp(scale * ks_t q . K_t),   t < L_i, causal: t <= L_i - n_i + j.
// The reference has neither a cache nor ragged batches; the dense form it builds is
// src/Optimizer/Optimizer.cc:2606-2860.
//
// `cached_split_kernel` serves few query rows per request (decoding).  There the cost is reading the cache:
// 2 L D bytes per key / value head, each read once and used for the G query heads of its group.
//   - The G heads and n_i queries of a key / value head share its keys as the columns of one tile of 8 NQ rows of Q,
//     so a byte is loaded and converted once.  Products run on mma.sync m16n8k16 with the cache as the 16-row
//     operand (S^T = K Q^T, O^T = V^T P^T): eight query rows cost no padding, where a tcgen05 tile would want 128.
//   - Work is cut in units of 128 keys of one (request, head, 16 rows); the units of the whole batch, numbered in
//     that order, are dealt to a fixed grid in equal contiguous ranges, whatever the lengths: every block finds its
//     range by a prefix sum over the requests.  A block leaves a partial result (running maximum, sum, output) for
//     at most its first and its last item; cached_join_kernel merges those in a fixed order.
//   - A warp owns 32 keys of a unit and a ring of its own in shared memory, which one of its lanes fills by TMA
//     (boxes of 16 or 32 rows of a page) ahead of use and across item borders; no block barrier stands in the loop.
//   - Codes become f16 in registers (exact: e4m3 is a subset of f16), bf16 queries too, each row scaled by a power
//     of two.  K's scale multiplies the scores, V's scale the product of its keys: no operand is rounded again but
//     P, to f16.
#include "common.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace kcg {

int* device_status_word();
int encode_tmap(CUtensorMap* out, int dtype, const void* base, int rank, const uint64_t* dims,
                const uint64_t* strides_bytes, const uint32_t* box, int swizzle_bytes);

namespace {
using namespace sm100;

constexpr int WARPS = 4;
constexpr int WKEYS = 32;           // keys of a warp's tile
constexpr int UNIT = WARPS * WKEYS; // keys of a unit
constexpr float kLazy = 8.0f;       // rescale only when the maximum grew by more than 2^8 (p <= 2^8 fits f16)

struct CachedParams {
  const void* Q;
  int64_t q_st, q_sh;
  void* O;
  int64_t o_st, o_sh;
  const float* ks;
  const float* vs;
  const int32_t* table;
  int64_t table_stride, width;
  const int32_t* lengths;
  const int32_t* cu;                // NULL: `uniform` queries each
  int64_t T, uniform, num_pages;
  int B, Hkv, G, page, causal;
  int box;                          // rows of a TMA box: 32 where a page is a multiple of that, else 16
  float scale_log2;
  float* part_o;                    // [grid][2][NQ D / 4][32 lanes]
  float* part_ml;                   // [grid][2][8 NQ][2]
  int* meta;                        // [grid][8]
  int* status;
};

// What a request contributes: its queries [t0, t0 + n), keys [0, len).
struct Request { int t0, n, len; };
__device__ __forceinline__ Request request_of(const CachedParams& p, int i) {
  Request r;
  int64_t a, b;
  if (p.cu) {
    a = p.cu[i];
    b = p.cu[i + 1];
    const int64_t a1 = min(max(a, static_cast<int64_t>(0)), p.T), b1 = min(max(b, a1), p.T);
    if ((a1 != a || b1 != b) && p.status) *p.status = KCG_ERR_INVALID_ARG;
    a = a1;
    b = b1;
  } else {
    a = i * p.uniform;
    b = a + p.uniform;
  }
  const int64_t len = p.lengths[i], most = p.width * p.page;
  const int64_t l1 = min(max(len, static_cast<int64_t>(0)), most);
  if (l1 != len && p.status) *p.status = KCG_ERR_INVALID_ARG;
  r.t0 = static_cast<int>(a);
  r.n = static_cast<int>(b - a);
  r.len = static_cast<int>(l1);
  return r;
}
__device__ __forceinline__ int unit_tiles(int len) { return len > 0 ? (len + UNIT - 1) / UNIT : 1; }
template <int ROWS> __device__ __forceinline__ int row_blocks(const CachedParams& p, int n) { return (n * p.G + ROWS - 1) / ROWS; }
template <int ROWS> __device__ __forceinline__ int64_t request_units(const CachedParams& p, const Request& r) {
  return static_cast<int64_t>(p.Hkv) * row_blocks<ROWS>(p, r.n) * unit_tiles(r.len);
}

// A place in the batch's sequence of units.
template <int ROWS> struct Cursor {
  Request r;
  int i, h, rb, tile, tiles, nrb;
  __device__ __forceinline__ void enter(const CachedParams& p, int req, int64_t offset) {
    i = req;
    r = request_of(p, i);
    tiles = unit_tiles(r.len);
    nrb = row_blocks<ROWS>(p, r.n);
    const int64_t item = offset / tiles;
    tile = static_cast<int>(offset - item * tiles);
    h = static_cast<int>(item / nrb);
    rb = static_cast<int>(item - static_cast<int64_t>(h) * nrb);
  }
  // to the next unit; true when it begins another item (only called while there is one)
  __device__ __forceinline__ bool next(const CachedParams& p) {
    if (++tile < tiles) return false;
    tile = 0;
    if (++rb == nrb) {
      rb = 0;
      if (++h == p.Hkv) {
        h = 0;
        do {
          ++i;
          r = request_of(p, i);
        } while (r.n == 0);
        tiles = unit_tiles(r.len);
        nrb = row_blocks<ROWS>(p, r.n);
      }
    }
    return true;
  }
};

__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t (&r)[2]) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
}

// The low / high two e4m3 codes of a word as two f16.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // c = a b
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 8x8 16-bit transpose across the warp: lane (g, t) gives row g, columns 2t and 2t + 1, and gets column g, rows 2t, 2t + 1
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// over the eight lanes that share t = lane % 4
__device__ __forceinline__ float column_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float column_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Byte offset of 16-byte chunk c of row r inside a tile of D-byte rows: TMA's swizzle of D bytes (the chunk's number
// xor that of its 128-byte line).  K is read by (row = lane / 4, chunk = lane % 4 (x 2 + c)), V by (row = 2 (lane % 4) + const, chunk = lane / 4):
// at D = 128 both are free of bank conflicts, at D = 64 V's 8-byte reads meet in pairs.
template <int D> __device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  if constexpr (D == 128) return r * 128 + ((c ^ (r & 7)) << 4);
  else return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// Blocks per SM and ring stages: what the registers of 8 NQ rows leave room for.
template <int NQ> struct SplitShape { static constexpr int BLOCKS = NQ == 1 ? 3 : 2, STAGES = NQ == 1 ? 2 : 3; };

template <int D, int NQ> struct SplitSmem {
  static constexpr int STAGES = SplitShape<NQ>::STAGES;
  static constexpr int TILE = WKEYS * D;              // bytes of a K or V tile of one warp
  static constexpr int NREG = NQ * D / 4;             // output registers of a lane
  uint8_t ring[WARPS][STAGES][2][TILE];
  static constexpr int FOLDS = NQ == 1 ? 2 : 1;       // (two do not fit beside a ring of three stages)
  float fold[FOLDS][NREG][32];                        // a warp's output on its way into another's
  float fold_ml[FOLDS][8 * NQ][2];
  float side[WARPS][STAGES][8];                       // per half tile: k scale (2), v scale (2), keys (2)
  uint64_t full[WARPS][STAGES];
  int64_t scan[WARPS];
  int64_t start_off;
  int start_i;
  int abort;
};

// Query fragments of an item: lane (g, t) holds row 8 q + g of tile q, for every 16-wide step s of the product the four
// dims that lane t's K words of that step hold, (D / 4) t + 4 s and on.  bf16 rows are scaled to f16's range by a power of two; f[q] receives
// its inverse for rows 8 q + 2 t and 8 q + 2 t + 1, the columns of S^T this lane will hold.
template <typename T, int D, int NQ>
__device__ __forceinline__ void load_queries(const CachedParams& p, const Cursor<8 * NQ>& c, int lane, uint32_t (&qb)[NQ][D / 16][2],
                                             float (&f)[NQ][2]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int R = c.rb * (8 * NQ) + 8 * q + g;
    uint4 v[D / 32];
    const bool live = R < c.r.n * p.G;
    const int j = live ? R / p.G : 0;
    const T* src = static_cast<const T*>(p.Q) + (c.r.t0 + j) * p.q_st + (c.h * p.G + (live ? R - j * p.G : 0)) * p.q_sh;
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
      v[k] = live ? __ldg(reinterpret_cast<const uint4*>(src + (D / 4) * t) + k) : make_uint4(0, 0, 0, 0);
    f[q][0] = f[q][1] = 1.f;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __vmaxu2(m, w[e] & 0x7fff7fffu);
      }
      m = max(m & 0xffffu, m >> 16);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // largest element to [2^13, 2^14); an element 2^-27 of it or more keeps all of its bits
      int e = static_cast<int>(m >> 7) - 127 - 13;
      e = e < -113 ? -113 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      f[q][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      f[q][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = pack_f16(__uint_as_float(w[x] << 16) * up, __uint_as_float(w[x] & 0xffff0000u) * up);
      }
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const uint4 x = v[s / 2];
      qb[q][s][0] = (s & 1) ? x.z : x.x;
      qb[q][s][1] = (s & 1) ? x.w : x.y;
    }
  }
}

// A lane's share of an item's output, divided by the row sums.  Lane (g, t) holds of tile q rows 8 q + 2 t + e (e = 0, 1),
// dims (D / 8) g + 2 j + half in o[j][2 half + e]; here tiles j0 .. j0 + N - 1.
template <typename T, int D, int N>
__device__ __forceinline__ void store_rows(const CachedParams& p, int t0, int n, int h, int row, int lane, const float (&o)[N][4],
                                           const float (&l)[2], int j0) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int R = row + 2 * t + e;
    if (R >= n * p.G) continue;
    const int j = R / p.G;
    T* dst = static_cast<T*>(p.O) + (t0 + j) * p.o_st + (h * p.G + (R - j * p.G)) * p.o_sh + g * (D / 8) + 2 * j0;
    const float inv = l[e] == 0.f ? 0.f : 1.0f / l[e];    // a row that sees no key is zero
    uint32_t w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float v[2] = {o[k][e] * inv, o[k][2 + e] * inv};
      w[k] = Words<T>::pack(v);
    }
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int k = 0; k < N; k += 4) reinterpret_cast<uint4*>(dst)[k / 4] = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) reinterpret_cast<uint32_t*>(dst)[k] = w[k];
    }
  }
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(WARPS * 32, SplitShape<NQ>::BLOCKS)
cached_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CachedParams p) {
  extern __shared__ uint8_t smem_raw[];
  using Smem = SplitSmem<D, NQ>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  constexpr int ROWS = 8 * NQ, STAGES = Smem::STAGES, NREG = Smem::NREG;
  constexpr int MT = D / 16;                // output tiles of 16 dims
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  grid_launch_dependents();
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&sm.full[warp][s], 1);
    if (warp == 0) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
      sm.abort = 0;
    }
    mbar_fence_init();
  }
  grid_dependency_wait();

  // ---- this block's range of units ----
  const int per = (p.B + WARPS * 32 - 1) / (WARPS * 32);
  const int i_lo = min(tid * per, p.B), i_hi = min(i_lo + per, p.B);
  int64_t mine = 0;
  for (int i = i_lo; i < i_hi; ++i) mine += request_units<ROWS>(p, request_of(p, i));
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) sm.scan[warp] = upto;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) upto += sm.scan[w];
    total += sm.scan[w];
  }
  const int64_t grid = min(static_cast<int64_t>(gridDim.x), total);   // blocks at work: none is without a unit
  int* meta = p.meta + blockIdx.x * 8;
  if (tid == 0) meta[0] = -1;
  if (blockIdx.x >= grid) return;
  const int64_t u0 = total * blockIdx.x / grid, u1 = total * (blockIdx.x + 1) / grid;
  if (upto - mine <= u0 && u0 < upto) {     // one thread's requests hold the first unit
    int64_t off = u0 - (upto - mine);
    int i = i_lo;
    for (;; ++i) {
      const int64_t n = request_units<ROWS>(p, request_of(p, i));
      if (off < n) break;
      off -= n;
    }
    sm.start_i = i;
    sm.start_off = off;
  }
  __syncthreads();

  Cursor<ROWS> cur;
  cur.enter(p, sm.start_i, sm.start_off);
  const int units = static_cast<int>(u1 - u0);

  // ---- loading: a cursor of its own, running ahead ----
  Cursor<ROWS> ld = cur;
  int ld_unit = 0;
  // this lane's look-ahead: page, row in it and scales of half lane & 1 of tile pid_tile + lane / 2
  int pid = -1, pid_row = 0, pid_tile = -1 << 20;
  float pid_ks = 0.f, pid_vs = 0.f;
  auto load_next = [&](int stage) {
    if (ld_unit >= units) return;
    if (ld.tile < pid_tile || ld.tile >= pid_tile + 16) {
      pid_tile = ld.tile;
      const int key = (ld.tile + (lane >> 1)) * UNIT + warp * WKEYS + (lane & 1) * 16;
      pid = -1;
      pid_row = 0;
      if (key < ld.r.len) {
        const int w = key / p.page;
        pid_row = key - w * p.page;
        pid = p.table[ld.i * p.table_stride + w];
        if (pid < 0 || pid >= p.num_pages) {
          pid = -1;
          if (p.status) *p.status = KCG_ERR_INVALID_ARG;
        }
      }
      pid_ks = pid_vs = 0.f;
      if (pid >= 0) {
        pid_ks = p.ks[static_cast<int64_t>(pid) * p.Hkv + ld.h];
        pid_vs = p.vs[static_cast<int64_t>(pid) * p.Hkv + ld.h];
      }
    }
    const int at = ld.tile - pid_tile;
    if ((lane >> 1) == at) {
      float* s = sm.side[warp][stage] + (lane & 1);
      s[0] = pid_ks;
      s[2] = pid_vs;
      reinterpret_cast<int*>(s)[4] = pid >= 0 ? min(16, ld.r.len - (ld.tile * UNIT + warp * WKEYS + (lane & 1) * 16)) : 0;
    }
    const int pg0 = __shfl_sync(0xffffffffu, pid, 2 * at), pg1 = __shfl_sync(0xffffffffu, pid, 2 * at + 1);
    const int in0 = __shfl_sync(0xffffffffu, pid_row, 2 * at), in1 = __shfl_sync(0xffffffffu, pid_row, 2 * at + 1);
    if (lane == 0) {
      // rows behind the last token are loaded with their page and left out by the reader; a half tile of no page is not
      // loaded at all (with boxes of 32 rows both halves are one page's, and the second may only lie behind the end)
      uint8_t* kdst = sm.ring[warp][stage][0];
      uint8_t* vdst = sm.ring[warp][stage][1];
      uint64_t* bar = &sm.full[warp][stage];
      const bool second = pg1 >= 0 && p.box == 16;
      mbar_expect_tx(bar, 2 * D * ((pg0 >= 0 ? p.box : 0) + (second ? 16 : 0)));
      if (pg0 >= 0) {
        tma_load_4d(kdst, &tmK, bar, 0, in0, ld.h, pg0);
        tma_load_4d(vdst, &tmV, bar, 0, in0, ld.h, pg0);
      }
      if (second) {
        tma_load_4d(kdst + 16 * D, &tmK, bar, 0, in1, ld.h, pg1);
        tma_load_4d(vdst + 16 * D, &tmV, bar, 0, in1, ld.h, pg1);
      }
    }
    if (++ld_unit < units) {
      if (ld.next(p)) pid_tile = -1 << 20;
    }
  };
  __syncwarp();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_next(s);

  uint32_t qb[NQ][D / 16][2];
  float cq[NQ][2];                          // what a score of this lane's columns is multiplied with, but for K's scale
  float o[NQ][MT][4], m[NQ][2], l[NQ][2];
  bool fresh = true;
  int stage = 0;
  bool first_item = true;
  int item_tile0 = cur.tile;                // of the part of the item this block has
  int lim0 = 0;                             // first key the item's first row must not see
  uint32_t parity = 0;
  for (int u = 0; u < units; ++u) {
    __syncwarp();                           // every lane has read the tile that is replaced now
    load_next(stage == 0 ? STAGES - 1 : stage - 1);
    if (fresh) {
      load_queries<T, D, NQ>(p, cur, lane, qb, cq);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int j = 0; j < MT; ++j) o[q][j][0] = o[q][j][1] = o[q][j][2] = o[q][j][3] = 0.f;
        m[q][0] = m[q][1] = -INFINITY;
        l[q][0] = l[q][1] = 0.f;
        cq[q][0] *= p.scale_log2;
        cq[q][1] *= p.scale_log2;
      }
      fresh = false;
      item_tile0 = cur.tile;
      lim0 = p.causal ? cur.r.len - cur.r.n + 1 + cur.rb * ROWS / p.G : INT32_MAX;
    }
    // A wait that runs out of time marks the launch as failed and goes on with what is there: the barriers that follow
    // need every warp, and the status tells the host that the result is void.
    if (!mbar_wait(&sm.full[warp][stage], parity, &sm.abort) && !*static_cast<volatile int*>(&sm.abort)) {
      *static_cast<volatile int*>(&sm.abort) = 1;
      if (p.status) *p.status = KCG_ERR_TIMEOUT;
    }
    __syncwarp();
    const uint32_t kt = smem_u32(sm.ring[warp][stage][0]), vt = smem_u32(sm.ring[warp][stage][1]);
    const float* side = sm.side[warp][stage];
    const int key0 = cur.tile * UNIT + warp * WKEYS;
    const int have0 = reinterpret_cast<const int*>(side)[4], have1 = reinterpret_cast<const int*>(side)[5];
    const int R0 = cur.rb * ROWS;
    if ((have0 | have1) > 0) {
    // ---- scores, S^T: element x of half u is key 16 u + g + 8 (x / 2), row 2 t + (x & 1) of its tile ----
    float s[NQ][2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t w0[4], w1[4];
        lds128(kt + tile_offset<D>(16 * half + g, (D / 64) * t + c), w0);
        lds128(kt + tile_offset<D>(16 * half + 8 + g, (D / 64) * t + c), w1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t a[4];
          e4m3x4_to_f16(w0[x], a[0], a[2]);
          e4m3x4_to_f16(w1[x], a[1], a[3]);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (c == 0 && x == 0) mma16816_first(s[q][half], a, qb[q][0][0], qb[q][0][1]);
            else mma16816(s[q][half], a, qb[q][4 * c + x][0], qb[q][4 * c + x][1]);
          }
        }
      }
      const float ks = side[half];
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[q][half][x] *= cq[q][x & 1] * ks;
    }
    // ---- mask: keys a row must not see, keys that are not there ----
    const bool ragged = have0 < 16 || have1 < 16;
    if (ragged || key0 + WKEYS > lim0) {
      const int past = cur.r.len - cur.r.n + 1;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int lim = p.causal ? past + (R0 + 8 * q + 2 * t + e) / p.G : cur.r.len;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int in = g + 8 * (k & 1);
            if (in >= (k < 2 ? have0 : have1) || key0 + 16 * (k >> 1) + in >= lim) s[q][k >> 1][2 * (k & 1) + e] = -INFINITY;
          }
        }
    }
    // ---- running maximum: changed only when some row outgrows it by 2^kLazy (or has its first keys) ----
    bool outgrown = false;
    float top[NQ][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[q][e] = fmaxf(fmaxf(s[q][0][e], s[q][0][2 + e]), fmaxf(s[q][1][e], s[q][1][2 + e]));
        outgrown = outgrown || top[q][e] > m[q][e] + kLazy;
      }
    if (__any_sync(0xffffffffu, outgrown)) {
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = fmaxf(m[q][e], column_max(top[q][e]));
          const float grow = x == m[q][e] ? 1.f : exp2f_approx(m[q][e] - x);      // 0 for the first keys
          m[q][e] = x;
          l[q][e] *= grow;
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[q][j][e] *= grow;
            o[q][j][2 + e] *= grow;
          }
        }
    }
    uint32_t pb[NQ][2][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const float b0 = m[q][0] == -INFINITY ? 0.f : m[q][0], b1 = m[q][1] == -INFINITY ? 0.f : m[q][1];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float p0 = exp2f_approx(s[q][k >> 1][2 * (k & 1)] - b0), p1 = exp2f_approx(s[q][k >> 1][2 * (k & 1) + 1] - b1);
        l[q][0] += p0;
        l[q][1] += p1;
        pb[q][k >> 1][k & 1] = transpose8x8(pack_f16(p0, p1));
      }
    }
    // ---- output, O^T: the product of each half tile with its page's scale ----
    const float vs0 = side[2], vs1 = side[3];
    constexpr int VW = D / 32;              // words of a lane's share of a V row
    uint32_t v[2][4][VW];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = half * 16 + 2 * t + (k & 1) + 8 * (k >> 1);
        if constexpr (D == 128) lds128(vt + tile_offset<D>(row, g), v[half][k]);
        else lds64(vt + tile_offset<D>(row, g >> 1) + (g & 1) * 8, v[half][k]);
      }
    if (ragged) {   // what lies behind the last token may be anything: P is zero there, and so must V be
      asm volatile("" ::: "memory");        // (a branch, not thirty-two selects in every tile)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (2 * t + (k & 1) + 8 * (k >> 1) >= (half ? have1 : have0))
#pragma unroll
            for (int c = 0; c < VW; ++c) v[half][k][c] = 0;
    }
    auto output = [&](auto same_scale) {
#pragma unroll
      for (int c = 0; c < VW; ++c) {        // word c: output tiles 2 c and 2 c + 1
        uint32_t a[2][2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int k = 0; k < 2; ++k) {     // keys 2 t, 2 t + 1, then those + 8
            const uint32_t x = v[half][2 * k][c], y = v[half][2 * k + 1][c];
            e4m3x4_to_f16(__byte_perm(x, y, 0x5140), a[half][0][2 * k], a[half][0][2 * k + 1]);
            e4m3x4_to_f16(__byte_perm(x, y, 0x7362), a[half][1][2 * k], a[half][1][2 * k + 1]);
          }
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float acc[4];
            float (&out)[4] = o[q][2 * c + e];
            mma16816_first(acc, a[0][e], pb[q][0][0], pb[q][0][1]);
            if constexpr (decltype(same_scale)::value) {
              mma16816(acc, a[1][e], pb[q][1][0], pb[q][1][1]);
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) out[x] = fmaf(acc[x], vs0, out[x]);
              mma16816_first(acc, a[1][e], pb[q][1][0], pb[q][1][1]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) out[x] = fmaf(acc[x], vs1, out[x]);
          }
      }
    };
    if (vs0 == vs1) output(std::true_type{}); else output(std::false_type{});
    }
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
    const bool last = u + 1 == units;
    if (cur.tile + 1 < cur.tiles && !last) {
      ++cur.tile;
      continue;
    }
    // ---- end of the item, or of this block's part of it: the four warps' results into warp 0 ----
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      l[q][0] = column_sum(l[q][0]);
      l[q][1] = column_sum(l[q][1]);
    }
    auto give = [&](int to) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) sm.fold[to][(q * MT + j) * 4 + x][lane] = o[q][j][x];
        if (g == 0)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sm.fold_ml[to][8 * q + 2 * t + e][0] = m[q][e];
            sm.fold_ml[to][8 * q + 2 * t + e][1] = l[q][e];
          }
      }
    };
    auto take = [&](int from) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float mine_w[2], other_w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m2 = sm.fold_ml[from][8 * q + 2 * t + e][0], l2 = sm.fold_ml[from][8 * q + 2 * t + e][1];
          const float hi = fmaxf(m[q][e], m2), base = hi == -INFINITY ? 0.f : hi;
          mine_w[e] = exp2f_approx(m[q][e] - base);
          other_w[e] = exp2f_approx(m2 - base);
          l[q][e] = l[q][e] * mine_w[e] + l2 * other_w[e];
          m[q][e] = hi;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            o[q][j][x] = o[q][j][x] * mine_w[x & 1] + sm.fold[from][(q * MT + j) * 4 + x][lane] * other_w[x & 1];
      }
    };
    __syncthreads();                        // the fold buffers are free
    if constexpr (Smem::FOLDS == 2) {
      if (warp >= 2) give(warp - 2);
      __syncthreads();
      if (warp < 2) take(warp);
      __syncthreads();
    } else {
#pragma unroll
      for (int w = 3; w > 1; --w) {
        if (warp == w) give(0);
        __syncthreads();
        if (warp == 0) take(0);
        __syncthreads();
      }
    }
    if (warp == 1) give(0);
    __syncthreads();
    if (warp == 0) {
      take(0);
      const bool whole = item_tile0 == 0 && cur.tile + 1 == cur.tiles;
      if (whole) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) store_rows<T, D, MT>(p, cur.r.t0, cur.r.n, cur.h, R0 + 8 * q, lane, o[q], l[q], 0);
      } else {
        const int slot = first_item ? 0 : 1;
        float* po = p.part_o + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * (NREG * 32) + lane;
        float* pm = p.part_ml + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * (ROWS * 2);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) po[((q * MT + j) * 4 + x) * 32] = o[q][j][x];
          if (g == 0)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              pm[2 * (8 * q + 2 * t + e)] = m[q][e];
              pm[2 * (8 * q + 2 * t + e) + 1] = l[q][e];
            }
        }
        if (item_tile0 == 0 && lane == 0) {
          // the item begins in this block, which lists the parts.  Its last unit is x_end; block c holds unit x
          // when c = floor(((x + 1) grid - 1) / total).
          const int64_t x_end = u0 + u + (cur.tiles - 1 - cur.tile);
          meta[1] = static_cast<int>(((x_end + 1) * grid - 1) / total);
          meta[2] = slot;
          meta[3] = cur.r.t0;
          meta[4] = cur.r.n;
          meta[5] = cur.h;
          meta[6] = cur.rb;
          meta[0] = 1;
        }
      }
    }
    fresh = true;
    first_item = false;
    if (!last) cur.next(p);
  }
  // every tile that was asked for has been waited for; after a timeout, give the rest a little longer to land
  if (*static_cast<volatile int*>(&sm.abort)) {
    int zero = 0;
    for (int s = 0; s < STAGES; ++s) mbar_wait(&sm.full[warp][s], s < stage ? parity : parity ^ 1, &zero, 2000000ull);
  }
}

// Merges the parts of items that several blocks worked on; block (c, y) takes share y of the output tiles (16 dims x 8
// rows) of the item that begins in block c of the split kernel and ends behind it.  Its warps share the tiles, and
// where there are fewer tiles than warps, the parts of a tile; sums are taken in an order that depends on sizes alone.
constexpr int JOIN_WARPS = 8;
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(JOIN_WARPS * 32) cached_join_kernel(const CachedParams p) {
  extern __shared__ float join_w[];                   // [parts][ROWS]: weight of each part
  __shared__ float s_l[8 * NQ];
  __shared__ float s_acc[JOIN_WARPS][4][32];
  constexpr int MT = D / 16, ROWS = 8 * NQ, NREG = NQ * MT * 4;
  grid_launch_dependents();
  grid_dependency_wait();
  const int* meta = p.meta + blockIdx.x * 8;
  if (meta[0] < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x, parts = meta[1] - c0 + 1, slot = meta[2];
  auto part_of = [&](int i) { return static_cast<int64_t>(c0 + i) * 2 + (i ? 0 : slot); };
  // weights: one warp per row
  for (int r = warp; r < ROWS; r += JOIN_WARPS) {
    float m = -INFINITY;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, p.part_ml[(part_of(i) * ROWS + r) * 2]);
    m = warp_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int i = lane; i < parts; i += 32) {
      const float2 ml = *reinterpret_cast<const float2*>(&p.part_ml[(part_of(i) * ROWS + r) * 2]);
      const float w = exp2f_approx(ml.x - base);
      join_w[i * ROWS + r] = w;
      l += ml.y * w;
    }
    l = warp_sum(l);
    if (lane == 0) s_l[r] = l;
  }
  __syncthreads();
  const int tiles = NQ * MT / gridDim.y;              // of this block
  const int per_tile = tiles < JOIN_WARPS ? JOIN_WARPS / tiles : 1;   // warps that share a tile's parts
  const int t = lane & 3;
  for (int k0 = 0; k0 < tiles; k0 += JOIN_WARPS / per_tile) {
    const int k = blockIdx.y * tiles + k0 + warp / per_tile, q = k / MT;
    float acc[1][4] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 8
    for (int i = warp % per_tile; i < parts; i += per_tile) {
      const float* po = p.part_o + part_of(i) * (NREG * 32) + k * 128 + lane;
      const float w0 = join_w[i * ROWS + 8 * q + 2 * t], w1 = join_w[i * ROWS + 8 * q + 2 * t + 1];
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[0][x] = fmaf(po[32 * x], x & 1 ? w1 : w0, acc[0][x]);
    }
    if (per_tile > 1) {
#pragma unroll
      for (int x = 0; x < 4; ++x) s_acc[warp][x][lane] = acc[0][x];
      __syncthreads();
      if (warp % per_tile == 0)
        for (int o = 1; o < per_tile; ++o)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[0][x] += s_acc[warp + o][x][lane];
    }
    if (warp % per_tile == 0) {
      const float l[2] = {s_l[8 * q + 2 * t], s_l[8 * q + 2 * t + 1]};
      store_rows<T, D, 1>(p, meta[3], meta[4], meta[5], meta[6] * ROWS + 8 * q, lane, acc, l, k % MT);
    }
  }
}

// Workspace of the split kernel with 8 NQ rows: two parts per block, each the lanes' output registers and (m, l) of
// every row, and eight ints per block.
size_t split_workspace(int64_t D, int nq, int grid) {
  return static_cast<size_t>(grid) * (2 * (nq * D / 4 * 32 * 4) + 2 * (8 * nq * 2 * 4) + 32);
}
int split_grid(int nq) { return sm_count() * (nq == 1 ? SplitShape<1>::BLOCKS : SplitShape<2>::BLOCKS); }

// Tensor map of one cache: [page][head][row][D], boxes of `box` rows.
int cache_map(CUtensorMap* tm, const void* cache, const int64_t strides[3], int64_t D, const CachedParams& p) {
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.page), static_cast<uint64_t>(p.Hkv),
                            static_cast<uint64_t>(p.num_pages)};
  // the stride of a dim with one entry is never used, but has to be a valid one
  const uint64_t st[3] = {static_cast<uint64_t>(strides[2]), static_cast<uint64_t>(p.Hkv > 1 ? strides[1] : D),
                          static_cast<uint64_t>(p.num_pages > 1 ? strides[0] : D)};
  const uint32_t box[4] = {static_cast<uint32_t>(D), static_cast<uint32_t>(p.box), 1, 1};
  return encode_tmap(tm, KCG_F8E4M3, cache, 4, dims, st, box, static_cast<int>(D));   // a row is one swizzle span
}

template <typename T, int D, int NQ>
int launch_split(CachedParams& p, const CUtensorMap& tmK, const CUtensorMap& tmV, int64_t items, void* workspace, cudaStream_t stream) {
  const int grid = split_grid(NQ);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<size_t>(grid) * 2 * (NQ * D / 4 * 32);
  p.meta = reinterpret_cast<int*>(p.part_ml + static_cast<size_t>(grid) * 2 * (8 * NQ * 2));
  constexpr int SMEM = sizeof(SplitSmem<D, NQ>) + 1024;
  static_assert(SMEM <= 228 * 1024 / SplitShape<NQ>::BLOCKS - 1024, "the blocks of an SM do not fit its shared memory");
  auto kern = cached_split_kernel<T, D, NQ>;
  KCG_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  // Not as a programmatic dependent: a block that becomes resident beside the previous kernel's keeps its SM at that
  // kernel's split of L1 and shared memory, where one or two blocks fit, and the others queue behind it (142 instead
  // of 100 us for 64 requests of 4096 tokens).  The join may come early: it asks for the same split.
  kern<<<grid, WARPS * 32, SMEM, stream>>>(tmK, tmV, p);
  const int rc = check_launch("cached_split_kernel");
  if (rc) return rc;
  // Many items: few parts each, one block per item.  Few items: many parts each, whose reading is spread over a
  // block per output tile.
  const unsigned share = items * 8 <= grid ? NQ * D / 16 : NQ;
  KCG_CUDA_OK(cudaFuncSetAttribute(cached_join_kernel<T, D, NQ>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  launch_overlapped(cached_join_kernel<T, D, NQ>, dim3(grid, share), dim3(JOIN_WARPS * 32), (grid + 1) * 8 * NQ * sizeof(float), stream, p);
  return check_launch("cached_join_kernel");
}

template <typename T, int D>
int launch_cached(CachedParams& p, int64_t rows, const CUtensorMap& tmK, const CUtensorMap& tmV, void* workspace, cudaStream_t stream) {
  const int64_t items = static_cast<int64_t>(p.B) * p.Hkv;
  if (rows <= 8) return launch_split<T, D, 1>(p, tmK, tmV, items, workspace, stream);
  return launch_split<T, D, 2>(p, tmK, tmV, items * ((rows + 15) / 16), workspace, stream);
}

}  // namespace
}  // namespace kcg

extern "C" int kcg_fmha_cached_workspace(int64_t D, size_t* bytes) {
  using namespace kcg;
  clear_error();
  if (!bytes) return fail(KCG_ERR_INVALID_ARG, "fmha_cached_workspace: null pointer");
  if (D != 64 && D != 128) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: head dimension %lld has no kernel (64, 128)", static_cast<long long>(D));
  const size_t one = split_workspace(D, 1, split_grid(1)), two = split_workspace(D, 2, split_grid(2));
  *bytes = one > two ? one : two;
  return KCG_OK;
}

extern "C" int kcg_fmha_cached_fwd(int dtype, int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                                   float softmax_scale, int causal, const void* Q, const int64_t q_strides[2],
                                   const void* k_cache, const int64_t kc_strides[3], const float* k_scale,
                                   const void* v_cache, const int64_t vc_strides[3], const float* v_scale,
                                   int64_t num_pages, int64_t page_size, const int32_t* block_table, int64_t table_width,
                                   int64_t table_stride, const int32_t* lengths, const int32_t* cu_new, void* O,
                                   const int64_t o_strides[2], void* workspace, size_t workspace_bytes, void* stream) {
  using namespace kcg;
  clear_error();
  if (T < 0 || B < 0 || Hq < 0 || Hkv < 0 || num_pages < 0 || table_width < 0 || max_new < 0)
    return fail(KCG_ERR_INVALID_ARG, "fmha_cached: negative size");
  if (page_size < 16 || page_size % 16 || page_size > 65536)
    return fail(KCG_ERR_INVALID_ARG, "fmha_cached: page_size %lld is not a multiple of 16 up to 65536", static_cast<long long>(page_size));
  if (dtype != KCG_BF16 && dtype != KCG_F16) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: dtype %d has no kernel (bfloat16, float16)", dtype);
  if (D != 64 && D != 128) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: head dimension %lld has no kernel (64, 128)", static_cast<long long>(D));
  if (T == 0 || B == 0 || Hq == 0) return KCG_OK;
  if (Hkv == 0 || Hq % Hkv) return fail(KCG_ERR_INVALID_ARG, "fmha_cached: %lld query heads do not divide into %lld key heads", static_cast<long long>(Hq), static_cast<long long>(Hkv));
  if (!Q || !k_cache || !v_cache || !k_scale || !v_scale || !lengths || !O || !q_strides || !kc_strides || !vc_strides || !o_strides ||
      (table_width && !block_table))
    return fail(KCG_ERR_INVALID_ARG, "fmha_cached: null pointer");
  if (!cu_new && T % B) return fail(KCG_ERR_INVALID_ARG, "fmha_cached: without cu_new, %lld query rows must divide into %lld requests", static_cast<long long>(T), static_cast<long long>(B));
  if (table_stride < table_width) return fail(KCG_ERR_INVALID_ARG, "fmha_cached: the rows of the block table overlap");
  if (B > INT32_MAX / 2 || Hq > 65535 || T * Hq > INT32_MAX - 65536 || num_pages > INT32_MAX || table_width > INT32_MAX ||
      table_width * page_size > INT32_MAX - 65536)
    return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: sizes beyond 32 bits");
  bool ok = aligned16(Q) && aligned16(O) && aligned16(k_cache) && aligned16(v_cache) && aligned16(workspace);
  for (int i = 0; i < 2; ++i) ok = ok && q_strides[i] % 8 == 0 && o_strides[i] % 8 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && kc_strides[i] % 16 == 0 && vc_strides[i] % 16 == 0;
  if (num_pages == 0) return fail(KCG_ERR_INVALID_ARG, "fmha_cached: the cache has no pages");
  if ((Hkv > 1 && (kc_strides[1] <= 0 || vc_strides[1] <= 0)) || (num_pages > 1 && (kc_strides[0] <= 0 || vc_strides[0] <= 0)) ||
      kc_strides[2] <= 0 || vc_strides[2] <= 0)
    return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: the strides of the caches must be positive");
  if (!ok) return fail(KCG_ERR_ALIGNMENT, "fmha_cached: rows of Q, O, the caches and the workspace must start on 16-byte boundaries");
  size_t need = 0;
  const int rc = kcg_fmha_cached_workspace(D, &need);
  if (rc) return rc;
  if (!workspace || workspace_bytes < need)
    return fail(KCG_ERR_INVALID_ARG, "fmha_cached: the workspace has %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
  CachedParams p{};
  p.Q = Q; p.q_st = q_strides[0]; p.q_sh = q_strides[1];
  p.O = O; p.o_st = o_strides[0]; p.o_sh = o_strides[1];
  p.ks = k_scale; p.vs = v_scale;
  p.table = block_table; p.table_stride = table_stride; p.width = table_width;
  p.lengths = lengths; p.cu = cu_new;
  p.T = T; p.uniform = cu_new ? 0 : T / B; p.num_pages = num_pages;
  p.B = static_cast<int>(B); p.Hkv = static_cast<int>(Hkv); p.G = static_cast<int>(Hq / Hkv);
  p.page = static_cast<int>(page_size); p.causal = causal != 0;
  p.box = page_size % 32 == 0 ? 32 : 16;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.status = device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // query rows of a request and key head, which choose the kernel: from max_new, else the mean over the batch
  CUtensorMap tmK, tmV;
  int mrc = cache_map(&tmK, k_cache, kc_strides, D, p);
  if (!mrc) mrc = cache_map(&tmV, v_cache, vc_strides, D, p);
  if (mrc) return mrc;
  const int64_t rows = (max_new > 0 ? max_new : (T + B - 1) / B) * p.G;
  if (dtype == KCG_BF16)
    return D == 128 ? launch_cached<__nv_bfloat16, 128>(p, rows, tmK, tmV, workspace, s) : launch_cached<__nv_bfloat16, 64>(p, rows, tmK, tmV, workspace, s);
  return D == 128 ? launch_cached<__half, 128>(p, rows, tmK, tmV, workspace, s) : launch_cached<__half, 64>(p, rows, tmK, tmV, workspace, s);
}

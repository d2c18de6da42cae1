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
//   - The G heads and n_i queries of a key / value head share its keys as the rows of one 16-row tile, so a byte
//     is loaded and converted once.  Products run on mma.sync m16n8k16: at 16 rows a 128-row tcgen05 tile would be
//     seven eighths padding, and tensor time is not what bounds this kernel.
//   - Work is cut in units of 128 keys of one (request, head, 16 rows); the units of the whole batch, numbered in
//     that order, are dealt to a fixed grid in equal contiguous ranges, whatever the lengths: every block finds its
//     range by a prefix sum over the requests.  A block leaves a partial result (running maximum, sum, output) for
//     at most its first and its last item; cached_join_kernel merges those in a fixed order.
//   - A warp owns 32 keys of a unit and a ring of its own in shared memory, filled by cp.async two tiles ahead,
//     across item borders; no block barrier stands in the loop.  Masked rows are not loaded but zero-filled.
//   - Codes become f16 in registers (exact: e4m3 is a subset of f16), bf16 queries too, each row scaled by a power
//     of two.  K's scale multiplies the scores, V's scale the product of its keys: no operand is rounded again but
//     P, to f16.
#include "common.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace kcg {

int* device_status_word();

namespace {
using sm100::smem_u32;

constexpr int ROWS = 16;            // query rows of an item
constexpr int WARPS = 4;
constexpr int WKEYS = 32;           // keys of a warp's tile
constexpr int UNIT = WARPS * WKEYS; // keys of a unit
constexpr int STAGES = 3;
constexpr float kLazy = 8.0f;       // rescale only when the maximum grew by more than 2^8 (p <= 2^8 fits f16)

struct CachedParams {
  const void* Q;
  int64_t q_st, q_sh;
  void* O;
  int64_t o_st, o_sh;
  const uint8_t* kc;
  int64_t kc_p, kc_h, kc_t;
  const uint8_t* vc;
  int64_t vc_p, vc_h, vc_t;
  const float* ks;
  const float* vs;
  const int32_t* table;
  int64_t table_stride, width;
  const int32_t* lengths;
  const int32_t* cu;                // NULL: `uniform` queries each
  int64_t T, uniform, num_pages;
  int B, Hkv, G, page, causal;
  float scale_log2;
  float* part_o;                    // [grid][2][D/8 * 4][32 lanes]
  float* part_ml;                   // [grid][2][ROWS][2]
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
__device__ __forceinline__ int row_blocks(const CachedParams& p, int n) {
  return static_cast<int>((static_cast<int64_t>(n) * p.G + ROWS - 1) / ROWS);
}
__device__ __forceinline__ int64_t request_units(const CachedParams& p, const Request& r) {
  return static_cast<int64_t>(p.Hkv) * row_blocks(p, r.n) * unit_tiles(r.len);
}

// A place in the batch's sequence of units.
struct Cursor {
  Request r;
  int i, h, rb, tile, tiles, nrb;
  __device__ __forceinline__ void enter(const CachedParams& p, int req, int64_t offset) {
    i = req;
    r = request_of(p, i);
    tiles = unit_tiles(r.len);
    nrb = row_blocks(p, r.n);
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
        nrb = row_blocks(p, r.n);
      }
    }
    return true;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  const int bytes = take ? 16 : 0;   // 0: sixteen zero bytes, the source is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Byte offset of 16-byte chunk c of row r inside a tile of D-byte rows: chunks are permuted inside 128-byte lines so
// that both readings are free of bank conflicts: K by (row = lane / 4, chunk = lane % 4 (+ 4)), V by
// (row = 2 (lane % 4) + const, chunk = lane / 4).
template <int D> __device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  if constexpr (D == 128) {
    return r * 128 + ((c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2))) << 4);
  } else {
    const int line = r >> 1;
    return line * 128 + (((((r & 1) << 2) | c) ^ ((line & 3) << 1)) << 4);
  }
}

template <int D> struct SplitSmem {
  static constexpr int TILE = WKEYS * D;              // bytes of a K or V tile of one warp
  static constexpr int NREG = D / 2;                  // output registers of a lane
  uint8_t ring[WARPS][STAGES][2][TILE];
  float fold[2][NREG][32];                            // a warp's output on its way into another's
  float fold_ml[2][ROWS][2];
  float side[WARPS][STAGES][8];                       // per half tile: k scale, v scale, keys
  int64_t scan[WARPS];
  int64_t total;
  int64_t start_off;
  int start_i;
};

// Query fragments of an item: lane (g, t) holds rows g and g + 8, for every 16-wide step of the products four
// dims of each (the dims of step s are those lane t's K words of step s hold).  Scaled to f16's range by a power of
// two per row; `f` receives its inverse.
template <typename T, int D>
__device__ __forceinline__ void load_queries(const CachedParams& p, const Cursor& c, int lane, uint32_t (&qa)[D / 16][4], float (&f)[2]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int R = c.rb * ROWS + g + 8 * half;
    uint4 v[D / 32];
    const bool live = R < c.r.n * p.G;
    const int j = live ? R / p.G : 0;
    const T* q = static_cast<const T*>(p.Q) + (c.r.t0 + j) * p.q_st + (c.h * p.G + (live ? R - j * p.G : 0)) * p.q_sh;
#pragma unroll
    for (int k = 0; k < D / 64; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        v[2 * k + e] = live ? __ldg(reinterpret_cast<const uint4*>(q + 64 * k + 16 * t) + e) : make_uint4(0, 0, 0, 0);
    f[half] = 1.f;
    if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
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
      f[half] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = pack_f16(__uint_as_float(w[x] << 16) * up, __uint_as_float(w[x] & 0xffff0000u) * up);
      }
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {      // step s: word s % 4 of chunk s / 4, i.e. dims 64 (s / 4) + 16 t + 4 (s % 4) ..
      const uint4 x = v[2 * (s / 4) + ((s % 4) >> 1)];
      qa[s][half] = (s & 1) ? x.z : x.x;
      qa[s][2 + half] = (s & 1) ? x.w : x.y;
    }
  }
}

// Output tiles [j0, j0 + N) of an item, divided by the row sums.  Lane (g, t) holds of tile j rows g (registers 0, 1)
// and g + 8 (2, 3), dims 2 t (D / 8) + j and (2 t + 1) (D / 8) + j.
template <typename T, int D, int N>
__device__ __forceinline__ void store_rows(const CachedParams& p, int t0, int n, int h, int rb, int lane, const float (&o)[N][4],
                                           const float (&l)[2], int j0) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int R = rb * ROWS + g + 8 * half;
    if (R >= n * p.G) continue;
    const int j = R / p.G;
    T* dst = static_cast<T*>(p.O) + (t0 + j) * p.o_st + (h * p.G + (R - j * p.G)) * p.o_sh + 2 * t * (D / 8) + j0;
    const float inv = l[half] == 0.f ? 0.f : 1.0f / l[half];    // a row that sees no key is zero
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      if constexpr (N % 8 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 8) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v[2] = {o[k + 2 * e][2 * half + side] * inv, o[k + 2 * e + 1][2 * half + side] * inv};
            w[e] = Words<T>::pack(v);
          }
          *reinterpret_cast<uint4*>(dst + side * (D / 8) + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) dst[side * (D / 8) + k] = Conv<T>::from_f(o[k][2 * half + side] * inv);
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32, 2) cached_split_kernel(const CachedParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  SplitSmem<D>& sm = *reinterpret_cast<SplitSmem<D>*>(smem_raw);
  constexpr int NT = D / 8;                 // output tiles of 8 dims
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- this block's range of units ----
  const int per = (p.B + WARPS * 32 - 1) / (WARPS * 32);
  const int i_lo = min(tid * per, p.B), i_hi = min(i_lo + per, p.B);
  int64_t mine = 0;
  for (int i = i_lo; i < i_hi; ++i) mine += request_units(p, request_of(p, i));
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
      const int64_t n = request_units(p, request_of(p, i));
      if (off < n) break;
      off -= n;
    }
    sm.start_i = i;
    sm.start_off = off;
  }
  __syncthreads();

  Cursor cur;
  cur.enter(p, sm.start_i, sm.start_off);
  const int units = static_cast<int>(u1 - u0);

  // ---- loading: a cursor of its own, running ahead ----
  Cursor ld = cur;
  int ld_unit = 0;
  int pid = -1, pid_tile = -1 << 20;        // this lane's page (tile pid_tile + lane / 2, half lane & 1), and its scales
  float pid_ks = 0.f, pid_vs = 0.f;
  auto load_next = [&](int stage) {
    if (ld_unit < units) {
      if (ld.tile < pid_tile || ld.tile >= pid_tile + 16) {
        pid_tile = ld.tile;
        const int key = (ld.tile + (lane >> 1)) * UNIT + warp * WKEYS + (lane & 1) * 16;
        pid = -1;
        if (key < ld.r.len) {
          pid = p.table[ld.i * p.table_stride + key / p.page];
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
      const int key0 = ld.tile * UNIT + warp * WKEYS;
      if ((lane >> 1) == at) {
        float* s = sm.side[warp][stage] + (lane & 1);
        s[0] = pid_ks;
        s[2] = pid_vs;
        reinterpret_cast<int*>(s)[4] = pid >= 0 ? min(16, ld.r.len - (key0 + (lane & 1) * 16)) : 0;
      }
      const uint32_t kdst = smem_u32(sm.ring[warp][stage][0]), vdst = smem_u32(sm.ring[warp][stage][1]);
      constexpr int CPR = D / 16;           // chunks of a row
      constexpr int RPI = 32 / CPR;         // rows of one warp instruction
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int64_t pg = __shfl_sync(0xffffffffu, pid, 2 * at + half);
        const int key = key0 + half * 16;
        const int in = key % p.page;
        const uint8_t* ksrc = p.kc + (pg < 0 ? 0 : pg) * p.kc_p + ld.h * p.kc_h + (lane % CPR) * 16;
        const uint8_t* vsrc = p.vc + (pg < 0 ? 0 : pg) * p.vc_p + ld.h * p.vc_h + (lane % CPR) * 16;
        const int have = pg < 0 ? 0 : ld.r.len - key;
#pragma unroll
        for (int q = 0; q < 16 / RPI; ++q) {
          const int r = q * RPI + lane / CPR;
          const bool take = r < have;
          const int64_t row = take ? in + r : 0;
          const uint32_t at_s = tile_offset<D>(half * 16 + r, lane % CPR);
          cp_async16(kdst + at_s, ksrc + row * p.kc_t, take);
          cp_async16(vdst + at_s, vsrc + row * p.vc_t, take);
        }
      }
      if (++ld_unit < units) {
        if (ld.next(p)) pid_tile = -1 << 20;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_next(s);

  uint32_t qa[D / 16][4];
  float qf[2];
  float o[NT][4], m[2], l[2];
  bool fresh = true;
  int stage = 0;
  bool first_item = true;
  int item_tile0 = cur.tile;                // of the part of the item this block has
  for (int u = 0; u < units; ++u) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    load_next(stage == 0 ? STAGES - 1 : stage - 1);
    if (fresh) {
      load_queries<T, D>(p, cur, lane, qa, qf);
#pragma unroll
      for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      fresh = false;
      item_tile0 = cur.tile;
    }
    const uint32_t kt = smem_u32(sm.ring[warp][stage][0]), vt = smem_u32(sm.ring[warp][stage][1]);
    const float* side = sm.side[warp][stage];
    const int key0 = cur.tile * UNIT + warp * WKEYS;
    const int have0 = reinterpret_cast<const int*>(side)[4], have1 = reinterpret_cast<const int*>(side)[5];
    // ---- scores ----
    float s[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t w[4];
        lds128(kt + tile_offset<D>(8 * j + g, t + 4 * c), w);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t b0, b1;
          e4m3x4_to_f16(w[x], b0, b1);
          mma16816(s[j], qa[4 * c + x], b0, b1);
        }
      }
    }
    const float c0 = p.scale_log2 * qf[0], c1 = p.scale_log2 * qf[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float ks = side[j >> 1];
      const float f0 = c0 * ks, f1 = c1 * ks;
      s[j][0] *= f0;
      s[j][1] *= f0;
      s[j][2] *= f1;
      s[j][3] *= f1;
    }
    // ---- mask: keys this row must not see, keys that are not there ----
    const int R0 = cur.rb * ROWS;
    const int past = cur.r.len - cur.r.n + 1;
    if (have0 < 16 || have1 < 16 || (p.causal && key0 + WKEYS > past + R0 / p.G)) {
      int lim[2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
        lim[half] = p.causal ? past + (R0 + g + 8 * half) / p.G : cur.r.len;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = 8 * j + 2 * t + (e & 1);
          if ((k & 15) >= (j < 2 ? have0 : have1) || key0 + k >= lim[e >> 1]) s[j][e] = -INFINITY;
        }
    }
    // ---- running maximum ----
    float grow[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x = fmaxf(fmaxf(s[0][2 * half], s[0][2 * half + 1]), fmaxf(s[1][2 * half], s[1][2 * half + 1]));
      x = fmaxf(x, fmaxf(fmaxf(s[2][2 * half], s[2][2 * half + 1]), fmaxf(s[3][2 * half], s[3][2 * half + 1])));
      x = quad_max(x);
      grow[half] = 1.f;
      if (x > m[half] + kLazy || (m[half] == -INFINITY && x > -INFINITY)) {
        grow[half] = exp2f_approx(m[half] - x);      // 0 for the first keys
        m[half] = x;
      }
    }
    if (__any_sync(0xffffffffu, grow[0] != 1.f || grow[1] != 1.f)) {
      l[0] *= grow[0];
      l[1] *= grow[1];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        o[j][0] *= grow[0];
        o[j][1] *= grow[0];
        o[j][2] *= grow[1];
        o[j][3] *= grow[1];
      }
    }
    const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
    uint32_t pa[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p0 = exp2f_approx(s[j][0] - b0), p1 = exp2f_approx(s[j][1] - b0);
      const float p2 = exp2f_approx(s[j][2] - b1), p3 = exp2f_approx(s[j][3] - b1);
      l[0] += p0 + p1;
      l[1] += p2 + p3;
      pa[j >> 1][(j & 1) * 2] = pack_f16(p0, p1);
      pa[j >> 1][(j & 1) * 2 + 1] = pack_f16(p2, p3);
    }
    // ---- output: the product of each half with its page's scale ----
    const float vs0 = side[2], vs1 = side[3];
    const bool same = vs0 == vs1;
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
    auto product = [&](int half, int c, float (&acc)[4][4]) {   // += P_half V_half for output tiles 4 c .. 4 c + 3
      uint32_t b[4][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t x = v[half][2 * k][c], y = v[half][2 * k + 1][c];
        e4m3x4_to_f16(__byte_perm(x, y, 0x5140), b[0][k], b[1][k]);
        e4m3x4_to_f16(__byte_perm(x, y, 0x7362), b[2][k], b[3][k]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mma16816(acc[e], pa[half], b[e][0], b[e][1]);
    };
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      float acc[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
      product(0, c, acc);
      if (!same) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            o[4 * c + e][x] = fmaf(acc[e][x], vs0, o[4 * c + e][x]);
            acc[e][x] = 0.f;
          }
      }
      product(1, c, acc);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[4 * c + e][x] = fmaf(acc[e][x], vs1, o[4 * c + e][x]);
    }

    if (++stage == STAGES) stage = 0;
    const bool last = u + 1 == units;
    if (cur.tile + 1 < cur.tiles && !last) {
      ++cur.tile;
      continue;
    }
    // ---- end of the item, or of this block's part of it: the four warps' results into warp 0 ----
    l[0] = quad_sum(l[0]);
    l[1] = quad_sum(l[1]);
    auto give = [&](int to) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) sm.fold[to][4 * j + x][lane] = o[j][x];
      if (t == 0) {
        sm.fold_ml[to][g][0] = m[0];
        sm.fold_ml[to][g][1] = l[0];
        sm.fold_ml[to][g + 8][0] = m[1];
        sm.fold_ml[to][g + 8][1] = l[1];
      }
    };
    auto take = [&](int from) {
      float mine_w[2], other_w[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float m2 = sm.fold_ml[from][g + 8 * half][0], l2 = sm.fold_ml[from][g + 8 * half][1];
        const float top = fmaxf(m[half], m2), base = top == -INFINITY ? 0.f : top;
        mine_w[half] = exp2f_approx(m[half] - base);
        other_w[half] = exp2f_approx(m2 - base);
        l[half] = l[half] * mine_w[half] + l2 * other_w[half];
        m[half] = top;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          o[j][x] = o[j][x] * mine_w[x >> 1] + sm.fold[from][4 * j + x][lane] * other_w[x >> 1];
    };
    __syncthreads();                        // the fold buffers are free
    if (warp >= 2) give(warp - 2);
    __syncthreads();
    if (warp < 2) take(warp);
    __syncthreads();
    if (warp == 1) give(0);
    __syncthreads();
    if (warp == 0) {
      take(0);
      const bool whole = item_tile0 == 0 && cur.tile + 1 == cur.tiles;
      if (whole) {
        store_rows<T, D, NT>(p, cur.r.t0, cur.r.n, cur.h, cur.rb, lane, o, l, 0);
      } else {
        const int slot = first_item ? 0 : 1;
        float* po = p.part_o + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * (D / 2 * 32) + lane;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) po[(4 * j + x) * 32] = o[j][x];
        if (t == 0) {
          float* pm = p.part_ml + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * (ROWS * 2);
          pm[2 * g] = m[0];
          pm[2 * g + 1] = l[0];
          pm[2 * (g + 8)] = m[1];
          pm[2 * (g + 8) + 1] = l[1];
        }
        if (item_tile0 == 0 && lane == 0) {
          // the item begins in this block: it lists the parts.  Its units end before u0 + u + tiles - tile; block c
          // holds unit x when c = floor(((x + 1) grid - 1) / total).
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
  cp_async_wait<0>();
}

// Merges the parts of items that several blocks worked on; block c takes the item that begins in block c of the
// split kernel and ends behind it.  Warps take shares of the output registers; parts are added in order.
constexpr int JOIN_WARPS = 8;
template <typename T, int D>
__global__ void __launch_bounds__(JOIN_WARPS * 32) cached_join_kernel(const CachedParams p) {
  constexpr int NT = D / 8, MINE = NT / JOIN_WARPS;   // output tiles of a warp
  grid_launch_dependents();
  grid_dependency_wait();
  const int* meta = p.meta + blockIdx.x * 8;
  if (meta[0] < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2;
  const int last = meta[1];
  const float* part_o = p.part_o + lane + static_cast<int64_t>(warp) * MINE * 4 * 32;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float acc[MINE][4];
#pragma unroll
  for (int j = 0; j < MINE; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  // first the maximum over the parts, then one weighted sum
  for (int c = blockIdx.x; c <= last; ++c) {
    const float* pm = p.part_ml + (static_cast<int64_t>(c) * 2 + (c == static_cast<int>(blockIdx.x) ? meta[2] : 0)) * (ROWS * 2);
    m[0] = fmaxf(m[0], pm[2 * g]);
    m[1] = fmaxf(m[1], pm[2 * (g + 8)]);
  }
  const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll 4
  for (int c = blockIdx.x; c <= last; ++c) {
    const int64_t part = static_cast<int64_t>(c) * 2 + (c == static_cast<int>(blockIdx.x) ? meta[2] : 0);
    const float* pm = p.part_ml + part * (ROWS * 2);
    const float w0 = exp2f_approx(pm[2 * g] - b0), w1 = exp2f_approx(pm[2 * (g + 8)] - b1);
    l[0] += pm[2 * g + 1] * w0;
    l[1] += pm[2 * (g + 8) + 1] * w1;
    const float* po = part_o + part * (D / 2 * 32);
#pragma unroll
    for (int j = 0; j < MINE; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[j][x] = fmaf(po[(4 * j + x) * 32], x < 2 ? w0 : w1, acc[j][x]);
  }
  store_rows<T, D, MINE>(p, meta[3], meta[4], meta[5], meta[6], lane, acc, l, warp * MINE);
}

int split_grid() { return sm_count() * 2; }

template <int D> size_t workspace_of(int grid) {
  return static_cast<size_t>(grid) * (2 * (D / 2 * 32 * 4) + 2 * (ROWS * 2 * 4) + 32);
}

template <typename T, int D>
int launch_split(CachedParams& p, void* workspace, cudaStream_t stream) {
  const int grid = split_grid();
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<size_t>(grid) * 2 * (D / 2 * 32);
  p.meta = reinterpret_cast<int*>(p.part_ml + static_cast<size_t>(grid) * 2 * (ROWS * 2));
  constexpr int SMEM = sizeof(SplitSmem<D>);
  auto kern = cached_split_kernel<T, D>;
  KCG_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  launch_overlapped(kern, dim3(grid), dim3(WARPS * 32), SMEM, stream, p);
  const int rc = check_launch("cached_split_kernel");
  if (rc) return rc;
  launch_overlapped(cached_join_kernel<T, D>, dim3(grid), dim3(JOIN_WARPS * 32), 0, stream, p);
  return check_launch("cached_join_kernel");
}

}  // namespace
}  // namespace kcg

extern "C" int kcg_fmha_cached_workspace(int64_t D, size_t* bytes) {
  using namespace kcg;
  clear_error();
  if (!bytes) return fail(KCG_ERR_INVALID_ARG, "fmha_cached_workspace: null pointer");
  if (D != 64 && D != 128) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: head dimension %lld has no kernel (64, 128)", static_cast<long long>(D));
  *bytes = D == 128 ? workspace_of<128>(split_grid()) : workspace_of<64>(split_grid());
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
  if (!ok) return fail(KCG_ERR_ALIGNMENT, "fmha_cached: rows of Q, O, the caches and the workspace must start on 16-byte boundaries");
  size_t need = 0;
  const int rc = kcg_fmha_cached_workspace(D, &need);
  if (rc) return rc;
  if (!workspace || workspace_bytes < need)
    return fail(KCG_ERR_INVALID_ARG, "fmha_cached: the workspace has %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
  CachedParams p{};
  p.Q = Q; p.q_st = q_strides[0]; p.q_sh = q_strides[1];
  p.O = O; p.o_st = o_strides[0]; p.o_sh = o_strides[1];
  p.kc = static_cast<const uint8_t*>(k_cache); p.kc_p = kc_strides[0]; p.kc_h = kc_strides[1]; p.kc_t = kc_strides[2];
  p.vc = static_cast<const uint8_t*>(v_cache); p.vc_p = vc_strides[0]; p.vc_h = vc_strides[1]; p.vc_t = vc_strides[2];
  p.ks = k_scale; p.vs = v_scale;
  p.table = block_table; p.table_stride = table_stride; p.width = table_width;
  p.lengths = lengths; p.cu = cu_new;
  p.T = T; p.uniform = cu_new ? 0 : T / B; p.num_pages = num_pages;
  p.B = static_cast<int>(B); p.Hkv = static_cast<int>(Hkv); p.G = static_cast<int>(Hq / Hkv);
  p.page = static_cast<int>(page_size); p.causal = causal != 0;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.status = device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KCG_BF16)
    return D == 128 ? launch_split<__nv_bfloat16, 128>(p, workspace, s) : launch_split<__nv_bfloat16, 64>(p, workspace, s);
  return D == 128 ? launch_split<__half, 128>(p, workspace, s) : launch_split<__half, 64>(p, workspace, s);
}

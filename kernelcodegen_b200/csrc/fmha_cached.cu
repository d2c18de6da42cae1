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
//   - Four warps form a team; a team takes two heads of a request side by side (their rows of a token may be neighbours in
//     memory), or one where the heads do not pair up; two or all four of its warps share a head's keys.  Work is cut in
//     units of 32 keys a warp; the units of the whole batch, numbered by request, head group, rows and keys, are dealt to a
//     fixed number of teams in equal contiguous ranges, whatever the lengths: every team finds its range by a prefix sum over
//     the requests.  A team leaves a partial result (running maximum, sum, output) for at most its first and its last item,
//     which cached_join_kernel merges in a fixed order.
//   - A warp of its own feeds each team: it walks the range, looks pages up ahead of use, and fills the warps' rings by
//     TMA (boxes of 16 or 32 rows of a page), across item borders.  The team's warps know nothing of requests and pages:
//     a ring entry says what it holds.  They meet only where keys are shared, at the end of an item.
//   - Codes become f16 in registers (exact: e4m3 is a subset of f16), bf16 queries too, each row scaled by a power
//     of two.  K's scale multiplies the scores, V's scale the product of its keys: no operand is rounded again but
//     P, to f16.
// Measured (32 query heads of 128): 64 ragged requests of up to 4096 keys, 8 key heads: 63 us, 4.4 TB/s; 2 x 131072 keys, 4
// key heads: 58 us, 4.6 TB/s; 8 such requests 178 us, 92 % of the copy rate.  Bound by reading the cache, plus about 10 us per
// call whatever the size: the prefix sum over the requests, the first fill of the rings, the join.
#include "common.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <type_traits>

namespace kcg {

int* device_status_word();
int encode_tmap(CUtensorMap* out, int dtype, const void* base, int rank, const uint64_t* dims,
                const uint64_t* strides_bytes, const uint32_t* box, int swizzle_bytes);

namespace {
using namespace sm100;
#include "fmha_blocks.cuh"

// The kernels walk the requests one after another, half a microsecond each, while other warps wait for the next that has work, and
// those waits are limited to two seconds.
constexpr int kMaxRequests = 1 << 20;
constexpr int WARPS = 4;            // of a team
constexpr int WKEYS = 32;           // keys of a warp's tile
constexpr float kLazy = 14.0f;      // rescale only when the maximum grew by more than 2^14 (p <= 2^14 fits f16)

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
  int wk_log2;                      // 2^wk_log2 warps, 2 or 4, share a head's keys; of 2 pairs each has a head of its own
  int whole_items;                  // the many-row kernel: items are dealt whole, not in ranges of key blocks
  int o_by_32;                      // rows of O start on 32-byte boundaries
  int box;                          // rows of a TMA box: 32 where a page is a multiple of that, else 16
  float scale_log2;
  float* part_o;                    // [grid][2][WARPS][NQ D / 4][32 lanes]
  float* part_ml;                   // [grid][2][WARPS][8 NQ][2]
  int* meta;                        // [grid][8]
  int* status;
};

// What a request contributes: its queries [t0, t0 + n), keys [0, len).  Loading and checking are apart, so that a
// load can be under way while its value is not needed yet.
struct Request { int t0, n, len; };
struct RawRequest { int a, b, len; };
__device__ __forceinline__ RawRequest load_request(const CachedParams& p, int i) {
  RawRequest w{0, 0, p.lengths[i]};
  if (p.cu) {
    w.a = p.cu[i];
    w.b = p.cu[i + 1];
  }
  return w;
}
__device__ __forceinline__ Request check_request(const CachedParams& p, int i, const RawRequest& w) {
  Request r;
  int64_t a = w.a, b = w.b;
  if (p.cu) {
    const int64_t a1 = min(max(a, static_cast<int64_t>(0)), p.T), b1 = min(max(b, a1), p.T);
    if ((a1 != a || b1 != b) && p.status) *p.status = KCG_ERR_INVALID_ARG;
    a = a1;
    b = b1;
  } else {
    a = i * p.uniform;
    b = a + p.uniform;
  }
  const int64_t len = w.len, most = p.width * p.page;
  const int64_t l1 = min(max(len, static_cast<int64_t>(0)), most);
  if (l1 != len && p.status) *p.status = KCG_ERR_INVALID_ARG;
  r.t0 = static_cast<int>(a);
  r.n = static_cast<int>(b - a);
  r.len = static_cast<int>(l1);
  return r;
}
__device__ __forceinline__ Request request_of(const CachedParams& p, int i) { return check_request(p, i, load_request(p, i)); }
__device__ __forceinline__ int unit_keys(const CachedParams& p) { return WKEYS << p.wk_log2; }
__device__ __forceinline__ int unit_tiles(const CachedParams& p, int len) {
  return len > 0 ? (len + unit_keys(p) - 1) >> (5 + p.wk_log2) : 1;
}
__device__ __forceinline__ int head_groups(const CachedParams& p) { return p.Hkv >> (2 - p.wk_log2); }
template <int ROWS> __device__ __forceinline__ int row_blocks(const CachedParams& p, int n) { return (n * p.G + ROWS - 1) / ROWS; }
template <int ROWS> __device__ __forceinline__ int64_t request_units(const CachedParams& p, const Request& r) {
  return static_cast<int64_t>(head_groups(p)) * row_blocks<ROWS>(p, r.n) * unit_tiles(p, r.len);
}

// A place in the batch's sequence of units; h counts groups of heads.
template <int ROWS> struct Cursor {
  Request r;
  int i, h, rb, tile, tiles, nrb;
  __device__ __forceinline__ void set(const CachedParams& p, const Request& request) {
    r = request;
    tiles = unit_tiles(p, r.len);
    nrb = row_blocks<ROWS>(p, r.n);
  }
  __device__ __forceinline__ void enter(const CachedParams& p, int req, int64_t offset) {
    i = req;
    set(p, request_of(p, i));
    const int64_t item = offset / tiles;
    tile = static_cast<int>(offset - item * tiles);
    h = static_cast<int>(item / nrb);
    rb = static_cast<int>(item - static_cast<int64_t>(h) * nrb);
  }
  // to the next unit (only called while there is one); `raw`: the request behind this one, where it is known already.
  // True when another item begins.
  __device__ __forceinline__ bool next(const CachedParams& p, bool known = false, RawRequest raw = {0, 0, 0}) {
    if (++tile < tiles) return false;
    tile = 0;
    if (++rb == nrb) {
      rb = 0;
      if (++h == head_groups(p)) {
        h = 0;
        ++i;
        if (!known) raw = load_request(p, i);
        Request n = check_request(p, i, raw);
        while (n.n == 0) n = request_of(p, ++i);
        set(p, n);
      }
    }
    return true;
  }
};

// 4 or 16 bytes, or as many zero bytes without a look at the source
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool take) {
  const int bytes = take ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  const int bytes = take ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// an arrival on `bar` (counted in its initial count) once this thread's cp.async so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t (&r)[2]) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
}

__device__ __forceinline__ void sts128(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
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

// Teams of a block (one block per SM), ring stages, and the registers that setmaxnreg moves from the feeding warps to
// the teams: what 8 NQ rows of output per lane leave room for.
template <int NQ> struct SplitShape;
template <> struct SplitShape<1> { static constexpr int TEAMS = 3, STAGES = 2, REGS_TEAM = 152, REGS_FEED = 56, REGS_LAUNCH = 128; };
template <> struct SplitShape<2> { static constexpr int TEAMS = 2, STAGES = 3, REGS_TEAM = 216, REGS_FEED = 72, REGS_LAUNCH = 168; };
template <int NQ> constexpr int split_threads() { return (SplitShape<NQ>::TEAMS + 1) * 128; }
template <int NQ> constexpr bool split_regs_fit() {
  using S = SplitShape<NQ>;
  return S::TEAMS * S::REGS_TEAM + S::REGS_FEED <= (S::TEAMS + 1) * S::REGS_LAUNCH && split_threads<NQ>() * S::REGS_LAUNCH <= 65536;
}
static_assert(split_regs_fit<1>() && split_regs_fit<2>(), "register split exceeds the block's allocation");

// What a ring entry holds, beside its K and V tiles.
struct Entry {
  int have[2];      // keys of each half tile that are there
  int flags;
  int key0;         // first key
  int t0, n, len;   // the request: first row of Q, rows, keys
  int head;
  int rb;           // rows [8 NQ rb, ..) of the n G
  int last_team;    // ENTRY_BEGIN without ENTRY_END: the team that has the item's last unit
  int pad[2];
  float ks[2], vs[2];
};
static_assert(sizeof(Entry) == 64, "");
constexpr int ENTRY_FIRST = 1;    // first unit of the team's part of an item
constexpr int ENTRY_LAST = 2;     // last unit of it
constexpr int ENTRY_BEGIN = 4;    // the part holds the item's first unit
constexpr int ENTRY_END = 8;      // the part holds the item's last unit
constexpr int ENTRY_SLOT1 = 16;   // not the team's first item

template <int D, int NQ> struct TeamSmem {
  static constexpr int STAGES = SplitShape<NQ>::STAGES;
  static constexpr int TILE = WKEYS * D;              // bytes of a K or V tile of one warp
  static constexpr int NREG = NQ * D / 4;             // output registers of a lane
  static constexpr int FOLDS = NQ == 1 ? 2 : 1;       // (two do not fit beside a ring of three stages)
  uint8_t ring[WARPS][STAGES][2][TILE];
  float fold[FOLDS][NREG][32];                        // a warp's output on its way into another's
  float fold_ml[FOLDS][8 * NQ][2];
  Entry entry[WARPS][STAGES];
  uint64_t full[WARPS][STAGES], empty[WARPS][STAGES];
  uint64_t met;                                       // the team's warps meet here, with bounded waits
  int64_t start_off;
  int start_i;
  uint8_t align[1024 - (FOLDS * (NREG * 128 + 64 * NQ) + 80 * WARPS * STAGES + 24) % 1024];
};
template <int D, int NQ> struct SplitSmem {
  TeamSmem<D, NQ> team[SplitShape<NQ>::TEAMS];
  int64_t scan[16];
  int abort;
};

// Query fragments of an item: lane (g, t) holds row 8 q + g of tile q, for every 16-wide step s of the product the four
// dims that lane t's K words of that step hold, (D / 4) t + 4 s and on.  bf16 rows are scaled to f16's range by a power of two; f[q] receives
// its inverse for rows 8 q + 2 t and 8 q + 2 t + 1, the columns of S^T this lane will hold.
template <typename T, int D, int NQ>
__device__ __forceinline__ void load_queries(const CachedParams& p, int t0, int n, int head, int rb, int lane,
                                             uint32_t (&qb)[NQ][D / 16][2], float (&f)[NQ][2]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int R = rb * (8 * NQ) + 8 * q + g;
    uint4 v[D / 32];
    const bool live = R < n * p.G;
    const int j = live ? R / p.G : 0;
    const T* src = static_cast<const T*>(p.Q) + (t0 + j) * p.q_st + (head * p.G + (live ? R - j * p.G : 0)) * p.q_sh;
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

// The feeding warp of a team: fills the rings for the units [u0, u1).
template <typename T, int D, int NQ>
__device__ __forceinline__ void feed_team(const CachedParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV, TeamSmem<D, NQ>& sm,
                                          int* abort, int64_t u0, int units, int64_t total, int64_t teams, int lane) {
  constexpr int ROWS = 8 * NQ, STAGES = TeamSmem<D, NQ>::STAGES;
  const int sub = lane & ((1 << p.wk_log2) - 1), head_in_group = (lane & 3) >> p.wk_log2;   // of warp `lane`, for lanes 0 .. 3
  const int group_heads = WARPS >> p.wk_log2;
  Cursor<ROWS> c;
  c.enter(p, sm.start_i, sm.start_off);
  // Pages are looked up 32 groups of 16 keys at a time, one per lane: keys win_key + 16 lane of request win_i.  The window
  // that comes next is looked up in two steps (its request, then its pages) while the present one is worked on, so
  // that no load waits for another at an item's border.
  int win_i = -1, win_key = 0, pid = -1, pid_row = 0;
  int nx_i = -1, nx_key = 0, nx_step = 0, npid = -1, nrow = 0;
  RawRequest nx_raw{0, 0, 0};
  auto look_up = [&](int i, int len, int key0, int& page, int& row) {
    const int key = key0 + 16 * lane;
    page = -1;
    row = 0;
    if (key < len) {
      const int w = key / p.page;
      row = key - w * p.page;
      page = p.table[i * p.table_stride + w];
      if (page < 0 || page >= p.num_pages) page = -2;   // reported when the window is taken into use
    }
  };
  int part_tile0 = c.tile, slot = 0;
  bool first = true;
  int stage = 0;
  uint32_t parity = 1;                      // of the empty barriers: the first pass over the ring waits for nobody
  for (int u = 0; u < units; ++u) {
    const int key0 = c.tile * unit_keys(p);
    if (c.i != win_i || key0 < win_key || key0 + unit_keys(p) > win_key + 512) {
      if (nx_step == 2 && c.i == nx_i && key0 == nx_key) {
        pid = npid;
        pid_row = nrow;
      } else {
        look_up(c.i, c.r.len, key0, pid, pid_row);
      }
      win_i = c.i;
      win_key = key0;
      if (pid == -2 && p.status) *p.status = KCG_ERR_INVALID_ARG;
      nx_i = c.i;
      nx_key = win_key + 512;               // a multiple of the unit
      nx_step = 1;
      nx_raw.len = c.r.len;
      if (nx_key >= c.r.len) {
        nx_key = 0;
        if (c.h + 1 == head_groups(p) && c.rb + 1 == c.nrb) {
          if (++nx_i < p.B) nx_raw = load_request(p, nx_i);
          else nx_step = 0;
        }
      }
    } else if (nx_step == 1) {
      look_up(nx_i, nx_i == c.i ? c.r.len : check_request(p, nx_i, nx_raw).len, nx_key, npid, nrow);
      nx_step = 2;
    }
    // lane w < 4 fills warp w's entry
    const int key = key0 + sub * WKEYS, at = (key - win_key) >> 4;
    const int pg0 = __shfl_sync(0xffffffffu, pid, at & 31), pg1 = __shfl_sync(0xffffffffu, pid, (at + 1) & 31);
    const int in0 = __shfl_sync(0xffffffffu, pid_row, at & 31), in1 = __shfl_sync(0xffffffffu, pid_row, (at + 1) & 31);
    const int head = c.h * group_heads + head_in_group;
    const bool last_of_item = c.tile + 1 == c.tiles, last = last_of_item || u + 1 == units;
    bool ok = true;
    if (lane < WARPS) {
      ok = mbar_wait(&sm.empty[lane][stage], parity, abort);
      if (ok) {
        Entry& e = sm.entry[lane][stage];
        int4 d;
        d.x = pg0 >= 0 ? min(16, c.r.len - key) : 0;
        d.y = pg1 >= 0 ? min(16, c.r.len - key - 16) : 0;
        d.z = (first ? ENTRY_FIRST : 0) | (last ? ENTRY_LAST : 0) | (part_tile0 == 0 ? ENTRY_BEGIN : 0) | (last_of_item ? ENTRY_END : 0) | slot;
        d.w = key;
        *reinterpret_cast<int4*>(&e) = d;
        *reinterpret_cast<int4*>(&e.t0) = make_int4(c.r.t0, c.r.n, c.r.len, head);
        e.rb = c.rb;
        if (last) e.last_team = static_cast<int>(((u0 + u + (c.tiles - c.tile)) * teams - 1) / total);   // (k holds unit x when
        // k = floor(((x + 1) teams - 1) / total))
        // rows behind the last token are loaded with their page and left out by the reader; a half tile of no page is
        // not loaded at all (with boxes of 32 rows both halves are one page's, and the second may only lie behind the end)
        uint8_t* kdst = sm.ring[lane][stage][0];
        uint8_t* vdst = sm.ring[lane][stage][1];
        uint64_t* bar = &sm.full[lane][stage];
        const bool second = pg1 >= 0 && p.box == 16;
        mbar_expect_tx(bar, 2 * D * ((pg0 >= 0 ? p.box : 0) + (second ? 16 : 0)));
        if (pg0 >= 0) {
          tma_load_4d(kdst, tmK, bar, 0, in0, head, pg0);
          tma_load_4d(vdst, tmV, bar, 0, in0, head, pg0);
        }
        if (second) {
          tma_load_4d(kdst + 16 * D, tmK, bar, 0, in1, head, pg1);
          tma_load_4d(vdst + 16 * D, tmV, bar, 0, in1, head, pg1);
        }
      }
    }
    if (!__all_sync(0xffffffffu, ok)) {
      if (lane == 0 && !*static_cast<volatile int*>(abort)) {
        *static_cast<volatile int*>(abort) = 1;
        if (p.status) *p.status = KCG_ERR_TIMEOUT;
      }
      return;
    }
    // lane 4 w + k: scale k of warp w's entry (K's and V's of the two halves); its arrival is one of the entry's five
    {
      const int w = (lane >> 2) & 3, k = lane & 3;
      const int page0_of = __shfl_sync(0xffffffffu, pg0, w), page1_of = __shfl_sync(0xffffffffu, pg1, w);
      const int head_of = __shfl_sync(0xffffffffu, head, w);
      if (lane < 16) {
        const int page = k & 1 ? page1_of : page0_of;
        float* dst = (k & 2 ? sm.entry[w][stage].vs : sm.entry[w][stage].ks) + (k & 1);
        // (the scale of a half without keys is 0: it multiplies a product that is zero, and what stood there may be NaN)
        cp_async4(smem_u32(dst), (k & 2 ? p.vs : p.ks) + (page >= 0 ? static_cast<int64_t>(page) * p.Hkv + head_of : 0), page >= 0);
        cp_async_arrive(&sm.full[w][stage]);
      }
    }
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
    first = false;
    if (u + 1 < units && c.next(p, nx_step > 0 && nx_i == c.i + 1, nx_raw)) {
      first = true;
      part_tile0 = 0;
      slot = ENTRY_SLOT1;
      // the next item's queries on their way to L2
      for (int x = lane; x < group_heads * ROWS * (D / 64); x += 32) {
        const int R = c.rb * ROWS + x / (D / 64) % ROWS;
        if (R >= c.r.n * p.G) continue;
        const int j = R / p.G;
        const T* q = static_cast<const T*>(p.Q) + (c.r.t0 + j) * p.q_st +
                     ((c.h * group_heads + x / (D / 64 * ROWS)) * p.G + (R - j * p.G)) * p.q_sh + x % (D / 64) * 64;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
      }
    }
  }
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(split_threads<NQ>(), 1)
cached_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CachedParams p) {
  extern __shared__ uint8_t smem_raw[];
  using Shape = SplitShape<NQ>;
  SplitSmem<D, NQ>& all = *reinterpret_cast<SplitSmem<D, NQ>*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  constexpr int ROWS = 8 * NQ, STAGES = Shape::STAGES, NREG = TeamSmem<D, NQ>::NREG, THREADS = split_threads<NQ>();
  constexpr int MT = D / 16;                // output tiles of 16 dims
  const int tid = threadIdx.x, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  static_assert(sizeof(TeamSmem<D, NQ>) % 1024 == 0, "tiles start on swizzle boundaries");
  grid_launch_dependents();
  if (tid < Shape::TEAMS * WARPS) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&all.team[tid / WARPS].full[tid % WARPS][s], 5);
      mbar_init(&all.team[tid / WARPS].empty[tid % WARPS][s], 1);
    }
    if (tid % WARPS == 0) mbar_init(&all.team[tid / WARPS].met, WARPS);
    mbar_fence_init();
  }
  if (tid == 0) {
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    all.abort = 0;
  }
  grid_dependency_wait();

  // ---- the teams' ranges of units ----
  const int per = (p.B + THREADS - 1) / THREADS;
  const int i_lo = min(tid * per, p.B), i_hi = min(i_lo + per, p.B);
  int64_t mine = 0;
  for (int i = i_lo; i < i_hi; ++i) mine += request_units<ROWS>(p, request_of(p, i));
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) all.scan[tid >> 5] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < (tid >> 5)) upto += all.scan[w];
    total += all.scan[w];
  }
  const int64_t teams = min(static_cast<int64_t>(gridDim.x) * Shape::TEAMS, total);   // at work: none is without a unit
  auto range = [&](int64_t k) { return total * k / teams; };
  for (int s = 0; s < Shape::TEAMS; ++s) {
    const int64_t k = static_cast<int64_t>(s) * gridDim.x + blockIdx.x;   // (a few units are spread over all SMs)
    if (k >= teams) break;
    int64_t off = range(k) - (upto - mine);
    if (off < 0 || off >= mine) continue;   // one thread's requests hold the range's first unit
    int i = i_lo;
    for (;; ++i) {
      const int64_t n = request_units<ROWS>(p, request_of(p, i));
      if (off < n) break;
      off -= n;
    }
    all.team[s].start_i = i;
    all.team[s].start_off = off;
  }
  __syncthreads();

  const int group = tid >> 7;               // 0: the feeding warps
  const int warp = (tid >> 5) & 3;
  if (group == 0) {
    reg_dealloc<Shape::REGS_FEED>();
    const int64_t k = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
    if (warp < Shape::TEAMS && k < teams)
      feed_team<T, D, NQ>(p, &tmK, &tmV, all.team[warp], &all.abort, range(k), static_cast<int>(range(k + 1) - range(k)), total, teams, lane);
    return;
  }
  reg_alloc<Shape::REGS_TEAM>();
  const int team = group - 1;
  const int64_t k_team = static_cast<int64_t>(team) * gridDim.x + blockIdx.x;
  TeamSmem<D, NQ>& sm = all.team[team];
  int* meta = p.meta + k_team * 8;
  if (warp == 0 && lane == 0) meta[0] = -1;
  if (k_team >= teams) return;
  const int sub = warp & ((1 << p.wk_log2) - 1);      // this warp among those of its head
  const int units = static_cast<int>(range(k_team + 1) - range(k_team));

  uint32_t qb[NQ][D / 16][2];
  float cq[NQ][2];                          // what a score of this lane's columns is multiplied with, but for K's scale
  float o[NQ][MT][4], m[NQ][2], l[NQ][2];
  int R0 = 0, lim0 = 0;                     // the item's first row, and the first key that row must not see
  int stage = 0;
  uint32_t parity = 0, met_parity = 0;
  // A wait that runs out of time raises the block's abort flag, which ends every other wait and loop, and the status.
  auto give_up = [&]() {
    if (!*static_cast<volatile int*>(&all.abort)) {
      *static_cast<volatile int*>(&all.abort) = 1;
      if (p.status) *p.status = KCG_ERR_TIMEOUT;
    }
  };
  bool together = true;
  auto meet = [&]() {                       // the team's four warps
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.met);
    together = mbar_wait_warp(&sm.met, met_parity, &all.abort) && together;
    met_parity ^= 1;
  };
  for (int u = 0; u < units; ++u) {
    if (!mbar_wait_warp(&sm.full[warp][stage], parity, &all.abort)) {
      give_up();
      break;
    }
    const Entry& entry = sm.entry[warp][stage];
    const int4 head4 = *reinterpret_cast<const int4*>(&entry);
    const int have0 = head4.x, have1 = head4.y, flags = head4.z, key0 = head4.w;
    if (flags & ENTRY_FIRST) {
      R0 = entry.rb * ROWS;
      load_queries<T, D, NQ>(p, entry.t0, entry.n, entry.head, entry.rb, lane, qb, cq);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int j = 0; j < MT; ++j) o[q][j][0] = o[q][j][1] = o[q][j][2] = o[q][j][3] = 0.f;
        m[q][0] = m[q][1] = -INFINITY;
        l[q][0] = l[q][1] = 0.f;
        cq[q][0] *= p.scale_log2;
        cq[q][1] *= p.scale_log2;
      }
      lim0 = p.causal ? entry.len - entry.n + 1 + R0 / p.G : INT32_MAX;
    }
    if ((have0 | have1) > 0) {
    const uint32_t kt = smem_u32(sm.ring[warp][stage][0]), vt = smem_u32(sm.ring[warp][stage][1]);
    const float4 scales = *reinterpret_cast<const float4*>(entry.ks);
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
      const float ks = half ? scales.y : scales.x;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[q][half][x] *= cq[q][x & 1] * ks;
    }
    // ---- mask: keys a row must not see, keys that are not there ----
    const bool ragged = have0 < 16 || have1 < 16;
    if (ragged || key0 + WKEYS > lim0) {
      const int past = entry.len - entry.n + 1;
      const int len = entry.len;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int lim = p.causal ? past + (R0 + 8 * q + 2 * t + e) / p.G : len;
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
        outgrown = outgrown || top[q][e] - m[q][e] > kLazy;     // (m + kLazy may round up to a p that f16 does not hold)
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
    const float vs0 = scales.z, vs1 = scales.w;
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
    const bool last = flags & ENTRY_LAST;
    if (!last) {
      __syncwarp();                         // every lane has read the tile
      if (lane == 0) mbar_arrive(&sm.empty[warp][stage]);
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
      continue;
    }
    // ---- end of the item, or of this team's part of it: the results of a head's warps into the first of them ----
    const int4 item = *reinterpret_cast<const int4*>(&entry.t0);    // t0, n, len, head
    const int rb = entry.rb, last_team = entry.last_team;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.empty[warp][stage]);
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
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
    meet();                      // the fold buffers are free
    if constexpr (TeamSmem<D, NQ>::FOLDS == 2) {
      if (p.wk_log2 == 2) {               // 2, 3 into 0, 1
        if (warp >= 2) give(warp - 2);
        meet();
        if (warp < 2) take(warp);
        meet();
        if (warp == 1) give(0);
      } else if (warp & 1) {
        give(warp >> 1);
      }
      meet();
      if (sub == 0) take(warp >> 1);
    } else {                              // one at a time
      for (int w = WARPS - 1; w > 0; --w) {
        if ((w & ((1 << p.wk_log2) - 1)) == 0) continue;
        if (warp == w) give(0);
        meet();
        if (warp == (w >> p.wk_log2) << p.wk_log2) take(0);
        meet();
      }
    }
    if (!together) {
      give_up();
      break;
    }
    if (sub == 0) {
      if ((flags & ENTRY_BEGIN) && (flags & ENTRY_END)) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) store_rows<T, D, MT>(p, item.x, item.y, item.w, R0 + 8 * q, lane, o[q], l[q], 0);
      } else {
        const int slot = flags & ENTRY_SLOT1 ? 1 : 0;
        const int64_t part = (k_team * 2 + slot) * WARPS + (warp >> p.wk_log2);
        float* po = p.part_o + part * (NREG * 32) + t * 8 + g;    // (the lanes of a row side by side)
        float* pm = p.part_ml + part * (ROWS * 2);
        const int rows = item.y * p.G - R0;
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (8 * q + 2 * t + e < rows) {
#pragma unroll
              for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half) po[((q * MT + j) * 4 + 2 * half + e) * 32] = o[q][j][2 * half + e];
              if (g == 0) {
                pm[2 * (8 * q + 2 * t + e)] = m[q][e];
                pm[2 * (8 * q + 2 * t + e) + 1] = l[q][e];
              }
            }
        if ((flags & ENTRY_BEGIN) && warp == 0 && lane == 0) {    // the item begins in this team, which lists the parts
          meta[1] = last_team;
          meta[2] = slot;
          meta[3] = item.x;
          meta[4] = item.y;
          meta[5] = item.w;                 // the group's first head
          meta[6] = rb;
          meta[0] = 1;
        }
      }
    }
  }
  // every entry has been waited for; after a timeout, give what is under way a little longer to land
  if (*static_cast<volatile int*>(&all.abort)) {
    int zero = 0;
    for (int s = 0; s < STAGES; ++s) mbar_wait(&sm.full[warp][s], s < stage ? parity ^ 1 : parity, &zero, 2000000ull);
  }
}

// Merges the parts of items that several teams worked on.  A job is one output tile (16 dims x 8 rows) of one head of
// such an item; all jobs are numbered and dealt to the warps of the grid, and where there are fewer jobs than warps,
// up to a block's warps share a job's parts.  All it does is wait for memory, so it has two trips to make: every block
// reads the items of all teams, then a warp asks for EARLY parts and their maxima and sums at once.  The order of the
// sums depends on sizes alone.
constexpr int JWARPS = 8, EARLY = 8, MAX_TEAMS = 1024;
// Lists the teams whose last item goes on behind them (their first meta word is set); called by a block of JWARPS warps.
__device__ __forceinline__ int open_items(const CachedParams& p, int teams, uint16_t* s_team, int* s_count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int items = 0;
  for (int c0 = 0; c0 < teams; c0 += JWARPS * 32) {
    const int c = c0 + threadIdx.x;
    const bool open = c < teams && p.meta[c * 8] >= 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, open);
    if (lane == 0) s_count[warp] = __popc(mask);
    __syncthreads();
    int before = items;
#pragma unroll
    for (int w = 0; w < JWARPS; ++w) {
      if (w < warp) before += s_count[w];
      items += s_count[w];
    }
    if (open) s_team[before + __popc(mask & ((1u << lane) - 1))] = static_cast<uint16_t>(c);
    __syncthreads();
  }
  return items;
}
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(JWARPS * 32) cached_join_kernel(const CachedParams p, int teams) {
  constexpr int MT = D / 16, ROWS = 8 * NQ, NREG = NQ * MT * 4;
  __shared__ float s_acc[JWARPS][8][32];
  __shared__ uint16_t s_team[MAX_TEAMS];              // teams whose last item goes on behind them
  __shared__ int s_count[JWARPS];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int4* meta = reinterpret_cast<const int4*>(p.meta);   // set, last team, slot, t0; n, head, rb
  const int items = open_items(p, teams, s_team, s_count);
  const int heads = WARPS >> p.wk_log2, tiles = heads * NQ * MT, jobs = items * tiles;
  int split = static_cast<int>(gridDim.x) * JWARPS / max(jobs, 1);
  split = split >= 8 ? 8 : (split >= 4 ? 4 : (split >= 2 ? 2 : 1));
  const int at_once = static_cast<int>(gridDim.x) * (JWARPS / split);   // jobs
  for (int j0 = 0; j0 < jobs; j0 += at_once) {
    if (j0 + static_cast<int>(blockIdx.x) * (JWARPS / split) >= jobs) break;
    const int job = j0 + blockIdx.x * (JWARPS / split) + warp / split, first = warp % split;
    const bool mine = job < jobs;
    const int c0 = mine ? s_team[job / tiles] : 0;
    const int4 a = meta[2 * c0], b = meta[2 * c0 + 1];
    const int parts = mine ? a.y - c0 + 1 : 0, n = b.x, rb = b.z, rows = n * p.G - rb * ROWS;
    const int head_in_group = job % tiles / (NQ * MT), k = job % (NQ * MT), q = k / MT;
    const bool live0 = mine && 8 * q + 2 * t < rows, live1 = mine && 8 * q + 2 * t + 1 < rows;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[1][4] = {{0.f, 0.f, 0.f, 0.f}};
    for (int i0 = first; i0 < parts; i0 += EARLY * split) {
      float v[EARLY][4];
      float2 ml[EARLY][2];
#pragma unroll
      for (int e = 0; e < EARLY; ++e) {
        const int i = i0 + e * split;
        const bool in = i < parts;
        const int part = ((c0 + i) * 2 + (i ? 0 : a.z)) * WARPS + head_in_group;
        const float2* pm = reinterpret_cast<const float2*>(p.part_ml) + part * ROWS + 8 * q + 2 * t;
        const float* po = p.part_o + static_cast<int64_t>(part) * (NREG * 32) + k * 128 + t * 8 + g;
        ml[e][0] = in && live0 ? pm[0] : make_float2(-INFINITY, 0.f);
        ml[e][1] = in && live1 ? pm[1] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int x = 0; x < 4; ++x) v[e][x] = in && (x & 1 ? live1 : live0) ? po[32 * x] : 0.f;
      }
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        float top = m[e2];
#pragma unroll
        for (int e = 0; e < EARLY; ++e) top = fmaxf(top, ml[e][e2].x);
        const float base = top == -INFINITY ? 0.f : top, keep = exp2f_approx(m[e2] - base);
        m[e2] = top;
        l[e2] *= keep;
        acc[0][e2] *= keep;
        acc[0][2 + e2] *= keep;
#pragma unroll
        for (int e = 0; e < EARLY; ++e) {
          const float w = exp2f_approx(ml[e][e2].x - base);
          l[e2] = fmaf(ml[e][e2].y, w, l[e2]);
          acc[0][e2] = fmaf(v[e][e2], w, acc[0][e2]);
          acc[0][2 + e2] = fmaf(v[e][2 + e2], w, acc[0][2 + e2]);
        }
      }
    }
    if (split > 1) {
      if (first > 0) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s_acc[warp][x][lane] = acc[0][x];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s_acc[warp][4 + e][lane] = m[e];
          s_acc[warp][6 + e][lane] = l[e];
        }
      }
      __syncthreads();
      if (first == 0)
        for (int o = 1; o < split; ++o)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m2 = s_acc[warp + o][4 + e][lane], top = fmaxf(m[e], m2), base = top == -INFINITY ? 0.f : top;
            const float w1 = exp2f_approx(m[e] - base), w2 = exp2f_approx(m2 - base);
            m[e] = top;
            l[e] = l[e] * w1 + s_acc[warp + o][6 + e][lane] * w2;
            acc[0][e] = acc[0][e] * w1 + s_acc[warp + o][e][lane] * w2;
            acc[0][2 + e] = acc[0][2 + e] * w1 + s_acc[warp + o][2 + e][lane] * w2;
          }
      __syncthreads();
    }
    if (first == 0 && mine) store_rows<T, D, 1>(p, a.w, n, b.y + head_in_group, rb * ROWS + 8 * q, lane, acc, l, k % MT);
  }
}

// Kernel attributes are set once per device: `done` is a bit per device of one kernel.
int once_per_device(std::atomic<uint64_t>& done, cudaError_t (*set)()) {
  int dev = 0;
  KCG_CUDA_OK(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return KCG_OK;
  KCG_CUDA_OK(set());
  if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return KCG_OK;
}

// Workspace of the split kernel with 8 NQ rows: two parts per team and head of a group, each the lanes' output registers
// and (m, l) of every row, and eight ints per team.
size_t split_workspace(int64_t D, int nq, int teams) {
  return static_cast<size_t>(teams) * (2 * WARPS * (nq * D / 4 * 32 * 4) + 2 * WARPS * (8 * nq * 2 * 4) + 32);
}
int split_teams(int nq) { return sm_count() * (nq == 1 ? SplitShape<1>::TEAMS : SplitShape<2>::TEAMS); }

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
int launch_split(CachedParams& p, const CUtensorMap& tmK, const CUtensorMap& tmV, void* workspace, cudaStream_t stream) {
  const int teams = split_teams(NQ), blocks = sm_count();
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<size_t>(teams) * 2 * WARPS * (NQ * D / 4 * 32);
  p.meta = reinterpret_cast<int*>(p.part_ml + static_cast<size_t>(teams) * 2 * WARPS * (8 * NQ * 2));
  constexpr int SMEM = sizeof(SplitSmem<D, NQ>) + 1024;
  static_assert(SMEM <= 227 * 1024, "a block does not fit an SM's shared memory");
  auto kern = cached_split_kernel<T, D, NQ>;
  static std::atomic<uint64_t> done{0};
  // (the join may become resident early, so it asks for the split kernel's division of L1 and shared memory)
  int rc = once_per_device(done, []() {
    const cudaError_t e = cudaFuncSetAttribute(cached_split_kernel<T, D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(cached_join_kernel<T, D, NQ>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  });
  if (rc) return rc;
  if (teams > MAX_TEAMS) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: a device of %d SMs", blocks);
  // Not as a programmatic dependent: a block that becomes resident beside the previous kernel's keeps its SM at that
  // kernel's split of L1 and shared memory, where this one does not fit, and queues behind it (142 instead of 100 us for
  // 64 requests of 4096 tokens).
  kern<<<blocks, split_threads<NQ>(), SMEM, stream>>>(tmK, tmV, p);
  rc = check_launch("cached_split_kernel");
  if (rc) return rc;
  launch_overlapped(cached_join_kernel<T, D, NQ>, dim3(2 * blocks), dim3(JWARPS * 32), 0, stream, p, teams);
  return check_launch("cached_join_kernel");
}

#include "fmha_cached_tiles_kernel.cuh"

template <typename T, int D>
int launch_cached(CachedParams& p, int64_t rows, const CUtensorMap& tmK, const CUtensorMap& tmV, void* workspace, cudaStream_t stream) {
  // Two heads side by side where there are two: as fast as four or one with a head's page in one piece, and 20 % faster
  // than one where a token's heads stand together (8 x 4096 tokens of 32 heads, token-major: 54.8 us, one head 68.2).
  p.wk_log2 = p.Hkv % 2 == 0 ? 1 : 2;
  // Up to 48 rows the split kernel reads the cache once per 16 of them and is still faster than a 256-row item that is
  // mostly empty: 16 requests x 4000 keys x 8 heads, 32 rows 73 against 112 us, 64 rows 125 against 113; 64 x 1000 keys 85
  // against 134 and 148 against 137.
  if (rows > 48) return launch_tiles<T, D>(p, static_cast<int64_t>(p.B) * p.Hkv * ((rows + 255) / 256), tmK, tmV, workspace, stream);
  if (rows <= 8) return launch_split<T, D, 1>(p, tmK, tmV, workspace, stream);
  return launch_split<T, D, 2>(p, tmK, tmV, workspace, stream);
}

}  // namespace
}  // namespace kcg

extern "C" int kcg_fmha_cached_workspace(int64_t D, size_t* bytes) {
  using namespace kcg;
  clear_error();
  if (!bytes) return fail(KCG_ERR_INVALID_ARG, "fmha_cached_workspace: null pointer");
  if (D != 64 && D != 128) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: head dimension %lld has no kernel (64, 128)", static_cast<long long>(D));
  const size_t one = split_workspace(D, 1, split_teams(1)), two = split_workspace(D, 2, split_teams(2));
  const size_t many = tiles_workspace(D, sm_count());
  // The many-row kernel stores its parts 32 bytes at a time, the caller's address is a multiple of 16: 16 bytes to spare.
  *bytes = std::max({one, two, many}) + 16;
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
  if (B > kMaxRequests) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: at most %d requests (got %lld)", kMaxRequests, static_cast<long long>(B));
  if (Hq > 65535 || T * Hq > INT32_MAX - 65536 || num_pages > INT32_MAX || table_width > INT32_MAX ||
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
  workspace = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(workspace) + 31) & ~static_cast<uintptr_t>(31));
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
  p.o_by_32 = (reinterpret_cast<uintptr_t>(O) & 31u) == 0 && o_strides[0] % 16 == 0 && o_strides[1] % 16 == 0;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.status = device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // query rows of a request and key head, which choose the kernel: from max_new, else the mean over the batch
  CUtensorMap tmK, tmV;
  int mrc = cache_map(&tmK, k_cache, kc_strides, D, p);
  if (!mrc) mrc = cache_map(&tmV, v_cache, vc_strides, D, p);
  if (mrc) return mrc;
  const int64_t rows = (max_new > 0 ? std::min(max_new, T) : (T + B - 1) / B) * p.G;
  if (dtype == KCG_BF16)
    return D == 128 ? launch_cached<__nv_bfloat16, 128>(p, rows, tmK, tmV, workspace, s) : launch_cached<__nv_bfloat16, 64>(p, rows, tmK, tmV, workspace, s);
  return D == 128 ? launch_cached<__half, 128>(p, rows, tmK, tmV, workspace, s) : launch_cached<__half, 64>(p, rows, tmK, tmV, workspace, s);
}

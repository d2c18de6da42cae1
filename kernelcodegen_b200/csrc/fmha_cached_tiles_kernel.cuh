// Attention over the paged 8-bit cache for many query rows per request (included by fmha_cached.cu inside its anonymous
// namespace).  Here the two matrix products are the cost, so they run on tcgen05 with 128-row tiles, in the order of the
// two-tile kernel of fmha_tcgen05.cu:
//
//   An item is a pair of 128-row tiles of one (request, key / value head): rows are (token, query head of the group) in
//   token-major order, so a block of 128 keys is loaded and converted once for 256 rows, whatever the group.  Where there
//   are many, items are dealt whole, in turn; where there are few, the key blocks of all items, numbered by request, head,
//   pair and keys, are dealt in equal contiguous ranges, as the split kernel deals its units, so that a short chunk against
//   a long context is spread over all SMs.  A range's first and last item may be parts, which cached_tiles_join_kernel
//   merges.
//   warps 0-3, 4-7  softmax of tile 0 / 1, one thread per row (scores, P and O in tensor memory); before that, the row
//                   of Q, as f16 scaled by a power of two, into the swizzled tile the products read; afterwards, O out
//   warp 8          one thread issues the products: S_i = Q_i K^T, O_i += P_i V, S_i(j + 1) right behind P_i V(j)
//   warp 9          walks the items, looks pages and scales up (a record per key block) and loads the codes of K and V by
//                   TMA (boxes of 16 or 32 rows of a page)
//   warps 10, 11    turn codes into f16 tiles in the swizzled layout tcgen05 wants, the same for K and V
// Every ring and barrier runs on across items: records, codes and the first tiles of the next item are on their way while
// the last blocks of this one are worked on.
//
// tcgen05 multiplies f16 with f16 or e4m3 with e4m3, not one with the other, and P in e4m3 would keep four bits; so the
// codes are widened on the way.  Scales: a page's is 2^e f with f in [1, 2).  The power of two, relative to the block's
// largest (K) or the item's largest so far (V), is multiplied into the codes, exactly where a page lies up to
// 2^15 below (e4m3's smallest step is 2^-9, f16's 2^-24); further down a code is rounded once, to f16, and off by up to 2^-25
// of the reference, which beside the reference's own codes is less than the f16 rounding of P.  The references go into the
// softmax constant and the output.  Where some f is not 1 (scales this library did not write) the softmax multiplies the
// scores of a page's 16-key groups with it, and V is multiplied with it (and what is left of the power of two) in fp32 and
// rounded once, to f16.
// Tensor memory (512 columns): S0, S1, O0, O1; P_i overwrites the first half of S_i.
// Measured (32 / 8 heads of 128, causal): 4 prompts of 4096 tokens 800 us (750 to 840 from run to run), 690 TFLOP/s; 3 chunks of up
// to 513 rows over up to 8704 keys 336 us.  A block of 128 keys takes both tiles 3.1 us on the fullest SM of the prompts, whose
// items are dealt whole and whose neighbours read the same keys, and 4.8 us in the chunks, dealt in ranges (start, parts and join
// included).  The tensor pipe is busy 36 and 30 % of the time, a scheduler issues in 32 and 27 % of the clocks; a warp's time
// goes to waits for barriers, tensor memory and loads (31, 34 %), fixed latencies (21, 18 %) and the fetching of instructions (18,
// 23 %: the roles' code is long, and straight).  The codes have one stage per side, so that a load's latency and the conversion of a
// block follow one another; where no other SM has just read the keys, as in ranges, that chain is the longer one.
#pragma once

constexpr int TM = 128;                 // rows of a tile; BN keys of a block
constexpr int TILES_THREADS = 384, CONVERT_WARPS = 2;
constexpr int TILES_REGS_SOFTMAX = 216, TILES_REGS_OTHER = 72;
static_assert(TILES_THREADS / 32 == 10 + CONVERT_WARPS, "warps 10 and up convert");
static_assert(256 * TILES_REGS_SOFTMAX + (TILES_THREADS - 256) * TILES_REGS_OTHER <= TILES_THREADS * 168, "register split exceeds the block's allocation");
// A record is written when the codes of the K tile before it have been converted, which is at most two blocks (the ring of f16
// tiles) before the softmax is through with that block: it is read at most four blocks after it is written.
constexpr int RECORDS = 6, ITEMS = 4;

// What the look-up says about a key block.
struct BlockRecord {
  float kref;                           // scores are to be multiplied with this
  float vshift;                         // what the output so far is to be multiplied with (V's reference has grown)
  float vref;                           // V's reference
  int plain;                            // every group's page is there, every f of K is 1
  uint32_t gone;                        // groups whose page is not in the pool: their keys are left out
  int have;                             // keys up to the request's last token; -1: there is no block and none will come
  int mode[2];                          // of K, V: 0: codes become f16 as they are, 1: times r, 2: there is more to it
  uint32_t r[2][8];                     // of K, V, per group of 16 keys: what its codes are multiplied with, exactly: two f16
  float g[2][8];                        // and then, in fp32 with a rounding to f16: what f16 products cannot do
  float fk[8];                          // f of K, which multiplies the scores
};
struct TilesItem {
  int t0, n, len, head, row0;           // the request's first row of Q, rows, keys; key head; first row of the pair
  int go;                               // 0: there is no item and none will come
  int block0, blocks;                   // the part: its first key block, and how many it has
  int part;                             // where the result goes: -1: O, else the workspace's part
  int pad[3];
};

template <int D> struct TilesSmem {
  static constexpr int DB = D / 64;
  static constexpr int TILE = DB * 16384;               // bytes of a 128 x D f16 tile: DB blocks of 128 rows x 128 bytes
  uint8_t q[2][TILE], k[2][TILE], v[2][TILE];
  uint8_t raw[2][BN * D];                               // codes of K, V, as TMA's swizzle leaves them
  BlockRecord rec[RECORDS];
  TilesItem item[ITEMS];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], rec_full[RECORDS], raw_full[2], raw_empty[2], item_full[ITEMS], item_empty[ITEMS];
  uint64_t q_full[2], s_full[2], p_full[4], o_full[2], drain;
  int64_t scan[16], start_off;
  int start_i;
  uint32_t tmem;
  int abort;
};

// A score times its constant less the running maximum m is one fused operation in the softmax, while m is a rounded product: they differ by
// up to half of m's last place, an exponent of 16 from |m| = 2^28 on.  A score is less than 2^30 (D elements of Q below 2^14, codes
// up to 448), so with a constant below this one products are less than 2^20; others are rounded, as m is, before the softmax.
constexpr float kWideFactor = 0.0009765625f;
constexpr int kF16MinExp = -14;         // of f16's normal numbers; a code times 2^e, e >= kF16MinExp, is exact in f16
__device__ __forceinline__ uint32_t f16x2_pow2(int e) { return static_cast<uint32_t>(e + 15) * 0x04000400u; }   // 2^e twice, kF16MinExp <= e <= 0
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// pv4_peek with a second barrier tested along.
__device__ __forceinline__ bool pv4_peek2(uint32_t d_o, uint32_t a_p, uint64_t vd, uint32_t idesc, uint32_t acc_first, uint32_t peek1,
                                          uint32_t par1, uint32_t peek2, uint32_t par2, bool& ok2) {
  uint32_t r1, r2;
  asm volatile(
      "{\n\t.reg .pred P, Q1, Q2, T;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 v1, v2, v3;\n\t"
      "setp.ne.b32 P, %6, 0;\n\t"
      "setp.eq.b32 T, %6, %6;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 Q1, [%7], %8;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 Q2, [%9], %10;\n\t"
      "add.u32 a1, %3, 8;\n\tadd.u32 a2, %3, 16;\n\tadd.u32 a3, %3, 24;\n\t"
      "add.s64 v1, %4, 128;\n\tadd.s64 v2, %4, 256;\n\tadd.s64 v3, %4, 384;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%2], [%3], %4, %5, P;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%2], [a1], v1, %5, T;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%2], [a2], v2, %5, T;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%2], [a3], v3, %5, T;\n\t"
      "selp.u32 %0, 1, 0, Q1;\n\tselp.u32 %1, 1, 0, Q2;\n\t}"
      : "=r"(r1), "=r"(r2)
      : "r"(d_o), "r"(a_p), "l"(vd), "r"(idesc), "r"(acc_first), "r"(peek1), "r"(par1), "r"(peek2), "r"(par2)
      : "memory");
  ok2 = r2 != 0;
  return r1 != 0;
}

// Key blocks of the tile of rows that begins at `first`: up to the last key its last row sees.
__device__ __forceinline__ int tile_blocks(const CachedParams& p, int first, int n, int len) {
  const int last = min(first + TM, n * p.G) - 1;
  if (last < first) return 0;
  const int end = p.causal ? min(len, len - n + 1 + last / p.G) : len;
  return end > 0 ? (end + BN - 1) / BN : 0;
}
__device__ __forceinline__ int pair_blocks(const CachedParams& p, int row0, int n, int len) {
  return max(tile_blocks(p, row0, n, len), tile_blocks(p, row0 + TM, n, len));
}
__device__ __forceinline__ int pairs_of(const CachedParams& p, const Request& r) { return (r.n * p.G + 2 * TM - 1) / (2 * TM); }
// sum over i < n of floor((a i + b) / m), by the steps of Euclid's algorithm on (m, a).
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t sum = 0;
  while (n > 0) {
    sum += (n - 1) * n / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const int64_t top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const int64_t s = m;
    m = a;
    a = s;
  }
  return sum;
}
// Units (key blocks, but one at least: a pair that sees nothing still has to write its zeros) of pairs 0 .. k - 1 of one
// head.  Under a causal mask pair i ends with row 256 i + 255 (the last pair, of fewer rows, is counted by itself) and sees
// len - n + 1 + floor((256 i + 255) / G) keys, in floor((256 i + 255 + G (len - n + 128)) / (128 G)) blocks.
__device__ __forceinline__ int64_t units_before(const CachedParams& p, const Request& r, int k) {
  if (k == 0) return 0;
  if (!p.causal) return static_cast<int64_t>(k) * max(1, pair_blocks(p, 0, r.n, r.len));
  if (r.len >= r.n) {
    const int full = min(k, pairs_of(p, r) - 1);
    const int64_t G = p.G;
    return floor_sum(full, 128 * G, 256, 255 + G * (r.len - r.n + 128)) + (k > full ? pair_blocks(p, full * 2 * TM, r.n, r.len) : 0);
  }
  int64_t units = 0;                        // rows before the request's first key: rare, counted one by one
  for (int i = 0; i < k; ++i) units += max(1, pair_blocks(p, i * 2 * TM, r.n, r.len));
  return units;
}
__device__ __forceinline__ int64_t head_units(const CachedParams& p, const Request& r) { return units_before(p, r, pairs_of(p, r)); }

template <typename T, int D>
__global__ void __launch_bounds__(TILES_THREADS, 1)
cached_tiles_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CachedParams p,
                    const uint32_t idesc_qk, const uint32_t idesc_pv) {
  extern __shared__ uint8_t smem_raw[];
  using Smem = TilesSmem<D>;
  constexpr int DB = Smem::DB, TILE = Smem::TILE;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &sm.abort;
  if (tid == 0) {
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.raw_full[s], 1);
      mbar_init(&sm.raw_empty[s], CONVERT_WARPS * 32);
      mbar_init(&sm.k_full[s], CONVERT_WARPS * 32);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], CONVERT_WARPS * 32);
      mbar_init(&sm.v_empty[s], 1);
      mbar_init(&sm.q_full[s], 4);
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.o_full[s], 1);
      mbar_init(&sm.p_full[2 * s], 4);
      mbar_init(&sm.p_full[2 * s + 1], 4);
    }
    for (int s = 0; s < RECORDS; ++s) mbar_init(&sm.rec_full[s], 1);
    for (int s = 0; s < ITEMS; ++s) {
      mbar_init(&sm.item_full[s], 1);
      mbar_init(&sm.item_empty[s], 9);      // eight softmax warps and the issuing thread
    }
    mbar_init(&sm.drain, 1);
    sm.abort = 0;
    mbar_fence_init();
  }
  if (warp == 8) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  auto give_up = [&]() {
    if (!*abort_flag) {
      *abort_flag = 1;
      if (p.status) *p.status = KCG_ERR_TIMEOUT;
    }
  };
  // A wait may run out in some lanes of a warp and not in others, and lanes must not leave while others count on them.  Where they do
  // something together behind a wait they vote on its end; the softmax warps, which a vote per wait would cost time, go on whatever
  // its end (what they work on is then meaningless, and the status says so) and leave together at the next block's vote, which they
  // have anyway.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_wait(bar, parity, abort_flag)) give_up();
  };
  auto over = [&]() -> bool { return __any_sync(0xffffffffu, *abort_flag); };
  // ---- this block's range of units ----
  const int per = (p.B + TILES_THREADS - 1) / TILES_THREADS;
  const int i_lo = min(tid * per, p.B), i_hi = min(i_lo + per, p.B);
  int64_t total = 0, first_unit = 0;
  int units = 0;
  if (!p.whole_items) {
    int64_t mine = 0;
    for (int i = i_lo; i < i_hi; ++i) mine += p.Hkv * head_units(p, request_of(p, i));
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    if (lane == 31) sm.scan[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TILES_THREADS / 32; ++w) {
      if (w < warp) upto += sm.scan[w];
      total += sm.scan[w];
    }
    const int64_t grid = min(static_cast<int64_t>(gridDim.x), total);   // blocks at work
    if (blockIdx.x < grid) {
      first_unit = total * blockIdx.x / grid;
      units = static_cast<int>(total * (blockIdx.x + 1) / grid - first_unit);
    }
    int64_t off = first_unit - (upto - mine);
    if (units > 0 && off >= 0 && off < mine) {           // one thread's requests hold the first unit
      int i = i_lo;
      for (;; ++i) {
        const int64_t n = p.Hkv * head_units(p, request_of(p, i));
        if (off < n) break;
        off -= n;
      }
      sm.start_i = i;
      sm.start_off = off;
    }
    if (tid == 0) p.meta[blockIdx.x * 8] = -1;
    __syncthreads();
  }
  // blocks of tile i in an item's part
  auto blocks_of = [&](int i, const TilesItem& it) {
    return min(max(tile_blocks(p, it.row0 + i * TM, it.n, it.len) - it.block0, 0), it.blocks);
  };

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax
    reg_alloc<TILES_REGS_SOFTMAX>();
    const int i = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    // (Registers are what this role is short of: an item's description stays in shared memory until its output is out.)
    const uint32_t s_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + i * BN, o_addr = s_addr + 256;
    static_assert(BN == TM, "O_i stands 256 columns behind S_i");
    uint32_t b = 0, phases = 0;             // key block; phases of s_full (bit 0) and o_full (bit 1)
    // Rows of Q and O cross global memory whole: PPR lanes with 16 bytes each take a row, RPI rows at a time.
    constexpr int PPR = D / 8, RPI = 32 / PPR;
    // A thread works out where its own row is (a division) and the others ask it.  (Strides may be negative.)
    constexpr int64_t NO_ROW = INT64_MIN;
    auto offset_of = [&](const TilesItem& it, int64_t by_token, int64_t by_head) -> int64_t {
      const int R = it.row0 + i * TM + r;
      if (R >= it.n * p.G) return NO_ROW;
      const int token = R / p.G;
      return (it.t0 + token) * by_token + (it.head * p.G + R - token * p.G) * by_head;
    };
    // The warp's 32 rows of Q: fetched as they are, straight to where they will be read, and turned into f16 there, every
    // thread its own row.  Returns what the row's scores are to be multiplied with.
    auto fetch_q = [&](const TilesItem& it) {
      const int64_t mine = offset_of(it, p.q_st, p.q_sh);
#pragma unroll
      for (int k = 0; k < 32 / RPI; ++k) {
        const int64_t at = __shfl_sync(0xffffffffu, mine, k * RPI + lane / PPR);
        const int row = quarter * 32 + k * RPI + lane / PPR, ch = lane % PPR;
        cp_async16(smem_u32(sm.q[i]) + (ch >> 3) * 16384 + row * 128 + (((ch & 7) ^ (row & 7)) << 4),
                   static_cast<const T*>(p.Q) + (at == NO_ROW ? 0 : at) + ch * 8, at != NO_ROW);
      }
    };
    auto convert_q = [&]() -> float {
      cp_async_wait_all();
      __syncwarp();                         // (a thread's row was fetched by its neighbours)
      const uint32_t row = smem_u32(sm.q[i]) + r * 128;
      auto piece = [&](int k) { return row + (k >> 3) * 16384 + (((k & 7) ^ (r & 7)) << 4); };
      const bool negative = p.scale_log2 < 0.f;          // the softmax's constant is not negative
      uint32_t w[PPR][4];
#pragma unroll
      for (int k = 0; k < PPR; ++k) lds128(piece(k), w[k]);
      uint32_t big = 0;
#pragma unroll
      for (int k = 0; k < PPR; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) big = __vmaxu2(big, w[k][x] & 0x7fff7fffu);
      big = max(big & 0xffffu, big >> 16);
      float top[2];
      Words<T>::unpack(big, top);
      int e = static_cast<int>(__float_as_uint(top[0]) >> 23) - 127 - 13;       // largest element to [2^13, 2^14)
      e = e < -113 ? -113 : e;
      const float up = __uint_as_float((static_cast<uint32_t>(127 - e) << 23) | (negative ? 0x80000000u : 0u));
      const float factor = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int k = 0; k < PPR; ++k) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float f[2];
          Words<T>::unpack(w[k][x], f);
          w[k][x] = pack_f16(f[0] * up, f[1] * up);
        }
        sts128(piece(k), w[k]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[i]);
      return factor * fabsf(p.scale_log2);
    };
    bool ok = true, have_q = false;
    float c = 0.f;
    for (uint32_t k_item = 0; ok; ++k_item) {
      if (!mbar_wait_warp(&sm.item_full[k_item % ITEMS], (k_item / ITEMS) & 1u, abort_flag)) { ok = false; break; }
      const TilesItem& it = sm.item[k_item % ITEMS];
      if (!it.go) break;
      // key blocks of this tile and of the other; keys this row sees from block b on
      const int n_mine = blocks_of(i, it), n_other = blocks_of(1 - i, it);
      int seen = 0;
      {
        const int R = it.row0 + i * TM + r;
        if (R < it.n * p.G) seen = (p.causal ? min(it.len, it.len - it.n + 1 + R / p.G) : it.len) - it.block0 * BN;
      }
      // A tile without key blocks has no queries either: its warps run on to later items, up to the ring's length, and
      // phases of q_full count the items that use them, which nobody can run ahead of.
      if (!have_q && n_mine > 0) {
        fetch_q(it);
        c = convert_q();
      }
      have_q = false;
      float m = -INFINITY, l = 0.f, vref = 1.f;
      for (int j = 0; j < n_mine; ++j, ++b, phases ^= 1u) {
        const BlockRecord& rec = sm.rec[b % RECORDS];
        wait(&sm.rec_full[b % RECORDS], (b / RECORDS) & 1u);
        float cj = c * rec.kref;
        // cj of 0, or so large that a score may be wide (one comparison for both)
        const bool odd = __any_sync(0xffffffffu, rec.plain == 0 || __float_as_uint(cj) - 1u >= __float_as_uint(kWideFactor) - 1u || *abort_flag);
        if (odd && over()) { ok = false; break; }
        const float vshift = rec.vshift;
        vref = rec.vref;
        wait(&sm.s_full[i], phases & 1u);
        tc_fence_after();
        if (j + 1 == n_mine) {
          // the tile's last scores are there, so its Q is free: the next item's, if that is known already
          const uint32_t next = k_item + 1;
          if (__all_sync(0xffffffffu, mbar_try_wait(&sm.item_full[next % ITEMS], (next / ITEMS) & 1u)) && sm.item[next % ITEMS].go &&
              blocks_of(i, sm.item[next % ITEMS]) > 0) {
            fetch_q(sm.item[next % ITEMS]);
            have_q = true;
          }
        }
        if (odd) {
          // scores that a block-wide constant does not serve are put right in place, in pieces that leave registers alone
          const bool wide = cj >= kWideFactor;
#pragma unroll 1
          for (int cc = 0; cc < BN / 32; ++cc) {
            uint32_t x[32];
            tmem_ld32(s_addr + cc * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float f = cj == 0.f ? 0.f : rec.fk[2 * cc + (k >> 4)], y = __fmul_rn(__uint_as_float(x[k]) * f, wide ? cj : 1.f);
              x[k] = (rec.gone >> (2 * cc + (k >> 4))) & 1u ? 0xff800000u : __float_as_uint(y);
            }
            tmem_st32(s_addr + cc * 32, x);
            tmem_wait_st();
          }
          if (cj == 0.f || wide) cj = 1.f;               // (-inf times 0 is not -inf)
        }
        // the scores being complete means that P V of the block before is, too: O may be changed
        if (j > 0 && vshift != 1.f) {
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t x[32];
            tmem_ld32(o_addr + cc * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * vshift);
            tmem_st32(o_addr + cc * 32, x);
            tmem_wait_st();
          }
        }
        softmax_block<__half, D, 0, static_cast<int>(kLazy), true>(s_addr, o_addr, j, seen - j * BN, cj, m, l, lane, [&](int half) { mbar_arrive(&sm.p_full[2 * i + half]); });
      }
      // The next item's scores may be computed while this one's output leaves.
      if (ok && have_q) c = convert_q();
      if (ok && n_mine > 0) {
        wait(&sm.o_full[i], phases >> 1);
        ok = !over();
        phases ^= 2u;
        tc_fence_after();
      }
      if (!ok) break;
      {
        const int part = it.part;
        // a row that sees no key is zero; a part keeps its sums as they are
        const float inv = l == 0.f ? 0.f : (part < 0 ? vref / l : vref);
        const int64_t at = part < 0 ? offset_of(it, p.o_st, p.o_sh) : 0;
        float* po = p.part_o + (static_cast<int64_t>(part) * 2 * TM + i * TM + r) * D;
        if (part >= 0) *reinterpret_cast<float2*>(p.part_ml + (static_cast<int64_t>(part) * 2 * TM + i * TM + r) * 2) = make_float2(m, l);
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t x[32];
          if (n_mine > 0) {
            tmem_ld32(o_addr + cc * 32, x);
            tmem_wait_ld();
          }
          if (part >= 0) {
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(x[k]) * inv);
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              st_256(po + cc * 32 + k, make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]), make_uint4(x[k + 4], x[k + 5], x[k + 6], x[k + 7]));
            continue;
          }
          uint4 w[4];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float f[2] = {__uint_as_float(x[2 * k]) * inv, __uint_as_float(x[2 * k + 1]) * inv};
            reinterpret_cast<uint32_t*>(w)[k] = l == 0.f ? 0u : Words<T>::pack(f);
          }
          if (at != NO_ROW) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.O) + at + cc * 32);
            if (p.o_by_32) {                // whole sectors
              st_256(dst, w[0], w[1]);
              st_256(dst + 2, w[2], w[3]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) dst[k] = w[k];
            }
          }
        }
        tc_fence_before();                  // (the next item's first product overwrites O behind this thread's first P)
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.item_empty[k_item % ITEMS]);
      b += max(n_other - n_mine, 0);
    }
    if (!ok) {
      give_up();
      cp_async_wait_all();                  // queries on their way into this block's memory
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ products
    reg_dealloc<TILES_REGS_OTHER>();
    if (lane == 0) {
      const uint64_t qd = make_smem_desc(smem_u32(sm.q[0]), 16, 1024), kd = make_smem_desc(smem_u32(sm.k[0]), 16, 1024);
      const uint64_t vd = make_smem_desc(smem_u32(sm.v[0]), 16384, 1024);
      const uint32_t kf = smem_u32(sm.k_full), vf = smem_u32(sm.v_full), pf = smem_u32(sm.p_full), sf = smem_u32(sm.s_full),
                     of = smem_u32(sm.o_full);
      uint32_t blocks = 0, cp0 = 0, cp1 = 0;             // key blocks before this item, P blocks of the tiles so far
      uint32_t q_phase = 0;                              // phases of q_full: bit i
      bool ok = true;
      for (uint32_t k_item = 0; ok; ++k_item) {
        if (!mbar_wait(&sm.item_full[k_item % ITEMS], (k_item / ITEMS) & 1u, abort_flag)) { ok = false; break; }
        const TilesItem& it = sm.item[k_item % ITEMS];
        const bool go = it.go;
        const int n0 = blocks_of(0, it), n1 = blocks_of(1, it), nmax = it.blocks;
        mbar_arrive(&sm.item_empty[k_item % ITEMS]);
        if (!go) break;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((i == 0 ? n0 : n1) > 0) {
            if (!mbar_wait(&sm.q_full[i], (q_phase >> i) & 1u, abort_flag)) ok = false;
            q_phase ^= 1u << i;
          }
        if (!ok) break;
        if (nmax > 0) {
          if (!mbar_wait(&sm.k_full[blocks & 1u], (blocks >> 1) & 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if ((i == 0 ? n0 : n1) > 0) {
#pragma unroll
              for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_ss<Kind::F16>(tmem + i * BN, qd + ((i * TILE + d * 16384 + k * 32) >> 4),
                                    kd + (((blocks & 1u) * TILE + d * 16384 + k * 32) >> 4), idesc_qk, (d | k) != 0 ? 1u : 0u);
              mma_commit(&sm.s_full[i]);
            }
          mma_commit(&sm.k_empty[blocks & 1u]);
        }
        // barriers already seen complete by a test that rode along with an earlier batch of products
        bool r_v = false, r_p00 = false, r_p10 = false;
        for (int j = 0; j < nmax && ok; ++j) {
          const uint32_t b = blocks + j, slot = b & 1u, next = slot ^ 1u;
          if (!r_v && !mbar_wait(&sm.v_full[slot], (b >> 1) & 1u, abort_flag)) { ok = false; break; }
          r_v = false;
          bool r_k = false;
          const uint64_t v = vd + ((slot * TILE) >> 4), k = kd + ((next * TILE) >> 4);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n_i = i == 0 ? n0 : n1;
            if (j >= n_i) continue;
            uint32_t& cp = i == 0 ? cp0 : cp1;
            bool& r_p = i == 0 ? r_p00 : r_p10;
            const uint32_t pj = cp & 1u;
            if (!r_p && !mbar_wait(&sm.p_full[2 * i], pj, abort_flag)) { ok = false; break; }
            r_p = false;
            tc_fence_after();
            const uint32_t d_o = tmem + 256 + i * TM, a_p = tmem + i * BN;
            bool seen_k;
            const bool seen_p = pv4_peek2(d_o, a_p, v, idesc_pv, j != 0 ? 1u : 0u, pf + (2 * i + 1) * 8, pj, kf + next * 8, ((b + 1) >> 1) & 1u, seen_k);
            if (!seen_p && !mbar_wait(&sm.p_full[2 * i + 1], pj, abort_flag)) { ok = false; break; }
            ++cp;
            bool t1, t2;
            // tested meanwhile: behind tile 0 the first half of tile 1's P, behind tile 1 the next V and tile 0's next P
            const uint32_t peek1 = i == 0 ? pf + 2 * 8 : vf + next * 8, par1 = i == 0 ? (cp1 & 1u) : (((b + 1) >> 1) & 1u);
            const uint32_t peek2 = pf, par2 = cp0 & 1u;
            const uint64_t q = qd + ((i * TILE) >> 4);
            if (j + 1 < n_i) {
              if (!r_k && !seen_k && !mbar_wait(&sm.k_full[next], ((b + 1) >> 1) & 1u, abort_flag)) { ok = false; break; }
              r_k = true;
              tc_fence_after();
              pv4_s_commit_peek2<D, true>(d_o, a_p + 32, v + 512, idesc_pv, tmem + i * BN, q, k, idesc_qk, sf + i * 8, peek1, par1, peek2, par2, t1, t2);
            } else {
              tc_fence_after();
              pv4_s_commit_peek2<D, false>(d_o, a_p + 32, v + 512, idesc_pv, tmem + i * BN, q, k, idesc_qk, of + i * 8, peek1, par1, peek2, par2, t1, t2);
            }
            if (i == 0) {
              r_p10 = t1 && j < n1;
            } else {
              r_v = t1 && j + 1 < nmax;
              r_p00 = t2 && j + 1 < n0;
            }
          }
          if (!ok) break;
          mma_commit(&sm.v_empty[slot]);
          if (j + 1 < nmax) mma_commit(&sm.k_empty[next]);
        }
        blocks += nmax;
      }
      if (!ok) give_up();
      int zero = 0;
      mma_commit(&sm.drain);                // what was issued must end before the block does
      mbar_wait(&sm.drain, 0, &zero, 20000000ull);
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------ items, pages, scales
    // Lane g < 8 looks after a block's keys 16 g .. 16 g + 15.
    reg_dealloc<TILES_REGS_OTHER>();
    int req = 0, head = 0, pair = 0, block0 = 0;         // the walk's place: the next unit to be done
    Request r{0, 0, 0};
    if (units > 0) {
      req = sm.start_i;
      r = request_of(p, req);
      const int64_t per_head = head_units(p, r);
      head = static_cast<int>(sm.start_off / per_head);
      int64_t off = sm.start_off - head * per_head;
      int above = pairs_of(p, r);           // the last pair with no more than `off` units before it
      while (pair + 1 < above) {
        const int mid = (pair + above) >> 1;
        if (units_before(p, r, mid) <= off) pair = mid; else above = mid;
      }
      block0 = static_cast<int>(off - units_before(p, r, pair));
    }
    // Whole items instead, one in gridDim.x: to the block's next one, the last rows of a head (the longest) first.
    int64_t left = blockIdx.x;
    bool another = units > 0;
    auto next_whole = [&]() {
      another = false;
      for (; req < p.B; ++req) {
        r = request_of(p, req);
        const int pairs = pairs_of(p, r);
        const int64_t n = static_cast<int64_t>(p.Hkv) * pairs;
        if (left < n) {
          head = static_cast<int>(left) / pairs;
          pair = pairs - 1 - static_cast<int>(left) % pairs;
          left += gridDim.x;
          another = true;
          return;
        }
        left -= n;
      }
    };
    if (p.whole_items) next_whole();
    int done = 0;                           // units
    uint32_t blocks = 0;
    bool ok = true;
    for (uint32_t k_item = 0; ok; ++k_item) {
      const bool go = another;
      const int row0 = pair * 2 * TM;
      const int in_item = go ? pair_blocks(p, row0, r.n, r.len) : 0, item_units = max(1, in_item);
      const int take = go ? (p.whole_items ? item_units : min(item_units - block0, units - done)) : 0;
      const int nmax = go ? min(take, in_item - block0) : 1;             // key blocks (none, where the pair sees nothing)
      const bool whole = block0 == 0 && take == item_units;
      if (!mbar_wait_warp(&sm.item_empty[k_item % ITEMS], ((k_item / ITEMS) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
      if (lane == 0) {
        const int slot = k_item == 0 ? 0 : 1;
        sm.item[k_item % ITEMS] = TilesItem{r.t0, r.n, r.len, head, row0, go, block0, max(nmax, 0), whole ? -1 : static_cast<int>(blockIdx.x) * 2 + slot, {0, 0, 0}};
        mbar_arrive(&sm.item_full[k_item % ITEMS]);
        if (go && !whole && block0 == 0) {   // the item begins here and ends in a later block's range: this one lists the parts
          const int64_t grid = min(static_cast<int64_t>(gridDim.x), total), last_unit = first_unit + done + item_units - 1;
          int* meta = p.meta + blockIdx.x * 8;
          meta[1] = static_cast<int>(((last_unit + 1) * grid - 1) / total);
          meta[2] = slot;
          meta[3] = r.t0;
          meta[4] = r.n;
          meta[5] = head;
          meta[6] = row0;
          meta[0] = 1;
        }
      }
      // the item's queries on their way to L2
      for (int R = row0 + lane; go && R < min(row0 + 2 * TM, r.n * p.G); R += 32) {
        const int token = R / p.G;
        const T* q = static_cast<const T*>(p.Q) + (r.t0 + token) * p.q_st + (head * p.G + R - token * p.G) * p.q_sh;
#pragma unroll
        for (int k = 0; k < D; k += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + k));
      }
      // Two loads follow one another (page, then scales), and a block takes hardly longer than either: a block's page is
      // asked for two blocks ahead, its scales one.
      struct Place { int pid, row; };
      auto page_of = [&](int j) -> Place {
        const int key = (block0 + j) * BN + 16 * lane;
        Place x{-1, 0};
        if (go && lane < 8 && j < nmax && key < r.len) {
          const int w = key / p.page;
          x.row = key - w * p.page;
          x.pid = p.table[req * p.table_stride + w];
          if (x.pid < 0 || x.pid >= p.num_pages) x.pid = -2;
        }
        return x;
      };
      auto scale_of = [&](const float* scales, const Place& x) { return x.pid >= 0 ? scales[static_cast<int64_t>(x.pid) * p.Hkv + head] : 0.f; };
      Place now = page_of(0), next = page_of(1);
      float ks = scale_of(p.ks, now), vs = scale_of(p.vs, now);
      int vexp = -1000;
      for (int j = 0; j < nmax; ++j) {
        const uint32_t b = blocks + j;
        const int page = now.pid, at = now.row;
        const float ks_now = ks, vs_now = vs;
        if (page == -2 && p.status) *p.status = KCG_ERR_INVALID_ARG;
        now = next;
        ks = scale_of(p.ks, now);
        vs = scale_of(p.vs, now);
        next = page_of(j + 2);
        // scale = f 2^e; zero, subnormal, infinite and NaN scales go into f, at the reference's exponent
        auto exponent = [](float s) {
          const int x = static_cast<int>((__float_as_uint(s) >> 23) & 255u);
          return x == 0 || x == 255 ? -1000 : x - 127;
        };
        auto rest = [](float s, int e, int ref) {
          if (e != -1000) return __uint_as_float((__float_as_uint(s) & 0x807fffffu) | 0x3f800000u);
          return s * pow2f(-ref / 2) * pow2f(-ref + ref / 2);
        };
        const bool there = page >= 0;
        const int ek = there ? exponent(ks_now) : -1000, ev = there ? exponent(vs_now) : -1000;
        const int kmax = __reduce_max_sync(0xffffffffu, ek), vmax = __reduce_max_sync(0xffffffffu, ev);
        const int kref = kmax == -1000 ? 0 : kmax, vold = vexp;
        vexp = max(vexp, vmax);
        const int vnow = vexp == -1000 ? 0 : vexp;
        const float fk = there ? rest(ks_now, ek, kref) : 1.f, fv = there ? rest(vs_now, ev, vnow) : 1.f;
        // the power of two, relative to the reference: an f16 factor where that is exact, else a part of the fp32 one
        const int dk = ek == -1000 ? 0 : ek - kref, dv = ev == -1000 ? 0 : ev - vnow;
        const float gk = dk < kF16MinExp ? pow2f(dk) : 1.f, gv = dv < kF16MinExp ? fv * pow2f(dv) : fv;
        const uint32_t gone = __ballot_sync(0xffffffffu, page == -2);
        const bool plain = __all_sync(0xffffffffu, page != -2 && fk == 1.f);
        const int have = r.len - (block0 + j) * BN;
        const bool full = gone == 0 && have >= BN;
        const bool unit_k = __all_sync(0xffffffffu, !there || ek == kref), unit_v = __all_sync(0xffffffffu, !there || ev == vnow);
        const bool plain_gk = __all_sync(0xffffffffu, gk == 1.f), plain_gv = __all_sync(0xffffffffu, gv == 1.f);
        // (with boxes of 32 rows an even group brings the odd one behind it)
        const bool issue = there && (p.box == 16 || (lane & 1) == 0);
        const uint32_t bytes = __reduce_add_sync(0xffffffffu, issue ? p.box * D : 0);
        if (!mbar_wait_warp(&sm.raw_empty[0], (b & 1u) ^ 1u, abort_flag)) { ok = false; break; }
        if (lane == 0 && go) mbar_expect_tx(&sm.raw_full[0], bytes);
        BlockRecord& rec = sm.rec[b % RECORDS];
        if (lane < 8) {
          rec.r[0][lane] = f16x2_pow2(dk < kF16MinExp ? 0 : dk);
          rec.r[1][lane] = f16x2_pow2(dv < kF16MinExp ? 0 : dv);
          rec.g[0][lane] = gk;
          rec.g[1][lane] = gv;
          rec.fk[lane] = fk;
        }
        if (lane == 0) {
          rec.kref = pow2f(kref);
          rec.vref = pow2f(vnow);
          rec.vshift = j == 0 || vold == vexp ? 1.f : (vold == -1000 ? pow2f(-vexp) : pow2f(vold - vexp));
          rec.plain = plain;
          rec.gone = gone;
          rec.mode[0] = !full || !plain_gk ? 2 : (unit_k ? 0 : 1);
          rec.mode[1] = !full || !plain_gv ? 2 : (unit_v ? 0 : 1);
          rec.have = go ? min(have, BN) : -1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.rec_full[b % RECORDS]);
        if (!go) break;
        if (issue) tma_load_4d(sm.raw[0] + lane * 16 * D, &tmK, &sm.raw_full[0], 0, at, head, page);
        if (!mbar_wait_warp(&sm.raw_empty[1], (b & 1u) ^ 1u, abort_flag)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(&sm.raw_full[1], bytes);
        __syncwarp();
        if (issue) tma_load_4d(sm.raw[1] + lane * 16 * D, &tmV, &sm.raw_full[1], 0, at, head, page);
      }
      if (!ok || !go) break;
      blocks += max(nmax, 0);
      if (p.whole_items) {
        next_whole();
        continue;
      }
      done += take;
      another = done < units;
      block0 += take;
      if (block0 == item_units) {           // on to the next pair, head, request
        block0 = 0;
        if (++pair == pairs_of(p, r)) {
          pair = 0;
          if (++head == p.Hkv) {
            head = 0;
            if (done < units)
              do r = request_of(p, ++req);
              while (r.n == 0);
          }
        }
      }
    }
    if (!ok) give_up();
    if (over()) {
      int zero = 0;                         // let the copies that were issued land before the block goes away
      for (int s = 0; s < 2; ++s) {
        mbar_wait(&sm.raw_full[s], 0, &zero, 2000000ull);
        mbar_wait(&sm.raw_full[s], 1, &zero, 2000000ull);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ codes to f16
    // A thread turns 16-byte pieces into two: of row r0 + STEP x, always the same column.  STEP is a multiple of 8, so
    // the swizzle is the same in every row it meets and its addresses differ by constants.
    reg_dealloc<TILES_REGS_OTHER>();
    constexpr int CPR = D / 16;             // pieces of a row
    constexpr int STEP = CONVERT_WARPS * 32 / CPR, PIECES = BN / STEP;
    static_assert(STEP % 8 == 0 && BN % STEP == 0 && PIECES % 4 == 0, "");
    const int ct = tid - (TILES_THREADS - CONVERT_WARPS * 32), r0 = ct / CPR, ch = ct % CPR;
    // The two 128-byte lines a row of D = 128 becomes share banks: threads of the second write their halves in the other order.
    const int swap = D == 128 ? ch >> 2 : 0;
    const uint32_t src0 = smem_u32(sm.raw[0]) + tile_offset<D>(r0, ch) + swap * 8;
    const uint32_t dst0 = smem_u32(sm.k[0]) + (ch >> 2) * 16384 + r0 * 128;
    const uint32_t first = ((2 * (ch & 3) + swap) ^ (r0 & 7)) << 4, second = ((2 * (ch & 3) + 1 - swap) ^ (r0 & 7)) << 4;
    static_assert(offsetof(Smem, v) - offsetof(Smem, k) == 2 * TILE, "V's tiles stand behind K's");
    bool ok = true;
    for (uint32_t b = 0; ok; ++b) {
      if (!mbar_wait(&sm.rec_full[b % RECORDS], (b / RECORDS) & 1u, abort_flag)) { ok = false; break; }
      const BlockRecord& rec = sm.rec[b % RECORDS];
      if (rec.have < 0) break;
      const uint32_t slot = b & 1u;
      const int have = rec.have;
      const uint32_t gone = rec.gone;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        if (!mbar_wait(&sm.raw_full[side], b & 1u, abort_flag) ||
            !mbar_wait(side ? &sm.v_empty[slot] : &sm.k_empty[slot], ((b >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
        const uint32_t src = src0 + side * (BN * D), dst = dst0 + (side * 2 + slot) * TILE;
        auto convert = [&](auto how) {
          constexpr int kMode = decltype(how)::value;
#pragma unroll 1
          for (int x0 = 0; x0 < PIECES; x0 += 4) {       // four pieces at once: the loads first
            uint32_t w[4][2][2];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              lds64(src + (x0 + x) * STEP * D, w[x][0]);
              lds64((src + (x0 + x) * STEP * D) ^ 8u, w[x][1]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int r = r0 + STEP * (x0 + x);
              uint32_t h[2][4];
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int y = 0; y < 2; ++y) e4m3x4_to_f16(w[x][e][y], h[e][2 * y], h[e][2 * y + 1]);
              if constexpr (kMode > 0) {
                const uint32_t f = rec.r[side][r >> 4];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int y = 0; y < 4; ++y) h[e][y] = hmul2(h[e][y], f);
              }
              if constexpr (kMode == 2) {
                const float g = rec.g[side][r >> 4];
                const bool nothing = r >= have || ((gone >> (r >> 4)) & 1u);   // (the bytes may be anything)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int y = 0; y < 4; ++y) {
                    uint32_t v = h[e][y];
                    if (g != 1.f) {
                      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v));
                      v = pack_f16(a.x * g, a.y * g);
                    }
                    h[e][y] = nothing ? 0u : v;
                  }
              }
              sts128(dst + (x0 + x) * STEP * 128 + first, h[0]);
              sts128(dst + (x0 + x) * STEP * 128 + second, h[1]);
            }
          }
        };
        const int mode = rec.mode[side];
        if (mode == 0) convert(std::integral_constant<int, 0>{});
        else if (mode == 1) convert(std::integral_constant<int, 1>{});
        else convert(std::integral_constant<int, 2>{});
        fence_proxy_async_smem();
        mbar_arrive(&sm.raw_empty[side]);
        mbar_arrive(side ? &sm.v_full[slot] : &sm.k_full[slot]);
      }
    }
    if (!ok) give_up();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merges the parts of items that several blocks worked on, in a fixed order.  A warp takes ROWS8 rows of an item at once and
// asks for two parts of all of them before it adds any: all it does is wait for memory.
constexpr int ROWS8 = 8;
template <typename T, int D>
__global__ void __launch_bounds__(JWARPS * 32) cached_tiles_join_kernel(const CachedParams p, int blocks) {
  __shared__ uint16_t s_block[MAX_TEAMS];             // blocks whose last item goes on behind them
  __shared__ int s_count[JWARPS];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int items = open_items(p, blocks, s_block, s_count);
  constexpr int VL = D / 32, JOBS = 2 * TM / ROWS8;   // floats of a lane; jobs of an item
  for (int job = blockIdx.x * JWARPS + warp; job < items * JOBS; job += gridDim.x * JWARPS) {
    const int c0 = s_block[job / JOBS], r = job % JOBS * ROWS8;
    const int4* meta = reinterpret_cast<const int4*>(p.meta + c0 * 8);   // set, last block, slot, t0; n, head, row0
    const int4 a = meta[0], b = meta[1];
    const int rows = b.x * p.G - b.z - r;             // that there are, from r on
    if (rows <= 0) continue;
    float m[ROWS8], l[ROWS8], acc[ROWS8][VL];
#pragma unroll
    for (int x = 0; x < ROWS8; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int k = 0; k < VL; ++k) acc[x][k] = 0.f;
    }
    for (int c = c0; c <= a.y; c += 2) {
      float2 ml[2][ROWS8];
      float v[2][ROWS8][VL];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t row = (static_cast<int64_t>(c + e) * 2 + (c + e == c0 ? a.z : 0)) * 2 * TM + r;
        const bool in = c + e <= a.y;
#pragma unroll
        for (int x = 0; x < ROWS8; ++x) {
          ml[e][x] = in ? *reinterpret_cast<const float2*>(p.part_ml + (row + x) * 2) : make_float2(-INFINITY, 0.f);
          const float* src = p.part_o + (row + x) * D + lane * VL;
          if constexpr (VL == 4) {
            const float4 f = in ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[e][x][0] = f.x;
            v[e][x][1] = f.y;
            v[e][x][2] = f.z;
            v[e][x][3] = f.w;
          } else {
            const float2 f = in ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
            v[e][x][0] = f.x;
            v[e][x][1] = f.y;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < ROWS8; ++x) {
        const float top = fmaxf(m[x], fmaxf(ml[0][x].x, ml[1][x].x)), base = top == -INFINITY ? 0.f : top;
        const float keep = exp2f_approx(m[x] - base), w0 = exp2f_approx(ml[0][x].x - base), w1 = exp2f_approx(ml[1][x].x - base);
        m[x] = top;
        l[x] = fmaf(ml[1][x].y, w1, fmaf(ml[0][x].y, w0, l[x] * keep));
#pragma unroll
        for (int k = 0; k < VL; ++k) acc[x][k] = fmaf(v[1][x][k], w1, fmaf(v[0][x][k], w0, acc[x][k] * keep));
      }
    }
#pragma unroll
    for (int x = 0; x < ROWS8; ++x) {
      if (x >= rows) break;
      const int R = b.z + r + x, token = R / p.G;
      const float inv = l[x] == 0.f ? 0.f : 1.0f / l[x];
      T* dst = static_cast<T*>(p.O) + (a.w + token) * p.o_st + (b.y * p.G + R - token * p.G) * p.o_sh + lane * VL;
#pragma unroll
      for (int k = 0; k < VL; k += 2) {
        const float f[2] = {acc[x][k] * inv, acc[x][k + 1] * inv};
        reinterpret_cast<uint32_t*>(dst)[k / 2] = Words<T>::pack(f);
      }
    }
  }
}

// Two parts per block, each 256 rows of D sums and (m, l), and eight ints per block.
size_t tiles_workspace(int64_t D, int blocks) { return static_cast<size_t>(blocks) * (2 * 2 * TM * (D + 2) * 4 + 32); }

template <typename T, int D>
int launch_tiles(CachedParams& p, int64_t items, const CUtensorMap& tmK, const CUtensorMap& tmV, void* workspace, cudaStream_t stream) {
  constexpr int SMEM = sizeof(TilesSmem<D>) + 1024;
  static_assert(SMEM <= 227 * 1024, "a block does not fit an SM's shared memory");
  const int blocks = sm_count();
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<size_t>(blocks) * 2 * 2 * TM * D;
  p.meta = reinterpret_cast<int*>(p.part_ml + static_cast<size_t>(blocks) * 2 * 2 * TM * 2);
  // Whole items take as many rounds as the fullest SM has items; ranges of key blocks fill all SMs alike, at a block's cost 1.4
  // times as high (no two SMs then work on the same keys at a time) and a tenth of a round for the join.  Whole items are not
  // dealt quite evenly under a causal mask (the fullest SM of 2048 has 258 blocks, the average 228), so the calls compare at 1.25.
  // Measured: 2048 items 810 whole, 1012 us in ranges; 512 items 128, 183; 128 items 88, 110; 160 items 323, 332; 32 items 636, 197.
  // `items` is what B requests of max_new rows would have: an upper bound, so a call with one long chunk among single tokens
  // is dealt whole although it has fewer.
  const int64_t rounds = (items + blocks - 1) / blocks;
  p.whole_items = static_cast<double>(rounds) <= 1.25 * static_cast<double>(items) / blocks + 0.1;
  static std::atomic<uint64_t> done{0};
  int rc = once_per_device(done, []() {
    const cudaError_t e = cudaFuncSetAttribute(cached_tiles_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(cached_tiles_join_kernel<T, D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  });
  if (rc) return rc;
  if (blocks > MAX_TEAMS) return fail(KCG_ERR_UNSUPPORTED, "fmha_cached: a device of %d SMs", blocks);
  cached_tiles_kernel<T, D><<<blocks, TILES_THREADS, SMEM, stream>>>(tmK, tmV, p, make_idesc(0, 0, 0, 0, TM, BN), make_idesc(0, 0, 0, 1, TM, D));
  rc = check_launch("cached_tiles_kernel");
  if (rc || p.whole_items) return rc;
  launch_overlapped(cached_tiles_join_kernel<T, D>, dim3(4 * blocks), dim3(JWARPS * 32), 0, stream, p, blocks);
  return check_launch("cached_tiles_join_kernel");
}

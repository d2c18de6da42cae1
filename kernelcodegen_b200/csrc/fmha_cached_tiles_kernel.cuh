// Attention over the paged 8-bit cache for many query rows per request (included by fmha_cached.cu inside its anonymous
// namespace).  Here the two matrix products are the cost, so they run on tcgen05 with 128-row tiles:
//
//   An item is a pair of 128-row tiles of one (request, key / value head): rows are (token, query head of the group) in
//   token-major order, so a block of 128 keys is loaded and converted once for 256 rows, whatever the group.
//   warps 0-3, 4-7  softmax of tile 0 / 1, one thread per row (scores, P and O in tensor memory); before that, the row
//                   of Q, as f16 scaled by a power of two, into the swizzled tile the products read; afterwards, O out
//   warp 8          one thread issues the products: S_i = Q_i K^T, O_i += P_i V, S_i(j + 1) right behind P_i V(j)
//   warp 9          looks pages up and loads the codes of K and V by TMA (boxes of 16 or 32 rows of a page)
//   warps 12-15     turn codes into f16 tiles in the swizzled layout tcgen05 wants (the same for K and V)
// tcgen05 multiplies f16 with f16 or e4m3 with e4m3, not one with the other, and P in e4m3 would keep four bits; so the
// codes are widened on the way.  Scales: a page's is 2^e f with f in [1, 2).  The power of two, relative to the block's
// largest (K) or the item's largest so far (V), is multiplied into the codes, exactly down to f16's smallest step (a
// page would have to lie 2^20 below to lose a bit that counts); the references go into the softmax constant and the
// output.  Where some f is not 1 (scales this library did not write) the softmax multiplies the scores of a page's 16-key
// groups with it, and V is multiplied with it, rounding once more, to f16.
// Tensor memory (512 columns): S0, S1, O0, O1; P_i overwrites the first half of S_i.
#pragma once

constexpr int TM = 128;                 // rows of a tile
constexpr int TN = 128;                 // keys of a block
constexpr int TILES_THREADS = 512;
constexpr int TILES_REGS_SOFTMAX = 200, TILES_REGS_OTHER = 56;
static_assert(2 * 128 * (TILES_REGS_SOFTMAX + TILES_REGS_OTHER) <= TILES_THREADS * 128, "register split exceeds the block's allocation");
constexpr int RECORDS = 8;

// What the loader says about a key block.
struct BlockRecord {
  float kref;                           // scores are to be multiplied with this
  float vshift;                         // what the output so far is to be multiplied with (V's reference has grown)
  float vref;                           // V's reference
  int plain;                            // every group's page is there, every f of K is 1
  uint32_t rk[8], rv[8];                // per group of 16 keys: what its codes are multiplied with, two f16
  float fk[8], fv[8];                   // f
  uint32_t gone;                        // groups whose page is not in the pool: their keys are left out
};

template <int D> struct TilesSmem {
  static constexpr int DB = D / 64;
  static constexpr int TILE = DB * 16384;               // bytes of a 128 x D f16 tile: DB blocks of 128 rows x 128 bytes
  uint8_t q[2][TILE], k[2][TILE], v[2][TILE];
  uint8_t raw[2][TN * D];                               // codes of K, V
  BlockRecord rec[RECORDS];
  uint64_t raw_full[2], raw_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], rec_full[RECORDS];
  uint64_t q_full, s_full[2], p_full[4], o_full[2], drain;
  int item[8];                                          // t0, n, len, head, pair, go
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ uint32_t f16x2_pow2(int e) {   // 2^e twice, e <= 0, 0 below f16's smallest step
  const uint32_t h = e >= -14 ? static_cast<uint32_t>(e + 15) << 10 : (e >= -24 ? 1u << (e + 24) : 0u);
  return h | (h << 16);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Items of a request; the longest (under a causal mask the last rows) come first.
__device__ __forceinline__ int64_t request_items(const CachedParams& p, const Request& r) {
  return static_cast<int64_t>(p.Hkv) * ((r.n * p.G + 2 * TM - 1) / (2 * TM));
}

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
      mbar_init(&sm.raw_empty[s], 4);
      mbar_init(&sm.k_full[s], 4);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], 4);
      mbar_init(&sm.v_empty[s], 1);
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.o_full[s], 1);
      mbar_init(&sm.p_full[2 * s], 4);
      mbar_init(&sm.p_full[2 * s + 1], 4);
    }
    for (int s = 0; s < RECORDS; ++s) mbar_init(&sm.rec_full[s], 1);
    mbar_init(&sm.q_full, 8);
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

  // Items are dealt round-robin.  All warps meet before and behind an item (every wait in between is bounded, so every
  // warp gets there); the loader's first thread walks the requests.
  auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(TILES_THREADS) : "memory"); };
  int64_t left = blockIdx.x;              // items between the walk's place and this block's next item
  int walk_i = 0;
  auto find_item = [&]() {
    bool go = false;
    Request r{0, 0, 0};
    for (; walk_i < p.B; ++walk_i) {
      r = request_of(p, walk_i);
      const int64_t n = request_items(p, r);
      if (left < n) {
        go = true;
        break;
      }
      left -= n;
    }
    sm.item[5] = go;
    if (go) {
      const int pairs = (r.n * p.G + 2 * TM - 1) / (2 * TM);
      const int idx = static_cast<int>(left);
      sm.item[0] = r.t0;
      sm.item[1] = r.n;
      sm.item[2] = r.len;
      sm.item[3] = idx / pairs;
      sm.item[4] = pairs - 1 - idx % pairs;
      sm.item[6] = walk_i;
      left += gridDim.x;
    }
  };
  uint32_t blocks = 0;                    // key blocks done before this item (phases of the rings and records)
  struct Item {
    int t0, n, len, head, row0, req, rows, n0, n1, nmax;
  };
  auto begin_item = [&](Item& it) {
    meet();
    if (!sm.item[5] || *abort_flag) return false;
    it.t0 = sm.item[0];
    it.n = sm.item[1];
    it.len = sm.item[2];
    it.head = sm.item[3];
    it.row0 = sm.item[4] * 2 * TM;
    it.req = sm.item[6];
    it.rows = it.n * p.G;
    // key blocks of the two tiles: up to the last key their last row sees
    auto blocks_of = [&](int first) {
      const int last = min(first + TM, it.rows) - 1;
      if (last < first) return 0;
      const int end = p.causal ? min(it.len, it.len - it.n + 1 + last / p.G) : it.len;
      return end > 0 ? (end + TN - 1) / TN : 0;
    };
    it.n0 = blocks_of(it.row0);
    it.n1 = blocks_of(it.row0 + TM);
    it.nmax = max(it.n0, it.n1);
    return true;
  };

    if (warp < 8) {
      // ------------------------------------------------------------------ softmax
      reg_alloc<TILES_REGS_SOFTMAX>();
      uint32_t cs = 0, cf = 0;              // score tiles and outputs of this tile so far
      Item it;
      while (begin_item(it)) {
      const int t0 = it.t0, n = it.n, len = it.len, head = it.head, row0 = it.row0, rows = it.rows;
      const int i = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
      const int R = row0 + i * TM + r;
      const bool live = R < rows;
      const int j_row = live ? R / p.G : 0;
      const int64_t q_at = (t0 + j_row) * p.q_st + (head * p.G + (live ? R - j_row * p.G : 0)) * p.q_sh;
      float c = fabsf(p.scale_log2);
      {
        // this thread's row of Q: in two passes, largest magnitude, then f16
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.Q) + q_at);
        float up = p.scale_log2 < 0.f ? -1.f : 1.f;      // the softmax's constant is not negative
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          uint32_t m = 0;
          if (live)
#pragma unroll
            for (int k = 0; k < D / 8; ++k) {
              const uint4 x = __ldg(src + k);
              m = __vmaxu2(__vmaxu2(__vmaxu2(__vmaxu2(m, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu), x.z & 0x7fff7fffu), x.w & 0x7fff7fffu);
            }
          m = max(m & 0xffffu, m >> 16);
          int e = static_cast<int>(m >> 7) - 127 - 13;
          e = e < -113 ? -113 : e;
          up *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          c *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        }
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          const uint4 x = live ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f[2];
            Words<T>::unpack(w[e], f);
            h[e] = pack_f16(f[0] * up, f[1] * up);
          }
          *reinterpret_cast<uint4*>(sm.q[i] + (k >> 3) * 16384 + r * 128 + (((k & 7) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full);
      }
      const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t s_addr = tmem + lane_base + i * TN, o_addr = tmem + lane_base + 256 + i * TM;
      const int n_mine = i == 0 ? it.n0 : it.n1;
      const int end = live ? (p.causal ? min(len, len - n + 1 + j_row) : len) : 0;   // keys this row sees
      float m = -INFINITY, l = 0.f, vref = 1.f;
      bool ok = true;
      for (int j = 0; j < n_mine; ++j, ++cs) {
        const BlockRecord& rec = sm.rec[(blocks + j) % RECORDS];
        if (!mbar_wait(&sm.rec_full[(blocks + j) % RECORDS], ((blocks + j) / RECORDS) & 1u, abort_flag) ||
            !mbar_wait(&sm.s_full[i], cs & 1u, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float cj = c * rec.kref;
        const bool plain = rec.plain != 0;
        const float vshift = rec.vshift;
        vref = rec.vref;
        if (__any_sync(0xffffffffu, !plain || cj == 0.f)) {
          // scores that a block-wide constant does not serve are put right in place, in pieces that leave registers alone
#pragma unroll 1
          for (int cc = 0; cc < TN / 32; ++cc) {
            uint32_t x[32];
            tmem_ld32(s_addr + cc * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float f = cj == 0.f ? 0.f : rec.fk[2 * cc + (k >> 4)];
              x[k] = (rec.gone >> (2 * cc + (k >> 4))) & 1u ? 0xff800000u : __float_as_uint(__uint_as_float(x[k]) * f);
            }
            tmem_st32(s_addr + cc * 32, x);
          }
          tmem_wait_st();
          if (cj == 0.f) cj = 1.f;                       // (-inf times 0 is not -inf)
        }
        uint32_t s[TN];
        tmem_ld64(s_addr, reinterpret_cast<uint32_t(&)[64]>(s[0]));
        tmem_ld64(s_addr + 64, reinterpret_cast<uint32_t(&)[64]>(s[64]));
        tmem_wait_ld();
        const int limit = end - j * TN;
        if (limit < TN) {
#pragma unroll
          for (int k = 0; k < TN; ++k)
            if (k >= limit) s[k] = 0xff800000u;
        }
        float mx[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) mx[a] = fmaxf(__uint_as_float(s[2 * a]), __uint_as_float(s[2 * a + 1]));
#pragma unroll
        for (int k = 16; k < TN; k += 16)
#pragma unroll
          for (int a = 0; a < 8; ++a) mx[a] = max3f(mx[a], __uint_as_float(s[k + 2 * a]), __uint_as_float(s[k + 2 * a + 1]));
        const float top = max3f(max3f(mx[0], mx[1], mx[2]), max3f(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
        const float mt = top * cj;
        float alpha = 1.f;
        if (mt > m + kLazy) {
          alpha = exp2f_approx(m - mt);                  // 0 for the first keys
          m = mt;
        }
        // the scores being complete means that P V of the block before is, too: O may be changed
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f || vshift != 1.f)) {
          const float a = alpha * vshift;
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t x[32];
            tmem_ld32(o_addr + cc * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * a);
            tmem_st32(o_addr + cc * 32, x);
          }
          tmem_wait_st();
        }
        const float base = m == -INFINITY ? 0.f : m;
        const uint64_t c2 = pk_make(cj, cj), nb2 = pk_make(-base, -base);
        uint64_t sum_a = 0ull, sum_b = 0ull;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int k = half * 64; k < half * 64 + 64; k += 2) {
            float x0, x1;
            pk_split(pk_fma(pk_make(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), c2, nb2), x0, x1);
            float p0 = exp2f_approx(x0), p1 = exp2f_approx(x1);
            if ((k >> 1) & 1) sum_b = pk_add(sum_b, pk_make(p0, p1));
            else sum_a = pk_add(sum_a, pk_make(p0, p1));
            s[k >> 1] = pack_f16(p0, p1);                // word k / 2 is not read again
          }
          tmem_st32(s_addr + half * 32, reinterpret_cast<uint32_t(&)[32]>(s[half * 32]));
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[2 * i + half]);
        }
        float l0, l1;
        pk_split(pk_add(sum_a, sum_b), l0, l1);
        l = l * alpha + (l0 + l1);
      }
      if (ok && n_mine > 0) {
        ok = mbar_wait(&sm.o_full[i], cf & 1u, abort_flag);
        ++cf;
        tc_fence_after();
      }
      if (!ok) give_up();
      if (ok) {
        const float inv = l == 0.f ? 0.f : vref / l;     // a row that sees no key is zero
        T* dst = static_cast<T*>(p.O) + (t0 + j_row) * p.o_st + (head * p.G + (live ? R - j_row * p.G : 0)) * p.o_sh;
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t x[32];
          if (n_mine > 0) {
            tmem_ld32(o_addr + cc * 32, x);
            tmem_wait_ld();
          }
          if (live) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float f[2] = {l == 0.f ? 0.f : __uint_as_float(x[k + 2 * e]) * inv, l == 0.f ? 0.f : __uint_as_float(x[k + 2 * e + 1]) * inv};
                w[e] = Words<T>::pack(f);
              }
              *reinterpret_cast<uint4*>(dst + cc * 32 + k) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        tc_fence_before();
      }
      blocks += it.nmax;
      meet();
      }
    } else if (warp == 8) {
      // ------------------------------------------------------------------ products
      reg_dealloc<TILES_REGS_OTHER>();
      uint32_t items = 0, cp0 = 0, cp1 = 0; // items, P blocks of the tiles so far
      Item it;
      while (begin_item(it)) {
      const int n0 = it.n0, n1 = it.n1, nmax = it.nmax;
      if (lane == 0) {
        bool ok = mbar_wait(&sm.q_full, items & 1u, abort_flag);
        ++items;
        const uint64_t qd = make_smem_desc(smem_u32(sm.q[0]), 16, 1024), kd = make_smem_desc(smem_u32(sm.k[0]), 16, 1024);
        const uint64_t vd = make_smem_desc(smem_u32(sm.v[0]), 16384, 1024);
        auto scores = [&](int i, uint32_t slot) {
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss<Kind::F16>(tmem + i * TN, qd + ((i * TILE + d * 16384 + k * 32) >> 4), kd + ((slot * TILE + d * 16384 + k * 32) >> 4),
                                idesc_qk, (d | k) != 0 ? 1u : 0u);
          mma_commit(&sm.s_full[i]);
        };
        auto output = [&](int i, int half, uint32_t slot, uint32_t first) {
#pragma unroll
          for (int k = 4 * half; k < 4 * half + 4; ++k)
            mma_ts_f16(tmem + 256 + i * TM, tmem + i * TN + k * 8, vd + ((slot * TILE + k * 2048) >> 4), idesc_pv, (first | k) != 0 ? 1u : 0u);
        };
        if (ok && nmax > 0) {
          ok = mbar_wait(&sm.k_full[blocks & 1u], (blocks >> 1) & 1u, abort_flag);
          tc_fence_after();
          if (ok) {
            if (n0 > 0) scores(0, blocks & 1u);
            if (n1 > 0) scores(1, blocks & 1u);
            mma_commit(&sm.k_empty[blocks & 1u]);
          }
        }
        for (int j = 0; j < nmax && ok; ++j) {
          const uint32_t b = blocks + j, slot = b & 1u, next = (b + 1) & 1u;
          ok = mbar_wait(&sm.v_full[slot], (b >> 1) & 1u, abort_flag);
          bool k_ready = false;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n_i = i == 0 ? n0 : n1;
            if (!ok || j >= n_i) continue;
            uint32_t& cp = i == 0 ? cp0 : cp1;
            if (!mbar_wait(&sm.p_full[2 * i], cp & 1u, abort_flag)) { ok = false; break; }
            tc_fence_after();
            output(i, 0, slot, j);
            if (!mbar_wait(&sm.p_full[2 * i + 1], cp & 1u, abort_flag)) { ok = false; break; }
            tc_fence_after();
            output(i, 1, slot, j);
            ++cp;
            if (j + 1 < n_i) {
              if (!k_ready && !mbar_wait(&sm.k_full[next], ((b + 1) >> 1) & 1u, abort_flag)) { ok = false; break; }
              k_ready = true;
              tc_fence_after();
              scores(i, next);
            } else {
              mma_commit(&sm.o_full[i]);
            }
          }
          if (!ok) break;
          mma_commit(&sm.v_empty[slot]);
          if (j + 1 < nmax) mma_commit(&sm.k_empty[next]);
        }
        if (!ok) {
          give_up();
          int zero = 0;
          mma_commit(&sm.drain);          // what was issued must end before the block does
          mbar_wait(&sm.drain, 0, &zero, 20000000ull);
        }
      }
      __syncwarp();
      blocks += it.nmax;
      meet();
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------------ pages and codes
      // lane g < 8 looks after the block's keys 16 g .. 16 g + 15; the next block's page and scales are asked for
      // before this one's ring entries are waited for
      reg_dealloc<TILES_REGS_OTHER>();
      if (lane == 0) find_item();
      Item it;
      while (begin_item(it)) {
      const int len = it.len, head = it.head, nmax = it.nmax, req = it.req;
      int pid = -1, row = 0;
      float ks = 0.f, vs = 0.f;
      auto look_up = [&](int j) {
        const int key = j * TN + 16 * lane;
        pid = -1;
        ks = vs = 0.f;
        if (lane < 8 && j < nmax && key < len) {
          const int w = key / p.page;
          row = key - w * p.page;
          pid = p.table[req * p.table_stride + w];
          if (pid < 0 || pid >= p.num_pages) {
            pid = -2;
            if (p.status) *p.status = KCG_ERR_INVALID_ARG;
          } else {
            ks = p.ks[static_cast<int64_t>(pid) * p.Hkv + head];
            vs = p.vs[static_cast<int64_t>(pid) * p.Hkv + head];
          }
        }
      };
      look_up(0);
      int vexp = -1000;
      bool ok = true;
      for (int j = 0; j < nmax && ok; ++j) {
        const uint32_t b = blocks + j;
        const int page = pid, at = row;
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
        const int ek = there ? exponent(ks) : -1000, ev = there ? exponent(vs) : -1000;
        const int kmax = __reduce_max_sync(0xffffffffu, ek), vmax = __reduce_max_sync(0xffffffffu, ev);
        const int kref = kmax == -1000 ? 0 : kmax, vold = vexp;
        vexp = max(vexp, vmax);
        const int vnow = vexp == -1000 ? 0 : vexp;
        const float fk = there ? rest(ks, ek, kref) : 1.f, fv = there ? rest(vs, ev, vnow) : 1.f;
        const uint32_t gone = __ballot_sync(0xffffffffu, page == -2);
        const bool all_plain = __all_sync(0xffffffffu, page != -2 && fk == 1.f);
        look_up(j + 1);
        ok = mbar_wait(&sm.raw_empty[0], (b & 1u) ^ 1u, abort_flag);
        BlockRecord& rec = sm.rec[b % RECORDS];
        if (lane < 8) {
          rec.rk[lane] = f16x2_pow2(ek == -1000 ? 0 : ek - kref);
          rec.rv[lane] = f16x2_pow2(ev == -1000 ? 0 : ev - vnow);
          rec.fk[lane] = fk;
          rec.fv[lane] = fv;
        }
        if (lane == 0) {
          rec.kref = pow2f(kref);
          rec.vref = pow2f(vnow);
          rec.vshift = j == 0 || vold == vexp ? 1.f : (vold == -1000 ? pow2f(-vexp) : pow2f(vold - vexp));
          rec.plain = all_plain;
          rec.gone = gone;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.rec_full[b % RECORDS]);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          if (side == 1) ok = ok && mbar_wait(&sm.raw_empty[1], (b & 1u) ^ 1u, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          const bool issue = there && lane < 8 && (p.box == 16 || (lane & 1) == 0);
          const uint32_t bytes = __reduce_add_sync(0xffffffffu, issue ? p.box * D : 0);
          if (lane == 0) mbar_expect_tx(&sm.raw_full[side], bytes);
          __syncwarp();
          if (issue) tma_load_4d(sm.raw[side] + lane * 16 * D, side ? &tmV : &tmK, &sm.raw_full[side], 0, at, head, page);
        }
      }
      if (!ok) {
        give_up();
        int zero = 0;
        for (int s = 0; s < 2; ++s) mbar_wait(&sm.raw_full[s], blocks & 1u, &zero, 2000000ull);
      }
      __syncwarp();
      blocks += nmax;
      meet();                               // (the item's description is not read any more)
      if (lane == 0) find_item();
      }
    } else if (warp >= 12) {
      // ------------------------------------------------------------------ codes to f16
      reg_dealloc<TILES_REGS_OTHER>();
      Item it;
      while (begin_item(it)) {
      const int len = it.len, nmax = it.nmax;
      const int ct = tid - 384;
      constexpr int CPR = D / 16;           // 16-code chunks of a row
      bool ok = true;
      for (int j = 0; j < nmax && ok; ++j) {
        const uint32_t b = blocks + j, slot = b & 1u;
        const BlockRecord& rec = sm.rec[b % RECORDS];
        const int have = len - j * TN;      // rows behind the last token become zero
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          uint64_t* empty = side ? &sm.v_empty[slot] : &sm.k_empty[slot];
          if (side == 0) ok = mbar_wait(&sm.rec_full[b % RECORDS], (b / RECORDS) & 1u, abort_flag);
          ok = ok && mbar_wait(&sm.raw_full[side], b & 1u, abort_flag) && mbar_wait(empty, ((b >> 1) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          const uint8_t* raw = sm.raw[side];
          uint8_t* tile = side ? sm.v[slot] : sm.k[slot];
          const uint32_t* ratio = side ? rec.rv : rec.rk;
          const uint32_t gone = rec.gone;
#pragma unroll 4
          for (int it = 0; it < TN * CPR / 128; ++it) {
            const int idx = it * 128 + ct, r = idx / CPR, ch = idx % CPR;
            uint32_t w[4], h[8];
            lds128(smem_u32(raw) + tile_offset<D>(r, ch), w);
            const uint32_t f = ratio[r >> 4];
            const bool nothing = r >= have || ((gone >> (r >> 4)) & 1u);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              e4m3x4_to_f16(w[x], h[2 * x], h[2 * x + 1]);
              h[2 * x] = hmul2(h[2 * x], f);
              h[2 * x + 1] = hmul2(h[2 * x + 1], f);
            }
            if (side == 1 && rec.fv[r >> 4] != 1.f) {
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[x]));
                h[x] = pack_f16(v.x * rec.fv[r >> 4], v.y * rec.fv[r >> 4]);
              }
            }
            if (nothing) {                  // (the bytes may be anything)
#pragma unroll
              for (int x = 0; x < 8; ++x) h[x] = 0u;
            }
            // chunks 2 c, 2 c + 1 of the row's 128-byte line in block ch / 4; the lines of the two blocks share banks, so
            // the second block's are written in the other order
            uint8_t* line = tile + (ch >> 2) * 16384 + r * 128;
            const int swap = D == 128 ? ch >> 2 : 0, c0 = 2 * (ch & 3) + swap, c1 = 2 * (ch & 3) + 1 - swap;
            const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
            *reinterpret_cast<uint4*>(line + ((c0 ^ (r & 7)) << 4)) = swap ? hi : lo;
            *reinterpret_cast<uint4*>(line + ((c1 ^ (r & 7)) << 4)) = swap ? lo : hi;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sm.raw_empty[side]);
            mbar_arrive(side ? &sm.v_full[slot] : &sm.k_full[slot]);
          }
        }
      }
      if (!ok) give_up();
      __syncwarp();
      blocks += it.nmax;
      meet();
      }
    } else {
      reg_dealloc<TILES_REGS_OTHER>();      // warps 10, 11
      Item it;
      while (begin_item(it)) meet();
    }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D>
int launch_tiles(const CachedParams& p, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t stream) {
  constexpr int SMEM = sizeof(TilesSmem<D>) + 1024;
  static_assert(SMEM <= 227 * 1024, "a block does not fit an SM's shared memory");
  auto kern = cached_tiles_kernel<T, D>;
  KCG_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  kern<<<sm_count(), TILES_THREADS, SMEM, stream>>>(tmK, tmV, p, make_idesc(0, 0, 0, 0, TM, TN), make_idesc(0, 0, 0, 1, TM, D));
  return check_launch("cached_tiles_kernel");
}

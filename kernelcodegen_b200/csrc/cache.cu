// Paged 8-bit key / value cache: planning a step's pages and slots, and writing keys and values.
//
// The cache is a pool of pages of `page_size` tokens.  A page holds, for every key / value head,
// page_size rows of D e4m3 codes and one fp32 scale; a stored value is code * scale.  Request i
// owns the pages its row of the block table lists, in order; token p of the request lives in page
// table[i][p / page_size] at offset p % page_size, and its "slot" is page * page_size + offset.
//
// Nothing like it exists in the reference, whose attention reads dense tensors of one length
// (src/Optimizer/Optimizer.cc:2606-2860).
#include "common.cuh"

namespace kcg {

int* device_status_word();

namespace {

// ---- planning -------------------------------------------------------------------------------------
// With c_i cached and n_i new tokens, pages of P tokens:
//   have_i = ceil(c_i / P), need_i = ceil((c_i + n_i) / P) - have_i,
//   E_i = need_0 + .. + need_i, C_i = n_0 + .. + n_i,
// request i takes entries F-1-(E_i - need_i) downwards of the free list (a stack of F pages), and
// token t of the step belongs to the request with C_{i-1} <= t < C_i.
//
// The work is a prefix sum over the requests and one store per token; it is bound by latency, not by
// bytes.  Every thread block computes the whole prefix sum into its shared memory (a few loads per
// thread) and then fills its own share of the tokens and requests, so a step is one launch and no
// block waits for another.
// 64 requests of one token each, or 500 with 292379 tokens: 16 us a call from Python, most of it on the host.
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 16384;   // 12 bytes of shared memory each
constexpr int kPlanTokensPerBlock = 2048; // 4 tokens per thread

struct PlanParams {
  const int32_t* cached;
  const int32_t* fresh;      // new tokens per request
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lengths;
  int32_t* cu_new;
  int64_t* slots;
  int32_t* free_left;
  int64_t table_stride, width, free_cap, max_tokens;
  int B, page;
  int what;                  // 1: table and slots, 2: lengths, cu_new and free_left, 3: both
  int* status;
};

__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const PlanParams p) {
  extern __shared__ int32_t plan_smem[];
  int32_t* s_stop = plan_smem;            // C_i, cut at max_tokens
  int32_t* s_base = s_stop + p.B;         // E_i - need_i of a served request, -1 of a refused one
  int32_t* s_cached = s_base + p.B;
  __shared__ int64_t s_part[2][kPlanThreads / 32];
  __shared__ int64_t s_carry[2];
  __shared__ int s_taken, s_bad;
  grid_launch_dependents();
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t F = *p.free_count;
  bool bad_free = F < 0 || F > p.free_cap;
  F = F < 0 ? 0 : (F > p.free_cap ? p.free_cap : F);
  if (tid == 0) { s_carry[0] = 0; s_carry[1] = 0; s_taken = 0; s_bad = bad_free; }
  __syncthreads();

  for (int i0 = 0; i0 < p.B; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t need = 0, toks = 0;
    int c = 0;
    bool bad = true;
    if (i < p.B) {
      c = p.cached[i];
      const int n = p.fresh[i];
      const int64_t total = static_cast<int64_t>(c) + n;
      bad = c < 0 || n < 0 || total > p.width * p.page || total > INT32_MAX;
      if (c < 0 || n < 0) s_bad = 1;
      toks = n > 0 ? n : 0;
      if (!bad) need = (total + p.page - 1) / p.page - (static_cast<int64_t>(c) + p.page - 1) / p.page;
    }
    int64_t a = need, b = toks;           // inclusive prefix sums over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) { a += ua; b += ub; }
    }
    if (lane == 31) { s_part[0][warp] = a; s_part[1][warp] = b; }
    __syncthreads();
    int64_t pa = s_carry[0], pb = s_carry[1];
    for (int w = 0; w < warp; ++w) { pa += s_part[0][w]; pb += s_part[1][w]; }
    a += pa;
    b += pb;
    if (i < p.B) {
      const bool served = !bad && b <= p.max_tokens && (need == 0 || a <= F);
      s_stop[i] = static_cast<int32_t>(b < p.max_tokens ? b : p.max_tokens);
      // (a refused request may stand behind sums that do not fit 32 bits; they are not stored)
      s_base[i] = served ? static_cast<int32_t>(need ? a - need : 0) : -1;
      s_cached[i] = c;
      if (served && need > 0) atomicMax(&s_taken, static_cast<int>(a));
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) { s_carry[0] = a; s_carry[1] = b; }
    __syncthreads();
  }

  // (every read of `cached`, `fresh` and `free_count` is behind the barriers above, so in a launch of
  // one block `lengths` may be `cached` and `free_left` may be `free_count`)
  if (p.what & 1) {
    const int64_t t_end = p.B ? s_stop[p.B - 1] : 0;
    // new pages into the table: one warp per request
    for (int i = blockIdx.x * (kPlanThreads / 32) + warp; i < p.B; i += gridDim.x * (kPlanThreads / 32)) {
      const int base = s_base[i];
      if (base < 0) continue;
      const int c = s_cached[i];
      const int n = s_stop[i] - (i ? s_stop[i - 1] : 0);   // served: not cut
      const int have = static_cast<int>((static_cast<int64_t>(c) + p.page - 1) / p.page);
      const int need = static_cast<int>((static_cast<int64_t>(c) + n + p.page - 1) / p.page) - have;
      for (int k = lane; k < need; k += 32) p.table[i * p.table_stride + have + k] = p.free_pages[F - 1 - base - k];
    }
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid; t < p.max_tokens;
         t += static_cast<int64_t>(gridDim.x) * kPlanThreads) {
      int64_t slot = -1;
      if (t < t_end) {
        int lo = 0, hi = p.B - 1;          // first request whose tokens end behind t
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (s_stop[mid] > t) hi = mid; else lo = mid + 1;
        }
        const int base = s_base[lo], c = s_cached[lo];
        if (base >= 0) {
          const int pos = c + static_cast<int>(t - (lo ? s_stop[lo - 1] : 0));
          const int pi = pos / p.page, have = static_cast<int>((static_cast<int64_t>(c) + p.page - 1) / p.page);
          // a page the request already had, or one of those it has just been given
          const int page = pi < have ? p.table[lo * p.table_stride + pi] : p.free_pages[F - 1 - base - (pi - have)];
          slot = page < 0 ? -1 : static_cast<int64_t>(page) * p.page + (pos - pi * p.page);
        }
      }
      p.slots[t] = slot;
    }
  }
  if ((p.what & 2) && blockIdx.x == 0) {
    for (int i = tid; i < p.B; i += kPlanThreads) {
      const int n = s_stop[i] - (i ? s_stop[i - 1] : 0);
      p.lengths[i] = s_base[i] < 0 ? s_cached[i] : s_cached[i] + n;
      p.cu_new[i + 1] = s_stop[i];
    }
    if (tid == 0) {
      p.cu_new[0] = 0;
      *p.free_left = static_cast<int32_t>(F) - s_taken;
      if (s_bad && p.status) *p.status = KCG_ERR_INVALID_ARG;
    }
  }
}

// ---- appending ------------------------------------------------------------------------------------
// Neighbouring tokens of one page in ascending slots, with fewer than 32 skipped tokens between two of
// them, form a run.  A run of one head of K or V is written by one warp, or by the four of a block where it has more rows
// than a warp holds.  With amax the largest finite magnitude of the run,
//   s = 2^k, the smallest power of two with amax / s <= 448 (e4m3's largest value), k >= -110;
// a run that does not begin at its page's first row keeps max(s, old scale), and the rows before it are
// rounded again when the scale has grown.  The scale is a power of two because e4m3 has an exponent of
// its own: a finer scale would gain no significant bit, and x / s, code * s and a change of scale are
// then exact, so that the only rounding is the one to e4m3's four significant bits.
//
// Bound by memory: each 16-bit element is read once and leaves as one byte.  A run stays in registers between
// finding amax and rounding (up to kVecs 16-byte vectors per lane: 64 rows of D = 128 in a block), with all
// of its loads in flight at once; longer runs are read twice.  8 prompts of 4096 tokens, 8 heads of 128: 51 us, 0.60 of the
// copy rate (one warp per run with 32 vectors per lane left six warps on an SM: 83 us).  What is left: slots, old scale and rows
// are three trips to memory that nothing overlaps within a block, five blocks of four warps are in flight on an SM, the 96
// registers of a thread spill about 50 words of the 16-bit kernels, and warps wait at barriers, for the one that finds the runs
// and for each other's maxima.  37 chunks of 419 tokens on average, 5 heads of 64: 28 us, where each of the ten blocks that
// share the heads finds the same runs again and 39 % of a warp's time is spent at barriers.
constexpr int kVecs = 8;
constexpr int kAppendWarps = 4;

struct AppendSide {
  const void* x;          // [T, Hkv, D]
  int64_t st, sh;         // element strides of x
  uint8_t* cache;
  int64_t cp, ch, ct;     // page, head and row strides of the cache
  float* scale;           // [pages, Hkv]
};
struct AppendParams {
  AppendSide side[2];     // K, V
  const int64_t* slots;
  int64_t T, slot_end;    // slots are in [0, slot_end)
  int heads, page, chunk; // chunk: tokens one block looks at
  int per;                // of the 2 * heads sides and heads, what one block writes
  int* status;
};

// Largest magnitude of the values of a word as an unsigned integer that orders like the magnitude.
template <typename T> __device__ __forceinline__ uint32_t mag_max(uint32_t m, uint32_t w) {
  if constexpr (sizeof(T) == 4) return max(m, w & 0x7fffffffu);
  else return __vmaxu2(m, w & 0x7fff7fffu);
}
template <typename T> struct MagInf;
template <> struct MagInf<float> { static constexpr uint32_t v = 0x7f800000u; };
template <> struct MagInf<__nv_bfloat16> { static constexpr uint32_t v = 0x7f80u; };
template <> struct MagInf<__half> { static constexpr uint32_t v = 0x7c00u; };

template <typename T> __device__ __forceinline__ float mag_to_float(uint32_t m) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(m);
  else {
    float f[2];
    Words<T>::unpack(m & 0xffffu, f);
    return f[0];
  }
}

// Exponent k of the scale for a finite amax (1.75 * 2^8 = 448).
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int k = static_cast<int>(b >> 23) - 127 - ((b & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return k < -110 ? -110 : k;
}
__device__ __forceinline__ float exp2i(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// The codes of one 16-byte vector.  kSpecial: infinities become NaN (e4m3 has none); without it every
// value is known to be finite.  Magnitudes are at most 448 after scaling, so nothing saturates.
template <typename T, bool kSpecial>
__device__ __forceinline__ void encode(const uint4& v, float inv, uint32_t (&code)[4 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float f[16 / sizeof(T)];
  constexpr int EPW = Words<T>::EPW;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float u[EPW];
    Words<T>::unpack(w[i], u);
#pragma unroll
    for (int e = 0; e < EPW; ++e) f[i * EPW + e] = kSpecial ? fmaf(u[e], inv, u[e] - u[e]) : u[e] * inv;
  }
#pragma unroll
  for (int i = 0; i < static_cast<int>(4 / sizeof(T)); ++i)
    code[i] = to_e4m3x2(f[4 * i], f[4 * i + 1]) | (to_e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16);
}

// A page's first `off` rows, from scale `old` to `scale`: `parts` warps, this one is `part`.
template <int D>
__device__ __forceinline__ void round_again(uint8_t* rows, int64_t stride, int off, float old, float scale, int lane, int part, int parts) {
  const float ratio = old / scale;
  for (int r = part * (128 / D) + lane / (D / 4); r < off; r += parts * (128 / D)) {
    uint32_t* q = reinterpret_cast<uint32_t*>(rows + r * stride) + lane % (D / 4);
    const uint32_t w = *q;
    uint32_t o = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * k)), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      o |= to_e4m3x2(f.x * ratio, f.y * ratio) << (16 * k);
    }
    *q = o;
  }
}
template <int CW> __device__ __forceinline__ void store_codes(uint8_t* q, const uint32_t (&code)[CW]) {
  if constexpr (CW == 2) *reinterpret_cast<uint2*>(q) = make_uint2(code[0], code[1]);
  else *reinterpret_cast<uint32_t*>(q) = code[0];
}

// What a run is: a block finds it once for all heads.
struct Run {
  int64_t slot0, page;    // of the page
  int at, n, off, dense;  // first token in the block's chunk, tokens, first row; dense: token r goes to row off + r
};

// The rare run, by one warp and a vector at a time: tokens are left out, or there are infinities or NaN.
template <typename T, int D>
__device__ __forceinline__ void append_odd(const AppendSide& a, int head, int heads, const int64_t* slots, int64_t t0, const Run& run, int page_size, int lane) {
  constexpr int VE = 16 / sizeof(T), VR = D / VE, RPI = 32 / VR, CW = 4 / sizeof(T);
  const int col = lane % VR;
  const T* x = static_cast<const T*>(a.x) + t0 * a.st + head * a.sh + col * VE;
  uint8_t* rows = a.cache + run.page * a.cp + head * a.ch;
  float* sp = a.scale + run.page * heads + head;
  const float old = run.off ? *sp : 0.f;
  float amax = 0.f;
  for (int r = lane / VR; r < run.n; r += RPI) {
    const int64_t s = slots[r] - run.slot0;
    if (s < 0 || s >= page_size) continue;
    for (int e = 0; e < VE; ++e) {
      const float f = fabsf(Conv<T>::to_f(x[r * a.st + e]));
      if (f < INFINITY) amax = fmaxf(amax, f);
    }
  }
  const float scale = fmaxf(exp2i(scale_exponent(warp_max(amax))), old), inv = 1.0f / scale;
  if (run.off && scale != old) round_again<D>(rows, a.ct, run.off, old, scale, lane, 0, 1);
  for (int r = lane / VR; r < run.n; r += RPI) {
    const int64_t s = slots[r] - run.slot0;
    if (s < 0 || s >= page_size) continue;
    uint32_t code[CW];
    encode<T, true>(*reinterpret_cast<const uint4*>(x + r * a.st), inv, code);
    store_codes<CW>(rows + s * a.ct + col * VE, code);
  }
  if (lane == 0) *sp = scale;
}

// A dense run; kParts warps (this one is `part`) share it.  False: it has values that are not finite, and nothing was written.
template <typename T, int D, int kParts>
__device__ __forceinline__ bool append_run(const AppendSide& a, int head, int heads, int64_t t0, const Run& run, int lane, int part,
                                           uint32_t* s_max) {
  constexpr int VE = 16 / sizeof(T);        // elements of a vector
  constexpr int VR = D / VE;                // vectors of a row
  constexpr int RPI = 32 / VR;              // rows one warp instruction covers
  constexpr int CAP = kVecs * RPI * kParts; // rows held in registers
  constexpr int CW = 4 / sizeof(T);         // words of codes per vector
  const int first = part * RPI + lane / VR, col = lane % VR, n = run.n;
  const T* x = static_cast<const T*>(a.x) + (t0 + first) * a.st + head * a.sh + col * VE;
  const int64_t x_step = a.st * (RPI * kParts), out_step = a.ct * (RPI * kParts);
  uint8_t* rows = a.cache + run.page * a.cp + head * a.ch;
  float* sp = a.scale + run.page * heads + head;
  const float old = run.off ? *sp : 0.f;    // a run at a page's first row: the page is new
  uint4 v[kVecs];
  auto load = [&](int base) {
    const T* at = x + base * a.st;
#pragma unroll
    for (int i = 0; i < kVecs; ++i, at += x_step)
      v[i] = base + first + i * RPI * kParts < n ? __ldcs(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
  };
  uint32_t mag = 0;
  for (int base = 0; base < n; base += CAP) {
    load(base);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) mag = mag_max<T>(mag_max<T>(mag_max<T>(mag_max<T>(mag, v[i].x), v[i].y), v[i].z), v[i].w);
  }
  if (sizeof(T) == 2) mag = max(mag & 0xffffu, mag >> 16);
  mag = __reduce_max_sync(0xffffffffu, mag);
  if (kParts > 1) {
    __syncthreads();                        // the values of the run before have been read
    if (lane == 0) s_max[part] = mag;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kParts; ++w) mag = max(mag, s_max[w]);
  }
  if (mag >= MagInf<T>::v) return false;    // (the same answer in all of the run's warps)
  const float scale = fmaxf(exp2i(scale_exponent(mag_to_float<T>(mag))), old);
  if (run.off && scale != old) round_again<D>(rows, a.ct, run.off, old, scale, lane, part, kParts);
  const float inv = 1.0f / scale;           // a power of two, unless the caller's own scale is kept
  uint8_t* out = rows + (run.off + first) * a.ct + col * VE;
  for (int base = 0; base < n; base += CAP) {
    if (n > CAP) load(base);
    uint8_t* at = out + base * a.ct;
#pragma unroll
    for (int i = 0; i < kVecs; ++i, at += out_step) {
      uint32_t code[CW];
      encode<T, false>(v[i], inv, code);
      if (base + first + i * RPI * kParts < n) store_codes<CW>(at, code);
    }
  }
  if (lane == 0 && part == 0 && (!run.off || scale != old)) *sp = scale;
  return true;
}

// Finding the runs costs more than a head's share of a short run, so one warp finds a block's and the block writes them for
// several heads.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kAppendWarps, 5) cache_append_kernel(const AppendParams p) {
  grid_launch_dependents();
  grid_dependency_wait();
  __shared__ Run s_run[32];
  __shared__ int s_runs;
  __shared__ uint32_t s_max[kAppendWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.chunk;
  const int count = static_cast<int>(min(static_cast<int64_t>(p.chunk), p.T - t0));   // <= 32
  if (warp == 0) {
    auto in_pool = [&](int64_t s) { return s >= 0 && s < p.slot_end; };
    auto page_of = [&](int64_t s) -> int64_t {   // (a 64-bit division is several times a 32-bit one)
      return p.slot_end <= UINT32_MAX ? static_cast<int64_t>(static_cast<uint32_t>(s) / static_cast<uint32_t>(p.page)) : s / p.page;
    };
    int64_t slot = -1, before = -1;
    if (lane < count) {
      slot = p.slots[t0 + lane];
      if (!in_pool(slot) && slot != -1 && p.status) *p.status = KCG_ERR_INVALID_ARG;
    }
    const bool valid = in_pool(slot);
    if (valid)                              // the last token before this one that is not skipped
      for (int64_t k = t0 + lane - 1; k >= 0 && k > t0 + lane - 33 && !in_pool(before); --k) before = p.slots[k];
    const int64_t page = valid ? page_of(slot) : -1;
    const bool first = valid && !(in_pool(before) && before < slot && page_of(before) == page);   // of a run
    int runs = 0;
    for (uint32_t left = __ballot_sync(0xffffffffu, first); left; left &= left - 1, ++runs) {
      const int at = __ffs(left) - 1;
      const int64_t s0 = __shfl_sync(0xffffffffu, slot, at), page0 = __shfl_sync(0xffffffffu, page, at);
      const int64_t slot0 = page0 * p.page, tr = t0 + at;
      // the run's last token, looking 32 tokens on from the last one found
      int n = 1, found = 1;
      int64_t s_last = s0;
      for (bool more = true; more;) {
        const int64_t k = tr + n + lane;
        const int64_t s = k < p.T ? p.slots[k] : -1;
        const bool in = in_pool(s);
        const uint32_t others = __ballot_sync(0xffffffffu, in && !(s > s0 && s < slot0 + p.page));
        uint32_t ours = __ballot_sync(0xffffffffu, in && s > s0 && s < slot0 + p.page);
        if (others) ours &= (1u << (__ffs(others) - 1)) - 1;
        more = ours != 0 && others == 0 && n < p.T;
        if (ours) {
          const int top = 31 - __clz(ours);
          s_last = __shfl_sync(0xffffffffu, s, top);
          found += __popc(ours);
          n += top + 1;
        }
      }
      // ascending slots of one page: nothing is left out when they span as many as they are
      if (lane == 0) s_run[runs] = Run{slot0, page0, at, n, static_cast<int>(s0 - slot0), found == n && s_last == s0 + n - 1};
    }
    if (lane == 0) s_runs = runs;
  }
  __syncthreads();
  const int runs = s_runs, h0 = blockIdx.y * p.per, mine = min(p.per, 2 * p.heads - h0);
  constexpr int ALONE = kVecs * 32 / (D * static_cast<int>(sizeof(T)) / 16);   // rows one warp holds
  int turn = 0;
  for (int k = 0; k < runs; ++k) {
    const Run& r = s_run[k];
    for (int h = h0; h < h0 + mine; ++h) {
      const AppendSide& a = p.side[h >= p.heads];
      const int head = h >= p.heads ? h - p.heads : h;
      const int64_t* slots = p.slots + t0 + r.at;
      // a long run is the whole block's, short ones are dealt to the warps in turn
      bool written = false, mine_too = warp == 0;
      if (r.dense && r.n > ALONE) {
        written = append_run<T, D, kAppendWarps>(a, head, p.heads, t0 + r.at, r, lane, warp, s_max);
      } else {
        mine_too = turn++ % kAppendWarps == warp;
        if (mine_too && r.dense) written = append_run<T, D, 1>(a, head, p.heads, t0 + r.at, r, lane, 0, s_max);
      }
      if (!written && mine_too) append_odd<T, D>(a, head, p.heads, slots, t0 + r.at, r, p.page, lane);
    }
  }
}

template <typename T>
int launch_append(const AppendParams& p, int64_t D, cudaStream_t stream) {
  const int64_t blocks = (p.T + p.chunk - 1) / p.chunk;
  const int64_t shares = (2 * p.heads + p.per - 1) / p.per;
  if (blocks > INT32_MAX || shares > 65535) return fail(KCG_ERR_UNSUPPORTED, "cache_append: too many tokens or heads");
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(shares)), block(32 * kAppendWarps);
  if (D == 128) launch_overlapped(cache_append_kernel<T, 128>, grid, block, 0, stream, p);
  else launch_overlapped(cache_append_kernel<T, 64>, grid, block, 0, stream, p);
  return check_launch("cache_append_kernel");
}

}  // namespace
}  // namespace kcg

extern "C" int kcg_cache_plan(int64_t requests, int64_t page_size, int64_t max_tokens, const int32_t* cached,
                              const int32_t* fresh, int32_t* block_table, int64_t table_width, int64_t table_stride,
                              const int32_t* free_pages, int64_t free_capacity, const int32_t* free_count,
                              int32_t* lengths, int32_t* cu_new, int64_t* slot_map, int32_t* free_left, void* stream) {
  using namespace kcg;
  clear_error();
  if (requests < 0 || max_tokens < 0 || table_width < 0 || free_capacity < 0)
    return fail(KCG_ERR_INVALID_ARG, "cache_plan: negative size");
  if (page_size < 1 || page_size > 65536) return fail(KCG_ERR_INVALID_ARG, "cache_plan: page_size %lld", static_cast<long long>(page_size));
  if (table_stride < table_width) return fail(KCG_ERR_INVALID_ARG, "cache_plan: the rows of the block table overlap");
  if (requests > kPlanMaxRequests)
    return fail(KCG_ERR_UNSUPPORTED, "cache_plan: at most %d requests (got %lld)", kPlanMaxRequests, static_cast<long long>(requests));
  if (max_tokens > INT32_MAX || table_width > INT32_MAX || free_capacity > INT32_MAX)
    return fail(KCG_ERR_UNSUPPORTED, "cache_plan: sizes beyond 2^31 - 1");
  if (!cu_new || !free_count || !free_left || (max_tokens && !slot_map) || (free_capacity && !free_pages) ||
      (requests && (!cached || !fresh || !lengths || (table_width && !block_table))))
    return fail(KCG_ERR_INVALID_ARG, "cache_plan: null pointer");
  PlanParams p{cached, fresh, block_table, free_pages, free_count, lengths, cu_new, slot_map, free_left,
               table_stride, table_width, free_capacity, max_tokens, static_cast<int>(requests),
               static_cast<int>(page_size), 3, device_status_word()};
  const size_t smem = static_cast<size_t>(requests) * 12;
  if (smem > 48 * 1024)
    KCG_CUDA_OK(cudaFuncSetAttribute(cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanMaxRequests * 12));
  int64_t blocks = (max_tokens + kPlanTokensPerBlock - 1) / kPlanTokensPerBlock;
  const int sms = sm_count();
  blocks = blocks < 1 ? 1 : (blocks > sms ? sms : blocks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Updating in place: with several blocks, `lengths` and `free_left` are written by a second launch, once
  // every block of the first has read what they overwrite.
  auto touch = [](const int32_t* a, int64_t na, const int32_t* b, int64_t nb) { return a < b + nb && b < a + na; };
  auto over_input = [&](const int32_t* o, int64_t n) {
    return touch(o, n, cached, requests) || touch(o, n, fresh, requests) || touch(o, n, free_count, 1);
  };
  const bool in_place = over_input(lengths, requests) || over_input(cu_new, requests + 1) || over_input(free_left, 1);
  if (in_place && blocks > 1) {
    p.what = 1;
    launch_overlapped(cache_plan_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kPlanThreads), smem, s, p);
    const int rc = check_launch("cache_plan_kernel");
    if (rc) return rc;
    p.what = 2;
    blocks = 1;
  }
  launch_overlapped(cache_plan_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kPlanThreads), smem, s, p);
  return check_launch("cache_plan_kernel");
}

extern "C" int kcg_cache_append(int dtype, int64_t T, int64_t Hkv, int64_t D, const void* K, const int64_t k_strides[2],
                                const void* V, const int64_t v_strides[2], const int64_t* slot_map, int64_t num_pages,
                                int64_t page_size, void* k_cache, const int64_t kc_strides[3], void* v_cache,
                                const int64_t vc_strides[3], float* k_scale, float* v_scale, void* stream) {
  using namespace kcg;
  clear_error();
  if (T < 0 || Hkv < 0 || D < 0 || num_pages < 0) return fail(KCG_ERR_INVALID_ARG, "cache_append: negative size");
  if (page_size < 16 || page_size % 16 || page_size > 65536)
    return fail(KCG_ERR_INVALID_ARG, "cache_append: page_size %lld is not a multiple of 16 up to 65536", static_cast<long long>(page_size));
  if (T == 0 || Hkv == 0) return KCG_OK;
  if (D != 64 && D != 128) return fail(KCG_ERR_UNSUPPORTED, "cache_append: head dimension %lld has no kernel (64, 128)", static_cast<long long>(D));
  if (!K || !V || !k_strides || !v_strides || !slot_map || !k_cache || !v_cache || !kc_strides || !vc_strides || !k_scale || !v_scale)
    return fail(KCG_ERR_INVALID_ARG, "cache_append: null pointer");
  if (num_pages > INT32_MAX || Hkv > 32767) return fail(KCG_ERR_UNSUPPORTED, "cache_append: too many pages or heads");
  const size_t es = kcg_dtype_size(dtype);
  if (dtype != KCG_BF16 && dtype != KCG_F16 && dtype != KCG_F32)
    return fail(KCG_ERR_UNSUPPORTED, "cache_append: dtype %d has no kernel (float32, bfloat16, float16)", dtype);
  bool ok = aligned16(K) && aligned16(V) && aligned16(k_cache) && aligned16(v_cache);
  for (int i = 0; i < 2; ++i) ok = ok && (k_strides[i] * es) % 16 == 0 && (v_strides[i] * es) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && kc_strides[i] % 16 == 0 && vc_strides[i] % 16 == 0;
  if (!ok) return fail(KCG_ERR_ALIGNMENT, "cache_append: rows of K, V and the caches must start on 16-byte boundaries");
  AppendParams p;
  p.side[0] = {K, k_strides[0], k_strides[1], static_cast<uint8_t*>(k_cache), kc_strides[0], kc_strides[1], kc_strides[2], k_scale};
  p.side[1] = {V, v_strides[0], v_strides[1], static_cast<uint8_t*>(v_cache), vc_strides[0], vc_strides[1], vc_strides[2], v_scale};
  p.slots = slot_map;
  p.T = T;
  p.slot_end = num_pages * page_size;
  p.heads = static_cast<int>(Hkv);
  p.page = static_cast<int>(page_size);
  // Blocks enough to fill the GPU a few times over: first tokens are put together (a block looks at up to 32), then heads.
  const int64_t blocks = static_cast<int64_t>(sm_count()) * 32;
  const int64_t chunk = (T * 2 * Hkv + blocks - 1) / blocks;
  p.chunk = static_cast<int>(chunk > 32 ? 32 : chunk);
  const int64_t per = (T + p.chunk - 1) / p.chunk * 2 * Hkv / blocks;
  p.per = static_cast<int>(per < 1 ? 1 : (per > 2 * Hkv ? 2 * Hkv : per));
  p.status = device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KCG_F32: return launch_append<float>(p, D, s);
    case KCG_BF16: return launch_append<__nv_bfloat16>(p, D, s);
    default: return launch_append<__half>(p, D, s);
  }
}

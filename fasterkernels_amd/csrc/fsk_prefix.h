// fsk_prefix.h -- paged decode of a batch whose sequences share their first
// pages: the shared tokens' attention, once for all sequences.  Part of
// fsk_decode.hip's translation unit (included once, inside its anonymous
// namespace, before run_decode).
//
// Over the shared tokens every sequence's query heads meet the same keys, so for
// one KV head they are a matrix of M = B G query rows (row b G + g: sequence b,
// head g of the KV head's G) against one K and V, and the decode's
// matrix-vector products become matrix products: K and V are read once per
// M-tile instead of once per sequence.  Softmax over shared and own tokens is
// the log-sum-exp merge of the two parts, which the reduce kernel does with the
// prefix's partials beside each sequence's own.

struct PrefixParams {
  const uint8_t* q;
  int64_t q_sb, q_sh;                     // bytes
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_sp, k_sh, k_st;               // bytes
  int64_t v_sp, v_sh, v_st;
  const int32_t* pages;                   // the shared pages (the first sequence's table row)
  FastDiv page;                           // divisor page_size
  int num_pages;
  const int32_t* lens;                    // [B] whole lengths
  int max_len;                            // ... clamped to [0, max_len]
  int32_t* own_lens;                      // [B] out: tokens past the prefix
  const float* k_scale;
  const float* v_scale;
  float score_scale;                      // sm_scale * log2(e)
  int B, G, Hkv, rows;                    // rows: M = B G
  FastDiv g_div, hkv_div, rt_div;         // divisors G, Hkv, row tiles
  int tokens, tiles, chunk;               // shared tokens, their tiles, tiles of a work item
  int units;                              // (chunk, KV head) pairs
  float* part_ml;                         // [chunks, Hkv, M, 2]
  float* part_acc;                        // [chunks, Hkv, M, D]
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4_w;

template <bool kBf16>
__device__ __forceinline__ f32x16 mfma32x32x16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The other half-wave's value (lane l ^ 32) folded in.
__device__ __forceinline__ float half_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(a[0]), u2f(a[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return u2f(a[0]) + u2f(a[1]);
}

// (Kept out of the templates, as lds_dma16 is.)
__device__ __forceinline__ u32x2 lds_read_tr16(uint32_t off) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)off));
}

// Tile geometry.  K and V tiles of kTile tokens lie in LDS as 16-bit rows (e4m3
// codes are widened on the way in: both widenings are exact), each row's
// 16-byte chunks in an order that spreads the operand reads over the banks.
template <int D>
struct PrefixTile {
  static constexpr int kTile = D <= 128 ? 64 : 32;
  static constexpr int kRow = 2 * D;             // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPlane = kTile * kRow;    // one tile of K or V
  static constexpr int kHalves = kTile / 16;     // 16-token pieces, each inside one page
  static constexpr int kBlocks = kTile / 32;     // 32-token score blocks
};
// V chunk m of row R is stored at m ^ v_swizzle(R): the transposing reads take
// 8 consecutive rows x 64 bytes, which land on all banks twice (512 bytes over
// 64 banks of 4).
template <int kChunks>
__device__ __forceinline__ int v_swizzle(int row) {
  return kChunks >= 16 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
}

// One work item: kWaves x 32 query rows of one KV head against `chunk` tiles.
//
// Lane l = 32 h + c.  S^T = K Q^T per 32 tokens (v_mfma_f32_32x32x16: A = K rows,
// B = query columns): lane (h, c) gets the scores of query c with tokens
// 8 (i / 4) + 4 h + i % 4, i = 0..15.  O^T += V^T P^T: k-slot e of half h is
// given token 16 s + 4 h + e (e < 4) or 16 s + 4 h + 4 + e, which is where the
// score block left P, so P needs no movement; V^T comes from LDS through the
// transposing read (16 lanes read 4 token rows of 16 dims, lane i gets dim i).
template <int D, bool kQBf16, bool kVBf16, bool kFp8, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void prefix_kernel(PrefixParams p) {
  using T = PrefixTile<D>;
  constexpr int kSteps = D / 16;    // QK k-steps
  constexpr int kDb = D / 32;       // output blocks of 32 dims
  constexpr int kPv = T::kTile / 16;  // PV k-steps
  extern __shared__ __attribute__((aligned(16))) uint8_t s_prefix[];  // [2 buffers][K, V]
  const uint32_t lds = (uint32_t)(uintptr_t)s_prefix;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = uniform((int)threadIdx.x / kWave);
  const int h = lane >> 5, c = lane & 31;

  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < p.B; b += 64 * kWaves) p.own_lens[b] = max(clampi(p.lens[b], 0, p.max_len) - p.tokens, 0);
  }
  // Row tiles of one (chunk, head) on one XCD, one after the other: they read
  // the same K and V through its L2.
  const uint32_t xcd = blockIdx.x & 7, in_xcd = blockIdx.x >> 3;
  const uint32_t group = fdiv(in_xcd, p.rt_div);
  const int rt = (int)(in_xcd - group * p.rt_div.d);
  const uint32_t unit = group * 8 + xcd;
  if (unit >= (uint32_t)p.units) return;
  const int jc = (int)fdiv(unit, p.hkv_div);
  const int kvh = (int)unit - jc * p.Hkv;
  const int tile0 = jc * p.chunk, tile1 = min(tile0 + p.chunk, p.tiles);

  // ---- this lane's query column
  const int row0 = (rt * kWaves + wave) * 32;
  const bool live = row0 < p.rows;                // any column of the wave is a query row
  const int row = min(row0 + c, p.rows - 1);
  const bool row_ok = row0 + c < p.rows;
  const int b = (int)fdiv((uint32_t)row, p.g_div);
  const int lim = row_ok ? min(clampi(p.lens[b], 0, p.max_len), p.tokens) : p.tokens;  // shared tokens it attends
  u32x4 qop[kSteps];
  {
    const uint8_t* qrow = p.q + (int64_t)b * p.q_sb + (int64_t)(kvh * p.G + (row - b * p.G)) * p.q_sh;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const u32x4 x = *(const u32x4*)(qrow + 32 * i + 16 * h);
      qop[i] = row_ok ? x : u32x4{0, 0, 0, 0};
    }
  }
  const float sscale = p.score_scale * (kFp8 ? *p.k_scale : 1.0f);
  int lim_min = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lim_min = min(lim_min, __shfl_xor(lim_min, o));
  lim_min = uniform(lim_min);

  // ---- staging: 16-token pieces dealt to the waves.  Pages of the next 64
  // pieces in one register (lane i: piece base + i).
  const uint8_t* kbase = p.k + (int64_t)kvh * p.k_sh;
  const uint8_t* vbase = p.v + (int64_t)kvh * p.v_sh;
  int win = 0, win_base = -64;
  auto piece_at = [&](int piece, int64_t& ko, int64_t& vo, bool& ok) {  // byte offsets of a piece's first rows
    if (piece - win_base >= 64) {  // (pieces come in order)
      win_base = piece;
      const int t = 16 * (piece + lane);
      win = t < p.tokens ? clampi(p.pages[fdiv((uint32_t)t, p.page)], 0, p.num_pages - 1) : 0;
    }
    const int t = 16 * piece;
    ok = t < p.tokens;
    const int page = __builtin_amdgcn_readlane(win, piece - win_base);
    const int off = t - (int)fdiv((uint32_t)t, p.page) * (int)p.page.d;
    ko = (int64_t)page * p.k_sp + (int64_t)off * p.k_st;
    vo = (int64_t)page * p.v_sp + (int64_t)off * p.v_st;
  };
  constexpr int kPieces = (T::kHalves + kWaves - 1) / kWaves;  // of this wave, per tile
  // 16-bit: DMA, 1 KB (64 / kChunks rows) a load.  e4m3: 16 codes a lane and load,
  // 1 KB = 1024 / D rows, kept in registers until the buffer is free.
  constexpr int kDma = 16 * T::kRow / 1024;
  constexpr int kCodeLoads = 16 * D / 1024 > 0 ? 16 * D / 1024 : 1;
  u32x4 codes[kFp8 ? 2 * kPieces * kCodeLoads : 1];
  int k_off[kDma], v_off[kDma];
  if constexpr (!kFp8) {
#pragma unroll
    for (int r = 0; r < kDma; ++r) {
      const int R = r * (64 / T::kChunks) + lane / T::kChunks;
      const int m = lane % T::kChunks;
      k_off[r] = R * (int)p.k_st + 16 * (m ^ k_swizzle<T::kChunks>(R));
      v_off[r] = R * (int)p.v_st + 16 * (m ^ v_swizzle<T::kChunks>(R));
    }
  }
  auto load = [&](int tile, uint32_t buf) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int hp = wave + i * kWaves;  // piece of the tile
      if (T::kHalves % kWaves != 0 && hp >= T::kHalves) break;
      int64_t ko, vo;
      bool ok;
      piece_at(tile * T::kHalves + hp, ko, vo, ok);
      // (pieces past the prefix read as zeros)
      const auto rk = make_rsrc(kbase + ko, ok ? 15 * (int)p.k_st + (kFp8 ? D : 2 * D) : 0);
      const auto rv = make_rsrc(vbase + vo, ok ? 15 * (int)p.v_st + (kFp8 ? D : 2 * D) : 0);
      if constexpr (!kFp8) {
#pragma unroll
        for (int r = 0; r < kDma; ++r) {
          lds_dma16(rk, buf + hp * 16 * T::kRow + r * 1024, k_off[r]);
          lds_dma16(rv, buf + T::kPlane + hp * 16 * T::kRow + r * 1024, v_off[r]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < kCodeLoads; ++r) {
          const int R = r * (1024 / D) + lane * 16 / D, d0 = lane * 16 % D;
          const auto x = buf_load<16>(rk, R * (int)p.k_st + d0), y = buf_load<16>(rv, R * (int)p.v_st + d0);
          codes[2 * (i * kCodeLoads + r)] = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
          codes[2 * (i * kCodeLoads + r) + 1] = u32x4{y.w[0], y.w[1], y.w[2], y.w[3]};
        }
      }
    }
  };
  // e4m3: the loaded codes, widened, into the buffer.
  auto store = [&](uint32_t buf) {
    if constexpr (kFp8) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int hp = wave + i * kWaves;
        if (T::kHalves % kWaves != 0 && hp >= T::kHalves) break;
#pragma unroll
        for (int r = 0; r < kCodeLoads; ++r) {
          const int R = r * (1024 / D) + lane * 16 / D, m = lane * 16 % D / 8;
          const u32x4 kc = codes[2 * (i * kCodeLoads + r)], vc = codes[2 * (i * kCodeLoads + r) + 1];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x2 k0 = e4m3x4_to<kQBf16>(kc[2 * e]), k1 = e4m3x4_to<kQBf16>(kc[2 * e + 1]);
            const u32x2 v0 = e4m3x4_to<kVBf16>(vc[2 * e]), v1 = e4m3x4_to<kVBf16>(vc[2 * e + 1]);
            const uint32_t at = buf + (hp * 16 + R) * T::kRow;
            *(lds_u32x4_w*)(uintptr_t)(at + 16 * ((m + e) ^ k_swizzle<T::kChunks>(R))) = u32x4{k0[0], k0[1], k1[0], k1[1]};
            *(lds_u32x4_w*)(uintptr_t)(at + T::kPlane + 16 * ((m + e) ^ v_swizzle<T::kChunks>(R))) =
                u32x4{v0[0], v0[1], v1[0], v1[1]};
          }
        }
      }
    }
  };

  // ---- operand addresses: XOR with a constant picks the chunk
  const uint32_t k_lane = c * T::kRow + 16 * (h ^ k_swizzle<T::kChunks>(c));
  const int vj = lane & 15, vr = 4 * h + vj / 4;
  const uint32_t v_lane = T::kPlane + vr * T::kRow +
                          16 * ((2 * (c >> 4) + (vj & 3) / 2) ^ v_swizzle<T::kChunks>(vr)) + 8 * (vj & 1);

  float m_ref = -INFINITY, l_run = 0.f;
  f32x16 acc[kDb];
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

  auto compute = [&](int tile, uint32_t buf) {
    const int t0 = tile * T::kTile;
    // scores, log2 domain
    f32x16 s[T::kBlocks];
#pragma unroll
    for (int tb = 0; tb < T::kBlocks; ++tb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[tb][i] = 0.f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const u32x4 kop = *(lds_u32x4*)(uintptr_t)(buf + tb * 32 * T::kRow + (k_lane ^ (32 * i)));
        s[tb] = mfma32x32x16<kQBf16>(kop, qop[i], s[tb]);
      }
    }
#pragma unroll
    for (int tb = 0; tb < T::kBlocks; ++tb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[tb][i] *= sscale;
    if (t0 + T::kTile > lim_min) {
#pragma unroll
      for (int tb = 0; tb < T::kBlocks; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t0 + 32 * tb + 8 * (i / 4) + 4 * h + i % 4 >= lim) s[tb][i] = -INFINITY;
    }
    float mt = s[0][0];
#pragma unroll
    for (int tb = 0; tb < T::kBlocks; ++tb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[tb][i]);
    mt = half_max(mt);
    // The exponentials are taken relative to m_ref, which follows the running
    // maximum only when that has grown by more than 2^8: the sums stay in fp32
    // and P below 2^8 keeps its relative precision in 16 bits, while the
    // rescaling of the accumulators is left out of nearly every tile.
    if (__builtin_amdgcn_ballot_w64(mt > m_ref + 8.f) != 0) {
      const float m_new = fmaxf(m_ref, mt);
      const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_ref - m_new);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
      m_ref = m_new;
    }
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
    // P^T operands; bf16 P as hi + lo parts, as in the split kernel
    u32x4 pop[kPv], plo[kVBf16 ? kPv : 1];
#pragma unroll
    for (int st = 0; st < kPv; ++st) {
      float pv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pv[e] = __builtin_amdgcn_exp2f(s[st / 2][8 * (st & 1) + e] - m_use);
        l_run += pv[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kVBf16) {
          const uint32_t hi = pack_bf16x2(pv[2 * e], pv[2 * e + 1]);
          pop[st][e] = hi;
          plo[st][e] = pack_bf16x2(pv[2 * e] - bf16_lo_to_f32(hi), pv[2 * e + 1] - bf16_hi_to_f32(hi));
        } else {
          pop[st][e] = pack_f16x2(pv[2 * e], pv[2 * e + 1]);
        }
      }
    }
    auto v_operand = [&](int st, int d) {
      const uint32_t at = buf + st * 16 * T::kRow + (v_lane ^ (64 * d));
      const u32x2 lo = lds_read_tr16(at), hi = lds_read_tr16(at + 8 * T::kRow);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    if (lim_min >= min(t0 + T::kTile, p.tokens)) {
#pragma unroll
      for (int st = 0; st < kPv; ++st)
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
          const u32x4 vop = v_operand(st, d);
          acc[d] = mfma32x32x16<kVBf16>(vop, pop[st], acc[d]);
          if constexpr (kVBf16) acc[d] = mfma32x32x16<true>(vop, plo[st], acc[d]);
        }
    } else {
      // Columns that end inside the prefix: V rows past a column's end may hold
      // anything, and 0 x inf is NaN, so the tile is multiplied once per
      // different end, with V's rows zeroed past it, and only the columns of
      // that end take the sum.
      uint64_t todo = __builtin_amdgcn_ballot_w64(lim > t0);
      while (todo) {
        const int end = __builtin_amdgcn_readlane(lim, __builtin_ctzll(todo));
        const bool mine = lim == end;
        todo &= ~__builtin_amdgcn_ballot_w64(mine);
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
          f32x16 sum;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll
          for (int st = 0; st < kPv; ++st) {
            u32x4 vop = v_operand(st, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dword e: tokens t, t + 1
              const int t = t0 + 16 * st + 4 * h + 8 * (e >> 1) + 2 * (e & 1);
              const uint32_t keep = (t < end ? 0xffffu : 0u) | (t + 1 < end ? 0xffff0000u : 0u);
              vop[e] &= keep;
            }
            sum = mfma32x32x16<kVBf16>(vop, pop[st], sum);
            if constexpr (kVBf16) sum = mfma32x32x16<true>(vop, plo[st], sum);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] += mine ? sum[i] : 0.f;
        }
      }
    }
  };

  // ---- tiles: while one is computed, the next one's loads are in flight.  One
  // barrier a tile: past it every wave's part of the tile is in LDS, and every
  // wave has done with the other buffer.
  load(tile0, lds);
  store(lds);
  for (int tile = tile0; tile < tile1; ++tile) {
    const uint32_t cur = lds + (uint32_t)((tile - tile0) & 1) * (2 * T::kPlane);
    const uint32_t nxt = lds + (uint32_t)((tile - tile0 + 1) & 1) * (2 * T::kPlane);
    __builtin_amdgcn_s_waitcnt(vm_wait_imm(0));  // (the compiler does not see the DMA's LDS writes)
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tile + 1 < tile1) load(tile + 1, nxt);
    if (live) compute(tile, cur);
    if (tile + 1 < tile1) store(nxt);
  }

  // ---- partials
  const float v_scale = kFp8 ? *p.v_scale : 1.0f;
  const float l_tot = half_sum(l_run);
  if (row_ok) {
    const int64_t idx = ((int64_t)jc * p.Hkv + kvh) * p.rows + row;
    float* dst = p.part_acc + idx * D + 4 * h;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f32x4*)(dst + 32 * d + 8 * i) = f32x4{acc[d][4 * i] * v_scale, acc[d][4 * i + 1] * v_scale,
                                                acc[d][4 * i + 2] * v_scale, acc[d][4 * i + 3] * v_scale};
    if (h == 0) *(f32x2*)(p.part_ml + 2 * idx) = f32x2{m_ref, l_tot};
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// The prefix's work split: waves of a workgroup, row tiles, tiles of an item and
// items per KV head (chunks).
struct PrefixPlan {
  int waves, row_tiles, tiles, chunk, chunks;
};
PrefixPlan plan_prefix(int64_t rows, int Hkv, int D, int64_t tokens, int cus) {
  PrefixPlan pl;
  pl.waves = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  pl.row_tiles = (int)cdiv(rows, 32 * pl.waves);
  pl.tiles = (int)cdiv(tokens, D <= 128 ? 64 : 32);
  // workgroups that fit the chip at once: by LDS two of 64 KB a CU (head_dim 64: four of 32 KB)
  const int64_t slots = (int64_t)cus * (D == 64 ? 4 : 2);
  const int64_t want = std::max<int64_t>(1, slots / ((int64_t)Hkv * pl.row_tiles));
  pl.chunk = (int)cdiv(pl.tiles, std::min<int64_t>(want, pl.tiles));
  pl.chunks = (int)cdiv(pl.tiles, pl.chunk);
  return pl;
}

// The prefix partials that a decode's reduce kernel takes in.
struct SharedParts {
  const float* ml;
  const float* acc;
  int n;
};

template <int D, bool kQBf16, bool kVBf16, bool kFp8>
int launch_prefix_waves(const PrefixParams& p, int waves, unsigned grid, const Launch& s) {
  using T = PrefixTile<D>;
  constexpr uint32_t lds = 4 * T::kPlane;
  auto go = [&](auto kernel) {
    launch(kernel, dim3(grid), dim3(64 * waves), lds, s, p);
    return FSK_OK;
  };
  if (waves == 1) return go(prefix_kernel<D, kQBf16, kVBf16, kFp8, 1>);
  if (waves == 2) return go(prefix_kernel<D, kQBf16, kVBf16, kFp8, 2>);
  return go(prefix_kernel<D, kQBf16, kVBf16, kFp8, 4>);
}
template <int D>
int launch_prefix(const PrefixParams& p, int q_dt, int kv_dt, int waves, unsigned grid, const Launch& s) {
  if (kv_dt == FSK_F16) return launch_prefix_waves<D, false, false, false>(p, waves, grid, s);
  if (kv_dt == FSK_BF16) return launch_prefix_waves<D, true, true, false>(p, waves, grid, s);
  if (q_dt == FSK_F16) return launch_prefix_waves<D, false, false, true>(p, waves, grid, s);
  return launch_prefix_waves<D, true, false, true>(p, waves, grid, s);
}

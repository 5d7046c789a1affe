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
//
// Work: 4 M Hkv D flops a shared token against 2 Hkv D elements of K and V, so the
// matrix cores bound long prefixes of wide batches and HBM the others.  Kernel /
// whole call, us (the floor is the larger of the bytes at a copy's 4.9 TB/s and the
// flops at a large product's 1.28 PF): 32 heads on 8 x 128, 32 sequences with 8192
// shared bf16 tokens and 16 to 1024 own 28 / 34 (floor 18, bytes); 64 on 32768 e4m3
// 57 / 62 (27, flops: 0.6 PF); 256 on 4096 f16 44 / 50 (33, bytes: 3.7 TB/s).  As
// many single sequences (paged_flash_decode) these take 112, 601 and 303.  What a
// prefix costs beyond its products is the serial part of each tile (barrier, first
// operand reads, widening) and the ends of the kernel (work plan and first loads 4,
// partials 6): without the softmax the second takes 56, with operands that are read
// once 59, with K and V from the caches no less.

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
  const float* k_scale;
  const float* v_scale;
  float score_scale;                      // sm_scale * log2(e)
  int B, G, Hkv, rows;                    // rows: M = B G
  FastDiv g_div, hkv_div, rt_div;         // divisors G, Hkv, row tiles
  int tokens, tiles, chunk;               // shared tokens, their tiles, tiles of a work item
  int blocks;                             // workgroups of the prefix
  int units;                              // (chunk, KV head) pairs
  float* part_ml;                         // [chunks, Hkv, M, 2]
  float* part_acc;                        // [chunks, Hkv, M, D]
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4_w;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

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

// Tile geometry.  K and V tiles of 64 tokens lie in LDS as 16-bit rows (e4m3
// codes are widened on the way in: both widenings are exact), each row's
// 16-byte chunks in an order that spreads the operand reads over the banks.
// LDS: two K tiles, then two V tiles.
template <int D>
struct PrefixTile {
  static constexpr int kTile = 64;
  static constexpr int kRow = 2 * D;             // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPlane = kTile * kRow;    // one tile of K or V
  static constexpr int kBlock = 32 * kRow;       // a score block's rows
  static constexpr int kPieces = kTile / 16;     // 16-token pieces, each inside one page
  // Waves of a workgroup: four of 32 query rows; at head_dim 256 four pairs, each
  // wave of a pair with half of the output dims (and all of the products: their
  // sums and Q together are too many registers for one wave of a SIMD's two).
  static constexpr int kSplit = D <= 128 ? 1 : 2;
  static constexpr int kWaves = 4 * kSplit;
};
// V chunk m of row R is stored at m ^ v_swizzle(R): a transposing read takes 4
// rows x 64 bytes a half-wave, which land on different banks (64 of 4 bytes).
template <int kChunks>
__device__ __forceinline__ int v_swizzle(int row) {
  return kChunks >= 16 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
}

// One work item: kWaves x 32 query rows of one KV head against `chunk` tiles.
//
// Lane l = 32 h + c.  S^T = K Q^T per 32 tokens (v_mfma_f32_32x32x16: A = K rows,
// B = query columns): lane (h, c) gets the scores of query c with tokens
// 8 (i / 4) + 4 h + i % 4, i = 0..15.  O^T += V^T P^T: k-slot e of half h is
// given token 16 s + 4 h + e (e < 4) or 16 s + 4 h + 4 + e, which is where the
// score block left P, so P needs no movement; V^T comes from LDS through the
// transposing read (16 lanes read 4 token rows of 16 dims, lane i gets dim i).
//
// Three score blocks are in work at once, so that matrix and vector instructions
// of one wave overlap (a wave's MFMA holds the matrix pipe for 32 cycles, in
// which it issues up to five vector instructions): while block i goes through
// the softmax, the products of block i + 1 and the values of block i - 1 are
// multiplied.  Tile t's K is therefore needed one stage before its V, and their
// buffers are refilled at different times: with one barrier a tile, K of tile
// t + 2 and V of tile t + 1 are loaded while blocks 2 t + 1 and 2 t + 2 go through.
template <int D, bool kQBf16, bool kVBf16, bool kFp8>
__device__ __forceinline__ void prefix_work(const PrefixParams& p, const uint32_t block, const uint32_t lds) {
  using T = PrefixTile<D>;
  constexpr int kRows = 128;        // query rows of a workgroup
  constexpr int kSteps = D / 16;    // QK k-steps
  constexpr int kDb = D / 32 / T::kSplit;  // the wave's output blocks of 32 dims
  const int lane = threadIdx.x & (kWave - 1);
  const int wave_id = uniform((int)threadIdx.x / kWave);
  const int wave = wave_id & 3, part = wave_id >> 2;  // 32 rows, and with kSplit a half of the dims
  const int h = lane >> 5, c = lane & 31;

  // Row tiles of one (chunk, head) on one XCD, one after the other: they read
  // the same K and V through its L2.
  const uint32_t xcd = block & 7, in_xcd = block >> 3;
  const uint32_t group = fdiv(in_xcd, p.rt_div);
  const int rt = (int)(in_xcd - group * p.rt_div.d);
  const uint32_t unit = group * 8 + xcd;
  if (unit >= (uint32_t)p.units) return;
  const int jc = (int)fdiv(unit, p.hkv_div);
  const int kvh = (int)unit - jc * p.Hkv;
  const int tile0 = jc * p.chunk, tile1 = min(tile0 + p.chunk, p.tiles);

  // ---- first loads, in flight together: the pages of the wave's first 64
  // 16-token pieces (lane i: piece base + i), the query rows and the lengths.
  // The wave stages piece `wave` of every tile (with kSplit K or V of it).
  int win_base = tile0 * T::kPieces;
  auto page_of = [&](int piece) {
    const int t = min(16 * piece, p.tokens - 1);  // (pieces past the prefix are not staged)
    return p.pages[fdiv((uint32_t)t, p.page)];
  };
  const int first_page = page_of(win_base + lane);
  const int row0 = rt * kRows + wave * 32;
  const bool live = row0 < p.rows;                // any column of the wave is a query row
  const int row = min(row0 + c, p.rows - 1);
  const bool row_ok = row0 + c < p.rows;
  const int b = (int)fdiv((uint32_t)row, p.g_div);
  u32x4 qop[kSteps];
  {
    const uint8_t* qrow = p.q + (int64_t)b * p.q_sb + (int64_t)(kvh * p.G + (row - b * p.G)) * p.q_sh;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qop[i] = *(const u32x4*)(qrow + 32 * i + 16 * h);
  }
  float sscale = p.score_scale * (kFp8 ? *p.k_scale : 1.0f);

  // ---- staging
  const uint8_t* kbase = p.k + (int64_t)kvh * p.k_sh;
  const uint8_t* vbase = p.v + (int64_t)kvh * p.v_sh;
  // Byte offsets of the pieces' first rows, in the lanes.
  int64_t k_piece, v_piece;
  auto place = [&](int page) {
    page = clampi(page, 0, p.num_pages - 1);
    const int t = 16 * (win_base + lane);
    const int row_in = t - (int)fdiv((uint32_t)t, p.page) * (int)p.page.d;
    k_piece = (int64_t)page * p.k_sp + (int64_t)row_in * p.k_st;
    v_piece = (int64_t)page * p.v_sp + (int64_t)row_in * p.v_st;
  };
  place(first_page);
  // 16-bit: DMA, 1 KB (64 / kChunks rows) a load.  e4m3: 16 codes a lane and load,
  // 1 KB = 1024 / D rows, kept in registers until the buffer is free.
  constexpr int kDma = 16 * T::kRow / 1024;
  constexpr int kCodeLoads = 16 * D / 1024;
  constexpr int kCodes = kFp8 ? kCodeLoads : 1;
  u32x4 k_codes[kCodes], v_codes[kCodes];
  // Byte offsets of the lane's 16 bytes in DMA load r of a piece, kept in registers
  // but at head_dim 256, which has none to spare.
  auto dma_off = [&](auto is_v, int r) {
    constexpr bool kV = decltype(is_v)::value;
    const int R = r * (64 / T::kChunks) + lane / T::kChunks, m = lane % T::kChunks;
    return R * (int)(kV ? p.v_st : p.k_st) + 16 * (m ^ (kV ? v_swizzle<T::kChunks>(R) : k_swizzle<T::kChunks>(R)));
  };
  constexpr int kOffs = D <= 128 ? kDma : 1;
  int k_off[kOffs], v_off[kOffs];
  if constexpr (!kFp8 && D <= 128) {
#pragma unroll
    for (int r = 0; r < kDma; ++r) {
      k_off[r] = dma_off(std::false_type{}, r);
      v_off[r] = dma_off(std::true_type{}, r);
    }
  }
  // This wave's pieces of a tile's K or V into a plane (16-bit), or into registers
  // (e4m3) from which put() widens them into it.  Pieces past the prefix read as zeros.
  auto load = [&](auto is_v, const uint8_t* base, int64_t at, int64_t st, const int (&off)[kOffs],
                  u32x4 (&codes)[kCodes], int tile, uint32_t plane) {
    const int piece = tile * T::kPieces + wave;
    const int from = (piece - win_base) & 63;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, from);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at >> 32), from);
    const auto rs = make_rsrc(base + (int64_t)(((uint64_t)hi << 32) | lo),
                              16 * piece < p.tokens ? 15 * (int)st + (kFp8 ? D : 2 * D) : 0);
#pragma unroll
    for (int r = 0; r < (kFp8 ? kCodeLoads : kDma); ++r) {
      if constexpr (!kFp8) {
        lds_dma16(rs, plane + wave * 16 * T::kRow + r * 1024, D <= 128 ? off[r % kOffs] : dma_off(is_v, r));
      } else {
        const int R = r * (1024 / D) + lane * 16 / D, d0 = lane * 16 % D;
        const auto x = buf_load<16>(rs, R * (int)st + d0);
        codes[r] = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
      }
    }
  };
  auto put = [&](auto is_v, const u32x4 (&codes)[kCodes], uint32_t plane) {
    if constexpr (kFp8) {
      constexpr bool kV = decltype(is_v)::value;
#pragma unroll
      for (int r = 0; r < kCodeLoads; ++r) {
        const int R = r * (1024 / D) + lane * 16 / D, m = lane * 16 % D / 8;
        const int swz = kV ? v_swizzle<T::kChunks>(R) : k_swizzle<T::kChunks>(R);
        const u32x4 x = codes[r];
        const uint32_t at = plane + (wave * 16 + R) * T::kRow;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x2 lo = e4m3x4_to<kV ? kVBf16 : kQBf16>(x[2 * e]), hi = e4m3x4_to<kV ? kVBf16 : kQBf16>(x[2 * e + 1]);
          *(lds_u32x4_w*)(uintptr_t)(at + 16 * ((m + e) ^ swz)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      }
    }
  };
  // (the window moves on when K, which runs a tile ahead of V, leaves it; V's pieces
  // of the tile before are still in it: 64 pieces are 16 tiles, kept from the
  // tile before the one that moves it)
  auto window = [&](int tile) {
    if ((tile + 1) * T::kPieces - win_base > 64) {
      win_base = (tile - 1) * T::kPieces;
      place(page_of(win_base + lane));
    }
  };
  auto load_k = [&](int tile) {
    window(tile);
    if (T::kSplit == 1 || part == 0) load(std::false_type{}, kbase, k_piece, p.k_st, k_off, k_codes, tile, lds + ((tile - tile0) & 1) * T::kPlane);
  };
  auto load_v = [&](int tile) {
    if (T::kSplit == 1 || part == 1) load(std::true_type{}, vbase, v_piece, p.v_st, v_off, v_codes, tile, lds + (2 + ((tile - tile0) & 1)) * T::kPlane);
  };
  auto put_k = [&](int tile) { if (T::kSplit == 1 || part == 0) put(std::false_type{}, k_codes, lds + ((tile - tile0) & 1) * T::kPlane); };
  auto put_v = [&](int tile) { if (T::kSplit == 1 || part == 1) put(std::true_type{}, v_codes, lds + (2 + ((tile - tile0) & 1)) * T::kPlane); };
  load_k(tile0);
  load_v(tile0);

  const int len = p.lens[b];
  // Whether a row of the workgroup's tile ends inside this chunk (every wave looks
  // at all of them: the waves take one path, which holds barriers).
  const int first = tile0 * T::kTile, end = min(tile1 * T::kTile, p.tokens);  // the chunk's tokens
  bool ends_inside = false;
  for (int r = lane; r < kRows; r += kWave) {
    const int rr = min(rt * kRows + r, p.rows - 1);
    const int l = p.lens[fdiv((uint32_t)rr, p.g_div)];
    ends_inside = ends_inside || (l > first && l < end);
  }
  const int lim = row_ok ? min(clampi(len, 0, p.max_len), p.tokens) : p.tokens;  // shared tokens the column attends
  const bool ragged = __builtin_amdgcn_ballot_w64(ends_inside) != 0;
  // The scale's sign goes to Q (exactly), so that the largest product is the
  // largest score; a scale of zero becomes the smallest normal number, which
  // scores every finite product as zero and keeps masked ones at -inf.
  {
    const uint32_t sign = sscale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) qop[i][e] = row_ok ? qop[i][e] ^ sign : 0u;
  }
  sscale = fabsf(sscale) < 1.17549435e-38f ? 1.17549435e-38f : fabsf(sscale);

  // ---- operand addresses: the chunk of a k-step (dim block) is an XOR away, tile
  // row and buffer a constant offset
  constexpr int kKeep = D <= 128 ? kSteps : 1;  // (head_dim 256: worked out where they are used)
  uint32_t k_at[kKeep], v_at[kDb];
  {
    const int vj = lane & 15, vr = 4 * h + vj / 4;
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
      k_at[i] = lds + ((c * T::kRow + 16 * (h ^ k_swizzle<T::kChunks>(c))) ^ (32 * i));
#pragma unroll
    for (int d = 0; d < kDb; ++d)
      v_at[d] = lds + 2 * T::kPlane + ((vr * T::kRow + 16 * ((2 * (c >> 4) + (vj & 3) / 2) ^ v_swizzle<T::kChunks>(vr)) +
                                    8 * (vj & 1)) ^ (64 * (part * kDb + d)));
  }
  // (at head_dim 256 the tile starts at a multiple of 512 past `lds`: the XOR stays within its row)
  auto k_operand = [&](uint32_t off, int i) {
    const uint32_t at = kKeep == kSteps ? k_at[i % kKeep] : lds + ((k_at[0] - lds) ^ (32 * i));
    return *(lds_u32x4*)((lds_u8*)(uintptr_t)at + off);
  };
  auto v_operand = [&](uint32_t off, int st, int d) {
    const u32x2 lo = lds_read_tr16(v_at[d] + (off + st * 16 * T::kRow));
    const u32x2 hi = lds_read_tr16(v_at[d] + (off + st * 16 * T::kRow + 8 * T::kRow));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  auto turn_k = [&](int by) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i) k_at[i] += by;
  };
  auto turn_v = [&](int by) {
#pragma unroll
    for (int d = 0; d < kDb; ++d) v_at[d] += by;
  };

  float m_ref = -INFINITY, m_max = -INFINITY, l_run = 0.f;
  f32x16 acc[kDb];
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

  // off: the block's offset in the two K (V) planes
  auto scores = [&](uint32_t off) {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) s = mfma32x32x16<kQBf16>(k_operand(off, i), qop[i], s);
    return s;
  };
  // Block's reference point (log2 domain).  The exponentials are taken relative
  // to m_ref, which follows the running maximum only when that has grown by
  // more than 2^8: the sums stay in fp32 and P below 2^8 keeps its relative
  // precision in 16 bits, while rescaling is left out of nearly every block.
  auto reference = [&](const f32x16& s) {
    float mt = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[i]);
    mt = half_max(mt) * sscale;
    m_max = fmaxf(m_max, mt);
    return mt > m_ref + 8.f ? mt : m_ref;
  };
  // P^T operands of a block's two k-steps relative to m_new, and the sum of P;
  // bf16 P as hi + lo parts, as in the split kernel.
  struct Weights {
    u32x4 hi[2], lo[2];
    float sum;
  };
  // Two weights, rounded into operands, and added to their sum.
  auto weight_pair = [&](uint32_t& hi, uint32_t& lo, float& sum, float a, float z) {
    if constexpr (kVBf16) {
      hi = pack_bf16x2(a, z);
      lo = pack_bf16x2(a - bf16_lo_to_f32(hi), z - bf16_hi_to_f32(hi));
      sum += a;
      sum += z;
    } else {
      // the sum of the weights as they are multiplied (fp32 sum of the f16 pair)
      hi = pack_f16x2(a, z);
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, hi), f16x2{(f16)1.f, (f16)1.f}, sum, false);
    }
  };
  auto weights = [&](const f32x16& s, float m_new) {
    Weights w;
    w.sum = 0.f;
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t hi, lo = 0;
      weight_pair(hi, lo, w.sum, __builtin_amdgcn_exp2f(fmaf(s[2 * j], sscale, -m_use)),
                  __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], sscale, -m_use)));
      w.hi[j / 4][j % 4] = hi;
      w.lo[j / 4][j % 4] = lo;
    }
    return w;
  };
  auto rescale = [&](float m_new) {
    if (__builtin_amdgcn_ballot_w64(m_new != m_ref) != 0) {
      const float alpha = m_new != m_ref ? __builtin_amdgcn_exp2f(m_ref - m_new) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
      m_ref = m_new;
    }
  };
  auto values = [&](uint32_t off, const Weights& w) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
        const u32x4 vop = v_operand(off, st, d);
        acc[d] = mfma32x32x16<kVBf16>(vop, w.hi[st], acc[d]);
        if constexpr (kVBf16) acc[d] = mfma32x32x16<true>(vop, w.lo[st], acc[d]);
      }
  };
  // One stage: products of the next block into s_next, softmax of s, values of
  // the block before (weights w_prev).  Returns s's weights; m: their reference.
  // Written slot by slot, one matrix instruction with the operand reads of two
  // slots on and its share of the softmax in each (left to itself the compiler
  // puts the reads next to their use and the exponentials in a row): the steps
  // are the maximum of 8 and 8 scores, the reference, then pair by pair the
  // exponent, the exponential and the rounding, one step apart.
  auto stage = [&](auto qk, auto pv, uint32_t k_blk, uint32_t v_blk, f32x16& s_next, const f32x16& s,
                   const Weights& w_prev, float& m) {
    constexpr bool kQk = decltype(qk)::value, kPv = decltype(pv)::value;
    constexpr int kVs = 2 * kDb, kRatio = kSteps / kVs;  // V operands, and QK k-steps for each
    constexpr int kPer = kVBf16 ? 2 : 1;                  // matrix instructions of a V operand
    constexpr int kSlots = (kQk ? kSteps : 0) + (kPv ? kVs * kPer : 0), kTimes = 13, kAhead = 2;
    u32x4 kop[kSteps], vop[kVs];
    float x[16], mt = -INFINITY, m_use = 0.f;
    Weights w;
    w.sum = 0.f;
    auto step = [&](int t) {
      if (t == 0 || t == 1) {
        float a = fmaxf(fmaxf(s[8 * t], s[8 * t + 1]), s[8 * t + 2]);
        a = fmaxf(fmaxf(a, s[8 * t + 3]), s[8 * t + 4]);
        a = fmaxf(fmaxf(a, s[8 * t + 5]), s[8 * t + 6]);
        mt = fmaxf(fmaxf(a, s[8 * t + 7]), mt);
        asm volatile("" : "+v"(mt));  // (here and below: keeps the step in its slot)
      }
      if (t == 2) {
        mt = half_max(mt) * sscale;
        m_max = fmaxf(m_max, mt);
        m = mt > m_ref + 8.f ? mt : m_ref;
        m_use = m == -INFINITY ? 0.f : m;
        asm volatile("" : "+v"(m_use));
      }
      if (t >= 3 && t < 11) {
        const int j = 2 * (t - 3);
        x[j] = fmaf(s[j], sscale, -m_use);
        x[j + 1] = fmaf(s[j + 1], sscale, -m_use);
        asm volatile("" : "+v"(x[j]), "+v"(x[j + 1]));
      }
      if (t >= 4 && t < 12) {
        const int j = 2 * (t - 4);
        x[j] = __builtin_amdgcn_exp2f(x[j]);
        x[j + 1] = __builtin_amdgcn_exp2f(x[j + 1]);
        asm volatile("" : "+v"(x[j]), "+v"(x[j + 1]));
      }
      if (t >= 5) {
        const int j = t - 5;
        uint32_t hi, lo = 0;
        weight_pair(hi, lo, w.sum, x[2 * j], x[2 * j + 1]);
        asm volatile("" : "+v"(hi), "+v"(lo), "+v"(w.sum));
        w.hi[j / 4][j % 4] = hi;
        w.lo[j / 4][j % 4] = lo;
      }
    };
    auto read = [&](int i) {
      if (i >= kSteps) return;
      if constexpr (kQk) kop[i] = k_operand(k_blk, i);
      if (kPv && i % kRatio == 0) vop[i / kRatio] = v_operand(v_blk, i / kRatio / kDb, i / kRatio % kDb);
    };
    int n = 0;
    auto rest = [&]() {  // of slot n
#pragma unroll
      for (int t = n * kTimes / kSlots; t < (n + 1) * kTimes / kSlots; ++t) step(t);
      ++n;
      __builtin_amdgcn_sched_barrier(0);
    };
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(i);
    if constexpr (kQk) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s_next[i] = 0.f;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if constexpr (kQk) {
        s_next = mfma32x32x16<kQBf16>(kop[i], qop[i], s_next);
        read(i + kAhead);
        rest();
      }
      if (kPv && i % kRatio == kRatio - 1) {
        const int j = i / kRatio;
        acc[j % kDb] = mfma32x32x16<kVBf16>(vop[j], w_prev.hi[j / kDb], acc[j % kDb]);
        if constexpr (!kQk) {
#pragma unroll
          for (int k = 0; k < kRatio; ++k) read(i + 1 - kRatio + k + kAhead);
        }
        rest();
        if constexpr (kVBf16) {
          acc[j % kDb] = mfma32x32x16<true>(vop[j], w_prev.lo[j / kDb], acc[j % kDb]);
          rest();
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    return w;
  };
  // A tile whose tokens do not all count for every column (columns that end
  // inside the chunk, the prefix's last tile).  V rows past a column's end may
  // hold anything, and 0 x inf is NaN, so from the wave's first end on each block
  // is multiplied once per different end, with V's rows zeroed past it, and only
  // the columns of that end take the sum.
  int first_end = lim > first ? lim : p.tokens;  // (columns that end before the chunk are dropped at its end)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) first_end = min(first_end, __shfl_xor(first_end, o));
  first_end = uniform(first_end);
  auto compute_ends = [&](int tile) {
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
      const uint32_t off = ((tile - tile0) & 1) * T::kPlane + tb * T::kBlock;
      const int t0 = tile * T::kTile + 32 * tb;
      f32x16 s = scores(off);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (t0 + 8 * (i / 4) + 4 * h + i % 4 >= lim) s[i] = -INFINITY;
      const float m_new = reference(s);
      const Weights w = weights(s, m_new);
      rescale(m_new);
      l_run += w.sum;
      if (t0 + 32 <= first_end) {
        values(off, w);
        continue;
      }
      uint64_t todo = __builtin_amdgcn_ballot_w64(lim > t0);
      while (todo) {
        const int last = __builtin_amdgcn_readlane(lim, __builtin_ctzll(todo));
        const bool mine = lim == last;
        todo &= ~__builtin_amdgcn_ballot_w64(mine);
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
          f32x16 sum;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            u32x4 vop = v_operand(off, st, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dword e: tokens t, t + 1
              const int t = t0 + 16 * st + 4 * h + 8 * (e >> 1) + 2 * (e & 1);
              vop[e] &= (t < last ? 0xffffu : 0u) | (t + 1 < last ? 0xffff0000u : 0u);
            }
            sum = mfma32x32x16<kVBf16>(vop, w.hi[st], sum);
            if constexpr (kVBf16) sum = mfma32x32x16<true>(vop, w.lo[st], sum);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] += mine ? sum[i] : 0.f;
        }
      }
    }
  };

  // ---- tiles.  Past a barrier every wave's part of what was loaded before it is in
  // LDS, and every wave has done with what it read before it.
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(vm_wait_imm(0));  // (the compiler does not see the DMA's LDS writes)
    asm volatile("" ::: "memory");
    __syncthreads();
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  // The tiles that count whole for every column go through the stages; the chunk's
  // others (from `whole` on) one by one.
  const int whole = ragged ? tile0 : max(tile0, min(tile1, p.tokens / T::kTile));
  put_k(tile0);
  put_v(tile0);
  int tile = tile0;
  if (tile < whole) {
    int side = T::kPlane;  // the other planes' distance
    f32x16 s0, s1;
    Weights w0, w1;
    float m;
    arrive();
    if (tile + 1 < whole) load_k(tile + 1);
    if (live) {
      s0 = scores(0);
      w0 = stage(yes, no, T::kBlock, 0, s1, s0, w1, m);
      rescale(m);
      l_run += w0.sum;
    }
    if (tile + 1 < whole) put_k(tile + 1);
    // Block 1 of `tile`, then block 0 of the next: K of the next tile, V of this one.
    // (One copy of the loop for both planes: the operands' addresses change sides,
    // 12 additions a tile, rather than the code.)
    while (tile + 1 < whole) {
      arrive();
      if (tile + 2 < whole) load_k(tile + 2);
      load_v(tile + 1);
      if (live) {
        turn_k(side);
        w1 = stage(yes, yes, 0, 0, s0, s1, w0, m);
        rescale(m);
        l_run += w1.sum;
        w0 = stage(yes, yes, T::kBlock, T::kBlock, s1, s0, w1, m);
        rescale(m);
        l_run += w0.sum;
        turn_v(side);
      }
      if (tile + 2 < whole) put_k(tile + 2);
      put_v(tile + 1);
      ++tile;
      side = -side;
    }
    if (tile > tile0) arrive();  // (the last tile's V)
    if (live) {
      w1 = stage(no, yes, 0, 0, s0, s1, w0, m);
      rescale(m);
      l_run += w1.sum;
      values(T::kBlock, w1);
      if (side < 0) {  // (back to the first planes)
        turn_k(side);
        turn_v(side);
      }
    }
    ++tile;
  }
  if (tile < tile1 && tile > tile0) {  // (the first tile is loaded)
    __syncthreads();
    load_k(tile);
    load_v(tile);
    put_k(tile);
    put_v(tile);
  }
  for (; tile < tile1; ++tile) {
    arrive();
    if (tile + 1 < tile1) {
      load_k(tile + 1);
      load_v(tile + 1);
    }
    if (live) compute_ends(tile);
    if (tile + 1 < tile1) {
      put_k(tile + 1);
      put_v(tile + 1);
    }
  }

  // ---- partials, relative to the maximum itself (the linear sink counts against it)
  const float to_max = m_max == m_ref ? 1.f : __builtin_amdgcn_exp2f(m_ref - m_max);
  const float v_scale = (kFp8 ? *p.v_scale : 1.0f) * to_max;
  const float l_tot = half_sum(l_run) * to_max;
  const bool none = lim <= first;  // the column ends before this chunk
  // The accumulators hold a row's sums in 16-byte pieces, 32 rows side by side:
  // stored like that, each instruction would touch 32 lines for 32 bytes each
  // (2.4 us of a 29 us kernel).  They go through LDS instead (piece m of row R at
  // m ^ R, so that neither side meets on a bank), a wave's rows in its own part.
  constexpr int kPieceRow = D / T::kSplit / 4;  // pieces of the wave's part of a row
  __syncthreads();  // (every wave has done with K and V)
  const uint32_t mine = lds + wave_id * (32 * kPieceRow * 16);
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = 8 * d + 2 * i + h;
      const f32x4 o = none ? f32x4{0.f, 0.f, 0.f, 0.f}
                           : f32x4{acc[d][4 * i] * v_scale, acc[d][4 * i + 1] * v_scale, acc[d][4 * i + 2] * v_scale,
                                   acc[d][4 * i + 3] * v_scale};
      *(lds_f32x4*)(uintptr_t)(mine + (c * kPieceRow + (m ^ (c & (kPieceRow - 1)))) * 16) = o;
    }
  const int64_t idx0 = ((int64_t)jc * p.Hkv + kvh) * p.rows + row0;  // the wave's first row
  if (row_ok && h == 0 && part == 0) *(f32x2*)(p.part_ml + 2 * (idx0 + c)) = none ? f32x2{-INFINITY, 0.f} : f32x2{m_max, l_tot};
  const int n_pieces = min(32, p.rows - row0) * kPieceRow;  // (<= 0: a wave without rows)
  float* dst = p.part_acc + idx0 * D + part * (D / T::kSplit);
#pragma unroll
  for (int k = 0; k < kPieceRow / 2; ++k) {
    const int i = k * kWave + lane, R = i / kPieceRow, m = i % kPieceRow;
    const f32x4 o = *(lds_f32x4*)(uintptr_t)(mine + (R * kPieceRow + (m ^ (R & (kPieceRow - 1)))) * 16);
    if (i < n_pieces) *(f32x4*)(dst + (int64_t)R * D + 4 * m) = o;
  }
}

// The whole of a shared decode but the merge: workgroups up to pp.blocks take the
// prefix, the others the sequences' own tokens (partial_work, a wave each), so
// that the own tokens' K and V stream in while the matrix cores are busy with
// the prefix.  Registers and LDS let eight waves on a CU: two workgroups (the
// first 256 of each kind share the CUs), at head_dim 256 one.  In turn instead
// (prefix, own tokens, merge) 256 x 4096 + 128 tokens took 34 + 31 us in the first
// two, together they take 44.
template <int D, int kKV>
constexpr uint32_t shared_stage() {
  constexpr uint32_t prefix = 4 * PrefixTile<D>::kPlane, own = PrefixTile<D>::kWaves * partial_stage<D, kKV>();
  return prefix > own ? prefix : own;
}
template <int D, int kQ, int kKV>
__global__ __launch_bounds__(64 * PrefixTile<D>::kWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
void shared_kernel(const int32_t* lens_arg, const int32_t* starts_arg, int B_arg, PrefixParams pp, Params pk) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_shared[];
  const uint32_t lds = (uint32_t)(uintptr_t)s_shared;
  if ((int)blockIdx.x < pp.blocks) {
    prefix_work<D, kQ == kBF16, kKV == kBF16, kKV == kE4M3>(pp, blockIdx.x, lds);
    return;
  }
  Params p = pk;
  p.lens = lens_arg;
  p.starts = starts_arg;
  p.B = B_arg;
  // (wave w of workgroup b is worker w S + b of kWaves S, S a multiple of 8: the
  // workers' numbers keep to the XCDs as those of one-wave workgroups do)
  const int b = (int)blockIdx.x - pp.blocks, S = (int)gridDim.x - pp.blocks;
  const int wave = uniform((int)threadIdx.x / kWave);
  partial_work<D, kQ, kKV, kPagedOwn, false, false, false>(
      p, nullptr, GivenWorker{(int)threadIdx.x & (kWave - 1), wave * S + b, PrefixTile<D>::kWaves * S},
      lds + wave * partial_stage<D, kKV>(), (int32_t*)(s_shared + shared_stage<D, kKV>()) + wave * 2 * (p.B + 1));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// The prefix's work split: row tiles, tiles of an item and items per KV head
// (chunks).
struct PrefixPlan {
  int row_tiles, tiles, chunk, chunks;
};
PrefixPlan plan_prefix(int64_t rows, int Hkv, int D, int64_t tokens, int cus) {
  PrefixPlan pl;
  pl.row_tiles = (int)cdiv(rows, 128);
  pl.tiles = (int)cdiv(tokens, 64);
  // One workgroup a CU, beside one of the own tokens': with two, the partials' way to
  // memory and back (twice as many) costs as much as the second wave a SIMD gives,
  // and the own tokens wait (us, with 0.5, 1, 2 a CU: 32 x 8192 bf16 39.5, 36.7, 47.4;
  // 64 x 32768 e4m3 94.5, 61.2, 60.6; 256 x 4096 f16 59.9, 56.1, 68.7).
  const int64_t slots = cus;
  const int64_t want = std::max<int64_t>(1, slots / ((int64_t)Hkv * pl.row_tiles));
  pl.chunk = (int)cdiv(pl.tiles, std::min<int64_t>(want, pl.tiles));
  pl.chunks = (int)cdiv(pl.tiles, pl.chunk);
  return pl;
}
// Sequences whose plan tables, one for each wave, fit LDS beside the tiles (160 KB
// a CU, 128 KB of tiles at head_dim 256).
constexpr int kSharedMaxBatch = 500;
template <int D>
constexpr uint32_t shared_tables(int B) { return PrefixTile<D>::kWaves * 8 * (uint32_t)(B + 1); }
static_assert(shared_stage<256, kF16>() + shared_tables<256>(kSharedMaxBatch) <= 160 * 1024, "tiles and tables fit LDS");

// The shared prefix of a decode (run_shared): the kernel's parameters and the
// prefix partials that the reduce kernel takes in.
struct SharedPrefix {
  PrefixParams p;
  int chunks;
};

template <int D, int kQ, int kKV>
void launch_shared_as(const SharedPrefix& sh, const Params& p, int own_blocks, const Launch& s) {
  launch(shared_kernel<D, kQ, kKV>, dim3((unsigned)(sh.p.blocks + own_blocks)), dim3(64 * PrefixTile<D>::kWaves),
         shared_stage<D, kKV>() + shared_tables<D>(p.B), s, p.lens, p.starts, p.B, sh.p, p);
}
template <int D>
void launch_shared(const SharedPrefix& sh, const Params& p, int own_blocks, int q_dt, int kv_dt, const Launch& s) {
  if (kv_dt == FSK_F16) launch_shared_as<D, kF16, kF16>(sh, p, own_blocks, s);
  else if (kv_dt == FSK_BF16) launch_shared_as<D, kBF16, kBF16>(sh, p, own_blocks, s);
  else if (q_dt == FSK_F16) launch_shared_as<D, kF16, kE4M3>(sh, p, own_blocks, s);
  else launch_shared_as<D, kBF16, kE4M3>(sh, p, own_blocks, s);
}

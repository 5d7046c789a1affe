// fsk_rope.h -- per-head RMS norm and position rotation of query and key rows,
// to tensors or on the way into the paged cache.  Part of fsk_decode.hip's
// translation unit (included once, inside its anonymous namespace, after the
// KV write's host side).
//
// For one head row x [D] of a token at position p, with the optional weight w:
//   y = x / sqrt(mean(x^2) + eps) * w                        (queries and keys)
//   y[i], y[j] = y[i] c - y[j] s, y[j] c + y[i] s            c, s = cos[p][t], sin[p][t]
// for the R / 2 pairs t: (i, j) = (t, t + R / 2), or (2 t, 2 t + 1) when
// interleaved; dims at R and past it are not rotated.  Everything is computed
// in fp32 from the row's own values and rounded once, to the type it is stored
// in; value rows are stored as they are (the KV write's rules).
//
// One pass: HBM holds each row once on the way in and once on the way out, and
// nothing else is large (a token's table row is R fp32 values for all its
// heads).  A thread owns 8 pairs of a row, both halves of each, so the rotation
// needs no exchange, and T = 4, 8 or 16 lanes own a row, so the norm's sum is
// DPP adds inside a 16-lane row.  A wave takes kRounds * 64 / T head rows of
// one token, so its position, slot and table row are read once, with the first
// rows' loads in flight.
//
// Bound by HBM at large sizes, by launch and two dependent round trips (position,
// table row) at small ones.  Kernel times, bf16: 16384 tokens of 32 + 8 heads of 128
// (344 MB) 59.5 us, 5.8 TB/s, above a plain copy's 4.9; into e4m3 pages 28001 tokens
// with values (646 MB) 117 us, 5.5 TB/s; one token 2.9 to 3.4 us.

struct RopeParams {
  const uint8_t* src[3];                 // q, k, v rows [n, H, D]
  int64_t s_st[3], s_sh[3];              // token / head strides, bytes
  uint8_t* out[2];                       // q and (without pools) k rows
  int64_t o_st[2], o_sh[2];
  uint8_t* pool[2];                      // k and v pools [P, Hkv, page_size, D], or null
  int64_t p_sp[2], p_sh[2], p_st[2];
  const float* scale[2];                 // e4m3 pools: quantisation scales, or null
  const int64_t* slots;                  // [n] page * page_size + row; out of range: skip
  uint32_t n_slots;
  FastDiv page;
  const uint8_t* weight[2];              // [D] norm weights of q and k, or null
  int w_dt;
  float eps, inv_d;                      // inv_d: 1 / D
  const uint8_t* cos;                    // [rows, R / 2]
  const uint8_t* sin;
  int64_t c_sr, n_sr;                    // their row strides, bytes
  int t_dt;
  uint32_t t_rows;
  const int64_t* positions;              // [n], or null: token i takes row i mod t_rows
  FastDiv rows_div;                      // divisor t_rows
  uint32_t n, heads, hq, hkv;            // heads: rows of a token (hq + hkv, with values + hkv)
  uint32_t lanes, rot_lanes;             // D / 16 and R / 16
  uint32_t t_log;                        // log2 of the lanes a row occupies
  int interleaved;
  uint32_t parts, items;                 // waves of a token, waves in all
  FastDiv parts_div;
  int32_t* bt;                           // block-table updates, as WriteParams
  int64_t bt_numel;
  const int64_t* upd;
  int n_upd;
};

constexpr int kRopeThreads = 256;
constexpr int kPlain = -1;  // kPool of a call without pools: k goes to a tensor of the source type

// Eight consecutive elements of type `dt` from p (16-byte aligned), widened.
template <int kDt>
__device__ __forceinline__ void rope_widen8(u32x4 lo, u32x4 hi, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = lo[j];
    const uint32_t w2 = hi[j];
    if constexpr (kDt == kF32) {
      x[j] = u2f(w);
      x[4 + j] = u2f(w2);
    } else if constexpr (kDt == kF16) {
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      x[2 * j] = (float)h[0];
      x[2 * j + 1] = (float)h[1];
    } else {
      x[2 * j] = bf16_lo_to_f32(w);
      x[2 * j + 1] = bf16_hi_to_f32(w);
    }
  }
}
// ... of a small operand (weights, tables), whose type is known at run time
__device__ __forceinline__ void rope_load8(const uint8_t* base, int64_t elem, int dt, float (&x)[8]) {
  const u32x4* p = (const u32x4*)(base + elem * (dt == FSK_F32 ? 4 : 2));
  const u32x4 lo = p[0];
  if (dt == FSK_F32) rope_widen8<kF32>(lo, p[1], x);
  else if (dt == FSK_F16) rope_widen8<kF16>(lo, lo, x);
  else rope_widen8<kBF16>(lo, lo, x);
}

// Sum over the 2^t_log lanes of a row (4, 8 or 16 lanes of a DPP row): each
// step adds the mirror image, whose lanes all hold the other half's sum.
__device__ __forceinline__ float rope_row_sum(float x, uint32_t t_log) {
  auto add = [](float a, int b) { return a + u2f((uint32_t)b); };
  x = add(x, __builtin_amdgcn_update_dpp(0, (int)f2u(x), 0xB1, 0xf, 0xf, true));    // quad_perm 1,0,3,2
  x = add(x, __builtin_amdgcn_update_dpp(0, (int)f2u(x), 0x4E, 0xf, 0xf, true));    // quad_perm 2,3,0,1
  const float y = add(x, __builtin_amdgcn_update_dpp(0, (int)f2u(x), 0x141, 0xf, 0xf, true));  // row_half_mirror
  if (t_log > 2) x = y;
  const float z = add(x, __builtin_amdgcn_update_dpp(0, (int)f2u(x), 0x140, 0xf, 0xf, true));  // row_mirror
  if (t_log > 3) x = z;
  return x;
}

// Eight fp32 values to p as kDt.
template <int kDt, bool kScaled>
__device__ __forceinline__ void rope_store8(uint8_t* p, const float (&x)[8], double rscale) {
  if constexpr (kDt == kF32) {
    row_store((u32x4*)p, u32x4{f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3])});
    row_store((u32x4*)(p + 16), u32x4{f2u(x[4]), f2u(x[5]), f2u(x[6]), f2u(x[7])});
  } else if constexpr (kDt == kE4M3) {
    u32x2 codes{encode_e4m3x4<kScaled>(x, rscale), encode_e4m3x4<kScaled>(x + 4, rscale)};
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) nan = nan || x[j] != x[j];
    if (__builtin_amdgcn_ballot_w64(nan) != 0) {
      codes[0] = nan_codes(codes[0], x);
      codes[1] = nan_codes(codes[1], x + 4);
    }
    row_store((u32x2*)p, codes);
  } else {
    row_store((u32x4*)p, u32x4{pack2<kDt>(x[0], x[1]), pack2<kDt>(x[2], x[3]), pack2<kDt>(x[4], x[5]),
                               pack2<kDt>(x[6], x[7])});
  }
}

template <int kSrc, int kPool, bool kScaled, int kRounds>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_kernel(RopeParams p) {
  constexpr int kSe = kSrc == kF32 ? 4 : 2;                          // source element bytes
  constexpr int kPe = kPool == kE4M3 ? 1 : kPool == kPlain ? kSe : 2;  // pool element bytes
  constexpr bool kPaged = kPool != kPlain;
  const int lane = threadIdx.x & (kWave - 1);
  const uint32_t item = (uint32_t)uniform((int)(blockIdx.x * (kRopeThreads / kWave) + threadIdx.x / kWave));
  if (kPaged && blockIdx.x == 0) {
    for (int j = threadIdx.x; j < p.n_upd; j += kRopeThreads) {
      const int64_t idx = p.upd[2 * j];
      if (idx >= 0 && idx < p.bt_numel) p.bt[idx] = (int32_t)p.upd[2 * j + 1];
    }
  }
  if (item >= p.items) return;
  const uint32_t tok = fdiv(item, p.parts_div);
  const uint32_t part = item - tok * p.parts;
  const uint32_t T = 1u << p.t_log;
  const uint32_t j = lane & (T - 1);
  const uint32_t row_slots = (uint32_t)kWave >> p.t_log;
  const uint32_t h0 = part * row_slots * kRounds + ((uint32_t)lane >> p.t_log);
  const bool rot = j < p.rot_lanes;
  const bool split = rot && !p.interleaved;      // the two chunks are the halves of R
  const uint32_t ea = split ? 8 * j : 16 * j;    // first elements of the thread's two chunks
  const uint32_t eb = split ? 8 * (p.rot_lanes + j) : 16 * j + 8;

  // All rows' loads first: they need nothing but the item.
  u32x4 raw[kRounds][kSe];  // chunk a, then chunk b: kSe / 2 loads of 16 bytes each
  uint32_t kind[kRounds], head[kRounds];
  bool ok[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t h = h0 + r * row_slots;
    ok[r] = h < p.heads && j < p.lanes;
    kind[r] = h < p.hq ? 0 : h < p.hq + p.hkv ? 1 : 2;
    head[r] = h - (kind[r] == 0 ? 0 : kind[r] == 1 ? p.hq : p.hq + p.hkv);
#pragma unroll
    for (int e = 0; e < kSe; ++e) raw[r][e] = u32x4{0, 0, 0, 0};
    if (!ok[r]) continue;
    const uint8_t* base = kind[r] == 0 ? p.src[0] : kind[r] == 1 ? p.src[1] : p.src[2];
    const int64_t st = kind[r] == 0 ? p.s_st[0] : kind[r] == 1 ? p.s_st[1] : p.s_st[2];
    const int64_t sh = kind[r] == 0 ? p.s_sh[0] : kind[r] == 1 ? p.s_sh[1] : p.s_sh[2];
    const uint8_t* a = base + (int64_t)tok * st + (int64_t)head[r] * sh;
#pragma unroll
    for (int e = 0; e < kSe / 2; ++e) {
      raw[r][e] = row_load((const u32x4*)(a + ea * kSe) + e);
      raw[r][kSe / 2 + e] = row_load((const u32x4*)(a + eb * kSe) + e);
    }
  }
  int64_t row = p.positions ? p.positions[tok] : (int64_t)(tok - fdiv(tok, p.rows_div) * p.t_rows);
  row = row < 0 ? 0 : row >= (int64_t)p.t_rows ? (int64_t)p.t_rows - 1 : row;  // (no read outside the table)
  uint8_t* dst_pool[2] = {nullptr, nullptr};
  bool stored = false;
  double rscale[2] = {1.0, 1.0};
  if constexpr (kPaged) {
    const int64_t slot = p.slots[tok];
    stored = slot >= 0 && slot < (int64_t)p.n_slots;
    const uint32_t page = stored ? fdiv((uint32_t)slot, p.page) : 0;
    const uint32_t prow = stored ? (uint32_t)slot - page * p.page.d : 0;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      dst_pool[kv] = p.pool[kv] + (int64_t)page * p.p_sp[kv] + (int64_t)prow * p.p_st[kv];
      if constexpr (kScaled) rscale[kv] = 1.0 / (double)*p.scale[kv];
    }
  }
  float c[8], s[8];
  if (rot) {
    rope_load8(p.cos + row * p.c_sr, 8 * j, p.t_dt, c);
    rope_load8(p.sin + row * p.n_sr, 8 * j, p.t_dt, s);
  }

#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    float x[2][8];
    rope_widen8<kSrc>(raw[r][0], raw[r][kSe / 2 - 1], x[0]);
    rope_widen8<kSrc>(raw[r][kSe / 2], raw[r][kSe - 1], x[1]);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(x[0][e], x[0][e], fmaf(x[1][e], x[1][e], sum));
    sum = rope_row_sum(j < p.lanes ? sum : 0.f, p.t_log);
    if (!ok[r]) continue;
    const uint8_t* wt = kind[r] == 0 ? p.weight[0] : kind[r] == 1 ? p.weight[1] : nullptr;
    if (wt) {
      const float rstd = 1.0f / sqrtf(fmaf(sum, p.inv_d, p.eps));
      float w[8];
      rope_load8(wt, ea, p.w_dt, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[0][e] = x[0][e] * rstd * w[e];
      rope_load8(wt, eb, p.w_dt, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[1][e] = x[1][e] * rstd * w[e];
    }
    if (rot && kind[r] < 2) {
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float& u = x[e >> 2][2 * (e & 3)];
          float& v = x[e >> 2][2 * (e & 3) + 1];
          const float y = fmaf(u, c[e], -v * s[e]);
          v = fmaf(v, c[e], u * s[e]);
          u = y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = fmaf(x[0][e], c[e], -x[1][e] * s[e]);
          x[1][e] = fmaf(x[1][e], c[e], x[0][e] * s[e]);
          x[0][e] = y;
        }
      }
    }
    if (kind[r] == 0 || !kPaged) {
      uint8_t* o = (kind[r] == 0 ? p.out[0] + (int64_t)tok * p.o_st[0] + (int64_t)head[r] * p.o_sh[0]
                                 : p.out[1] + (int64_t)tok * p.o_st[1] + (int64_t)head[r] * p.o_sh[1]);
      rope_store8<kSrc, false>(o + ea * kSe, x[0], 1.0);
      rope_store8<kSrc, false>(o + eb * kSe, x[1], 1.0);
    } else if constexpr (kPaged) {
      if (!stored) continue;
      const bool is_v = kind[r] == 2;
      uint8_t* o = (is_v ? dst_pool[1] + (int64_t)head[r] * p.p_sh[1] : dst_pool[0] + (int64_t)head[r] * p.p_sh[0]);
      if constexpr (kPool == kSrc) {
        if (is_v) {  // same type: a bit-exact copy
          row_store((u32x4*)(o + ea * kPe), raw[r][0]);
          row_store((u32x4*)(o + eb * kPe), raw[r][1]);
          continue;
        }
      }
      const double rs = is_v ? rscale[1] : rscale[0];
      rope_store8<kPool, kScaled>(o + ea * kPe, x[0], rs);
      rope_store8<kPool, kScaled>(o + eb * kPe, x[1], rs);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct RopeArgs {
  const void* src[3]; int64_t s_st[3], s_sh[3];  // q (null: none), k, v (null without pools)
  int64_t n;
  const int64_t* slots;
  const void* cos; int64_t c_sr; const void* sin; int64_t n_sr; int64_t t_rows; int t_dt;
  int rotary, interleaved;
  const int64_t* positions;
  const void* weight[2]; int w_dt; float eps;
  void* out[2]; int64_t o_st[2], o_sh[2];
  bool paged;
  void* pool[2]; int64_t p_sp[2], p_sh[2], p_st[2];
  int num_pages, page_size, Hq, Hkv, D, src_dt, pool_dt;
  const float* scale[2];
  int32_t* bt; int64_t bt_numel; const int64_t* upd; int64_t n_upd;
  hipStream_t stream;
};

template <int kSrc, int kPool, bool kScaled>
void launch_rope(const RopeParams& p, int rounds, unsigned grid, const Launch& s) {
  if (rounds == 1) launch(norm_rope_kernel<kSrc, kPool, kScaled, 1>, dim3(grid), dim3(kRopeThreads), 0, s, p);
  else launch(norm_rope_kernel<kSrc, kPool, kScaled, 2>, dim3(grid), dim3(kRopeThreads), 0, s, p);
}
template <int kSrc>
void dispatch_rope(const RopeParams& p, bool paged, int pool_dt, bool scaled, int rounds, unsigned grid, const Launch& s) {
  if (!paged) launch_rope<kSrc, kPlain, false>(p, rounds, grid, s);
  else if (pool_dt == FSK_F16) launch_rope<kSrc, kF16, false>(p, rounds, grid, s);
  else if (pool_dt == FSK_BF16) launch_rope<kSrc, kBF16, false>(p, rounds, grid, s);
  else if (scaled) launch_rope<kSrc, kE4M3, true>(p, rounds, grid, s);
  else launch_rope<kSrc, kE4M3, false>(p, rounds, grid, s);
}

bool is_float_dt(int dt) { return dt == FSK_F16 || dt == FSK_BF16 || dt == FSK_F32; }

// A row tensor's strides (elements) and alignment (bytes of 8 elements, at most 16).
int check_rope_rows(const char* name, const void* ptr, std::initializer_list<int64_t> strides, int elem) {
  const int a = elem == 1 ? 8 : 16;
  if (!ptr) return fail(FSK_ERR_INVALID, std::string(name) + ": null tensor pointer");
  if (!aligned(ptr, a)) return fail(FSK_ERR_INVALID, std::string(name) + " rows must be aligned to 16 bytes (e4m3: 8)");
  for (const int64_t st : strides) {
    if (st < 0) return fail(FSK_ERR_INVALID, std::string(name) + ": negative stride");
    if (st >= kMaxStride) return fail(FSK_ERR_UNSUPPORTED, std::string(name) + ": stride above 2^40 elements");
    if ((st * elem) % a) return fail(FSK_ERR_INVALID, std::string(name) + " rows must be aligned to 16 bytes (e4m3: 8)");
  }
  return FSK_OK;
}

int run_rope(const RopeArgs& a) {
  const bool with_q = a.Hq > 0;
  if (a.n < 0 || a.n_upd < 0) return fail(FSK_ERR_INVALID, "negative count");
  if (a.Hq < 0 || a.Hkv <= 0 || a.D <= 0) return fail(FSK_ERR_INVALID, "heads and head_dim must be positive");
  if (a.Hq > kMaxQHeads || a.Hkv > kMaxQHeads) return fail(FSK_ERR_UNSUPPORTED, "heads above 65536");
  if (a.D % 16 || a.D > 256) return fail(FSK_ERR_UNSUPPORTED, "head_dim must be a multiple of 16, at most 256");
  if (a.rotary < 0 || a.rotary > a.D) return fail(FSK_ERR_INVALID, "rotary_dim must be in [0, head_dim]");
  if (a.rotary % 16) return fail(FSK_ERR_UNSUPPORTED, "rotary_dim must be a multiple of 16");
  if (!is_float_dt(a.src_dt)) return fail(FSK_ERR_UNSUPPORTED, "q, k and v must be f16, bf16 or f32");
  const bool norm = a.weight[0] || a.weight[1];
  if (norm && !is_float_dt(a.w_dt)) return fail(FSK_ERR_UNSUPPORTED, "norm weights must be f16, bf16 or f32");
  for (int i = 0; i < 2; ++i)
    if (a.weight[i] && !aligned(a.weight[i], 16)) return fail(FSK_ERR_INVALID, "norm weights must be 16-byte aligned");
  if (norm && !(a.eps >= 0.f && std::isfinite(a.eps))) return fail(FSK_ERR_INVALID, "eps must be finite and >= 0");
  const int se = elem_bytes(a.src_dt);
  if (a.n >= ((int64_t)1 << 31)) return fail(FSK_ERR_UNSUPPORTED, "batch too large for one call");
  if (a.t_rows < 0 || a.t_rows >= ((int64_t)1 << 31)) return fail(FSK_ERR_UNSUPPORTED, "table rows out of int32 range");
  int st = FSK_OK;
  if (a.rotary > 0) {
    if (!is_float_dt(a.t_dt)) return fail(FSK_ERR_UNSUPPORTED, "cos and sin must be f16, bf16 or f32");
    if (a.n > 0) {
      if (a.t_rows == 0) return fail(FSK_ERR_INVALID, "cos and sin have no rows");
      if (!a.positions && a.n % a.t_rows) return fail(FSK_ERR_INVALID, "without positions the tokens must be a multiple of the table's rows");
      const int te = elem_bytes(a.t_dt);
      if ((st = check_rope_rows("cos", a.cos, {a.c_sr}, te)) != FSK_OK) return st;
      if ((st = check_rope_rows("sin", a.sin, {a.n_sr}, te)) != FSK_OK) return st;
    }
  }
  if (a.n > 0) {
    if (with_q && (st = check_rope_rows("q", a.src[0], {a.s_st[0], a.s_sh[0]}, se)) != FSK_OK) return st;
    if (with_q && (st = check_rope_rows("q_out", a.out[0], {a.o_st[0], a.o_sh[0]}, se)) != FSK_OK) return st;
    if ((st = check_rope_rows("k", a.src[1], {a.s_st[1], a.s_sh[1]}, se)) != FSK_OK) return st;
  }
  bool scaled = false;
  if (!a.paged) {
    if (a.n > 0 && (st = check_rope_rows("k_out", a.out[1], {a.o_st[1], a.o_sh[1]}, se)) != FSK_OK) return st;
  } else {
    if (a.n > 0 && (st = check_rope_rows("v", a.src[2], {a.s_st[2], a.s_sh[2]}, se)) != FSK_OK) return st;
    if (a.page_size <= 0 || a.num_pages <= 0) return fail(FSK_ERR_INVALID, "page_size and num_pages must be positive");
    if (a.pool_dt != FSK_F16 && a.pool_dt != FSK_BF16 && a.pool_dt != FSK_E4M3)
      return fail(FSK_ERR_UNSUPPORTED, "pools must be f16, bf16 or e4m3");
    scaled = a.scale[0] || a.scale[1];
    if (scaled && (!a.scale[0] || !a.scale[1])) return fail(FSK_ERR_INVALID, "pass both k_scale and v_scale or neither");
    if (scaled && a.pool_dt != FSK_E4M3) return fail(FSK_ERR_INVALID, "scales apply to e4m3 pools only");
    if (a.n_upd > 0 && (!a.bt || !a.upd || a.bt_numel <= 0)) return fail(FSK_ERR_INVALID, "block-table updates need block_table");
    if (a.n_upd >= (1 << 30)) return fail(FSK_ERR_UNSUPPORTED, "too many block-table updates");
    if ((int64_t)a.num_pages * a.page_size >= ((int64_t)1 << 31)) return fail(FSK_ERR_UNSUPPORTED, "pool above 2^31 slots");
    if (a.n > 0) {
      if (!a.slots) return fail(FSK_ERR_INVALID, "null slot_mapping");
      const int pe = elem_bytes(a.pool_dt);
      for (int kv = 0; kv < 2; ++kv) {
        st = check_rope_rows(kv ? "v_pool" : "k_pool", a.pool[kv], {a.p_sp[kv], a.p_sh[kv], a.p_st[kv]}, pe);
        if (st != FSK_OK) return st;
        if (a.page_size > 1 && a.p_st[kv] < a.D) return fail(FSK_ERR_INVALID, "pool row stride must be >= head_dim");
      }
    }
  }
  const int64_t heads = (int64_t)a.Hq + a.Hkv + (a.paged ? a.Hkv : 0);
  if (a.n * heads >= ((int64_t)1 << 31)) return fail(FSK_ERR_UNSUPPORTED, "batch too large for one call");
  if (a.n == 0 && a.n_upd == 0) return FSK_OK;

  RopeParams p;
  memset(&p, 0, sizeof(p));
  for (int i = 0; i < 3; ++i) {
    p.src[i] = (const uint8_t*)a.src[i];
    p.s_st[i] = a.s_st[i] * se; p.s_sh[i] = a.s_sh[i] * se;
  }
  for (int i = 0; i < 2; ++i) {
    p.out[i] = (uint8_t*)a.out[i];
    p.o_st[i] = a.o_st[i] * se; p.o_sh[i] = a.o_sh[i] * se;
    p.weight[i] = (const uint8_t*)a.weight[i];
  }
  if (a.paged) {
    const int pe = elem_bytes(a.pool_dt);
    for (int kv = 0; kv < 2; ++kv) {
      p.pool[kv] = (uint8_t*)a.pool[kv];
      p.p_sp[kv] = a.p_sp[kv] * pe; p.p_sh[kv] = a.p_sh[kv] * pe; p.p_st[kv] = a.p_st[kv] * pe;
      p.scale[kv] = a.scale[kv];
    }
    p.slots = a.slots;
    p.n_slots = (uint32_t)((int64_t)a.num_pages * a.page_size);
    p.page = make_fastdiv((uint32_t)a.page_size);
    p.bt = a.bt; p.bt_numel = a.bt_numel; p.upd = a.upd; p.n_upd = (int)a.n_upd;
  }
  p.w_dt = a.w_dt; p.eps = a.eps; p.inv_d = 1.0f / (float)a.D;
  p.cos = (const uint8_t*)a.cos; p.sin = (const uint8_t*)a.sin;
  p.t_dt = a.t_dt;
  const int te = a.rotary > 0 ? elem_bytes(a.t_dt) : 0;
  p.c_sr = a.c_sr * te; p.n_sr = a.n_sr * te;
  p.t_rows = (uint32_t)std::max<int64_t>(a.t_rows, 1);
  p.positions = a.positions;
  p.rows_div = make_fastdiv(p.t_rows);
  p.n = (uint32_t)a.n; p.heads = (uint32_t)heads; p.hq = (uint32_t)a.Hq; p.hkv = (uint32_t)a.Hkv;
  p.lanes = (uint32_t)a.D / 16; p.rot_lanes = (uint32_t)a.rotary / 16;
  p.t_log = p.lanes <= 4 ? 2 : p.lanes <= 8 ? 3 : 4;
  p.interleaved = a.interleaved != 0;
  const uint32_t slots_per_wave = (uint32_t)kWave >> p.t_log;
  // A second round of rows per wave where one leaves more waves than the card holds
  // at once (32 a CU), whose last ones would start late; for rows of four lanes, 16 to
  // a wave, of which one round wastes more of a token's last wave, from half of that.
  // Inputs from HBM, us, 1 / 2 rounds: bf16, 32 + 8 heads of 128: 64 tokens 3.3 / 3.7,
  // 1024 5.9 / 6.4, 1400 (7000 waves) 7.3 / 8.0, 1700 9.5 / 8.5, 2048 10.5 / 9.5, 16384
  // 64.5 / 60.7; into pages 820 6.1 / 6.4, 1365 9.6 / 8.0.  f16, 64 + 8 heads of 64: 600
  // (3000 waves) 4.8 / 4.8, 820 5.6 / 5.5, 1237 7.7 / 6.9, 3000 14.7 / 14.7.
  const int waves_a_cu = p.t_log == 2 ? 15 : 28;
  const int rounds = a.n * cdiv(heads, slots_per_wave) > waves_a_cu * (int64_t)device_cus() ? 2 : 1;
  p.parts = (uint32_t)cdiv(heads, slots_per_wave * rounds);
  p.parts_div = make_fastdiv(p.parts);
  p.items = (uint32_t)(a.n * p.parts);
  const unsigned grid = (unsigned)std::max<int64_t>(1, cdiv(p.items, kRopeThreads / kWave));
  if (grid >= (1u << 24)) return fail(FSK_ERR_UNSUPPORTED, "batch too large for one call");
  (void)hipGetLastError();
  hipEvent_t ev[3];
  timing_events(ev);
  const Launch l{a.stream, ev[0], ev[1]};
  if (a.src_dt == FSK_F16) dispatch_rope<kF16>(p, a.paged, a.pool_dt, scaled, rounds, grid, l);
  else if (a.src_dt == FSK_BF16) dispatch_rope<kBF16>(p, a.paged, a.pool_dt, scaled, rounds, grid, l);
  else dispatch_rope<kF32>(p, a.paged, a.pool_dt, scaled, rounds, grid, l);
  timing_keep(ev, !ev[0] || hipEventRecord(ev[2], a.stream) == hipSuccess);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FSK_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(e));
  return FSK_OK;
}

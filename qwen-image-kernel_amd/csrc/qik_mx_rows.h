// Attention of few query rows over a 4-bit slab and fresh keys (gfx950): a
// token's heads, or some tokens', against a cache of any length.
//
// The mathematics is the tile loop's of qik_attn_kernel.h (S^T = K.Q^T, online
// softmax in the exp2 domain with a lazy reference point, O^T = V^T.P^T), but such
// a call is bound by the slab's bytes: 17/32 of a byte per element of K and V,
// each read once.  So:
//   * an item is 16 or 32 query rows of one (b, KV head) -- the query heads that
//     share the KV head times the query positions -- and its keys in steps of
//     32.  Items are cut into pieces of the same number of steps, one a
//     workgroup, so that sequences of any lengths fill the device evenly.  With
//     lengths of several entries (SPREAD) every workgroup reads them all, takes
//     the number of steps that cuts their sum into as many pieces as the host
//     aims at, and finds its own among them (24 entries of up to 8192 keys, ten
//     draws: 33.0 us with the number that the longest gave for all, 30.5 so; the
//     same bytes in entries of one length 25.6 to 29).  The heads come first in the grid, so
//     that pieces without keys do not fall on the same XCDs;
//   * a workgroup's waves take its steps in turn, each with its own softmax state
//     and its own LDS, and never wait for each other before the end;
//   * a call lasts some microseconds, so that its instructions' way from memory
//     shows: the loop's and the merge's code stands once, what can be a loop is
//     one, and what can be divided on the host is;
//   * the products are v_mfma_f32_16x16x32: with 16 rows a lane holds half of the
//     scores and accumulators that a 32-row tile has;
//   * K goes from memory to the matrix cores through registers alone.  The
//     order of the head dim inside a dot product is free, as long as Q has the
//     same: lane (key, quarter) holds a quarter of its key's row, 4 to 32
//     contiguous bytes of codes, and every 4 bytes become one operand;
//   * V is turned into the element type in registers and goes through the
//     wave's own LDS, whose transpose read gives the V^T operand;
//   * the next step's codes are loaded as soon as this step's have been turned,
//     before its softmax;
//   * the pieces of a cut item leave their (m, l, O) in the workspace, and the
//     last to arrive combines them in the order of the keys, so that the result
//     does not depend on which one that is.
// 32 query heads on 8 KV heads of 128, MI355X: a token against 131072 keys 30.6 us,
// 4.6 TB/s of the slab (a large copy reaches 5.15); 24 tokens of sequences of up
// to 8192 keys 30 to 33 us, 3.7 to 4.0 TB/s, where the pieces are two a CU and not
// quite even, and the merge ends last; a token against 1501 keys 8.6 us, of which
// the bytes would be less than one: launch, a piece's loads and steps, and the merge
// one after the other.
#ifndef QIK_MX_ROWS_H
#define QIK_MX_ROWS_H

#include "qik_attn_kernel.h"

namespace qik {

constexpr int ROWS_N = 32;        // keys of a step
constexpr int ROWS_M = 16;        // query rows of a tile; an item has one or two tiles

// Waves of a workgroup; two workgroups share a CU (one at D = 256 or with two tiles).
constexpr int rows_waves(int D, int mt) { return D > 128 && mt > 1 ? 4 : 8; }

struct RowsParams {
  const char* q;
  const char* k_new;
  const char* v_new;
  const char* k_codes;
  const char* v_codes;
  const char* k_scales;
  const char* v_scales;
  const int32_t* lengths;    // NULL: P keys of the slab in every batch entry
  const int32_t* L;
  const uint8_t* key_valid;
  char* out;
  unsigned* ctl;             // arrivals per item, zero between launches
  float* part;               // per (item, piece): rows x D accumulators, then rows (m, l)
  int64_t sq[3], skn[3], svn[3], so[3];  // b, s, h in elements
  int64_t skc[3], svc[3], sks[3], svs[3];  // b, p, h in bytes
  int64_t svalid_b, sL_b;
  int R;                     // query rows of a KV head: SQ * G, row r is head r % G of position r / G
  int SN, P, HKV, G, KV;
  int uniform;
  int steps;                 // of a piece (SPREAD: at least)
  int B, spread;             // SPREAD: entries; pieces that all of them aim at
  unsigned by_G, by_HKV;     // ceil(2^32 / G), ceil(2^32 / HKV): see quotient
  int row_bits;              // log2 of the rows a piece keeps in the workspace, a power of two
  float qk_scale;
};

// LDS bytes of one wave: its V step, and at the end its share of a tile's O
template <int D>
constexpr int rows_wave_lds() { return D * 2 * ROWS_N; }
static_assert(ROWS_N * 2 == ROWS_M * 4, "a wave's O of 16 rows in fp32 takes the room of a step's V");
// bytes a piece of `rows` rows keeps in the workspace: O, then (m, l) of each row
__host__ __device__ constexpr int rows_slot(int D, int rows) { return (rows * (D + 2) + 3) / 4 * 16; }

template <bool FP16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (FP16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// x of the four lanes l, l ^ 16, l ^ 32, l ^ 48 together
__device__ __forceinline__ float quad_max(float x) {
  const unsigned u = __float_as_uint(pair_max(x));
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  const unsigned u = __float_as_uint(pair_sum(x));
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the sum over lanes 0 .. l in each lane l
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 to the next row, 31 to the upper half
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// n / d by ceil(2^32 / d) (0 for d = 1): exact while n * d < 2^32
__device__ __forceinline__ int quotient(int n, unsigned by) { return by == 0u ? n : (int)__umulhi((unsigned)n, by); }

// MT: 16-row tiles of an item.  SPREAD: the grid's z are the pieces of all entries
// of a head, one entry after the other; else its y are the entries and z the
// pieces of each.
template <int D, bool FP16, bool KV, int MT, bool SPREAD>
__global__ void __launch_bounds__(64 * rows_waves(D, MT), D <= 128 && MT == 1 ? 4 : 1) mx_rows_kernel(const RowsParams p) {
  constexpr int ROWS_WAVES = rows_waves(D, MT);
  constexpr int ROWS_THREADS = 64 * ROWS_WAVES;
  constexpr int CH = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int KSTEPS = D / 32;              // products of a 16-key block of S^T
  constexpr int DBLK = D / 16;                // 16-row blocks of O^T
  constexpr float TAU = 8.0f;
  constexpr int WORDS = D / 32;               // 4-byte words of codes in a quarter row
  constexpr int NB = D / 128 > 0 ? D / 128 : 1;  // scale bytes of a quarter row
  constexpr int WLDS = rows_wave_lds<D>();
  constexpr int ROWS = MT * ROWS_M;
  __shared__ u32x4 lds[ROWS_WAVES * WLDS / 16];
  __shared__ float sm[ROWS_WAVES][ROWS], sl[ROWS_WAVES][ROWS], smax[ROWS];
  __shared__ int slast;

  const int tid = (int)threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  char* const vS = reinterpret_cast<char*>(lds) + wave * WLDS;

  // ---- the item and its steps [t0, t1): the slab's, then the fresh keys'
  const int hr = (int)blockIdx.x;
  const int rt = quotient(hr, p.by_HKV);
  const int h = hr - rt * p.HKV;
  const int row_first = rt * ROWS;
  const int rows = min(p.R - row_first, ROWS);
  int b = (int)blockIdx.y, piece = (int)blockIdx.z, steps = p.steps, Pc = p.P;
  const int fresh = cdiv_i(p.SN, ROWS_N);
  if constexpr (SPREAD) {
    // lanes hold the entries first + lane
    auto length = [&](int first) { return first + lane < p.B ? min(max(gload_i32(p.lengths + first + lane), 0), p.P) : 0; };
    auto steps_of = [&](int first, int len) { return first + lane < p.B ? cdiv_i(len, ROWS_N) + fresh : 0; };
    const int own = length(0);
    int sum = steps_of(0, own);  // (the host: less than 2^30 in all)
    for (int first = 64; first < p.B; first += 64) sum += steps_of(first, length(first));
    sum = __builtin_amdgcn_readlane(wave_scan(sum), 63);
    // (so the pieces are spread + B at most, the grid's z)
    steps = max(__builtin_amdgcn_readfirstlane((int)((unsigned)(sum + p.spread - 1) / (unsigned)p.spread)), steps);
    int before = 0;
    b = -1;
    for (int first = 0; first < p.B && b < 0; first += 64) {
      const int len = first == 0 ? own : length(first);
      const int n = first + lane < p.B ? max((int)((unsigned)(steps_of(first, len) + steps - 1) / (unsigned)steps), 1) : 0;
      const int upto = wave_scan(n), all = __builtin_amdgcn_readlane(upto, 63);
      if (piece - before < all) {
        const int l = __builtin_ctzll(__ballot(upto > piece - before));
        b = first + l;
        piece -= before + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l);
        Pc = __builtin_amdgcn_readlane(len, l);
      }
      before += all;
    }
    if (b < 0) return;
  } else if (p.lengths != nullptr) {
    Pc = min(max(*((const __attribute__((address_space(4))) int32_t*)(p.lengths + b)), 0), p.P);
  }
  const int slab = cdiv_i(Pc, ROWS_N);
  const int T = slab + fresh;
  const int t0 = piece * steps;
  if (t0 >= T && t0 > 0) return;
  const int pieces = max((T + steps - 1) / steps, 1);
  const int s1 = p.P;  // absolute index of the first fresh key

  // Q as the B operand: lane holds Q[m, g * D/4 + 8j .. + 8], the order in which
  // the codes of a quarter row come; and each row's causal length
  u32x4 qreg[MT][KSTEPS];
  int Lrow[MT];
  int Lmax = p.KV - 1, Lmin = p.KV - 1;
  if (!p.uniform) Lmax = -1, Lmin = INT_MAX;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = row_first + mt * ROWS_M + l16;
    const bool live = m < p.R;
    const int mrd = live ? m : p.R - 1;
    const int tok = quotient(mrd, p.by_G);
    const int head = h * p.G + (mrd - tok * p.G);
    const char* qr = p.q + (b * p.sq[0] + (int64_t)tok * p.sq[1] + head * p.sq[2]) * 2 + g * (D / 2);
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) qreg[mt][j] = gload16(qr + 16 * j);
    Lrow[mt] = p.KV - 1;
    if (!p.uniform) {
      const int Lraw = max(gload_i32(p.L + b * p.sL_b + tok), -1);  // (any negative length: Lrow - kv0 stays in range)
      Lrow[mt] = live ? Lraw : -1;
      Lmax = max(Lmax, Lrow[mt]);
      Lmin = min(Lmin, live ? Lraw : INT_MAX);
    }
  }
  // the steps that a row sees
  int t1 = min(T, t0 + steps);
  if (!p.uniform) {
    Lmax = wave_reduce_i32<true>(Lmax);
    Lmin = wave_reduce_i32<false>(Lmin);
    t1 = min(t1, Lmax >= s1 ? slab + (Lmax - s1) / ROWS_N + 1 : min(slab, Lmax >= 0 ? Lmax / ROWS_N + 1 : 0));
  }

  const char* const kcb = p.k_codes + b * p.skc[0] + h * p.skc[2];
  const char* const vcb = p.v_codes + b * p.svc[0] + h * p.svc[2];
  const char* const ksb = p.k_scales + b * p.sks[0] + h * p.sks[2];
  const char* const vsb = p.v_scales + b * p.svs[0] + h * p.svs[2];
  const char* const knb = p.k_new + (b * p.skn[0] + h * p.skn[2]) * 2;
  const char* const vnb = p.v_new + (b * p.svn[0] + h * p.svn[2]) * 2;
  const int kcs = (int)p.skc[1], vcs = (int)p.svc[1], kss = (int)p.sks[1], vss = (int)p.svs[1];
  const int kns = (int)(p.skn[1] * 2), vns = (int)(p.svn[1] * 2);

  // a step's codes of this lane's two keys (l16 and l16 + 16) and quarter row
  // (g), and their scale bytes
  struct Step {
    unsigned kc[2][WORDS], vc[2][WORDS];
    unsigned ks[2], vs[2], valid[2];
  };
  auto rows_bytes = [](int n_in, int stride, int bytes) {
    const int n = min(n_in, ROWS_N);
    return n > 0 ? (n - 1) * stride + bytes : 0;
  };
  auto load_words = [&](unsigned (&w)[WORDS], const __amdgpu_buffer_rsrc_t rs, uint32_t off) {
    if constexpr (WORDS >= 4) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16 * i, 0, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
      }
    } else if constexpr (WORDS == 2) {
      const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
      w[0] = v[0];
      w[1] = v[1];
    } else {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
    }
  };
  auto load_scales = [&](const __amdgpu_buffer_rsrc_t rs, uint32_t row) -> unsigned {
    if constexpr (NB == 2) return __builtin_amdgcn_raw_buffer_load_b16(rs, row + 2 * g, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b8(rs, row + g * (D / 4) / 32, 0, 0);
  };
  auto load_valid = [&](int kv0, int n_in, unsigned (&valid)[2]) {
    if constexpr (KV) {
      const auto rs = make_rsrc(reinterpret_cast<const char*>(p.key_valid) + b * p.svalid_b + kv0,
                                __builtin_amdgcn_readfirstlane(min(n_in, ROWS_N)));
#pragma unroll
      for (int i = 0; i < 2; ++i) valid[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, (uint32_t)(l16 + 16 * i), 0, 0);
    }
  };
  auto load_step = [&](int t, Step& s) {
    const int row0 = t * ROWS_N, n_in = Pc - row0;
    const auto rk = make_rsrc(kcb + (int64_t)row0 * kcs, rows_bytes(n_in, kcs, D / 2));
    const auto rv = make_rsrc(vcb + (int64_t)row0 * vcs, rows_bytes(n_in, vcs, D / 2));
    const auto rks = make_rsrc(ksb + (int64_t)row0 * kss, rows_bytes(n_in, kss, D / 32));
    const auto rvs = make_rsrc(vsb + (int64_t)row0 * vss, rows_bytes(n_in, vss, D / 32));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load_words(s.kc[i], rk, (uint32_t)((l16 + 16 * i) * kcs + g * (D / 8)));
      s.ks[i] = load_scales(rks, (uint32_t)((l16 + 16 * i) * kss));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load_words(s.vc[i], rv, (uint32_t)((l16 + 16 * i) * vcs + g * (D / 8)));
      s.vs[i] = load_scales(rvs, (uint32_t)((l16 + 16 * i) * vss));
    }
    load_valid(row0, n_in, s.valid);
  };
  // 2^(byte - 127) of word j's block
  auto scale_of = [](unsigned bytes, int j) { return __uint_as_float(((bytes >> (8 * (j / 4))) & 0xffu) << 23); };

  float m_run[MT], l_run[MT];
  f32x4 oacc[MT][DBLK];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m_run[mt] = -INFINITY;
    l_run[mt] = 0.0f;
#pragma unroll
    for (int db = 0; db < DBLK; ++db) oacc[mt][db] = f32x4{};
  }

  // V^T operand: the transpose read gives lane l16 column 16 db + l16 of four
  // rows; rows 4g .. 4g + 3 and the same 16 on, whose chunks swz leaves at the
  // same places
  const int rq = 4 * g + (l16 >> 2);
  int voffs[DBLK];
#pragma unroll
  for (int db = 0; db < DBLK; ++db)
    voffs[db] = rq * ROWB + (((2 * db + ((l16 & 3) >> 1)) ^ swz<CH>(rq)) << 4) + 8 * (l16 & 1);
  auto put_v = [&](int i, int j, u32x4 v) {
    const int key = l16 + 16 * i;
    *reinterpret_cast<u32x4*>(vS + key * ROWB + (((g * WORDS + j) ^ swz<CH>(key)) << 4)) = v;
  };

  // softmax and PV of one step: sa holds S^T (lane: row l16, keys 16s + 4g + i),
  // the wave's LDS its V
  auto finish_step = [&](f32x4 (&sa)[MT][2], int kv0, int n_in, const unsigned (&valid)[2]) {
    [[maybe_unused]] unsigned vm = ~0u;
    if constexpr (KV) vm = ((unsigned)__ballot(valid[0] != 0u) & 0xffffu) | ((unsigned)__ballot(valid[1] != 0u) << 16);
    const bool masked = !(n_in >= ROWS_N && kv0 + ROWS_N - 1 <= Lmin && (!KV || vm == ~0u));
    u32x4 pb[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (masked) {
        const int lim = min(Lrow[mt] - kv0, n_in - 1) - 4 * g;
        const unsigned mine = vm >> (4 * g);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bool ok = 16 * s + i <= lim;
            if constexpr (KV) ok = ok && ((mine >> (16 * s + i)) & 1u) != 0;
            sa[mt][s][i] = ok ? sa[mt][s][i] : -INFINITY;
          }
      }
      float mx = sa[mt][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sa[mt][e / 4][e % 4]);
      mx = quad_max(mx) * p.qk_scale;
      if (__any(mx > m_run[mt] + TAU)) {
        const float m_new = fmaxf(m_run[mt], mx);
        const float alpha = (m_new == -INFINITY) ? 1.0f : __builtin_amdgcn_exp2f(m_run[mt] - m_new);
        l_run[mt] *= alpha;
#pragma unroll
        for (int db = 0; db < DBLK; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) oacc[mt][db][i] *= alpha;
        m_run[mt] = m_new;
      }
      const float m_safe = (m_run[mt] == -INFINITY) ? 0.0f : m_run[mt];
      float rs = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sa[mt][e / 4][e % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(sa[mt][e / 4][e % 4], p.qk_scale, -m_safe));
        rs += sa[mt][e / 4][e % 4];
      }
      l_run[mt] += rs;
      pb[mt] = u32x4{pack2<FP16>(sa[mt][0][0], sa[mt][0][1]), pack2<FP16>(sa[mt][0][2], sa[mt][0][3]),
                     pack2<FP16>(sa[mt][1][0], sa[mt][1][1]), pack2<FP16>(sa[mt][1][2], sa[mt][1][3])};
    }
    // the wave's own LDS stores are done in order before its reads; the empty
    // asm keeps the compiler from moving either across
    asm volatile("" ::: "memory");
#pragma unroll
    for (int db = 0; db < DBLK; ++db) {
      const u32x2 w0 = __builtin_bit_cast(u32x2, lds_read_tr16(vS + voffs[db]));
      const u32x2 w1 = __builtin_bit_cast(u32x2, lds_read_tr16(vS + voffs[db] + 16 * ROWB));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        oacc[mt][db] = mfma16<FP16>(u32x4{w0.x, w0.y, w1.x, w1.y}, pb[mt], oacc[mt][db]);
    }
    asm volatile("" ::: "memory");
  };

  Step cur = {};
  int t = t0 + wave;
  if (t < min(t1, slab)) load_step(t, cur);
  for (; t < t1; t += ROWS_WAVES) {
    f32x4 sa[MT][2];
    int kv0 = t * ROWS_N, n_in = Pc - kv0;
    unsigned valid[2] = {cur.valid[0], cur.valid[1]};
    if (t < slab) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j) {
          const u32x4 kw = dequant_fp4x8<FP16>(cur.kc[i][j], scale_of(cur.ks[i], j));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) sa[mt][i] = mfma16<FP16>(kw, qreg[mt][j], j == 0 ? f32x4{} : sa[mt][i]);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool on = !KV || valid[i] != 0u;  // a hidden key's V counts as zeros, whatever it held
#pragma unroll
        for (int j = 0; j < WORDS; ++j)
          put_v(i, j, dequant_fp4x8<FP16>(on ? cur.vc[i][j] : 0u, on ? scale_of(cur.vs[i], j) : 1.0f));
      }
      if (t + ROWS_WAVES < min(t1, slab)) load_step(t + ROWS_WAVES, cur);
    } else {
      // fresh keys
      const int row0 = (t - slab) * ROWS_N;
      kv0 = s1 + row0;
      n_in = p.SN - row0;
      const auto rk = make_rsrc(knb + (int64_t)row0 * kns, rows_bytes(n_in, kns, ROWB));
      const auto rv = make_rsrc(vnb + (int64_t)row0 * vns, rows_bytes(n_in, vns, ROWB));
      load_valid(kv0, n_in, valid);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j) {
          const u32x4 kw = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                         rk, (uint32_t)((l16 + 16 * i) * kns + g * (D / 2) + 16 * j), 0, 0));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) sa[mt][i] = mfma16<FP16>(kw, qreg[mt][j], j == 0 ? f32x4{} : sa[mt][i]);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool on = !KV || valid[i] != 0u;
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j) {
          const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                        rv, (uint32_t)((l16 + 16 * i) * vns + g * (D / 2) + 16 * j), 0, 0));
          put_v(i, j, on ? w : u32x4{0u, 0u, 0u, 0u});
        }
      }
    }
    finish_step(sa, kv0, n_in, valid);
  }

  // ---- the waves' states become the piece's: m through LDS, then O tile by
  // tile and l, scaled to the rows' largest m, each wave's in its own LDS, and
  // added in wave order
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
    if (g == 0) sm[wave][mt * ROWS_M + l16] = m_run[mt];
  __syncthreads();
  // 1 / l, 0 for a row without keys, NaN for a NaN
  auto inverse = [](float l) {
    const bool pos = l > 0.0f;
    return (1.0f / (pos ? l : 1.0f)) * (pos ? 1.0f : l - l);
  };
  constexpr int C4 = D / 4;                    // four-element pieces of a row
  constexpr int SC1 = 16;                      // cache policy: device scope
  // the output of piece c of the item's row r
  auto put_out = [&](int r, int c, f32x4 v, float l) {
    const float inv = inverse(l);
    const int m = row_first + r;
    const int tok = quotient(m, p.by_G);
    const int head = h * p.G + (m - tok * p.G);
    gstore8(p.out + (b * p.so[0] + (int64_t)tok * p.so[1] + head * p.so[2]) * 2 + c * 8,
            u32x2{pack2<FP16>(v[0] * inv, v[1] * inv), pack2<FP16>(v[2] * inv, v[3] * inv)});
  };
  const int item = b * (int)gridDim.x + hr;
  const int slot = rows_slot(D, 1 << p.row_bits);  // bytes of a piece
  const int ml_at = (D * 4) << p.row_bits;         // of its (m, l)
  // the item's pieces (gridDim.z at most, less than 2^31 bytes)
  const int64_t first_slot = SPREAD ? (int64_t)hr * (int)gridDim.z + ((int)blockIdx.z - piece) : (int64_t)item * (int)gridDim.z;
  const auto slots = make_rsrc(reinterpret_cast<const char*>(p.part) + first_slot * slot, pieces == 1 ? 0 : pieces * slot);
  const uint32_t mine = (uint32_t)(piece * slot);
  auto piece_at = [](int r, int c) { return r * (D * 4) + ((c ^ (r & (C4 - 1) & 15)) << 4); };
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r0 = mt * ROWS_M;
    float M = sm[0][r0 + l16];
#pragma unroll
    for (int w = 1; w < ROWS_WAVES; ++w) M = fmaxf(M, sm[w][r0 + l16]);
    const float a = (m_run[mt] == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f(m_run[mt] - M);
    const float l_tot = quad_sum(l_run[mt]) * a;
    if (g == 0) {
      sl[wave][r0 + l16] = l_tot;
      if (wave == 0) smax[r0 + l16] = M;
    }
    if (r0 + l16 < rows) {
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const f32x4 o = oacc[mt][db];
        *reinterpret_cast<f32x4*>(vS + piece_at(l16, 4 * db + g)) = f32x4{o[0] * a, o[1] * a, o[2] * a, o[3] * a};
      }
    }
    __syncthreads();
    for (int i = tid; i < min(rows - r0, ROWS_M) * C4; i += ROWS_THREADS) {
      const int r = i / C4, c = i % C4;
      f32x4 v = f32x4{};
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < ROWS_WAVES; ++w) {
        v += *reinterpret_cast<const f32x4*>(reinterpret_cast<char*>(lds) + w * WLDS + piece_at(r, c));
        l += sl[w][r0 + r];
      }
      if (pieces == 1) {
        put_out(r0 + r, c, v, l);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), slots, mine + (uint32_t)((r0 * C4 + i) * 16), 0, SC1);
        if (c == 0)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{smax[r0 + r], l}), slots,
                                                mine + (uint32_t)(ml_at + (r0 + r) * 8), 0, SC1);
      }
    }
    if (mt + 1 < MT) __syncthreads();
  }
  if (pieces == 1) return;

  // ---- the last piece of the item to arrive combines them.  Ordering at
  // device scope as in qik_attn_kernel.h: the stores above write through and
  // are complete (vmcnt 0, every wave, then the barrier) before the arrival;
  // the slots are read with device-scope loads issued after it.
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  if (tid == 0) {
    const bool last = g_fetch_add(p.ctl + item, 1u) == (unsigned)pieces - 1u;
    if (last) g_store(p.ctl + item, 0u);
    slast = last ? 1 : 0;
  }
  __syncthreads();
  if (slast == 0) return;

  // A thread takes four elements of a row; where those are fewer than the
  // threads, groups of threads take every ng-th piece each.  Every one runs the
  // online softmax over its pieces (no pass over the m first), and the groups' states are combined in group order.
  struct State {
    f32x4 v;
    float m, l;
  };
  static_assert(sizeof(State) * ROWS_THREADS <= sizeof(lds), "the groups' states fit");
  auto add = [](State& s, f32x4 v, float l, float x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s.v[e] = __builtin_fmaf(v[e], x, s.v[e]);
    s.l = __builtin_fmaf(l, x, s.l);
  };
  float* const states = reinterpret_cast<float*>(lds);  // [6][threads]
  const int n4_bits = __builtin_ctz(C4) + p.row_bits;   // log2 of the item's four-element pieces
  const int ng = max(ROWS_THREADS >> n4_bits, 1);
  for (int i = tid; i < (ng << n4_bits); i += ROWS_THREADS) {
    const int at = i & ((1 << n4_bits) - 1);
    State s = {f32x4{}, -INFINITY, 0.0f};
    // AHEAD pieces at a time (past the last: zeros, which the buffer's end gives,
    // of weight zero); one after the other they cost their latency each
    constexpr int AHEAD = 8;
    for (int n = i >> n4_bits; n < pieces; n += AHEAD * ng) {
      f32x4 v[AHEAD];
      f32x2 ml[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint32_t off = (uint32_t)((n + k * ng) * slot);
        v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(slots, off + (uint32_t)(at * 16), 0, SC1));
        ml[k] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(slots, off + (uint32_t)(ml_at + at / C4 * 8), 0, SC1));
      }
      float m = s.m;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (n + k * ng >= pieces) ml[k][0] = -INFINITY;
        m = fmaxf(m, ml[k][0]);
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      const float a = __builtin_amdgcn_exp2f(s.m - ref);  // 0 for -inf, as below
#pragma unroll
      for (int e = 0; e < 4; ++e) s.v[e] *= a;
      s.l *= a;
      s.m = m;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) add(s, v[k], ml[k][1], __builtin_amdgcn_exp2f(ml[k][0] - ref));
    }
    if (ng == 1) {
      if (at / C4 < rows) put_out(at / C4, at % C4, s.v, s.l);
      continue;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) states[e * ROWS_THREADS + i] = s.v[e];
    states[4 * ROWS_THREADS + i] = s.m;
    states[5 * ROWS_THREADS + i] = s.l;
  }
  if (ng == 1) return;
  __syncthreads();
  if (tid < (1 << n4_bits) && tid / C4 < rows) {
    const float* const x = states + tid;
    float m = -INFINITY;
    for (int n = 0; n < ng; ++n) m = fmaxf(m, x[4 * ROWS_THREADS + (n << n4_bits)]);
    const float ref = m == -INFINITY ? 0.0f : m;
    State s = {f32x4{}, m, 0.0f};
    for (int n = 0; n < ng; ++n) {
      const float* y = x + (n << n4_bits);
      add(s, f32x4{y[0], y[ROWS_THREADS], y[2 * ROWS_THREADS], y[3 * ROWS_THREADS]}, y[5 * ROWS_THREADS],
          __builtin_amdgcn_exp2f(y[4 * ROWS_THREADS] - ref));
    }
    put_out(tid / C4, tid % C4, s.v, s.l);
  }
}

}  // namespace qik

#endif  // QIK_MX_ROWS_H

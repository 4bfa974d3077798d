// Attention of few query rows over a 4-bit slab and fresh keys (gfx950): a
// token's heads, or some tokens', against a cache of any length.
//
// The mathematics is the tile loop's of qik_attn_kernel.h (S^T = K.Q^T, online
// softmax in the exp2 domain with a lazy reference point, O^T = V^T.P^T on
// v_mfma_f32_32x32x16), but such a call is bound by the slab's bytes: 17/32 of
// a byte per element of K and V, each read once.  So:
//   * a workgroup holds up to 32 query rows of one (b, KV head) -- the query heads
//     that share the KV head times the query positions -- and one slice of its
//     keys; its four waves take the slice's steps of 32 keys in turn, each with
//     its own softmax state, and never wait for each other before the end;
//   * K goes from memory to the matrix cores through registers alone.  The
//     order of the head dim inside a dot product is free, as long as Q has the
//     same: lane (key, half) holds its key's half row, 16 to 64 contiguous bytes
//     of codes, and every 4 bytes become one operand;
//   * V is turned into the element type in registers and goes through the
//     wave's own LDS, whose transpose read gives the V^T operand;
//   * the next step's codes are loaded before the present step is computed;
//   * the slices of a (b, KV head) leave their (m, l, O) in the workspace, and
//     the last to arrive combines them in slice order, so that the result does
//     not depend on which one that is.
#ifndef QIK_MX_ROWS_H
#define QIK_MX_ROWS_H

#include "qik_attn_kernel.h"

namespace qik {

constexpr int ROWS_WAVES = 4;
constexpr int ROWS_N = 32;        // keys of a step
constexpr int ROWS_M = 32;        // query rows of a workgroup
constexpr int ROWS_THREADS = ROWS_WAVES * 64;

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
  unsigned* ctl;             // arrivals per item, zero between launches (nsplit > 1)
  float* part;               // per (item, slice): rows x D accumulators, then rows (m, l)
  int64_t sq[3], skn[3], svn[3], so[3];  // b, s, h in elements
  int64_t skc[3], svc[3], sks[3], svs[3];  // b, p, h in bytes
  int64_t svalid_b, sL_b;
  int R;                     // query rows of a KV head: SQ * G, row r is head r % G of position r / G
  int SN, P, HKV, G, KV;
  int uniform;
  int nrt, nsplit;           // row tiles of a KV head, slices of its keys
  int prow;                  // rows a slice keeps in the workspace: min(R, ROWS_M)
  float qk_scale;
};

// LDS bytes of one wave: its V step, and at the end its share of O (half of the
// head dim at a time)
template <int D>
constexpr int rows_wave_lds() { return D * 2 * ROWS_N > 4096 ? D * 2 * ROWS_N : 4096; }
// the merge keeps (m, l) of every slice and row there, beside 16 bytes a thread
template <int D>
constexpr int rows_max_splits(int rows) { return (ROWS_WAVES * rows_wave_lds<D>() - 16 * ROWS_THREADS) / 8 / rows; }
// fp32 values a slice of `rows` rows keeps in the workspace: O, then (m, l) of each row
template <int D>
__host__ __device__ constexpr int rows_slot(int rows) { return (rows * (D + 2) + 3) / 4 * 4; }

template <int D, bool FP16, bool KV>
__global__ void __launch_bounds__(ROWS_THREADS, D <= 128 ? 2 : 1) mx_rows_kernel(const RowsParams p) {
  constexpr int CH = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int KSTEPS = D / 16;
  constexpr int DBLK = D / 32;
  constexpr float TAU = 8.0f;
  constexpr int WORDS = D / 16;               // 4-byte words of codes in half a row
  constexpr int NB = D >= 64 ? D / 64 : 1;    // blocks (scale bytes) of half a row
  constexpr int WLDS = rows_wave_lds<D>();
  __shared__ u32x4 lds[ROWS_WAVES * WLDS / 16];
  __shared__ float sm[ROWS_WAVES][ROWS_M], sl[ROWS_WAVES][ROWS_M];
  __shared__ int slast;

  const int tid = (int)threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, l32 = lane & 31;
  char* const vS = reinterpret_cast<char*>(lds) + wave * WLDS;

  // workgroup -> (row tile, slice, batch entry, KV head): the row tiles of one
  // slice are a multiple of the slices apart, so they share an XCD's L2 when
  // that is a multiple of the XCDs
  const int per = (int)(gridDim.x / (unsigned)p.nrt);
  const int rt = (int)blockIdx.x / per;
  const int rest = (int)blockIdx.x - rt * per;
  const int bh = rest / p.nsplit;
  const int slice = rest - bh * p.nsplit;
  const int b = bh / p.HKV;
  const int h = bh - b * p.HKV;

  const int m = rt * ROWS_M + l32;
  const bool live = m < p.R;
  const int mrd = live ? m : p.R - 1;
  const int tok = (int)((unsigned)mrd / (unsigned)p.G);
  const int head = h * p.G + (mrd - tok * p.G);
  const int rows = min(p.R - rt * ROWS_M, ROWS_M);

  int Pc = p.P;
  if (p.lengths != nullptr) Pc = __builtin_amdgcn_readfirstlane(min(max(gload_i32(p.lengths + b), 0), p.P));
  int Lrow = p.KV - 1, Lmax = p.KV - 1, Lmin = p.KV - 1;
  if (!p.uniform) {
    const int Lraw = gload_i32(p.L + b * p.sL_b + tok);
    Lrow = live ? Lraw : -1;
    Lmax = wave_reduce_i32<true>(Lrow);
    Lmin = wave_reduce_i32<false>(live ? Lraw : INT_MAX);
  }

  // Q as the B operand: lane holds Q[m, hf * D/2 + 8j .. + 8], the order in
  // which the codes of half a row come
  u32x4 qreg[KSTEPS];
  {
    const char* qr = p.q + (b * p.sq[0] + (int64_t)tok * p.sq[1] + head * p.sq[2]) * 2 + hf * D;
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) qreg[j] = gload16(qr + 16 * j);
  }

  const char* const kcb = p.k_codes + b * p.skc[0] + h * p.skc[2];
  const char* const vcb = p.v_codes + b * p.svc[0] + h * p.svc[2];
  const char* const ksb = p.k_scales + b * p.sks[0] + h * p.sks[2];
  const char* const vsb = p.v_scales + b * p.svs[0] + h * p.svs[2];
  const char* const knb = p.k_new + (b * p.skn[0] + h * p.skn[2]) * 2;
  const char* const vnb = p.v_new + (b * p.svn[0] + h * p.svn[2]) * 2;
  const int kcs = (int)p.skc[1], vcs = (int)p.svc[1], kss = (int)p.sks[1], vss = (int)p.svs[1];
  const int kns = (int)(p.skn[1] * 2), vns = (int)(p.svn[1] * 2);
  const int s1 = p.P;  // absolute index of the first fresh key

  // steps: the slab's, then the fresh keys'; this slice's, dealt to the waves in turn
  const int run0 = Lmax >= 0 ? min(cdiv_i(Pc, ROWS_N), Lmax / ROWS_N + 1) : 0;
  const int run1 = Lmax >= s1 ? min(cdiv_i(p.SN, ROWS_N), (Lmax - s1) / ROWS_N + 1) : 0;
  const int T = run0 + run1;
  const int t0 = (int)((int64_t)T * slice / p.nsplit);
  const int t1 = (int)((int64_t)T * (slice + 1) / p.nsplit);

  // a step's codes of this lane's key (l32) and half row (hf), and its scale bytes
  struct Step {
    unsigned kc[WORDS], vc[WORDS];
    unsigned ks, vs;
    unsigned valid;
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
    } else {
      const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
      w[0] = v[0];
      w[1] = v[1];
    }
  };
  auto load_scales = [&](const __amdgpu_buffer_rsrc_t rs, uint32_t row) -> unsigned {
    if constexpr (NB == 4) return __builtin_amdgcn_raw_buffer_load_b32(rs, row + 4 * hf, 0, 0);
    if constexpr (NB == 2) return __builtin_amdgcn_raw_buffer_load_b16(rs, row + 2 * hf, 0, 0);
    return __builtin_amdgcn_raw_buffer_load_b8(rs, row + (D == 32 ? 0 : hf), 0, 0);
  };
  auto load_valid = [&](int kv0, int n_in) -> unsigned {
    if constexpr (KV) {
      const auto rs = make_rsrc(reinterpret_cast<const char*>(p.key_valid) + b * p.svalid_b + kv0,
                                __builtin_amdgcn_readfirstlane(min(n_in, ROWS_N)));
      return __builtin_amdgcn_raw_buffer_load_b8(rs, (uint32_t)l32, 0, 0);
    }
    return 1u;
  };
  auto load_step = [&](int t, Step& s) {
    const int row0 = t * ROWS_N, n_in = Pc - row0;
    const auto rk = make_rsrc(kcb + (int64_t)row0 * kcs, rows_bytes(n_in, kcs, D / 2));
    const auto rv = make_rsrc(vcb + (int64_t)row0 * vcs, rows_bytes(n_in, vcs, D / 2));
    const auto rks = make_rsrc(ksb + (int64_t)row0 * kss, rows_bytes(n_in, kss, D / 32));
    const auto rvs = make_rsrc(vsb + (int64_t)row0 * vss, rows_bytes(n_in, vss, D / 32));
    load_words(s.kc, rk, (uint32_t)(l32 * kcs + hf * (D / 4)));
    s.ks = load_scales(rks, (uint32_t)(l32 * kss));
    load_words(s.vc, rv, (uint32_t)(l32 * vcs + hf * (D / 4)));
    s.vs = load_scales(rvs, (uint32_t)(l32 * vss));
    s.valid = load_valid(row0, n_in);
  };
  // 2^(byte - 127) of word j's block
  auto scale_of = [](unsigned bytes, int j) { return __uint_as_float(((bytes >> (8 * (j / 4))) & 0xffu) << 23); };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16 oacc[DBLK];
#pragma unroll
  for (int db = 0; db < DBLK; ++db) oacc[db] = f32x16{};

  const int j16 = lane & 15;
  const int rq = 4 * hf + (j16 >> 2);
  const int colq = 16 * ((lane >> 4) & 1) + 4 * (j16 & 3);
  int voffs[2][DBLK];
#pragma unroll
  for (int db = 0; db < DBLK; ++db) {
    const int col = db * 32 + colq;
    voffs[0][db] = rq * ROWB + (((col >> 3) ^ swz<CH>(rq)) << 4) + ((col & 7) << 1);
    voffs[1][db] = (rq + 8) * ROWB + (((col >> 3) ^ swz<CH>(rq + 8)) << 4) + ((col & 7) << 1);
  }
  auto put_v = [&](int j, u32x4 v) {
    *reinterpret_cast<u32x4*>(vS + l32 * ROWB + (((hf * WORDS + j) ^ swz<CH>(l32)) << 4)) = v;
  };

  // softmax and PV of one step: sa holds S^T (lane: row l32, keys 8(i/4) + 4hf
  // + i%4), the wave's LDS its V
  auto finish_step = [&](f32x16& sa, int kv0, int n_in, unsigned valid) {
    [[maybe_unused]] unsigned vm = ~0u;
    if constexpr (KV) vm = (unsigned)__ballot(valid != 0u);
    if (!(n_in >= ROWS_N && kv0 + ROWS_N - 1 <= Lmin && (!KV || vm == ~0u))) {
      const int lim = min(Lrow - kv0, n_in - 1) - 4 * hf;
      const unsigned mine = vm >> (4 * hf);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int na = 8 * (i >> 2) + (i & 3);
        bool ok = na <= lim;
        if constexpr (KV) ok = ok && ((mine >> na) & 1u) != 0;
        sa[i] = ok ? sa[i] : -INFINITY;
      }
    }
    float mx = sa[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sa[i]);
    mx = pair_max(mx) * p.qk_scale;
    if (__any(mx > m_run + TAU)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = (m_new == -INFINITY) ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DBLK; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[db][i] *= alpha;
      m_run = m_new;
    }
    const float m_safe = (m_run == -INFINITY) ? 0.0f : m_run;
    float rs = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sa[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sa[i], p.qk_scale, -m_safe));
      rs += sa[i];
    }
    l_run += rs;
    // the wave's own LDS stores are done in order before its reads; the empty
    // asm keeps the compiler from moving either across
    asm volatile("" ::: "memory");
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 pb;
      pb.x = pack2<FP16>(sa[8 * s + 0], sa[8 * s + 1]);
      pb.y = pack2<FP16>(sa[8 * s + 2], sa[8 * s + 3]);
      pb.z = pack2<FP16>(sa[8 * s + 4], sa[8 * s + 5]);
      pb.w = pack2<FP16>(sa[8 * s + 6], sa[8 * s + 7]);
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const u32x2 w0 = __builtin_bit_cast(u32x2, lds_read_tr16(vS + voffs[0][db] + 16 * s * ROWB));
        const u32x2 w1 = __builtin_bit_cast(u32x2, lds_read_tr16(vS + voffs[1][db] + 16 * s * ROWB));
        oacc[db] = mfma32<FP16>(u32x4{w0.x, w0.y, w1.x, w1.y}, pb, oacc[db]);
      }
    }
    asm volatile("" ::: "memory");
  };

  // ---- the slab's steps
  const int e0 = min(t1, run0);
  int t = t0 + wave;
  Step next;
  if (t < e0) load_step(t, next);
  for (; t < e0; t += ROWS_WAVES) {
    const Step cur = next;
    if (t + ROWS_WAVES < e0) load_step(t + ROWS_WAVES, next);
    const int n_in = Pc - t * ROWS_N;
    f32x16 sa = f32x16{};
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) sa = mfma32<FP16>(dequant_fp4x8<FP16>(cur.kc[j], scale_of(cur.ks, j)), qreg[j], sa);
    const bool on = !KV || cur.valid != 0u;  // a hidden key's V counts as zeros, whatever it held
#pragma unroll
    for (int j = 0; j < WORDS; ++j) put_v(j, dequant_fp4x8<FP16>(on ? cur.vc[j] : 0u, on ? scale_of(cur.vs, j) : 1.0f));
    finish_step(sa, t * ROWS_N, n_in, cur.valid);
  }
  // ---- the fresh keys'
  for (; t < t1; t += ROWS_WAVES) {
    const int row0 = (t - run0) * ROWS_N, n_in = p.SN - row0;
    const auto rk = make_rsrc(knb + (int64_t)row0 * kns, rows_bytes(n_in, kns, ROWB));
    const auto rv = make_rsrc(vnb + (int64_t)row0 * vns, rows_bytes(n_in, vns, ROWB));
    const unsigned valid = load_valid(s1 + row0, n_in);
    f32x16 sa = f32x16{};
    u32x4 kw[KSTEPS];
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j)
      kw[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, (uint32_t)(l32 * kns + hf * D + 16 * j), 0, 0));
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) sa = mfma32<FP16>(kw[j], qreg[j], sa);
    const bool on = !KV || valid != 0u;
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, (uint32_t)(l32 * vns + hf * D + 16 * j), 0, 0));
      put_v(j, on ? w : u32x4{0u, 0u, 0u, 0u});
    }
    finish_step(sa, s1 + row0, n_in, valid);
  }

  // ---- the waves' states become the slice's: m and l through LDS, then O in
  // halves of the head dim, each wave's rows in its own LDS, added in wave order
  const float l_tot = pair_sum(l_run);
  if (hf == 0) {
    sm[wave][l32] = m_run;
    sl[wave][l32] = l_tot;
  }
  __syncthreads();
  float M = sm[0][l32];
#pragma unroll
  for (int w = 1; w < ROWS_WAVES; ++w) M = fmaxf(M, sm[w][l32]);
  const float a = (m_run == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f(m_run - M);
  // l of the slice's row r, and of its reference point
  auto row_l = [&](int r, float* mrow) {
    float mm = sm[0][r], ll = 0.0f;
#pragma unroll
    for (int w = 1; w < ROWS_WAVES; ++w) mm = fmaxf(mm, sm[w][r]);
#pragma unroll
    for (int w = 0; w < ROWS_WAVES; ++w)
      ll += sl[w][r] * (sm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][r] - mm));
    *mrow = mm;
    return ll;
  };
  // 1 / l, 0 for a row without keys, NaN for a NaN
  auto inverse = [](float l) {
    const bool pos = l > 0.0f;
    return (1.0f / (pos ? l : 1.0f)) * (pos ? 1.0f : l - l);
  };
  auto out_row = [&](int r) {
    const int mm = rt * ROWS_M + r;
    const int tk = (int)((unsigned)mm / (unsigned)p.G);
    const int hd = h * p.G + (mm - tk * p.G);
    return p.out + (b * p.so[0] + (int64_t)tk * p.so[1] + hd * p.so[2]) * 2;
  };
  constexpr int DH = DBLK > 1 ? DBLK / 2 : 1;  // blocks of a pass
  constexpr int C4 = DH * 8;                   // four-element pieces of a row in a pass
  constexpr int SC1 = 16;                      // cache policy: device scope
  const int item = rt * (per / p.nsplit) + bh;
  const int slot = rows_slot<D>(p.prow) * 4;   // bytes of a slice
  const bool whole = p.nsplit == 1;
  // the item's slots (less than 2^31 bytes: rows_max_splits)
  const auto slots = make_rsrc(reinterpret_cast<const char*>(p.part) + (int64_t)item * p.nsplit * slot, whole ? 0 : p.nsplit * slot);
#pragma unroll
  for (int d0 = 0; d0 < DBLK; d0 += DH) {
    if (l32 < rows) {
#pragma unroll
      for (int db = 0; db < DH; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int c = db * 8 + 2 * q4 + hf;  // d = 4c .. 4c + 3 of the pass
          const f32x16& o = oacc[d0 + db];
          *reinterpret_cast<f32x4*>(vS + l32 * (C4 * 16) + ((c ^ (l32 & (C4 - 1))) << 4)) =
              f32x4{o[4 * q4] * a, o[4 * q4 + 1] * a, o[4 * q4 + 2] * a, o[4 * q4 + 3] * a};
        }
    }
    __syncthreads();
    for (int i = tid; i < rows * C4; i += ROWS_THREADS) {
      const int r = i / C4, c = i % C4;
      f32x4 v = f32x4{};
#pragma unroll
      for (int w = 0; w < ROWS_WAVES; ++w)
        v += *reinterpret_cast<const f32x4*>(reinterpret_cast<char*>(lds) + w * WLDS + r * (C4 * 16) + ((c ^ (r & (C4 - 1))) << 4));
      const int d = d0 * 32 + 4 * c;
      if (whole) {
        float mr;
        const float inv = inverse(row_l(r, &mr));
        gstore8(out_row(r) + d * 2, u32x2{pack2<FP16>(v[0] * inv, v[1] * inv), pack2<FP16>(v[2] * inv, v[3] * inv)});
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), slots, (uint32_t)(slice * slot + (r * D + d) * 4), 0, SC1);
      }
    }
    __syncthreads();
  }
  if (whole) return;
  if (tid < rows) {
    float mr;
    const float lr = row_l(tid, &mr);
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{mr, lr}), slots,
                                          (uint32_t)(slice * slot + (p.prow * D + 2 * tid) * 4), 0, SC1);
  }

  // ---- the last slice of the item to arrive combines them.  Ordering at
  // device scope as in qik_attn_kernel.h: the stores above write through and
  // are complete (vmcnt 0, every wave, then the barrier) before the arrival;
  // the slots are read with device-scope loads issued after it.
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  if (tid == 0) {
    const bool last = g_fetch_add(p.ctl + item, 1u) == (unsigned)p.nsplit - 1u;
    if (last) g_store(p.ctl + item, 0u);
    slast = last ? 1 : 0;
  }
  __syncthreads();
  if (slast == 0) return;

  f32x2* const ml = reinterpret_cast<f32x2*>(lds);  // [nsplit][rows]: (m, l), then (weight, -)
  f32x4* const sums = reinterpret_cast<f32x4*>(reinterpret_cast<char*>(lds) + ROWS_WAVES * WLDS - 16 * ROWS_THREADS);
  for (int i = tid; i < p.nsplit * rows; i += ROWS_THREADS) {
    const int s = i / rows, r = i - s * rows;
    ml[i] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(slots, (uint32_t)(s * slot + (p.prow * D + 2 * r) * 4), 0, SC1));
  }
  __syncthreads();
  if (tid < rows) {
    float mm = -INFINITY, ll = 0.0f;
    for (int s = 0; s < p.nsplit; ++s) mm = fmaxf(mm, ml[s * rows + tid][0]);
    for (int s = 0; s < p.nsplit; ++s) {
      const f32x2 x = ml[s * rows + tid];
      const float w = x[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[0] - mm);
      ll = __builtin_fmaf(x[1], w, ll);
      ml[s * rows + tid] = f32x2{w, 0.0f};
    }
    sm[0][tid] = inverse(ll);
  }
  __syncthreads();
  // one thread per four elements of a row; where they are fewer than the
  // threads, groups of threads take every ng-th slice each, and their sums are
  // added in group order
  const int n4 = rows * (D / 4);
  const int ng = max(ROWS_THREADS / n4, 1);
  for (int i = tid; i < n4 * ng; i += ROWS_THREADS) {
    const int g = i / n4, at = i - g * n4;
    const int r = at / (D / 4), c = at % (D / 4);
    f32x4 v = f32x4{};
#pragma unroll 8
    for (int s = g; s < p.nsplit; s += ng) {
      const f32x4 x = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(slots, (uint32_t)(s * slot + (r * D + 4 * c) * 4), 0, SC1));
      const float w = ml[s * rows + r][0];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(x[e], w, v[e]);
    }
    if (ng > 1) {
      sums[i] = v;
      continue;
    }
    const float inv = sm[0][r];
    gstore8(out_row(r) + c * 8, u32x2{pack2<FP16>(v[0] * inv, v[1] * inv), pack2<FP16>(v[2] * inv, v[3] * inv)});
  }
  if (ng == 1) return;
  __syncthreads();
  for (int i = tid; i < n4; i += ROWS_THREADS) {
    const int r = i / (D / 4), c = i % (D / 4);
    f32x4 v = sums[i];
    for (int g = 1; g < ng; ++g) v += sums[g * n4 + i];
    const float inv = sm[0][r];
    gstore8(out_row(r) + c * 8, u32x2{pack2<FP16>(v[0] * inv, v[1] * inv), pack2<FP16>(v[2] * inv, v[3] * inv)});
  }
}

}  // namespace qik

#endif  // QIK_MX_ROWS_H

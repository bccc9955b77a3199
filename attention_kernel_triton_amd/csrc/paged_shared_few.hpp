// Units of few rows in a launch with shared prefixes: own keys of sequences of few new tokens, and
// prefixes of groups of few tokens.  Included by paged_chunk.hip.
//
// A unit is the rows of one (sequence, kv head), at most 32, and its keys; the units stand on an axis
// as in chunk_range, each as long as its keys plus kWaveUnitCost, cut at multiples of kCkWaveBlock
// into equal ranges, one to a wave.  A wave's range is one stream of 32-key steps, whatever units they
// belong to: while a step is computed the next one's K and V are on their way and the page ids of the
// one after it, so a new unit costs its wave no idle round trip; its query rows are asked for as soon
// as the last step before it has used the old ones.  What a unit's part leaves, and how parts of
// a unit are joined: see state_row.
//
// Bound by memory (K and V once) in long launches, by the start in short ones: the sequences'
// places, the share, the wave's place on the axis, page ids, K and V stand one behind another, about 9 of the
// 23 us of a decode step of 32 sequences with 100 to 1,000 own keys.  With teams of four waves to a
// range, as without shared prefixes, units this short spend their time on a team's start, merge and
// barriers (that step: 50.6 us, 28.3 now; 33.7 with this stream and the join alone).

static_assert(kWaveUnitCost >= kCkWaveBlock, "a unit's last block lies before its end on the axis");

// Place of a wave on the axis: 32 keys of a unit.
struct FewStep {
  int b, kvh;      // sequence (B or more: a group's prefix) and kv head; b = -1: the range is done
  int64_t start;   // of the unit on the axis
  int len, ip0;    // its keys, its first page table entry
  int k0, k1, k;   // the part that the wave serves, and the step's first key
};

template <int D, bool BF16, bool LSE>
__device__ __forceinline__ void shared_few(const ChunkParams& p, char* lds, const int4* table,
                                           int block, int W, int64_t total) {
  constexpr int WAVES = chunk_waves(D);
  typedef Elt<BF16> E;
  typedef typename E::v8 v8;
  constexpr int KS = D / 16;
  constexpr int NT = D / 32;
  constexpr int ROWB = D * 2;
  const int wave = uniform((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;

  // ---- this wave's range.  Workgroup i runs on XCD i % 8, so consecutive ranges go to one XCD's
  // L2; the waves of a workgroup are far apart, so that a short axis takes one wave of many
  // workgroups.
  const int range = wave * W + (block % 8) * (W / 8) + block / 8;
  const int ns = num_seqs<true>(p);
  auto cost = [&](const Seq<true>& s) -> int {
    return s.n > 0 && s.n <= p.split_tokens ? s.len + kWaveUnitCost : 0;
  };
  auto seq_length = [&](int b) -> int64_t {
    return b < ns ? (int64_t)cost(load_seq<true>(p, b, table)) * p.Hkv : 0;
  };
  const int64_t Lw = max(div_range64(total + W * WAVES - 1, W * WAVES), (int64_t)kCkWaveKeys);
  const int64_t x0 = range * Lw;
  if (x0 >= total) return;
  const int64_t x1 = x0 + Lw < total ? x0 + Lw : total;

  // ---- lane (l32, g) has row l32: the same token and head of every unit.
  const int tok = (int)((uint32_t)l32 * p.g_magic >> 16);
  const int head = l32 - tok * p.G;

  // Keys of the unit from where a range starts that many axis keys behind it (see chunk_range).
  auto cut = [&](int64_t d, int keys) -> int {
    return uniform(d >= keys + kCkWaveBlock ? keys
                   : d < kCkWaveBlock       ? 0
                                            : min((int)d / kCkWaveBlock * kCkWaveBlock, keys));
  };
  // The first step of the unit that s names, or of the next one with keys in the range.
  Seq<true> ns_seq;  // of the unit that `enter` looks at
  auto enter = [&](FewStep& s) {
    for (;;) {
      if (s.start >= x1) {
        s.b = -1;
        return;
      }
      s.len = ns_seq.len;
      s.ip0 = ns_seq.ip0;
      s.k0 = cut(x0 - s.start, s.len);
      s.k1 = cut(x1 - s.start, s.len);
      s.k = s.k0;
      if (s.k0 < s.k1) return;
      if (s.len == 0 && x0 - s.start < kCkWaveBlock && x1 - s.start >= kCkWaveBlock) {
        // Nothing to see: left by the wave of what would be the first block.
        if (g == 0 && tok < ns_seq.n) {
          Unit<true> u;
          u.prefix = ns_seq.prefix;
          state_ml(p, u)[(int64_t)(ns_seq.q0 + tok) * p.Hq + s.kvh * p.G + head] =
              float4_t{AKT_C_NEG_INF, 0.f, 0.f, __int_as_float(ns_seq.more ? kStateMore : 0)};
        }
      }
      s.start += s.len + kWaveUnitCost;
      if (++s.kvh < p.Hkv) continue;
      s.kvh = 0;
      do {
        if (++s.b >= ns) {
          s.b = -1;
          return;
        }
        ns_seq = load_seq_uniform<true>(p, s.b, table);
      } while (cost(ns_seq) == 0);
    }
  };
  auto advance = [&](FewStep& s) {
    s.k += 32;
    if (s.k < s.k1) return;
    s.start += s.len + kWaveUnitCost;
    if (++s.kvh == p.Hkv) {
      s.kvh = 0;
      do {
        if (++s.b >= ns) {
          s.b = -1;
          return;
        }
        ns_seq = load_seq_uniform<true>(p, s.b, table);
      } while (cost(ns_seq) == 0);
    }
    enter(s);
  };

  FewStep lead;  // the step whose page ids are asked for
  {
    int64_t at = 0;
    for (int jb = 0;; jb += 64) {
      const int64_t len = seq_length(jb + lane), inc = wave_inclusive_scan64(len);
      const uint64_t m = __ballot(at + inc > x0);
      if (m) {
        const int l = __builtin_ctzll(m);
        lead.b = uniform(jb + l);
        at += read_lane64(inc - len, l);
        break;
      }
      at += read_lane64(inc, 63);
    }
    ns_seq = load_seq_uniform<true>(p, lead.b, table);
    const int unit = cost(ns_seq);
    lead.kvh = div_range(x0 - at, unit);
    lead.start = uniform64(at + (int64_t)lead.kvh * unit);
    enter(lead);
  }
  if (lead.b < 0) return;

  // ---- loads.  Lane (l32, g) takes chunks 2 k + g of the K and V rows of key l32 of a step.
  int id_next = 0, slot_next = 0;
  auto load_ids = [&](const FewStep& s) {
    const int key = min(s.k + l32, s.k1 - 1);
    const int lp = page_of(p, key);
    slot_next = key - lp * p.page_size;
    id_next = (s.b >= p.B ? p.prefix_indices : p.indices)[s.ip0 + lp];
  };
  uint32_t valid_next = 0;  // keys that can be read: in the pool, before the part's end
  const half_t* src = p.q;
  // A key that cannot be read takes a row of q (any readable row does: its score is masked, its V
  // zeroed).
  auto place = [&](const FewStep& s) {
    const bool ok = s.k + l32 < s.k1 && (uint32_t)id_next < (uint32_t)p.num_pool_pages;
    valid_next = (uint32_t)__ballot(ok);
    src = (ok ? p.pool + s.kvh * p.sh + id_next * p.sp + (int64_t)slot_next * p.ss : p.q) + 8 * g;
  };
  uint4_t kf[KS], vr[KS];
  auto load_k = [&]() {
#pragma unroll
    for (int k = 0; k < KS; ++k) kf[k] = ld16(src + 16 * k);
  };
  auto load_v = [&]() {
    if (valid_next == 0xffffffffu) {
#pragma unroll
      for (int k = 0; k < KS; ++k) vr[k] = ld16(src + p.skv + 16 * k);
    } else {
      const bool ok = (valid_next >> l32) & 1;
#pragma unroll
      for (int k = 0; k < KS; ++k) vr[k] = ok ? ld16(src + p.skv + 16 * k) : uint4_t{0, 0, 0, 0};
    }
  };
  v8 qf[KS];
  auto load_q = [&](const Unit<true>& u) {
    const half_t* q = p.q + (int64_t)(u.q0 + tok) * p.q_st + (int64_t)(u.kvh * p.G + head) * p.q_sh + 8 * g;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint4_t v = {0, 0, 0, 0};
      if (tok < u.ntok) v = ld16(q + 16 * k);
      if (p.neg_q) v ^= uint4_t{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
      qf[k] = E::as8(v);
    }
  };
  auto unit_of = [&](const FewStep& s) -> Unit<true> {
    const Seq<true> q = load_seq_uniform<true>(p, s.b, table);
    return Unit<true>{q.q0, q.n, s.kvh, q.len - q.n, q.len, q.len, q.ip0, q.prefix, q.more};
  };

  // ---- V^T through the transposing read: see prefill_kernel.
  char* const vst = lds + wave * (32 * ROWB);
  const int s16 = lane & 15;
  const int vrow = 4 * g + (s16 >> 2);
  const int vcl = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
  int voff[NT], voffh[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    voff[n] = vrow * ROWB + (((4 * n + vcl) ^ tswz<D>(vrow)) * 16) + (s16 & 1) * 8;
    voffh[n] = (vrow + 8) * ROWB + (((4 * n + vcl) ^ tswz<D>(vrow + 8)) * 16) + (s16 & 1) * 8;
  }
  auto frag = [&](int h, int n) -> v8 {
    const uint2 lo = ds_read_tr16(vst + voff[n] + h * 16 * ROWB);
    const uint2 hi = ds_read_tr16(vst + voffh[n] + h * 16 * ROWB);
    return E::as8(uint4_t{lo.x, lo.y, hi.x, hi.y});
  };

  // ---- the stream.
  FewStep cur = lead, next;
  Unit<true> u = unit_of(cur);
  load_ids(cur);
  load_q(u);
  place(cur);
  load_k();
  load_v();
  uint32_t valid = valid_next;
  next = cur;
  advance(next);
  lead = next;
  if (next.b >= 0) load_ids(next);

  float16_t oacc[NT];
  float m_run = kCkFloor, l_part = 0.f, x_part = 0.f;  // x: the sum of the unrounded P
  bool bad = false;
  const float c = p.qk_scale;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[n][i] = 0.f;
#pragma clang loop unroll(disable)
  for (;;) {
    const bool causal = p.causal && !u.prefix;
    const int lim = causal ? u.first + min(tok, u.ntok - 1) : u.len - 1;
    const int lim_min = causal ? u.first : u.len - 1;
    const bool end = next.b != cur.b || next.kvh != cur.kvh;  // of the unit's part
    Unit<true> un = u;
    if (end && next.b >= 0) un = unit_of(next);
    float16_t sv;
#pragma unroll
    for (int i = 0; i < 16; ++i) sv[i] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) sv = E::mfma(E::as8(kf[k]), qf[k], sv);
    if (next.b >= 0) {
      place(next);
      load_k();
      if (end) load_q(un);
    }
    if (causal && cur.k + 31 > u.first)  // keys that not every row sees
      bad |= zero_not_finite<BF16>(vr);
#pragma unroll
    for (int k = 0; k < KS; ++k)
      *reinterpret_cast<uint4_t*>(vst + l32 * ROWB + (((2 * k + g) ^ tswz<D>(l32)) * 16)) = vr[k];
    if (next.b >= 0) {
      load_v();
      lead = next;
      advance(lead);
      if (lead.b >= 0) load_ids(lead);
    }
    if (cur.k + 31 > lim_min || valid != 0xffffffffu)  // wave-uniform
      mask_scores(sv, valid, lim - cur.k, g);
    float mx = sv[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, sv[i]);
    float ma, mb;
    swap32(mx, ma, mb);
    const float m_new =
        __builtin_elementwise_maximum(m_run, __builtin_elementwise_maximum(ma, mb) * c);
    if (__any(!(m_new <= m_run + kCkSlack))) {
      // The slack leaves P below 2^kCkSlack.  The first keys' rise from the floor scales zeros.
      const float alpha = fast_exp2(m_run - m_new);
      l_part *= alpha;
      x_part *= alpha;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[n][i] *= alpha;
      m_run = m_new;
    }
    uint32_t pk[8];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float p0 = fast_exp2(__builtin_fmaf(sv[i], c, -m_run));
      const float p1 = fast_exp2(__builtin_fmaf(sv[i + 1], c, -m_run));
      pk[i >> 1] = E::pack2(p0, p1);
      if constexpr (LSE) x_part += p0 + p1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) l_part = E::dot2(pk[i], E::kOnes, l_part);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v8 bop = E::as8(uint4_t{pk[4 * h], pk[4 * h + 1], pk[4 * h + 2], pk[4 * h + 3]});
#pragma unroll
      for (int n = 0; n < NT; ++n) oacc[n] = E::mfma(frag(h, n), bop, oacc[n]);
    }
    if (end) {
      if (bad)
        for (int k = cur.k0; k < cur.k1; k += 32)
          if (k + 31 > u.first)  // a step that the values were taken out of
            add_not_finite<D, BF16, true>(p, u, k, min(k + 32, cur.k1), g, lim, oacc);
      const float l_row = xor32_sum(l_part), x_row = xor32_sum(x_part);
      if (tok < u.ntok) {
        const int64_t at = (int64_t)(u.q0 + tok) * p.Hq + u.kvh * p.G + head;
        const StateRow to = state_row<D>(p, u, at, cur.k0 == 0 && cur.k1 == cur.len, cur.k0 == 0,
                                         range, cur.start, Lw, kCkWaveBlock, false, 32, l32);
        if (g == 0) *to.ml = float4_t{m_run, l_row, x_row, to.tag};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            st16(to.o + 32 * n + 8 * k + 4 * g,
                 as_uint4f(float4_t{oacc[n][4 * k], oacc[n][4 * k + 1], oacc[n][4 * k + 2],
                                    oacc[n][4 * k + 3]}));
      }
      if (next.b < 0) return;
      bad = false;
      m_run = kCkFloor;
      l_part = x_part = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[n][i] = 0.f;
    }
    cur = next;
    next = lead;
    u = un;
    valid = valid_next;
  }
}

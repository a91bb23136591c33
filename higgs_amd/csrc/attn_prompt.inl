// attn_prompt.inl -- the body of the prompts' kernel.
//
// Block = (kv head, tile of 128 rows, part of its tiles of BN keys); a wave
// has 32 rows. As in the decode kernel S^T = K Q^T and O^T = V^T P^T, here on
// 32x32x16 instructions: a lane has half the scores of one row in registers,
// its weights are the second product's operand as they stand, and a row's
// reference and sum are one register each.
//
// K and V tiles come straight from memory to LDS, double buffered: the next
// tile's loads are issued before a tile is computed, one barrier a tile.
//
// 8 sequences of 2048, 32/8 heads of 128 bf16, causal (275 GFLOP): 341 to 352
// us, 780 to 806 TFLOP/s, where a large library product reaches 1260 (a card
// that clocks lower: up to 410). With two waves a SIMD the matrix units work 42
// % of the time and the vector units 50 (a score takes a multiply-add, an exp
// and half a conversion), each wave's own step one after the other. 8191 tokens
// in a window of 4096, soft cap, 16/8 heads of 256 (412 GFLOP): 575 to 582 us;
// registers allow one wave a SIMD there, and the tile's load instructions and
// its barrier stand beside the step. Deeper rings of tiles, 256 rows a block
// and loads spread over the step were no faster.
//
// Included where a kernel, or a function of one, stands over
//   T, D, BN, CAP   the type, the values of a row, a tile's keys and the soft cap's form
//   keys, a         which keys the block takes, the call's arguments
//   lds, words      prompt_lds<D>() bytes, 1024-byte aligned, and kPromptWords
//   x, grid_x, y, splits   the block's place, and the y there are
//   TWO             are weights multiplied in two parts?
// As a function of its arguments' type the kernel without a prefix was scheduled
// otherwise, with 4 registers more, and took 1.5 % longer (8191 tokens in a window of
// 4096, 16/8 heads of 256: 571 us for 562).
  constexpr int NT = 2 * kPromptRows, BM = kPromptRows, CH = D / 8, kUnits = BN * CH / NT;
  constexpr int kRow = 2 * D, kTile = BN * kRow;
  constexpr int KT = BN / 32, QS = D / 16, DT = D / 32, kAhead = 2;
  static_assert(BN == 64 && BN * CH % NT == 0, "two tiles of 32 keys, whole units per thread");
  typedef Mx<T> M;
  static_assert(prompt_lds<D>() == 4 * kTile, "two tiles of keys, two of values");
  int& odd = words[0];   // 1 + index of the last tile found to hold values that are not finite
  int& redo = words[1];  // a row's sums are not finite

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int place = x / a.p.kv_heads, hk = x - place * a.p.kv_heads, G = a.group;

  // which sequence's tile this is: tiles are counted over the sequences, from
  // the last one on (the longest ones of a prompt first)
  const int64_t want = grid_x / a.p.kv_heads - 1 - place;
  int seq = 0, tile = (int)want;
  KvSeq s{0, a.b.tokens, 0};  // the prefix: the rows of all sequences
  if (keys != kPrefix) {
    const Owner w = find_owner(
        a.b.batch, [&](int b) { return ((int64_t)kv_seq(a.b, b).n * G + BM - 1) / BM; }, [&](int64_t) { return want; });
    if (w.seq < 0) return;
    seq = __builtin_amdgcn_readfirstlane(w.seq);
    tile = __builtin_amdgcn_readfirstlane((int)(want - w.before));
    s = kv_seq(a.b, seq);
    s.first = __builtin_amdgcn_readfirstlane(s.first);
    s.n = __builtin_amdgcn_readfirstlane(s.n);
    s.len = __builtin_amdgcn_readfirstlane(s.len);
  }
  const int R = s.n * G, pos0 = s.len - s.n;  // pos0 may be negative: rows in front of the sequence

  const int row0 = tile * BM;
  int p_first = pos0 + row0 / G, p_last = pos0 + (min(row0 + BM, R) - 1) / G;
  // this lane's row
  const int wrow0 = row0 + 32 * wave;
  const int row = min(wrow0 + col, R - 1);
  const int qi = row / G, head = hk * G + row - qi * G;
  const bool in = wrow0 + col < R;
  int p = pos0 + qi, pw_first = 0, pw_last = 0;
  if (keys == kPrefix) {
    // every row has a sequence of its own; a row of none sees nothing
    int* const lowest_of = words + 2;
    int* const highest_of = lowest_of + NT / 64;
    const KvSeq of = kv_seq(a.b, kv_row_owner(a.b, qi));
    p = qi >= of.first && qi < of.first + of.n ? of.len - of.n + qi - of.first : -1;
    int lowest = p, highest = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {  // (the halves hold the same rows)
      lowest = min(lowest, __shfl_xor(lowest, o));
      highest = max(highest, __shfl_xor(highest, o));
    }
    pw_first = __builtin_amdgcn_readfirstlane(lowest);
    pw_last = __builtin_amdgcn_readfirstlane(highest);
    if (lane == 0) {
      lowest_of[wave] = pw_first;
      highest_of[wave] = pw_last;
    }
    __syncthreads();
    p_first = min(min(lowest_of[0], lowest_of[1]), min(lowest_of[2], lowest_of[3]));
    p_last = max(max(highest_of[0], highest_of[1]), max(highest_of[2], highest_of[3]));
    p_first = __builtin_amdgcn_readfirstlane(p_first);
    p_last = __builtin_amdgcn_readfirstlane(p_last);
  }
  // the block's keys, in tiles of BN: those of the first `sinks`, then the window's,
  // of the keys from .. cap - 1 that are the call's
  const int from = keys == kBehind && pre_of(a) > 0 ? prefix_of(a) : 0;
  const int64_t own = (int64_t)a.b.width << a.p.page_shift;
  const int64_t cap = keys == kOwn ? own : keys == kPrefix ? (int64_t)prefix_of(a) : max(own, (int64_t)prefix_of(a));
  const int hi = (int)min((int64_t)p_last + 1, cap);
  const int lo = a.window > 0 && p_first >= a.window ? p_first - a.window + 1 : 0;
  const int t_from = from / BN, t_hi = hi > 0 ? (hi + BN - 1) / BN : 0;
  const int t_lo = (keys == kBehind ? max(lo, from) : lo) / BN;
  // (at most 2^30 before it is rounded up: sinks and lo may both end at int32's end)
  int front = min((min(min(a.sinks, lo), max(hi, 0)) + BN - 1) / BN, t_lo);
  if (keys == kBehind) front = max(front - t_from, 0);
  const int tiles = a.p.n_pages > 0 ? front + max(t_hi - t_lo, 0) : 0;
  const int per = (tiles + splits - 1) / splits;
  const int it0 = min(per * y, tiles), it1 = min(it0 + per, tiles);
  auto tile_of = [&](int it) { return it < front ? t_from + it : t_lo + it - front; };
  if (keys != kPrefix) {  // the range of the wave's rows
    pw_first = pos0 + min(wrow0, R - 1) / G;
    pw_last = pos0 + min(wrow0 + 31, R - 1) / G;
  }

  const Scale sc = fold_scale<CAP>(a);

  // lane l looks up key l of a tile
  const int32_t* table = a.b.table + (int64_t)seq * a.b.table_stride;
  const char* kbase = a.p.k + 2 * hk * a.p.kst[2];
  const char* vbase = a.p.v + 2 * hk * a.p.vst[2];
  auto look_up = [&](int it) -> int32_t {
    if (it >= it1) return -1;
    const int key = tile_of(it) * BN + (lane & (BN - 1));
    if (keys == kPrefix) return key < hi ? page_of_prefix(a, key) : -1;
    if (keys == kBehind) return key >= from && key < hi ? page_behind(a, table, key) : -1;
    return key < hi ? table[key >> a.p.page_shift] : -1;
  };
  // Looked at a turn after the load was issued: a wait for it is a wait for
  // the tiles' loads before it.
  auto checked = [&](int32_t page) { return (uint32_t)page < (uint32_t)a.p.n_pages ? page : -1; };
  // One load instruction takes 64 pieces, of rows that lie in one page when
  // pages have 16 tokens or more: the address of its first row is then scalar,
  // and the lanes' offsets are the same for every tile. A key that does not
  // exist reads what is there (a page's end, or page 0); its score is masked
  // and its value, if not finite, taken out.
  const bool whole = a.p.page_shift >= 4 && a.p.kst[1] < (1 << 24) && a.p.vst[1] < (1 << 24);
  // But where the prefix ends inside such a run of rows, the rows in front of its
  // end and those behind it lie in two pages: that tile goes row by row.
  const int cut = keys == kBehind && (prefix_of(a) & 15) ? prefix_of(a) / BN : -1;
  // (rows i * NT / CH apart have the same offsets, where that is a multiple of 16)
  constexpr int kOffs = NT % (16 * CH) == 0 ? 1 : kUnits;
  uint32_t koff[kOffs], voff[kOffs];
#pragma unroll
  for (int i = 0; i < kOffs; ++i) {
    const int u0 = i * NT + 64 * wave, u = u0 + lane, r = u / CH, c = u - r * CH, r0 = u0 / CH;
    koff[i] = 2 * ((r - r0) * (uint32_t)a.p.kst[1] + 8 * key_piece<D>(r, c));
    voff[i] = 2 * ((r - r0) * (uint32_t)a.p.vst[1] + 8 * value_place<D>(r, c));
  }
  // Two parts of the weights of rows of 128 leave no register for what a lane needs a few
  // times a tile, and to get it back from memory would wait for the tiles' loads: it is kept in LDS.
  constexpr bool kLean = prompt_lean<D, TWO>();
  static_assert(!kLean || kOffs == 1, "one offset");
  int* const kept = words + kPromptWords + threadIdx.x;
  if constexpr (kLean) {
    kept[0] = koff[0];
    kept[NT] = voff[0];
    kept[2 * NT] = p;
  }
  const uint32_t lds0 = lds_address(lds) + 1024 * wave;
  auto load = [&](int it, uint32_t to, int32_t page, const char* base, int64_t page_step, int64_t row_step,
                  const uint32_t* off, auto piece) {
    const int key0 = tile_of(it) * BN;
    if (page < 0) page = 0;
    if (whole && (keys != kBehind || tile_of(it) != cut)) {
      const uint64_t at = (uint64_t)(base + 2 * (page * page_step + ((key0 + lane) & a.p.page_mask) * row_step));
      const int at_lo = (int)(uint32_t)at, at_hi = (int)(uint32_t)(at >> 32);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int r0 = (i * NT + 64 * wave) / CH;
        const uint64_t row = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, r0) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane(at_lo, r0);
        lds_load(to + 16 * NT * i, (const char*)row, off[i % kOffs]);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kUnits; ++i) {
        const int u = i * NT + threadIdx.x, r = u / CH, c = u - r * CH;
        const int64_t pg = __shfl(page, r), at = (key0 + r) & a.p.page_mask;
        lds_load(to + 16 * NT * i, base + 2 * (pg * page_step + at * row_step + 8 * piece(r, c)));
      }
    }
  };
  // keys and values have two slots each: tile it0 + i lies in slot i % 2
  auto load_keys = [&](int it, int slot, int32_t page) {
    load(it, lds0 + slot * kTile, page, kbase, a.p.kst[0], a.p.kst[1], kLean ? (uint32_t*)kept : koff, key_piece<D>);
  };
  auto load_values = [&](int it, int slot, int32_t page) {
    load(it, lds0 + (2 + slot) * kTile, page, vbase, a.p.vst[0], a.p.vst[1], kLean ? (uint32_t*)kept + NT : voff, value_place<D>);
  };
  // does some row of this range see only a part of the tile?
  auto part_seen = [&](int key0, int first, int last) {
    return !(key0 + BN - 1 <= first &&
             (a.window == 0 || key0 > last - a.window || key0 + BN - 1 < a.sinks));
  };
  auto position = [&]() { return kLean ? kept[2 * NT] : p; };
  // which keys of a tile this lane's row sees (bit i: key key0 + i)
  auto seen_keys = [&](int key0, uint64_t exist) {
    const int p = position();
    auto below = [&](int key) {  // the tile's keys below `key`
      const int n = key - key0;
      return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
    };
    uint64_t m = p >= 0 ? below(p + 1) & exist : 0ull;
    if (a.window > 0 && p >= a.window) m &= ~below(p - a.window + 1) | below(a.sinks);
    return m;
  };

  u32x4 qf[QS];
  auto load_rows = [&]() {  // behind the first keys' loads: one wait for both
    const char* qp = a.q + 2 * ((int64_t)(s.first + qi) * a.qst[0] + head * a.qst[1] + 8 * half);
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      qf[i] = *reinterpret_cast<const u32x4*>(qp + 32 * i);
      for (int w = 0; w < 4; ++w) qf[i][w] = (qf[i][w] & sc.keep) ^ sc.flip;
    }
  };
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = f32x16{};
  float ref = lowest_ref(sc.c), sum = 0.0f;
  const float slack = M::kSlack / sc.c;
  bool any = false;

  // A lane's places in a tile of keys (row col, piece 2 i + half) and of values
  // (row 4 half + (lane % 16) / 4, 8-byte pieces, read transposed). Rows are
  // whole multiples of 64 bytes (D = 96: 192) and the places differ by an
  // exclusive or: every piece's address is one register's, xor a constant.
  const int vr = 4 * half + (lane & 15) / 4, vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t kat = col * kRow + 16 * key_place<D>(col, half);
  const uint32_t vat = vr * kRow + 16 * value_place<D>(vr, vc) + 8 * (lane & 1);
  auto key_frag = [&](int slot, int t, int i) {
    const char* kt = lds + slot * kTile + 32 * t * kRow;
    if constexpr (D == 96) {
      const int r = 32 * t + col;
      return *reinterpret_cast<const u32x4*>(kt + col * kRow + 16 * key_place<D>(r, 2 * i + half));
    } else {
      return *reinterpret_cast<const u32x4*>(kt + (kat ^ (32 * i)));
    }
  };
  auto value_frag = [&](int slot, int t, int k) {
    const char* vt = lds + (2 + slot) * kTile + 16 * k * kRow +
                     (D == 96 ? vat + 64 * t : vat ^ (64 * t));
    const u32x2 v0 = lds_transposed(vt), v1 = lds_transposed(vt + 8 * kRow);
    return u32x4{v0[0], v0[1], v1[0], v1[1]};
  };

  // Scores of tile `it` ready in x: hides those that the wave's rows do not see,
  // and moves the references that others pass; `shrunk` is then the factor for
  // the sums so far (few tiles move any: most leave `moved` false).
  bool moved;
  float shrunk, base;  // base: of the weights' exponents, c x + base
  uint32_t see[KT];  // CAP, masked: the 32 keys' bits, at 8 (e / 4) + e % 4 for score e
  auto settle = [&](f32x16* x, int it, uint64_t exist, bool masked) {
    auto top_of = [&](const f32x16* x) {
      float part[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = max3(x[0][e], x[0][e + 4], x[0][e + 8]);
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = max3(part[e], x[0][e + 12], x[1][e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = max3(part[e], x[1][e + 4], x[1][e + 8]);
      part[0] = max3(part[0], x[1][12], x[1][13]);
      part[1] = max3(part[1], x[1][14], x[1][15]);
      return max3(max3(part[0], part[1], part[2]), part[3], part[3]);
    };
    float top;
    if (masked) {
      float hidden = -INFINITY;
      asm volatile("" : "+v"(hidden));  // no register for it but here
      const uint64_t bits = seen_keys(tile_of(it) * BN, exist) >> (4 * half);
      const bool some = (bits & 0x0f0f0f0f0f0f0f0full) != 0;
      any |= some;
      f32x16 h[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        see[t] = (uint32_t)(bits >> (32 * t));
#pragma unroll
        for (int e = 0; e < 16; ++e) h[t][e] = see[t] & (1u << (8 * (e / 4) + e % 4)) ? x[t][e] : hidden;
      }
      top = top_of(h);
      if constexpr (CAP) {
        // the scores stay: under tanh a hidden one would count, so the weights are cleared instead
        top = some ? cap_tanh<CAP>(top * sc.inner) : hidden;
      } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) x[t] = h[t];
      }
    } else {
      any = true;
      top = top_of(x);
      if constexpr (CAP) top = cap_tanh<CAP>(top * sc.inner);
    }
    moved = kLean ? __any((top - ref) * sc.c > M::kSlack) : __any(top > ref + slack);
    if (moved) {  // a row's own scores alone decide for it
      top = halves_max(top);
      const float to = (kLean ? (top - ref) * sc.c > M::kSlack : top > ref + slack) ? top : ref;
      shrunk = lesser((ref - to) * sc.c);
      sum *= shrunk;
      ref = to;
    }
    base = CAP == kWideCap ? M::kBias : fmaf(-ref, sc.c, M::kBias);
    if constexpr (CAP == kNoCap) {
      if (__any(fabsf(base) > kBaseMax)) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[t][e] -= fabsf(base) > kBaseMax ? ref : 0.0f;
        base = fabsf(base) > kBaseMax ? M::kBias : base;
      }
    }
  };
  // Weights of scores 2 i and 2 i + 1, rounded to the type: by half a step, as the
  // result is (a row's error against 64 bits is 1.3 times that of weights in f32).
  // A second part, as single tokens have (TWO: also of a pass over their prefix, so that
  // a row's bits are as good as without one), is half as many matrix
  // instructions again and a conversion a weight, where the two bound the kernel.
  // The sum takes the rounded ones, so that a row's weights add up to one as used.
  float add[4];
  uint32_t low;  // what the weights' first parts leave
  auto weigh = [&](const f32x16* x, int i) {
    float s0 = x[i / 8][2 * i % 16], s1 = x[i / 8][2 * i % 16 + 1];
    if constexpr (CAP) {
      s0 = cap_tanh<CAP>(s0 * sc.inner);
      s1 = cap_tanh<CAP>(s1 * sc.inner);
    }
    if constexpr (CAP == kWideCap) {  // such scores may be past kBaseMax
      s0 -= ref;
      s1 -= ref;
    }
    const float w0 = __builtin_amdgcn_exp2f(fmaf(s0, sc.c, base));
    const float w1 = __builtin_amdgcn_exp2f(fmaf(s1, sc.c, base));
    const uint32_t pair = M::pack(w0, w1);
    add[i & 3] = M::add_pair(pair, i < 4 ? 0.0f : add[i & 3]);
    if constexpr (TWO) {
      low = M::pack(w0 - T::lo(pair), w1 - T::hi(pair));
      add[i & 3] = M::add_pair(low, add[i & 3]);
    }
    return pair;
  };
  // Sums of what is not finite among a tile's values 32 t .. 32 t + 31 that the
  // lane's row sees (`see`): zero, an infinity or NaN.
  auto odd_sum = [&](int slot, int t, uint64_t see) {
    // constants of this path, kept out of the loop's registers
    uint32_t one = M::kOne, c128 = M::k128, c16384 = M::k16384, inf = 0x7f800000u;
    asm volatile("" : "+s"(one), "+s"(c128), "+s"(c16384), "+s"(inf));
    auto code = [&](uint32_t h) {
      const uint32_t e = h & M::kExp, f = h & 0x7fffu & ~M::kExp;
      return e != M::kExp ? 0u : f ? c16384 : h & 0x8000u ? c128 : one;
    };
    f32x16 n = f32x16{};
#pragma unroll 1
    for (int k = 0; k < 2 * KT; ++k) {
      const u32x4 v = value_frag(slot, t, k);
      u32x4 c, on;
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = (uint32_t)(see >> (16 * k + 8 * (i / 2) + 2 * (i & 1)));
        c[i] = code(v[i] & 0xffffu) | code(v[i] >> 16) << 16;
        on[i] = (two & 1 ? one : 0u) | (two & 2 ? one << 16 : 0u);
      }
      n = M::mma32x16(c, on, n);
    }
    f32x16 f;
    for (int e = 0; e < 16; ++e) {
      const int counts = (int)n[e], nan = counts >> 14, neg = (counts >> 7) & 127, pos = counts & 127;
      const uint32_t bits = nan || (neg && pos) ? inf | 0x400000u : neg ? inf | 0x80000000u : pos ? inf : 0u;
      f[e] = u2f(bits);
    }
    return f;
  };
  // values of tile `it` that are not finite, where some row sees only part of the tile
  auto odd_values = [&](int it, int slot, uint64_t exist, bool all) {
    const int key0 = tile_of(it) * BN;
    if (all && !part_seen(key0, p_first, p_last)) return;
    char* vt = lds + (2 + slot) * kTile;
    uint32_t bits = 0;
#pragma unroll 1
    for (int i = 0; i < kUnits; ++i) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(vt + 16 * (i * NT + threadIdx.x));
      bits |= odd_pair<M>(v[0]) | odd_pair<M>(v[1]) | odd_pair<M>(v[2]) | odd_pair<M>(v[3]);
    }
    if (bits) odd = it + 1;
    __syncthreads();
    if (odd != it + 1) return;
    const uint64_t see = seen_keys(key0, exist) >> (4 * half);
#pragma unroll 1
    for (int t = 0; t < DT; ++t) {
      const f32x16 f = odd_sum(slot, t, see);
#pragma unroll
      for (int u = 0; u < DT; ++u)
        if (u == t) o[u] += f;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < kUnits; ++i) {
      u32x4* v = reinterpret_cast<u32x4*>(vt + 16 * (i * NT + threadIdx.x));
      u32x4 t = *v;
      for (int j = 0; j < 4; ++j) t[j] = finite_pair<M>(t[j]);
      *v = t;
    }
    __syncthreads();
  };
  auto all_of = [&](uint64_t exist) { return exist == ~0ull; };

  // One step: the product of tile it - 1 with its weights w, the weights wn of
  // tile `it`, whose scores x are ready, and the scores of tile it + 1 into y:
  // independent pieces, so that the matrix cores and the vector units have
  // work side by side from every wave. The product comes first, so that w is
  // done with when y begins. Before the first tile the weights are zero; behind
  // the last one the scores are of stale keys and not used.
  // The operands of the matrix instructions are read kAhead ahead; nothing
  // moves across a pair of weights, or the reads would all come first and spill.
  constexpr int kPairs = 8 * KT, kQ = KT * QS, kP = DT * 2 * KT, kW = TWO ? 2 : 1;
  auto step = [&](const f32x16* x, f32x16* y, const u32x4* w, u32x4* wn, int slot) {
    u32x4 f[kAhead + 1];
    auto frag = [&](int n) {
      if constexpr (kLean && CAP) {  // with tanh no room for the places' variants either: worked out for each piece
        auto other = [](uint32_t at, uint32_t mask) {
          uint32_t r = at;
          if (mask) asm volatile("v_xor_b32 %0, %1, %2" : "=v"(r) : "v"(mask), "v"(at));
          return r;
        };
        if (n < kP) {
          const char* vt = lds + (2 + (slot ^ 1)) * kTile + 16 * (n / DT) * kRow + other(vat, 64 * (n % DT));
          const u32x2 v0 = lds_transposed(vt), v1 = lds_transposed(vt + 8 * kRow);
          return u32x4{v0[0], v0[1], v1[0], v1[1]};
        }
        const int j = n - kP;
        return *reinterpret_cast<const u32x4*>(lds + (slot ^ 1) * kTile + 32 * (j / QS) * kRow + other(kat, 32 * (j % QS)));
      }
      return n < kP ? value_frag(slot ^ 1, n % DT, n / DT) : key_frag(slot ^ 1, (n - kP) / QS, (n - kP) % QS);
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) f[j] = frag(j);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = i * (kQ + kW * kP) / kPairs; u < (i + 1) * (kQ + kW * kP) / kPairs; ++u) {
        // the product's pieces serve a weight's kW parts each
        const int n = u < kW * kP ? u / kW : u - (kW - 1) * kP, part = u < kW * kP ? u % kW : 0;
        if (part == 0 && n + kAhead < kQ + kP) f[(n + kAhead) % (kAhead + 1)] = frag(n + kAhead);
        const u32x4& v = f[n % (kAhead + 1)];
        const int j = n - kP;
        if (j < 0)
          o[n % DT] = M::mma32x16(v, w[2 * KT * part + n / DT], o[n % DT]);
        else
          y[j / QS] = M::mma32x16(v, qf[j % QS], j % QS ? y[j / QS] : f32x16{});
      }
      wn[i / 4][i & 3] = weigh(x, i);
      if constexpr (TWO) wn[2 * KT + i / 4][i & 3] = low;
      if (i % 4 == 3) {  // here, and not where they are used
        asm volatile("" : "+v"(wn[i / 4]));
        if constexpr (TWO) asm volatile("" : "+v"(wn[2 * KT + i / 4]));
        asm volatile("" : "+v"(add[0]), "+v"(add[1]), "+v"(add[2]), "+v"(add[3]));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    sum += (add[0] + add[1]) + (add[2] + add[3]);
  };

  if (threadIdx.x == 0) odd = redo = 0;
  if (it0 < it1) {
    // pages of the tiles it, it + 1 and it + 2, and which keys of it - 1 and it exist
    int32_t page0 = look_up(it0), page1 = look_up(it0 + 1), next = look_up(it0 + 2);
    page0 = checked(page0);
    page1 = checked(page1);
    uint64_t exist = __ballot(page0 >= 0), exist1 = 0;
    load_keys(it0, 0, page0);
    if (it0 + 1 < it1) load_keys(it0 + 1, 1, page1);
    load_rows();
#pragma unroll
    for (int i = 0; i < kUnits; ++i)  // the values in front of the first tile
      *reinterpret_cast<u32x4*>(lds + 3 * kTile + 16 * (i * NT + threadIdx.x)) = u32x4{0, 0, 0, 0};
    landed_barrier();
    f32x16 xa[KT], xb[KT];
    u32x4 wa[2 * KT * kW], wb[2 * KT * kW];  // all weights' first parts, then their second ones
#pragma unroll
    for (int k = 0; k < 2 * KT * kW; ++k) wb[k] = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      xa[t] = f32x16{};
#pragma unroll
      for (int i = 0; i < QS; ++i) xa[t] = M::mma32x16(key_frag(0, t, i), qf[i], xa[t]);
    }
    __syncthreads();  // its slot is loaded again below

    auto turn = [&](f32x16* x, f32x16* y, const u32x4* w, u32x4* wn, int it, int slot) {
      asm volatile("" : "+v"(next));  // waits here if it must, in front of the tiles' loads
      const int32_t page2 = checked(next);
      next = look_up(it + 3);
      load_values(it, slot, page0);
      if (it + 2 < it1) load_keys(it + 2, slot, page2);
      page0 = page1;
      page1 = page2;
      const bool masked = !all_of(exist) || part_seen(tile_of(it) * BN, pw_first, pw_last);
      settle(x, it, exist, masked);
      if (it > it0) odd_values(it - 1, slot ^ 1, exist1, all_of(exist1));
      const float before = sum;
      step(x, y, w, wn, slot);
      if (CAP && masked) {
        sum = before;
#pragma unroll
        for (int k = 0; k < 2 * KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t two = see[k / 2] >> (16 * (k & 1) + 8 * (i / 2) + 2 * (i & 1));
            wn[k][i] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
            sum = M::add_pair(wn[k][i], sum);
            if constexpr (TWO) {
              wn[2 * KT + k][i] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
              sum = M::add_pair(wn[2 * KT + k][i], sum);
            }
          }
      }
      if (moved) {
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= shrunk;
      }
      exist1 = exist;
      exist = __ballot(page0 >= 0);
      landed_barrier();
    };
    auto drain = [&](const u32x4* w, int slot) {
      odd_values(it1 - 1, slot, exist1, all_of(exist1));
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const u32x4 v = value_frag(slot, j % DT, j / DT);
        o[j % DT] = M::mma32x16(v, w[j / DT], o[j % DT]);
        if constexpr (TWO) o[j % DT] = M::mma32x16(v, w[2 * KT + j / DT], o[j % DT]);
      }
    };
    // two turns a round, so that no score or weight is moved between registers
    int it = it0;
    for (; it + 1 < it1; it += 2) {
      turn(xa, xb, wb, wa, it, 0);
      turn(xb, xa, wa, wb, it + 1, 1);
    }
    if (it < it1) {
      turn(xa, xb, wb, wa, it, 0);
      drain(wa, 0);
    } else {
      drain(wb, 1);
    }
  }
  sum = halves_sum(sum);
  any = halves_sum(any ? 1.0f : 0.0f) != 0.0f;
  // Sums that are not finite though the row's weights are: its values are not.
  bool bad;
  {
    float peak[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        peak[0] = peak3(peak[0], o[t][e], o[t][e + 1]);
        peak[1] = peak3(peak[1], o[t][e + 2], o[t][e + 3]);
      }
    bad = !(peak[0] < INFINITY && peak[1] < INFINITY) && sum > 0.0f && sum < INFINITY;
  }
  auto tell = [&]() {  // the block, whether a row is bad; without a wait for stores
    if (bad) redo = 1;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  // (in front of the stores 168 registers do for rows of 64, a third block a CU;
  // rows of 256 would move 32 of their sums to memory)
  if constexpr (D < 256) tell();
  // (a row's parts over the prefix come first)
  int64_t part_at = (int64_t)(s.first + qi) * a.q_heads + head;
  if (keys == kOwn) part_at = part_at * splits + y;
  else part_at = part_at * row_parts_of(a) + (keys == kBehind ? pre_of(a) : 0) + y;
  const bool parts = keys == kOwn ? splits > 1 : keys == kPrefix || row_parts_of(a) > 1;
  char* out_row = a.out + 2 * ((int64_t)(s.first + qi) * a.ost[0] + head * a.ost[1]);
  if (parts) {
    if (in && half == 0)
      *reinterpret_cast<f32x2*>(a.stat + 2 * part_at) = f32x2{any ? (keys == kOwn ? ref * sc.c : ref) : -INFINITY, sum};
    if (in && any) {
      float* dst = a.part + part_at * D + 4 * half;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4*>(dst + 32 * t + 2 * e) = f32x4{o[t][e], o[t][e + 1], o[t][e + 2], o[t][e + 3]};
    }
  } else {
    // a lane has 4 of every 8 values of its row: the halves trade, for 16-byte stores
    const float r = any ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        u32x4 v;
        for (int i = 0; i < 2; ++i) {
          const uint32_t b0 = T::pack(o[t][e + 2 * i] * r, o[t][e + 2 * i + 1] * r);
          const uint32_t b1 = T::pack(o[t][e + 4 + 2 * i] * r, o[t][e + 5 + 2 * i] * r);
          const auto x = __builtin_amdgcn_permlane32_swap(b0, b1, false, false);
          v[i] = x[0];
          v[2 + i] = x[1];
        }
        if (in) *reinterpret_cast<u32x4*>(out_row + 16 * half + 64 * t + 4 * e) = v;
      }
  }

  // Rows over values that are not finite, of which a weight may have been rounded
  // to zero: every column that holds such a value among the keys that the row sees
  // is written again, from the counts of every tile.
  if constexpr (D == 256) tell();
  if (!redo) return;
#pragma unroll 1
  for (int t = 0; t < DT; ++t) {
    f32x16 f = f32x16{};
#pragma unroll 1
    for (int it = it0; it < it1; ++it) {
      const int32_t page = checked(look_up(it));
      const uint64_t exist = __ballot(page >= 0);
      load_values(it, 0, page);
      landed_barrier();
      f += odd_sum(0, t, seen_keys(tile_of(it) * BN, exist) >> (4 * half));
      __syncthreads();
    }
    if (!bad || !in) continue;
#pragma unroll 1
    for (int e = 0; e < 16; e += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = e == 0 ? f[i] : e == 4 ? f[4 + i] : e == 8 ? f[8 + i] : f[12 + i];
        const int d = 32 * t + 2 * e + 4 * half + i;
        if (x == 0.0f) continue;
        if (parts) a.part[part_at * D + d] = x;
        else *reinterpret_cast<uint16_t*>(out_row + 2 * d) = (uint16_t)T::pack(x, x);
      }
  }

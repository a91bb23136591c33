// attn_walk.inl -- a wave's walk over a run of keys of a kv head, for up to 16 query heads
// that have one token each.
//
// The tiles begin, begin + STEP, ... below last of n keys; key_of(i) is the position of key
// i, page_of(position) its page.
//
// A tile's scores are S^T = K Q^T on 16x16x32 matrix instructions: keys are
// the rows, so K's 16-byte pieces go from memory straight into the operand,
// and a lane ends with 4 keys each of one head. That is also where the second
// product O^T = V^T P^T wants its weights: no weight crosses lanes. V^T comes
// through LDS (written row by row, read transposed). K and V of the next tile
// are in flight while a tile is computed.
//
// Weights are split in two 16-bit parts (hi + lo, both multiplied): the
// matrix cores have time to spare, and two parts keep 16 bits of a weight in
// bf16 and 22 in f16, well below the result's own rounding.
//
// Included where a kernel, or a function of one, stands over
//   T, D, CAP, STEP, NS, kKeys, kStep, kOut, kRow   the type, sizes and steps
//   a, sc, qf, kbase, vbase   the arguments, the scores' scale, the heads' q, the kv head's rows
//   begin, last, n, key_of, page_of, vt   the run, and room for a tile of values
//   m, j   the lane's head, and its quarter
// and leaves o, ref, sum and any: the sums, their reference and whether there was a key.
  // page of key i of the run (-1: none) and its place in the page
  auto look_up = [&](int tile, int32_t* page, int32_t* at) {
#pragma unroll
    for (int h = 0; h < NS; ++h) {
      const int i = tile * kKeys + 16 * h + m;
      page[h] = -1;
      at[h] = 0;
      if (tile < last && i < n) {
        const int32_t key = key_of(i);
        page[h] = page_of(key);
        at[h] = key & a.p.page_mask;
      }
    }
  };
  u32x4 kr[NS][kStep], vr[NS][kStep];
  uint32_t there = 0;  // bit i: key i of the loaded tile exists
  auto load = [&](const int32_t* page, const int32_t* at) {
    there = 0;
#pragma unroll
    for (int h = 0; h < NS; ++h) {
      const bool ok = (uint32_t)page[h] < (uint32_t)a.p.n_pages;
      there |= (uint32_t)(__ballot(ok) & 0xffffu) << (16 * h);
      // a key that does not exist reads the pool's begin row, and is masked below
      const int64_t pg = ok ? page[h] : 0, r = ok ? at[h] : 0;
      const char* kp = kbase + 2 * (pg * a.p.kst[0] + r * a.p.kst[1]);
      const char* vp = vbase + 2 * (pg * a.p.vst[0] + r * a.p.vst[1]);
#pragma unroll
      for (int s = 0; s < kStep; ++s) kr[h][s] = *reinterpret_cast<const u32x4*>(kp + 64 * s);
#pragma unroll
      for (int s = 0; s < kStep; ++s) vr[h][s] = *reinterpret_cast<const u32x4*>(vp + 64 * s);
    }
  };

  f32x4 o[kOut];
#pragma unroll
  for (int t = 0; t < kOut; ++t) o[t] = f32x4{0, 0, 0, 0};
  float ref = lowest_ref(sc.c), sum = 0.0f;
  const float slack = Mx<T>::kDecSlack / sc.c;
  bool any = false;
  constexpr uint32_t kAll = NS == 2 ? 0xffffffffu : 0xffffu;

  int32_t page[NS], at[NS];
  if (a.p.n_pages > 0 && begin < last) {
    look_up(begin, page, at);
    load(page, at);
    look_up(begin + STEP, page, at);
    for (int tile = begin; tile < last; tile += STEP) {
      // scores
      f32x4 s[NS];
#pragma unroll
      for (int h = 0; h < NS; ++h) {
        s[h] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < kStep; ++k) s[h] = Mx<T>::mma16x32(kr[h][k], qf[k], s[h]);
      }
      const uint32_t now = there;
      if (now != kAll) {  // values that do not exist must not be multiplied by their zero weight
#pragma unroll
        for (int h = 0; h < NS; ++h)
          if (!((now >> (16 * h + m)) & 1))
#pragma unroll
            for (int k = 0; k < kStep; ++k) vr[h][k] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int h = 0; h < NS; ++h)
#pragma unroll
        for (int k = 0; k < kStep; ++k)
          *reinterpret_cast<u32x4*>(vt + (16 * h + m) * kRow + 64 * k + 16 * j) = vr[h][k];
      if (tile + STEP < last) {
        load(page, at);
        look_up(tile + 2 * STEP, page, at);
      }
      // weights
      float x[4 * NS], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) {
        x[i] = s[i / 4][i % 4];
        if constexpr (CAP) x[i] = cap_tanh<CAP>(x[i] * sc.inner);
      }
      const uint32_t mine = now >> (4 * j);  // this lane's keys: bits 0..3 and 16..19
      if (now != kAll) {
#pragma unroll
        for (int i = 0; i < 4 * NS; ++i)
          if (!((mine >> (16 * (i / 4) + i % 4)) & 1)) x[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) top = fmaxf(top, x[i]);
      if (__any(top > ref + slack)) {  // a head's own scores alone decide for it
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = top > ref + slack ? top : ref, f = lesser((ref - to) * sc.c);
        sum *= f;
#pragma unroll
        for (int t = 0; t < kOut; ++t) o[t] *= f;
        ref = to;
      }
      const float base = fmaf(-ref, sc.c, Mx<T>::kDecBias);
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], sc.c, base));
      any |= now != 0;
      uint32_t hi[2 * NS], lo[2 * NS];
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        sum += x[2 * i] + x[2 * i + 1];
        hi[i] = Mx<T>::pack(x[2 * i], x[2 * i + 1]);
        lo[i] = Mx<T>::pack(x[2 * i] - T::lo(hi[i]), x[2 * i + 1] - T::hi(hi[i]));
      }
      // O^T += V^T P^T
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < kOut; ++t) {
        const char* p = vt + (4 * j + m / 4) * kRow + 32 * t + 8 * (m & 3);
        const u32x2 v0 = lds_transposed(p);
        if constexpr (NS == 2) {
          const u32x2 v1 = lds_transposed(p + 16 * kRow);
          const u32x4 v = {v0[0], v0[1], v1[0], v1[1]};
          o[t] = Mx<T>::mma16x32(v, u32x4{hi[0], hi[1], hi[2], hi[3]}, o[t]);
          o[t] = Mx<T>::mma16x32(v, u32x4{lo[0], lo[1], lo[2], lo[3]}, o[t]);
        } else {
          o[t] = Mx<T>::mma16x16(v0, u32x2{hi[0], hi[1]}, o[t]);
          o[t] = Mx<T>::mma16x16(v0, u32x2{lo[0], lo[1]}, o[t]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

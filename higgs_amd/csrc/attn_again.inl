// attn_again.inl -- the keys of a walk once more, of heads whose scores do not fit the walk's
// weights or whose sums are not finite: one after the other in f32. The reference is the
// maximum, subtracted before the scale, and an infinity or NaN among the values
// counts however small its key's weight is (the two parts of a weight would
// not do: the lesser one may be zero or negative). Lane: head m, a quarter of D.
//
// Included as attn_walk.inl, over the same names and
//   qp, hk, acc   the head's q from the lane's quarter on, the kv head, the sums [D / 4]
// and leaves r and l, the reference and the weights' sum.
  constexpr int kPieces = D / 32;
  float r = lowest_ref(sc.c), l = 0.0f;
#pragma unroll
  for (int d = 0; d < D / 4; ++d) acc[d] = 0.0f;
#pragma unroll 1
  for (int i = begin * kKeys; i < min(last * kKeys, n); i += (i + 1) % kKeys ? 1 : 1 + (STEP - 1) * kKeys) {
    const int32_t key = key_of(i), pg = page_of(key);
    if ((uint32_t)pg >= (uint32_t)a.p.n_pages) continue;
    const int64_t row = key & a.p.page_mask;
    const char* kp = a.p.k + 2 * (hk * a.p.kst[2] + pg * a.p.kst[0] + row * a.p.kst[1] + j * (D / 4));
    const char* vp = a.p.v + 2 * (hk * a.p.vst[2] + pg * a.p.vst[0] + row * a.p.vst[1] + j * (D / 4));
    float x = 0.0f;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const u32x4 kw = *reinterpret_cast<const u32x4*>(kp + 16 * c);
      const u32x4 qw = *reinterpret_cast<const u32x4*>(qp + 16 * c);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t qq = (qw[w] & sc.keep) ^ sc.flip;
        x = fmaf(T::hi(kw[w]), T::hi(qq), fmaf(T::lo(kw[w]), T::lo(qq), x));
      }
    }
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
    if constexpr (CAP) x = cap_tanh<CAP>(x * sc.inner);
    if (x > r) {
      const float f = lesser((r - x) * sc.c);
      l *= f;
#pragma unroll
      for (int d = 0; d < D / 4; ++d) acc[d] *= f;
      r = x;
    }
    const float w = __builtin_amdgcn_exp2f(fmaf(x - r, sc.c, Mx<T>::kDecBias));
    const float odd = x == -INFINITY ? w : fmaxf(w, 1.0e-44f);
    l += w;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const u32x4 vw = *reinterpret_cast<const u32x4*>(vp + 16 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = e & 1 ? T::hi(vw[e / 2]) : T::lo(vw[e / 2]);
        acc[8 * c + e] = fmaf(v, fabsf(v) < INFINITY ? w : odd, acc[8 * c + e]);
      }
    }
  }

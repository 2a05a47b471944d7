// fattn_decode_q4.cuh — split-KV decode over a Q4_0 cache (included by fattn_mma.cu, which has the staging, the merge and the launch).
//
// At most 8 query rows per KV head, no explicit mask, no softcap.  Like the kernel over a Q8_0 cache, the keys are on the M side of
// both products (S^T = K.Q^T, O^T = V^T.P^T: a block's scale belongs to an accumulator row of the thread that loaded it, or rides
// on P), every warp copies the raw bytes of its own 16 keys of a tile and there is no barrier in the key loop.  What four bits change:
//
//   * A nibble in the low byte of a half IS a number: bits 0..3 are n * 2^-24, bits 4..7 are n * 2^-20, F16 denormals that the tensor
//     cores multiply exactly.  A word of a key's quants gives its eight values to two MMAs with one shift and four ands.  The
//     block's -8 goes into the accumulators' start (scores: -8 * sum of the query row over the block, a constant per row) or is
//     subtracted from the halves (values: the sum of P over keys has no bound to cancel against).  Query rows are scaled by a power
//     of two to a largest value in [2^10, 2^11), and by another 2^-4 where they meet the upper nibbles, so none of their bits is lost.
//   * 18-byte blocks: in a pair of blocks (9 words) the second one's 16 bytes of quants are four words, the first one's lie in three
//     words and two halves.  Which dims a thread of a quad contracts is free, so thread t takes word 1 + t, and thread 3 the halves.
//   * The result is exact to a few 2^-24 of its size, not to the 2^-11 of F16 weights: P enters the second product as two F16 terms,
//     hi = f16(P d) and lo = f16(P d - hi), d the block's scale, each product formed and split by fused multiply-adds.  With at most
//     four query rows (FEW) the two terms are columns 0..3 and 4..7 of ONE MMA, whose other half would be padding; with more, two.
//     P is held up to 2^14 for that (its top is 2^10 at the running maximum plus the 2^4 by which the maximum may lag), so that lo keeps its
//     bits above F16's smallest value; a warp that meets a scale of 2 or more lowers the top to 2^-4, for good, so that P d stays
//     finite for every scale.  (Values whose scale is below 2^-17 lose some of the extra bits.)
constexpr int kDecQ4Stages = 3;
constexpr int kDecQ4Skew = 16;   // a head's rows start on any 4-byte boundary: the copies start on the 16-byte unit around it

template <int HD, int NW, bool FEW>
__global__ void __launch_bounds__(32 * NW, 16 / NW) fattn_decode_q4_kernel(const FattnArgs a) {
    constexpr int NBLK = HD / 32, RB = NBLK * 18;
    constexpr int KT = 16 * NW;                        // keys per tile
    constexpr int RAW = 16 * RB + kDecQ4Skew;          // a warp's raw K or V bytes of a stage
    constexpr int NS = kDecQ4Stages;
    constexpr float kTop = 10.0f, kLowTop = -4.0f, kGrow = 4.0f;   // log2: P at the running maximum, with scales of 2 and more, and how far the maximum may lag
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __half* sQ = reinterpret_cast<__half*>(smem_raw);   // [8][HD], in the order the quads read them
    uint8_t* sRaw = smem_raw + 8 * HD * sizeof(__half);  // [NS][NW][K | V]
    __shared__ float s_m[NW][kDecRows], s_l[NW][kDecRows];
    __shared__ float s_negc[8 * NBLK], s_c[8];
    __shared__ __align__(8) uint64_t s_bar[NW][NS];      // one barrier per (warp, stage)

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const int bk = b / a.bq;
    const int R = a.Tq * a.gqa;  // <= 8 (FEW: <= 4); row rr -> (iq = rr / gqa, head hk*gqa + rr % gqa)
    const float ninf = -INFINITY;
    cluster_announce(a);

    const uint8_t* kbase = a.k.p + (int64_t)hk * a.k.nb2 + (int64_t)bk * a.k.nb3;
    const uint8_t* vbase = a.v.p + (int64_t)hk * a.v.nb2 + (int64_t)bk * a.v.nb3;
    const int kskew = (int)((uintptr_t)kbase & 15), vskew = (int)((uintptr_t)vbase & 15);
    if (lane < NS) {
        mbar_init(smem_u32(&s_bar[warp][lane]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the kernels before this one have completed and flushed
    const int len_b = clamp_len(a, b);
    const int tq_b = q_rows_of(a, b);
    static_assert(8 * (HD / 8) <= 32 * NW, "one chunk of a query row per thread");
    const int q_row = tid / (HD / 8), q_ch = tid % (HD / 8);
    uint4 q_val = make_uint4(0u, 0u, 0u, 0u), q_hi = q_val;
    const bool q_f32 = a.q.type == B200_TYPE_F32 && a.q.vec16;
    const int q_src = FEW ? q_row & 3 : q_row;   // FEW: columns 4..7 repeat rows 0..3
    if (q_row < 8 && q_src < R) {
        int iq, hq;
        row_to_query(a, hk, q_src, iq, hq);
        const uint8_t* rowp = a.q.p + (int64_t)iq * a.q.nb1 + (int64_t)hq * a.q.nb2 + (int64_t)b * a.q.nb3;
        if (q_f32) {
            q_val = load_global(reinterpret_cast<const uint4*>(rowp) + 2 * q_ch);
            q_hi = load_global(reinterpret_cast<const uint4*>(rowp) + 2 * q_ch + 1);
        } else {
            q_val = load8_as_half(rowp, a.q.type, q_ch * 8, a.hd, a.q.vec16);
        }
    }
    int kmax = tq_b > 0 ? len_b : 0, full = len_b;   // keys below `full` are seen by every row
    const int n_past = n_past_of(a, len_b, tq_b);
    if (a.causal) kmax = min(kmax, n_past + tq_b), full = min(full, n_past + 1);
    const int n_tiles = (kmax + KT - 1) / KT;
    const int tps = div_splits(a, n_tiles + a.n_splits - 1);
    const int tile_lo = split * tps, tile_hi = min(n_tiles, tile_lo + tps);
    // lanes 2s (K) and 2s+1 (V) of a warp copy the raw bytes of the warp's 16 keys of tile `tile0 + s`, from the 16-byte unit that
    // holds the first to the one that holds the last; lane 2s announces both copies to the stage's barrier
    auto issue_lanes = [&](int tile0, int n_stages) {
        const int s_ = lane >> 1, tile = tile0 + s_;
        if (s_ < n_stages && tile < tile_hi) {
            const int stage = (tile - tile_lo) % NS;
            const int r0 = tile * KT + 16 * warp;
            const int n = min(16, max(0, len_b - r0));
            const uint32_t kbytes = n ? (uint32_t)((kskew + n * RB + 15) & ~15) : 0, vbytes = n ? (uint32_t)((vskew + n * RB + 15) & ~15) : 0;
            const uint32_t bar = smem_u32(&s_bar[warp][stage]);
            if ((lane & 1) == 0) mbar_expect_tx(bar, kbytes + vbytes);
            if (n) {
                const uint32_t dst = smem_u32(sRaw + (stage * NW + warp) * 2 * RAW) + (lane & 1) * RAW;
                bulk_g2s(dst, ((lane & 1) ? vbase - vskew : kbase - kskew) + (int64_t)r0 * RB, (lane & 1) ? vbytes : kbytes, bar);
            }
        }
    };
    issue_lanes(tile_lo, NS);
    if (q_f32) q_val = f32x8_to_half(q_val, q_hi);
    if (q_row < 8) {
        // the row's largest magnitude to [2^10, 2^11): its exponent field over the HD / 8 lanes that hold it
        uint32_t h[4] = {q_val.x, q_val.y, q_val.z, q_val.w}, top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) top = max(top, max(h[i] & 0x7C00u, (h[i] >> 16) & 0x7C00u));
#pragma unroll
        for (int m = 1; m < HD / 8; m <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
        const int e = (int)(top >> 10), shift = e == 31 ? 0 : 25 - max(e, 1);   // (an infinity or NaN leaves the row as it is)
        const float up = __int_as_float((127 + shift) << 23);
        float f[8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            f[2 * i] = x.x * up, f[2 * i + 1] = x.y * up;
            sum += f[2 * i] + f[2 * i + 1];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int blk = q_ch >> 2;
        if ((q_ch & 3) == 0) s_negc[q_row * NBLK + blk] = sum * (-8.0f * 0x1p-24f);
        if (q_ch == 0) s_c[q_row] = a.scale * kLog2e * __int_as_float((127 + 24 - shift) << 23);
        // value 16 ks + j of a block to the place where the quad's thread that has byte j finds it: even blocks bytes 2 + 4t .. 5 + 4t
        // for t < 3 and 0, 1, 14, 15 for t = 3, odd blocks 4t .. 4t + 3; a thread's bytes 0, 2 | 1, 3 are its two registers
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int v = (q_ch & 3) * 8 + i, ks = v >> 4, j = v & 15;
            const int byte = blk & 1 ? j : (j < 2 ? 12 + j : (j > 13 ? j : j - 2));
            const int place = (byte & ~3) | ((byte & 1) << 1) | ((byte & 2) >> 1);
            sQ[q_row * HD + blk * 32 + ks * 16 + place] = __float2half_rn(ks ? f[i] * 0.0625f : f[i]);
        }
    }
    __syncthreads();
    uint32_t qb[NBLK][2][2];
    float negc[NBLK][2];
#pragma unroll
    for (int blk = 0; blk < NBLK; blk++) {
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const uint2 w = *reinterpret_cast<const uint2*>(sQ + g * HD + blk * 32 + ks * 16 + 4 * t);
            qb[blk][ks][0] = w.x, qb[blk][ks][1] = w.y;
        }
        negc[blk][0] = s_negc[2 * t * NBLK + blk], negc[blk][1] = s_negc[(2 * t + 1) * NBLK + blk];
    }
    const float c[2] = {s_c[2 * t], s_c[2 * t + 1]};
    int last[2];   // the last key that the thread's rows see
#pragma unroll
    for (int j = 0; j < 2; j++) last[j] = a.causal ? n_past + (FEW ? (2 * t + j) & 3 : 2 * t + j) / a.gqa : len_b - 1;

    float top = kTop;
    float m_run[2] = {ninf, ninf}, l_run[2] = {0.0f, 0.0f};   // reference (running maximum - top) and sum of rows 2t, 2t+1; the same on the lanes that share t
    float o[NBLK][2][4];   // [block][m-tile]: c0 / c1 = dim 32blk + 2g + mt of columns 2t / 2t+1 (times 2^-24), c2 / c3 = dim + 16 (times 2^-20)
#pragma unroll
    for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
        for (int mt = 0; mt < 2; mt++) o[blk][mt][0] = o[blk][mt][1] = o[blk][mt][2] = o[blk][mt][3] = 0.0f;
    const uint32_t sel3 = t == 3 ? 0x5432u : 0x7654u;
    const uint32_t eight_lo = 0x80088008u, eight_hi = 0x80808080u;   // -8 * 2^-24, -8 * 2^-20
    // FEW: columns 4..7 are the second terms
    const bool second = FEW && g >= 4;
    auto rescale = [&](int j, float alpha) {
        l_run[j] *= alpha;
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
            for (int mt = 0; mt < 2; mt++) o[blk][mt][j] *= alpha, o[blk][mt][2 + j] *= alpha;
    };

    for (int tile = tile_lo; tile < tile_hi; tile++) {
        const int key0 = tile * KT + 16 * warp;   // this warp's 16 keys
        const int stage = (tile - tile_lo) % NS;
        if (!mbar_wait_bounded(smem_u32(&s_bar[warp][stage]), (uint32_t)((tile - tile_lo) / NS) & 1u)) break;
        const uint8_t* rawK = sRaw + (stage * NW + warp) * 2 * RAW + kskew;
        const uint8_t* rawV = sRaw + (stage * NW + warp) * 2 * RAW + RAW + vskew;
        const int rows_valid = len_b - key0;      // keys at or beyond it hold stale bytes

        // ---- S^T = K.Q^T: keys g and g+8, columns 2t and 2t+1 ----
        float st[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int pair = 0; pair < NBLK / 2; pair++) {
            uint32_t w[2][2];   // [block of the pair][key]
            float d[2][2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t* W = reinterpret_cast<const uint32_t*>(rawK + (g + 8 * i) * RB + 36 * pair);
                const uint32_t w0 = W[0], w4 = W[4], mine = t == 3 ? w4 : W[1 + t];
                w[0][i] = __byte_perm(w0, mine, sel3);
                w[1][i] = W[5 + t];
                d[0][i] = __half2float(__ushort_as_half((uint16_t)w0));
                d[1][i] = __half2float(__ushort_as_half((uint16_t)(w4 >> 16)));
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int blk = 2 * pair + u;
                float acc[4] = {negc[blk][0], negc[blk][1], negc[blk][0], negc[blk][1]};
                const uint32_t s0 = w[u][0] >> 8, s1 = w[u][1] >> 8;
                const uint32_t lo[4] = {w[u][0] & 0x000F000Fu, w[u][1] & 0x000F000Fu, s0 & 0x000F000Fu, s1 & 0x000F000Fu};
                const uint32_t hi[4] = {w[u][0] & 0x00F000F0u, w[u][1] & 0x00F000F0u, s0 & 0x00F000F0u, s1 & 0x00F000F0u};
                mma16816(acc, lo, qb[blk][0][0], qb[blk][0][1]);
                mma16816(acc, hi, qb[blk][1][0], qb[blk][1][1]);
                st[0] = fmaf(d[u][0], acc[0], st[0]), st[1] = fmaf(d[u][0], acc[1], st[1]);
                st[2] = fmaf(d[u][1], acc[2], st[2]), st[3] = fmaf(d[u][1], acc[3], st[3]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) st[e] *= c[e & 1];
        if (key0 + 16 > full) {   // not every key is seen by every row
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int key = key0 + g + 8 * (e >> 1);
                if (key >= len_b || key > last[e & 1]) st[e] = ninf;
            }
        }

        // ---- the block scales of V, keys 2t, 2t+1 | 2t+8, 2t+9; those of dead keys read as 0 ----
        uint32_t d01[NBLK], d23[NBLK], any_scale = 0;
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++) {
            uint32_t ds[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                ds[i] = *reinterpret_cast<const uint16_t*>(rawV + key * RB + blk * 18);
                if (rows_valid < 16 && key >= rows_valid) ds[i] = 0;
            }
            d01[blk] = __byte_perm(ds[0], ds[1], 0x5410), d23[blk] = __byte_perm(ds[2], ds[3], 0x5410);
            any_scale |= d01[blk] | d23[blk];
        }

        // ---- lazy running maximum, and the top of P: bit 14 of a half says 2 and more ----
        const float lm[2] = {fmaxf(st[0], st[2]), fmaxf(st[1], st[3])};
        const bool lower = top != kLowTop && (any_scale & 0x40004000u);
        if (__any_sync(0xffffffffu, lm[0] > m_run[0] + (top + kGrow) || lm[1] > m_run[1] + (top + kGrow) || lower)) {
            if (__any_sync(0xffffffffu, lower)) {
#pragma unroll
                for (int j = 0; j < 2; j++) m_run[j] += top - kLowTop, rescale(j, 0x1p-14f);
                static_assert(kTop - kLowTop == 14.0f, "");
                top = kLowTop;
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float rm = lm[j];
                rm = fmaxf(rm, __shfl_xor_sync(0xffffffffu, rm, 4));
                rm = fmaxf(rm, __shfl_xor_sync(0xffffffffu, rm, 8));
                rm = fmaxf(rm, __shfl_xor_sync(0xffffffffu, rm, 16));
                if (rm > m_run[j] + (top + kGrow)) {   // -inf > -inf is false: the first finite maximum is taken
                    rescale(j, exp2f(m_run[j] - (rm - top)));   // m_run = -inf -> 0
                    m_run[j] = rm - top;
                }
            }
        }
        const float muse[2] = {m_run[0] == ninf ? 0.0f : m_run[0], m_run[1] == ninf ? 0.0f : m_run[1]};
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            p[e] = fast_ex2(st[e] - muse[e & 1]);
            l_run[e & 1] += p[e];
        }
        // P^T as the B operand: (key g, columns 2t, 2t+1) -> (keys 2t, 2t+1, column g), the F16 values and what they leave of P
        const uint32_t h0 = pack_half2(p[0], p[1]), h1 = pack_half2(p[2], p[3]);
        const float2 r0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), r1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        uint32_t ph[2] = {movmatrix_trans(h0), movmatrix_trans(h1)};
        uint32_t pl[2] = {movmatrix_trans(pack_half2(p[0] - r0.x, p[1] - r0.y)), movmatrix_trans(pack_half2(p[2] - r1.x, p[3] - r1.y))};
        __half2 P[2], N[2], L[2];   // P, what P d is taken from (FEW: nothing for the first terms), the rest of P (FEW: nothing for the first terms)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            P[i] = *reinterpret_cast<const __half2*>(&ph[i]);
            if (FEW) {
                const uint32_t n = second ? ph[i] ^ 0x80008000u : 0u, l = second ? pl[i] : 0u;
                N[i] = *reinterpret_cast<const __half2*>(&n), L[i] = *reinterpret_cast<const __half2*>(&l);
            } else {
                L[i] = *reinterpret_cast<const __half2*>(&pl[i]);
            }
        }

        // ---- O^T += V^T.P^T: this thread's bytes are 2g, 2g+1 of each block ----
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const uint16_t*>(rawV + (2 * t + (i & 1) + 8 * (i >> 1)) * RB + blk * 18 + 2 + 2 * g);
            const uint32_t x01 = __byte_perm(w[0], w[1], 0x5410), x23 = __byte_perm(w[2], w[3], 0x5410);
            const __half2 d2[2] = {*reinterpret_cast<const __half2*>(&d01[blk]), *reinterpret_cast<const __half2*>(&d23[blk])};
            uint32_t first_term[2], second_term[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const __half2 hi = FEW ? __hmul2(N[i], d2[i]) : __hmul2(P[i], d2[i]);
                const __half2 lo = __hfma2(L[i], d2[i], __hfma2(P[i], d2[i], FEW ? hi : __hneg2(hi)));
                first_term[i] = *reinterpret_cast<const uint32_t*>(&hi), second_term[i] = *reinterpret_cast<const uint32_t*>(&lo);
            }
            auto minus = [](uint32_t x, uint32_t e) {
                const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&e));
                return *reinterpret_cast<const uint32_t*>(&v);
            };
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                const uint32_t y01 = mt ? x01 >> 8 : x01, y23 = mt ? x23 >> 8 : x23;
                const uint32_t af[4] = {minus(y01 & 0x000F000Fu, eight_lo), minus(y01 & 0x00F000F0u, eight_hi), minus(y23 & 0x000F000Fu, eight_lo),
                                        minus(y23 & 0x00F000F0u, eight_hi)};
                if (!FEW) mma16816(o[blk][mt], af, first_term[0], first_term[1]);
                mma16816(o[blk][mt], af, second_term[0], second_term[1]);
            }
        }
        __syncwarp();   // every lane is done with this stage's bytes
        issue_lanes(tile + NS, 1);
    }

    let_dependents_launch();
    // ---- merge the warps' (m, l, O) in shared memory ----
    constexpr int SLAB_STRIDE = HD + 4;
    static_assert(NW * 8 * SLAB_STRIDE * sizeof(float) <= 8 * HD * sizeof(__half) + NS * NW * 2 * RAW, "the slabs lie where the stages were");
    float* slab = reinterpret_cast<float*>(smem_raw);   // [NW][8][SLAB_STRIDE]
    float lq[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        float v = l_run[j];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        lq[j] = v;
    }
    if (g == 0) {
        s_m[warp][2 * t] = m_run[0], s_m[warp][2 * t + 1] = m_run[1];
        s_l[warp][2 * t] = lq[0], s_l[warp][2 * t + 1] = lq[1];
    }
    __syncthreads();  // the warps' (m, l) are visible, and all warps are done with the raw stages (the merge slabs alias them)
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if ((FEW ? (2 * t + j) & 3 : 2 * t + j) >= R) continue;
        float* row = slab + (warp * 8 + 2 * t + j) * SLAB_STRIDE + 2 * g;
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++) {
            *reinterpret_cast<float2*>(row + 32 * blk) = make_float2(o[blk][0][j] * 0x1p24f, o[blk][1][j] * 0x1p24f);
            *reinterpret_cast<float2*>(row + 32 * blk + 16) = make_float2(o[blk][0][2 + j] * 0x1p20f, o[blk][1][2 + j] * 0x1p20f);
        }
    }
    __syncthreads();
    decode_write_out<HD, NW, 8, FEW>(a, slab, s_m, s_l, sRaw + NS * NW * 2 * RAW, R, b, hk, split, tq_b, tid);
}

// fattn_decode_q4.cuh — split-KV decode over a Q4_0 cache (included by fattn_mma.cu, which has the staging, the merge and the launch).
//
// No explicit mask, no softcap; at most 8 query rows per CTA (9 to 16 rows of a KV head are two CTAs, the second of which finds the
// keys in L2).  Like the kernel over a Q8_0 cache, the keys are on the M side of
// both products (S^T = K.Q^T, O^T = V^T.P^T: a block's scale belongs to an accumulator row of the thread that loaded it, or rides
// on P), every warp copies the raw bytes of its own 16 keys of a tile and there is no barrier in the key loop.  What four bits change:
//
//   * A nibble becomes a number by a mask and one multiply-add: bits 0..3 of a half are the denormal n * 2^-24, bits 4..7 n * 2^-20, and
//     times 2^15 or 2^11 less 2^-6 either is (n - 8) * 2^-9, exactly.  A word of a key's quants is eight values in 1 shift, 4 masks, 4
//     multiply-adds; the block's -8 never enters a sum that would have to cancel it.
//   * 18-byte blocks: in a pair of blocks (9 words) the second one's 16 bytes of quants are four words, the first one's lie in three
//     words and two halves.  Which dims a thread of a quad contracts is free, so thread t takes word 1 + t, and thread 3 the halves.
//   * The result is that of fp32 arithmetic (relative L2 3e-7 against a 64-bit run; 3e-4 with P and V rounded to F16): P enters the second
//     product as two F16 terms, hi = f16(P d) and lo = f16(P d - hi), d the block's scale, formed and split by fused multiply-adds.
//     With at most four query rows (FEW) the two terms are columns 0..3 and 4..7 of ONE MMA, whose other half would be padding;
//     with more, two.  P is held up to 2^14 for that (its top is 2^10 at the running maximum plus the 2^4 by which the maximum may
//     lag), so that lo keeps its bits above F16's smallest value.  The scales have to fit that range: a warp that meets one of 2^e, e > 0, lowers the
//     top to 2^(10 - e), for good, so that P d stays finite; and where some run of 32 values of head_dim has only small scales (none of 2^-7 in the
//     warp's first keys, or what a lowered top leaves small), these are multiplied by a power of two that its accumulators keep until the end (V of 1e-6: relative
//     error 2e-7, without it 2e-4 to 7e-4).  Of a product of weight and scale what counts is kept to 2^-28 of the largest scale so far in its run of
//     32.  256 streams x 4096 keys 182.1 -> 185.4 us by it, 64 ragged streams of six rows 29.6 -> 30.6, 97 keys 3.2 -> 3.4; a second copy of the key loop for such
//     values, or scales rewritten in shared memory, cost 2 to 6 %.  The products of 32
//     keys are summed by themselves and then added: the tensor cores cut a sum off at its last bit, which over thousands of keys showed as
//     a shrinkage of 1e-6.
//
// What bounds it: the issue of instructions by four warps per scheduler, whose own fixed latencies leave a third of the slots empty (78 % of them used on a full SM,
// 67 % over the launch; no pipe is full: ALU 50 %, LSU 37, FMA 26, HMMA 22).  Per 16 keys of head_dim 128 a warp issues 388: 128 masks and multiply-adds of the nibbles, 52 from
// and to shared memory (18-byte blocks come in words and halves), 28 for the scales of V, 24 that split P d, 20 MMAs; masks, shifts, byte
// selections and half-precision arithmetic take two clocks each.  256 streams x 8 KV heads of up to 4096 keys (0.81 GB) 185 us, 4.4 TB/s or
// 0.68 of the measured copy rate; in a loop of seconds, at the power limit, 207.  Stages
// of 16 keys, whose waits, votes and addresses are per 16 keys, 238 us; 96 registers for a fifth CTA per SM, which leave no two m-tiles to
// overlap, 218 where 128 registers took 198.
constexpr int kDecQ4Stages = 2;
constexpr int kDecQ4Keys = 32;   // keys of a warp per stage: two m16 tiles, which share the waits, the votes and the addresses
constexpr int kDecQ4Skew = 16;   // a head's rows start on any 4-byte boundary: the copies start on the 16-byte unit around it

// d = a.b
__device__ __forceinline__ void mma16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// Nibbles n as (n - 8) * 2^-9.  (The tensor cores take the denormals as they are, too, but align products by the fields of their
// exponents: a score was then off by 2^-20 of itself instead of 2^-23.)
__device__ __forceinline__ uint32_t nibbles(uint32_t masked, uint32_t up) {
    const uint32_t less = 0xA400A400u;   // -2^-6
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&masked), *reinterpret_cast<const __half2*>(&up), *reinterpret_cast<const __half2*>(&less));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t low_nibbles(uint32_t x) { return nibbles(x & 0x000F000Fu, 0x78007800u); }    // 2^15
__device__ __forceinline__ uint32_t high_nibbles(uint32_t x) { return nibbles(x & 0x00F000F0u, 0x68006800u); }   // 2^11

template <int HD, int NW, bool FEW>
__global__ void __launch_bounds__(32 * NW, 16 / NW) fattn_decode_q4_kernel(const FattnArgs a) {
    constexpr int NBLK = HD / 32, RB = NBLK * 18, NS = kDecQ4Stages, WK = kDecQ4Keys, NT = WK / 16;
    constexpr int KT = WK * NW;                        // keys per tile
    constexpr int RAW = WK * RB + kDecQ4Skew;          // a warp's raw K or V bytes of a stage
    constexpr float kTop = 10.0f, kGrow = 4.0f;   // log2: P at the running maximum while every scale is below 2, and how far the maximum may lag
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __half* sQ = reinterpret_cast<__half*>(smem_raw);   // [8][HD], in the order the quads read them
    uint8_t* sRaw = smem_raw + 8 * HD * sizeof(__half);  // [NW][NS][K | V]
    __shared__ float s_m[NW][kDecRows], s_l[NW][kDecRows];
    __shared__ __align__(8) uint64_t s_bar[NW][NS];      // one barrier per (warp, stage)

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int all_rows = a.Tq * a.gqa;   // <= 16; row rr -> (iq = rr / gqa, head hk*gqa + rr % gqa)
    const int pair = !FEW && all_rows > 8, split = blockIdx.x, hk = blockIdx.y >> pair, b = blockIdx.z;
    const int bk = b / a.bq;
    const int row0 = pair ? 8 * (blockIdx.y & 1) : 0, R = min(8, all_rows - row0);   // this CTA's rows (FEW: <= 4)
    const float ninf = -INFINITY;
    cluster_announce(a);

    // lane 0 copies K, lane 1 V, each from the 16-byte unit around its first row on
    const uint8_t* base = (lane & 1 ? a.v.p + (int64_t)hk * a.v.nb2 + (int64_t)bk * a.v.nb3 : a.k.p + (int64_t)hk * a.k.nb2 + (int64_t)bk * a.k.nb3);
    const int skew = (int)((uintptr_t)base & 15);
    base -= skew;
    const int kskew = __shfl_sync(0xffffffffu, skew, 0), vskew = __shfl_sync(0xffffffffu, skew, 1);
    uint8_t* stages = sRaw + warp * NS * 2 * RAW;
    const uint32_t bar = smem_u32(&s_bar[warp][0]), my_stage = smem_u32(stages) + (lane & 1) * RAW;
    if (lane < NS) {
        mbar_init(bar + 8 * lane, 2);   // two lanes arrive, each with the bytes of its own copy
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
        row_to_query(a, hk, row0 + q_src, iq, hq);
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
    // The raw bytes of WK keys from the warp's next ones on, up to the 16-byte unit that holds the last valid row's end
    int key0 = tile_lo * KT + WK * warp;            // this warp's keys of the current tile
    const int key_end = min(tile_hi * KT, kmax);    // (a warp whose keys all lie behind the last visible one has nothing to do)
    const uint8_t* next = base + (int64_t)key0 * RB;
    constexpr uint32_t kWhole = WK * RB;            // a multiple of 16
    const uint32_t whole = kWhole + (uint32_t)((skew + 15) & ~15);
    auto issue = [&](int key, int stage) {
        if (lane < 2) {
            const uint32_t bytes = key + WK <= len_b ? whole : (uint32_t)((skew + (len_b - key) * RB + 15) & ~15);   // (key < key_end <= len_b)
            mbar_expect_tx(bar + 8 * stage, bytes);
            bulk_g2s(my_stage + stage * 2 * RAW, next, bytes, bar + 8 * stage);
        }
        next += (int64_t)KT * RB;
    };
#pragma unroll
    for (int i = 0; i < NS; i++)
        if (key0 + i * KT < key_end) issue(key0 + i * KT, i);
    if (q_f32) q_val = f32x8_to_half(q_val, q_hi);
    if (q_row < 8) {
        // rows behind q_len may hold anything: their result is a zero times what comes of them
        if ((row0 + q_src) / a.gqa >= tq_b) q_val = make_uint4(0u, 0u, 0u, 0u);
        const int blk = q_ch >> 2;
        const __half* h = reinterpret_cast<const __half*>(&q_val);
        // value 16 ks + j of a block to the place where the quad's thread that has byte j finds it: even blocks bytes 2 + 4t .. 5 + 4t
        // for t < 3 and 0, 1, 14, 15 for t = 3, odd blocks 4t .. 4t + 3; a thread's bytes 0, 2 | 1, 3 are its two registers
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int v = (q_ch & 3) * 8 + i, ks = v >> 4, j = v & 15;
            const int byte = blk & 1 ? j : (j < 2 ? 12 + j : (j > 13 ? j : j - 2));
            const int place = (byte & ~3) | ((byte & 1) << 1) | ((byte & 2) >> 1);
            sQ[q_row * HD + blk * 32 + ks * 16 + place] = h[i];
        }
    }
    __syncthreads();
    uint32_t qb[NBLK][2][2];
#pragma unroll
    for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const uint2 w = *reinterpret_cast<const uint2*>(sQ + g * HD + blk * 32 + ks * 16 + 4 * t);
            qb[blk][ks][0] = w.x, qb[blk][ks][1] = w.y;
        }
    const float c = a.scale * kLog2e * 512.0f;   // (quants enter as 2^-9 of themselves)
    int last[2];   // the last key that the thread's rows see
#pragma unroll
    for (int j = 0; j < 2; j++) last[j] = a.causal ? min(len_b - 1, n_past + (FEW ? (2 * t + j) & 3 : row0 + 2 * t + j) / a.gqa) : len_b - 1;

    float top = kTop;
    // Exponent fields of the largest scales so far, a byte per block of 32 values of head_dim; 15 (a scale of 1 to 2) stands for everything from 2^-7 on as
    // long as nothing else was met.  What is missing to the top of P d's range is made up for by scales that enter the second product times 2^raised.
    constexpr uint32_t kUnseen = 0x80808080u, kUsual = 0x0F0F0F0Fu;
    uint32_t fields = kUnseen;
    auto raised = [&](int blk) {   // (nothing has been summed while no scale was seen)
        const int room = 25 - (int)top - (int)(fields >> (8 * blk) & 31u);
        return fields != kUnseen && room > 3 ? room : 0;
    };
    float m_run[2] = {ninf, ninf}, l_run[2] = {0.0f, 0.0f};   // reference (running maximum - top) and sum of rows 2t, 2t+1; the same on the lanes that share t
    float minus_m[2] = {0.0f, 0.0f}, bound[2] = {ninf, ninf};  // what is added to a score (nothing while the reference is -inf), and the largest that needs no new one
    float o[NBLK][2][4];   // [block][m-tile]: c0 / c1 = dim 32blk + 2g + mt of columns 2t / 2t+1, c2 / c3 = dim + 16, all times 2^-9
#pragma unroll
    for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
        for (int mt = 0; mt < 2; mt++) o[blk][mt][0] = o[blk][mt][1] = o[blk][mt][2] = o[blk][mt][3] = 0.0f;
    const uint32_t sel3 = t == 3 ? 0x5432u : 0x7654u;
    const uint32_t second = FEW && g >= 4 ? 0xFFFFFFFFu : 0u;   // FEW: columns 4..7 are the second terms
    auto rescale = [&](int j, float alpha) {
        l_run[j] *= alpha;
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
            for (int mt = 0; mt < 2; mt++) o[blk][mt][j] *= alpha, o[blk][mt][2 + j] *= alpha;
    };

    for (int stage = 0, parity = 0; key0 < key_end; key0 += KT) {
        // (every lane has to have seen the phase complete itself: that is what orders the copied bytes before its reads, a vote orders none)
        if (!__all_sync(0xffffffffu, mbar_try_wait(bar + 8 * stage, (uint32_t)parity)) && !mbar_wait_bounded(bar + 8 * stage, (uint32_t)parity)) break;
        const uint8_t* rawK = stages + stage * 2 * RAW + kskew;
        const uint8_t* rawV = stages + stage * 2 * RAW + RAW + vskew;

        // ---- S^T = K.Q^T: per m-tile keys g and g+8, columns 2t and 2t+1 ----
        float st[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            st[nt][0] = st[nt][1] = st[nt][2] = st[nt][3] = 0.0f;
#pragma unroll
            for (int pair = 0; pair < NBLK / 2; pair++) {
                uint32_t w[2][2];   // [block of the pair][key]
                float d[2][2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t* W = reinterpret_cast<const uint32_t*>(rawK + (16 * nt + g + 8 * i) * RB + 36 * pair);
                    const uint32_t w0 = W[0], w4 = W[4];
                    w[0][i] = __byte_perm(w0, W[1 + t], sel3);
                    w[1][i] = W[5 + t];
                    d[0][i] = __half2float(__ushort_as_half((uint16_t)w0));
                    d[1][i] = __half2float(__ushort_as_half((uint16_t)(w4 >> 16)));
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int blk = 2 * pair + u;
                    float acc[4];
                    const uint32_t s0 = w[u][0] >> 8, s1 = w[u][1] >> 8;
                    const uint32_t lo[4] = {low_nibbles(w[u][0]), low_nibbles(w[u][1]), low_nibbles(s0), low_nibbles(s1)};
                    const uint32_t hi[4] = {high_nibbles(w[u][0]), high_nibbles(w[u][1]), high_nibbles(s0), high_nibbles(s1)};
                    mma16816_from(acc, lo, qb[blk][0][0], qb[blk][0][1]);
                    mma16816(acc, hi, qb[blk][1][0], qb[blk][1][1]);
                    st[nt][0] = fmaf(d[u][0], acc[0], st[nt][0]), st[nt][1] = fmaf(d[u][0], acc[1], st[nt][1]);
                    st[nt][2] = fmaf(d[u][1], acc[2], st[nt][2]), st[nt][3] = fmaf(d[u][1], acc[3], st[nt][3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 x = __fmul2_rn(make_float2(st[nt][2 * i], st[nt][2 * i + 1]), make_float2(c, c));
                st[nt][2 * i] = x.x, st[nt][2 * i + 1] = x.y;
            }
        }
        const bool edge = key0 + WK > full;
        if (edge) {   // not every key is seen by every row
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (key0 + 16 * nt + g + 8 * (e >> 1) > last[e & 1]) st[nt][e] = ninf;
        }

        // ---- the block scales of V, keys 2t, 2t+1 | 2t+8, 2t+9 of each m-tile; those of dead keys read as 0 ----
        uint32_t dv[NT][NBLK][2], any_scale = 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int blk = 0; blk < NBLK; blk++) {
                uint32_t ds[4];
#pragma unroll
                for (int i = 0; i < 4; i++) ds[i] = *reinterpret_cast<const uint16_t*>(rawV + (16 * nt + 2 * t + (i & 1) + 8 * (i >> 1)) * RB + blk * 18);
                dv[nt][blk][0] = __byte_perm(ds[0], ds[1], 0x5410), dv[nt][blk][1] = __byte_perm(ds[2], ds[3], 0x5410);
            }
        if (edge) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int key = key0 + 16 * nt + 2 * t + 8 * i;
                    const uint32_t live = (key < len_b ? 0x0000FFFFu : 0u) | (key + 1 < len_b ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int blk = 0; blk < NBLK; blk++) dv[nt][blk][i] &= live;
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int blk = 0; blk < NBLK; blk++) any_scale |= dv[nt][blk][0] | dv[nt][blk][1];

        // ---- lazy running maximum, and the top of P: bit 14 of a half says that a scale is 2 or more ----
        float lm[2] = {st[0][0], st[0][1]};
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = nt ? 0 : 2; e < 4; e++) lm[e & 1] = fmaxf(lm[e & 1], st[nt][e]);
        if (__any_sync(0xffffffffu, lm[0] > bound[0] || lm[1] > bound[1] || (any_scale & 0x40004000u))) {
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
                minus_m[j] = m_run[j] == ninf ? 0.0f : -m_run[j], bound[j] = m_run[j] + (top + kGrow);
            }
            bool fit = __any_sync(0xffffffffu, any_scale & 0x40004000u);
            if (fields != kUsual) {
                if (fields == kUnseen) {   // the warp's first keys
                    uint32_t usual = 0;
#pragma unroll
                    for (int blk = 0; blk < NBLK; blk++) {
                        uint32_t seen = 0;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) seen |= dv[nt][blk][0] | dv[nt][blk][1];
                        usual |= seen & 0x60006000u ? 1u << blk : 0u;
                    }
                    if (__reduce_or_sync(0xffffffffu, usual) == (1u << NBLK) - 1) fields = kUsual;
                    else fit = true;
                } else {
#pragma unroll
                    for (int blk = 0; blk < NBLK; blk++) fit |= raised(blk) > 0;
                }
            }
            if (fit) {   // exponent fields E of the largest scales: d < 2^(E - 14)
                int was[NBLK], field[NBLK], most = 0;
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) {
                    uint32_t largest = 0;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < 2; i++) largest = max(largest, max(dv[nt][blk][i] & 0x7C00u, (dv[nt][blk][i] >> 16) & 0x7C00u));
                    was[blk] = raised(blk);
                    field[blk] = max((int)(__reduce_max_sync(0xffffffffu, largest) >> 10), (int)(fields >> (8 * blk) & 31u));
                    most = max(most, min(field[blk], 30));   // (an infinite scale has no range)
                }
                const float lower = fminf(top, 25.0f - (float)most);
                if (lower < top) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        m_run[j] += top - lower, rescale(j, exp2f(lower - top));
                        minus_m[j] = m_run[j] == ninf ? 0.0f : -m_run[j], bound[j] = m_run[j] + (lower + kGrow);
                    }
                    top = lower;
                }
                fields = 0;
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) {
                    fields |= (uint32_t)field[blk] << (8 * blk);
                    const int up = raised(blk);
                    if (up != was[blk]) {
                        const float f = exp2f((float)(up - was[blk]));
#pragma unroll
                        for (int mt = 0; mt < 2; mt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[blk][mt][e] *= f;
                    }
                    if (up) {   // by two powers of two, of which F16 holds either
                        bound[0] = bound[1] = ninf;   // (the next keys' scales come here too)
                        const uint32_t a = (uint32_t)(15 + up / 2) << 10, b = (uint32_t)(15 + up - up / 2) << 10;
                        const uint32_t a2 = a | a << 16, b2 = b | b << 16;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const __half2 x = __hmul2(__hmul2(*reinterpret_cast<const __half2*>(&dv[nt][blk][i]), *reinterpret_cast<const __half2*>(&a2)), *reinterpret_cast<const __half2*>(&b2));
                                dv[nt][blk][i] = *reinterpret_cast<const uint32_t*>(&x);
                            }
                    }
                }
            }
        }
        // P^T as the B operand: (key g, columns 2t, 2t+1) -> (keys 2t, 2t+1, column g), the F16 values and what they leave of P
        __half2 P[NT][2], N[NT][2], L[NT][2];   // P, what P d is taken from (FEW: nothing for the first terms), the rest of P (FEW: nothing for the first terms)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 x = __fadd2_rn(make_float2(st[nt][2 * i], st[nt][2 * i + 1]), make_float2(minus_m[0], minus_m[1]));
                const float2 p = make_float2(fast_ex2(x.x), fast_ex2(x.y)), sum = __fadd2_rn(make_float2(l_run[0], l_run[1]), p);
                l_run[0] = sum.x, l_run[1] = sum.y;
                const uint32_t h = pack_half2(p.x, p.y);
                const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h)), rest = __fadd2_rn(p, make_float2(-r.x, -r.y));
                const uint32_t ph = movmatrix_trans(h), pl = movmatrix_trans(pack_half2(rest.x, rest.y));
                P[nt][i] = *reinterpret_cast<const __half2*>(&ph);
                const uint32_t n = (ph ^ 0x80008000u) & second, l = FEW ? pl & second : pl;
                N[nt][i] = *reinterpret_cast<const __half2*>(&n), L[nt][i] = *reinterpret_cast<const __half2*>(&l);
            }

        // ---- O^T += V^T.P^T: this thread's bytes are 2g, 2g+1 of each block ----
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++) {
            float part[2][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    w[i] = *reinterpret_cast<const uint16_t*>(rawV + (16 * nt + 2 * t + (i & 1) + 8 * (i >> 1)) * RB + blk * 18 + 2 + 2 * g);
                const uint32_t x01 = __byte_perm(w[0], w[1], 0x5410), x23 = __byte_perm(w[2], w[3], 0x5410);
                uint32_t first_term[2], second_term[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const __half2 d2 = *reinterpret_cast<const __half2*>(&dv[nt][blk][i]);
                    const __half2 hi = FEW ? __hmul2(N[nt][i], d2) : __hmul2(P[nt][i], d2);
                    const __half2 lo = __hfma2(L[nt][i], d2, __hfma2(P[nt][i], d2, FEW ? hi : __hneg2(hi)));
                    first_term[i] = *reinterpret_cast<const uint32_t*>(&hi), second_term[i] = *reinterpret_cast<const uint32_t*>(&lo);
                }
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    const uint32_t y01 = mt ? x01 >> 8 : x01, y23 = mt ? x23 >> 8 : x23;
                    const uint32_t af[4] = {low_nibbles(y01), high_nibbles(y01), low_nibbles(y23), high_nibbles(y23)};
                    // the keys' sum by itself: the tensor cores cut a sum off at its last bit, which over a long cache is a bias
                    if (nt == 0) mma16816_from(part[mt], af, second_term[0], second_term[1]);
                    else mma16816(part[mt], af, second_term[0], second_term[1]);
                    if (!FEW) mma16816(part[mt], af, first_term[0], first_term[1]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float2 sum = __fadd2_rn(make_float2(o[blk][mt][2 * i], o[blk][mt][2 * i + 1]), make_float2(part[mt][2 * i], part[mt][2 * i + 1]));
                    o[blk][mt][2 * i] = sum.x, o[blk][mt][2 * i + 1] = sum.y;
                }
        }
        __syncwarp();   // every lane is done with this stage's bytes
        if (key0 + NS * KT < key_end) issue(key0 + NS * KT, stage);
        static_assert(NS == 2, "");
        parity ^= stage, stage ^= 1;
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
    float unit[NBLK];
#pragma unroll
    for (int blk = 0; blk < NBLK; blk++) unit[blk] = __int_as_float((127 + 9 - raised(blk)) << 23);   // 2^(9 - raised)
    if (g == 0) {
#pragma unroll
        for (int j = 0; j < 2; j++) {   // (scores that are no numbers raise no maximum: the row must not pass for one without keys)
            s_m[warp][2 * t + j] = lq[j] == lq[j] ? m_run[j] : 0.0f;
            s_l[warp][2 * t + j] = lq[j];
        }
    }
    __syncthreads();  // the warps' (m, l) are visible, and all warps are done with the raw stages (the merge slabs alias them)
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if ((FEW ? (2 * t + j) & 3 : 2 * t + j) >= R) continue;
        float* row = slab + (warp * 8 + 2 * t + j) * SLAB_STRIDE + 2 * g;
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++) {
            *reinterpret_cast<float2*>(row + 32 * blk) = make_float2(o[blk][0][j] * unit[blk], o[blk][1][j] * unit[blk]);
            *reinterpret_cast<float2*>(row + 32 * blk + 16) = make_float2(o[blk][0][2 + j] * unit[blk], o[blk][1][2 + j] * unit[blk]);
        }
    }
    __syncthreads();
    decode_write_out<HD, NW, 8, FEW>(a, slab, s_m, s_l, sRaw + NW * NS * 2 * RAW, R, b, hk, split, tq_b, tid, row0);
}

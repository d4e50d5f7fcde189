// Low-rank adapters of many requests beside a shared projection (llattn_adapters_w4a8).
//
// Tokens come in segments, each with an adapter of a pool or none:
//   H[n][j] = c_a * sum_g s[n][g] * (sum_{k in group g} q[n][k] * A_a[j][k])       j < rank of adapter a
//   Y[n][row0 + i] += sum_j H[n][j] * B_a[i][j]
// from the int8 activations that the projection itself reads (codes in fragment order, one scale for each group of 128).
//
// A cluster takes up to 32 tokens of one segment. Each of its CTAs has a part of the groups in the first product and a part of the rows in the second;
// in between it stores its sums of H into the others' shared memory (st.async, counted in on a barrier there), and each adds all of them up in
// the CTAs' order.
//
// First product: the codes are exact in 16 bits, so mma.sync multiplies them with A as it is, and each group's sum takes its scale in fp32: nothing is
// rounded but the fp32 sums. A lane's word of the fragment order is four neighbouring values of a run of sixteen; the four K slots of a lane
// in an m16n8k16 are given to just these, and A is read to match, eight bytes a lane. Groups of A, codes and scales come through cp.async, two to four
// ahead.
//
// Second product: B is multiplied as it is, too, with H in parts that have all of its exponents: three of bf16 for bf16 (24 bits), two of tf32 for fp16 (22
// bits), whose B is widened (11 bits, exact). One part alone would leave 2^-8 or 2^-11 of the adapter's contribution, two of bf16 2^-17 = 8e-6, an order
// above the rest of the sums' error. Two of fp16 behind a power of two for the token, with fp16's B as it is, took 3 to 8 % less for 64 ranks (8 segments of
// 128 tokens 12.2 us, now 13.2) and 10 % less for 128, but fp16 has five bits of exponent: a rank whose sum is 2^-24 of the token's largest kept 14 bits, one
// of 2^-40 nothing, however much B makes of it. Up to 32 ranks with mma.sync, a warp for 32 rows: four for each of its eight row lanes, so that a token's
// 32 values of Y are one 128-byte line and a lane adds 16 bytes of it. More ranks on tcgen05: 128 rows of B as the A operand, 64 or 96 columns of all
// parts of the tokens' H as the B operand, B copied (or widened) into the swizzled tile in an order of rows that gives a thread four neighbouring ones
// from tensor memory.
// Y is added to by vector reductions in L2 and never comes to an SM: loading and storing it instead took 22 us in the place of 13 for 64 segments of 32 tokens.
//
// What bounds it is the length of a CTA's chain at two CTAs of eight warps an SM (three for 16 ranks). One token 4.9 us: launch, segment, operands, the
// cluster's exchange (1,600 of 8,000 cycles) and B. A full batch (64 segments of 32 tokens, adapters of rank 16) 13.3 us cold and 10.0 warm, 9.1 without the
// additions to Y: 256 CTAs work at once (as many more find no tile and leave), 19,000 cycles each, of which 3,400 to find the segment, 4,700 in the first
// product and 6,000 in the second; DRAM is at a quarter of its rate. 4096 tokens of rank 64 27.5 us, 38,000 cycles: 12,500 in the first product, 17,000 in
// the second; issue slots 42 %, shared memory 30 %, tensor cores 11 %. With tf32 pairs on mma.sync 45, with one CTA a tile and every operand from memory 205.
#pragma once

namespace llattn {

constexpr int AD_TOK = 32, AD_THREADS = 256, AD_WARPS = 8, AD_MAX_POOLS = LLATTN_MAX_ADAPTER_POOLS, AD_MAX_RANK = 128;

struct AdapterPoolDesc {
    const void* A;            // [n][rank][K]
    const void* B;            // [n][rows][rank]
    const float* scale;       // [n] or null
    const int32_t* ranks;     // [n] or null
    int n, rank, rows, row0;
};
struct AdapterParams {
    AdapterPoolDesc pool[AD_MAX_POOLS];
    const int8_t* q;
    const float* s;
    float* Y;
    const int32_t* first;     // [nseg + 1]
    const int32_t* adapter;   // [nseg]
    long long ldy;
    int ntokens, K, nseg, parts;
};

struct AdapterF16 {
    // four int8 values -> two pairs of fp16, exact: 1024 + (v + 128) is a half whose low byte is v + 128
    static __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const half2 off = __half2half2(__ushort_as_half(0x6480));        // 1152
        const half2 x = __hsub2(*reinterpret_cast<const half2*>(&a), off), y = __hsub2(*reinterpret_cast<const half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&x); hi = *reinterpret_cast<const uint32_t*>(&y);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static constexpr bool TF32 = true;         // the second product's type,
    static constexpr int PARTS = 2;            // and H's parts in it
};
struct AdapterBF16 {
    // a byte v behind 0x43 is the bf16 number 128 + (v & 127), and with its sign bit alone 128 or 256: their difference is v, exact
    static __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
        const uint32_t p = __byte_perm(w, 0x43434343u, 0x4140), q = __byte_perm(w, 0x43434343u, 0x4342);
        lo = minus(p & 0xff7fff7fu, p & 0xff80ff80u); hi = minus(q & 0xff7fff7fu, q & 0xff80ff80u);
    }
    static __device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
        const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&x);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static constexpr bool TF32 = false;
    static constexpr int PARTS = 3;
    static __device__ __forceinline__ uint32_t part(float& a, float& b) {      // two values rounded, what is left of them in their place
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
        a -= __low2float(x); b -= __high2float(x);
        return *reinterpret_cast<const uint32_t*>(&x);
    }
};
__device__ __forceinline__ float2 half2_floats(uint32_t w) { return __half22float2(*reinterpret_cast<const half2*>(&w)); }
__device__ __forceinline__ float to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return __uint_as_float(r);
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)),
          "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// A block of 64 ranks in bf16 or 32 in tf32: four K-steps over 128-byte-swizzle tiles (A: 128 rows of B, B: the parts of the tokens' H). One elected lane issues.
#define AD_MMA_BLOCK(KIND)                                                                                                                                    \
    asm volatile(                                                                                                                                             \
        "{\n\t.reg .pred pe, pf, pt;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\t"                                                                               \
        "elect.sync _|pe, 0xffffffff;\n\t"                                                                                                                    \
        "setp.ne.b32 pf, %5, 0;\n\t setp.eq.b32 pt, 0, 0;\n\t"                                                                                                \
        "mov.b64 da, {%1, %3};\n\t mov.b64 db, {%2, %3};\n\t"                                                                                                 \
        "@pe tcgen05.mma.cta_group::1.kind::" KIND " [%0], da, db, %4, pf;\n\t"                                                                               \
        "add.u32 x, %1, 2;\n\t add.u32 y, %2, 2;\n\t mov.b64 da, {x, %3};\n\t mov.b64 db, {y, %3};\n\t"                                                       \
        "@pe tcgen05.mma.cta_group::1.kind::" KIND " [%0], da, db, %4, pt;\n\t"                                                                               \
        "add.u32 x, %1, 4;\n\t add.u32 y, %2, 4;\n\t mov.b64 da, {x, %3};\n\t mov.b64 db, {y, %3};\n\t"                                                       \
        "@pe tcgen05.mma.cta_group::1.kind::" KIND " [%0], da, db, %4, pt;\n\t"                                                                               \
        "add.u32 x, %1, 6;\n\t add.u32 y, %2, 6;\n\t mov.b64 da, {x, %3};\n\t mov.b64 db, {y, %3};\n\t"                                                       \
        "@pe tcgen05.mma.cta_group::1.kind::" KIND " [%0], da, db, %4, pt;\n\t"                                                                               \
        "}\n" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate_first) : "memory")
template <bool TF32>
__device__ __forceinline__ void mma_adapter_block_warp(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate_first) {
    if constexpr (TF32) AD_MMA_BLOCK("tf32");
    else AD_MMA_BLOCK("f16");
}
#undef AD_MMA_BLOCK
// Sixteen bytes of which the first `bytes` are copied and the others become zeros.
__device__ __forceinline__ void cp_async16_some(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A CTA of RT sixteens of ranks and 32 tokens: its warps' shares and its shared memory.
template <int RT, bool TF32> struct AdapterTile {
    static constexpr int R = 16 * RT, TOK = AD_TOK;
    // First product: a warp takes RW x 4 tiles of (16 ranks, 8 tokens) and every WK-th run of sixteen values of a group
    static constexpr int RW = RT < 2 ? RT : 2, WR = RT / RW, WK = AD_WARPS / WR;
    // A stage: a group of A and of the codes, rows padded for conflict-free reads, and the tokens' scales
    static constexpr int LDA = 288, LDQ = 144, Q = R * LDA, SX = Q + TOK * LDQ, STAGE = SX + TOK * 4, STAGES = RT > 4 ? 2 : RT > 1 ? 3 : 5;
    // Then, in the same place: the warps' sums by share of the group, [WK][TOK][LDP], and H in parts. For few ranks [TOK] rows LDH bytes apart (bf16: the
    // first two parts side by side, then the third; tf32: one part, then the other); else the tensor cores' tiles, a block of ranks after the other, and behind them
    // tiles of 128 rows of B, the last one where the sums were (of tf32 one tile: half of its blocks there, half behind H). In front of all a
    // slot [TOK][R] for the sums of each other CTA of the cluster.
    static constexpr bool WIDE = RT >= 4;
    static constexpr int LDP = WIDE ? R : R + 4, LDH = 4 * R + (RT == 2 ? 64 : 0), LDH3 = LDH / 2, SLOT = R * TOK * 4, SUMS = WK * TOK * LDP * 4;
    static constexpr int BLOCK = TF32 ? 32 : 64, BLOCKS = (R + BLOCK - 1) / BLOCK, HBLOCK = (TF32 ? 2 : 3) * TOK * 128, WBLOCK = 128 * 128, WTILE = BLOCKS * WBLOCK, WTILES = RT > 4 ? 2 : 3;
    static constexpr int H_AT = WIDE ? (SUMS + 1023) / 1024 * 1024 : SUMS, W_AT = H_AT + BLOCKS * HBLOCK;
    static constexpr int AREA = !WIDE ? H_AT + TOK * (LDH + (TF32 ? LDH : LDH3)) : TF32 ? W_AT + WTILE / 2 : W_AT + (WTILES - 1) * WTILE;
    static_assert(!WIDE || (TF32 ? WTILE / 2 : WTILE) <= H_AT, "the last tile takes the place of the sums");
    static __device__ __forceinline__ int tile_at(int i) { return i % WTILES == WTILES - 1 ? 0 : W_AT + i % WTILES * WTILE; }
    static __device__ __forceinline__ int block_at(int k) { return k < BLOCKS / 2 ? k * WBLOCK : W_AT + (k - BLOCKS / 2) * WBLOCK; }      // of the one tile
    // Where a token's sum of a rank is: the rows of a warp's stores are two apart (padded, or swizzled: its ranks in eights)
    static __device__ __forceinline__ int sum_at(int row, int j) { return row * LDP + (WIDE ? j ^ ((row >> 1 & 3) << 3) : j); }
    static constexpr int HEAD = WIDE ? 1024 : 64;
    static constexpr int bytes(int ctas) { return HEAD + (ctas - 1) * SLOT + (STAGES * STAGE > AREA ? STAGES * STAGE : AREA); }
    static constexpr int MOST = bytes(8) <= 227 * 1024 ? 8 : 4;        // CTAs of a cluster
    static_assert(bytes(MOST) <= 227 * 1024, "shared memory of the largest cluster");
};

// Four neighbouring values added in L2: Y need not come here. Every value of a call is added to once, so no order matters; an fp32 addition rounded to
// nearest (numbers below 2^-126 count as zero).
__device__ __forceinline__ void add_to4(float* y, float a, float b, float c, float d) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(y), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// A run of bytes into L2, both multiples of 16.
__device__ __forceinline__ void l2_prefetch(const void* p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// The shared-memory address `addr` of this CTA in CTA `rank` of its cluster.
__device__ __forceinline__ uint32_t cluster_address(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// 16 bytes into another CTA's shared memory, counted on the barrier `bar` there.
__device__ __forceinline__ void cluster_store4(uint32_t addr, const float4& v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(addr), "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w)), "r"(bar) : "memory");
}
// Behind a wait for that barrier: what the other CTAs have stored is visible (the wait itself acquires for this CTA only).
__device__ __forceinline__ void cluster_acquire(uint32_t bar) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%0], 0;\n\t}\n" ::"r"(bar) : "memory");
}
// (Nothing is handed over by it: the barrier's initialisation has its own fence.)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Where tile `want` is, the tiles of the segments being counted through in order: the segment's adapter, or -1, first token and tokens (0: there is no
// such tile). A bound is cut to the tokens there are, and one below an earlier one counts as that one: a token is in one segment at most, and there
// are no more tiles than the grid has. Every warp for itself, a lane for a run of neighbouring segments: one load behind the launch, and no barrier.
// Every CTA looks at all bounds, so the search grows with their square: segments of one token (rank 16, K and rows 2048) 128 12.8 us, 512 43, 1024 102, 4096
// 775, 10,000 1.7 ms, 65,536 136 ms, where the bytes of the largest take 0.19.
struct AdapterPlace { int adapter, n0, live; };
__device__ __forceinline__ AdapterPlace adapter_place(const AdapterParams& p, int want, int lane) {
    const int per = (p.nseg + 31) / 32, s0 = min(lane * per, p.nseg), s1 = min(s0 + per, p.nseg);
    auto bound = [&](int i) { return min(max(__ldg(p.first + i), 0), p.ntokens); };
    auto tiles = [](int t0, int t1) { return t1 > t0 ? (t1 - t0 + AD_TOK - 1) / AD_TOK : 0; };
    int mine = 0, t0 = bound(s0);
    int a = s0 < s1 ? __ldg(p.adapter + s0) : -1;             // with up to 32 segments all there is to it
    bool back = false;                         // a lane sees its run's bounds and the next run's first one: all neighbours
    for (int i = s0, t = t0; i < s1; ++i) {
        const int t1 = bound(i + 1);
        back |= t1 < t;
        mine += tiles(t, t1);
        t = t1;
    }
    if (__any_sync(0xffffffffu, back)) {       // again, from the largest bound of the runs ahead
        int most = t0;
        for (int i = s0 + 1; i < s1; ++i) most = max(most, bound(i));
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, most, o);
            if (lane >= o) most = max(most, v);
        }
        const int ahead = __shfl_up_sync(0xffffffffu, most, 1);
        if (lane > 0) t0 = max(t0, ahead);
        mine = 0;
        for (int i = s0, t = t0; i < s1; ++i) {
            const int t1 = max(t, bound(i + 1));
            mine += tiles(t, t1);
            t = t1;
        }
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    int k = want - (upto - mine), live = 0;
    const bool found = k >= 0 && k < mine;
    if (found)
        for (int i = s0; i < s1; ++i) {
            const int t1 = max(t0, bound(i + 1)), n = tiles(t0, t1);
            if (k < n) {
                if (i > s0) a = __ldg(p.adapter + i);
                live = min(AD_TOK, t1 - t0 - AD_TOK * k);
                t0 += AD_TOK * k;
                break;
            }
            k -= n;
            t0 = t1;
        }
    const unsigned who = __ballot_sync(0xffffffffu, found);
    const int from = who ? __ffs(who) - 1 : 0;
    AdapterPlace at{__shfl_sync(0xffffffffu, a, from), __shfl_sync(0xffffffffu, t0, from), __shfl_sync(0xffffffffu, live, from)};
    return at;
}

template <typename T, int RT>
__global__ void __launch_bounds__(AD_THREADS, RT == 1 ? 3 : 2) adapters_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ __align__(1024) uint8_t ad_smem[];
    using C = AdapterTile<RT, T::TF32>;
    ptx::grid_dependency_wait();               // nothing is read or written before the kernel ahead has completed
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const AdapterPoolDesc& P = p.pool[blockIdx.y];
    const int parts = p.parts, part = blockIdx.x % parts;          // a cluster is the parts of one tile
    const AdapterPlace place = adapter_place(p, blockIdx.x / parts, lane);
    const int a = place.adapter, n0 = place.n0, live = place.live;
    if (live == 0 || a < 0 || a >= P.n) return;                    // the same for the whole cluster
    if (C::WIDE && ptx::smem_u32(ad_smem) & 1023) {                // the tensor cores' tiles would lie elsewhere than they say
        if (tid == 0) atomicOr(&g_dense_err, ERR_SMEM_ALIGN);
        return;
    }
    // ---- barriers: one counts the sums of the cluster's CTAs in (they may use it once all are here), two the tensor cores' products
    const uint32_t bar = ptx::smem_u32(ad_smem), slots_s = ptx::smem_u32(ad_smem + C::HEAD);
    volatile int* abort_flag = reinterpret_cast<int*>(ad_smem + 24);
    if (tid == 0) {
        *abort_flag = 0;
        ptx::mbar_init(bar, 1);
        ptx::mbar_init(bar + 8, 1);
        ptx::mbar_init(bar + 16, 1);
        ptx::fence_mbar_init();
        if (parts > 1) ptx::mbar_arrive_expect_tx(bar, (parts - 1) * C::SLOT);
    }
    if (parts > 1) cluster_arrive();
    uint8_t* area = ad_smem + C::HEAD + (parts - 1) * C::SLOT;
    const uint32_t area_s = ptx::smem_u32(area);
    const int groups = p.K / DN_GROUP, mygroups = part < groups ? (groups - part + parts - 1) / parts : 0;
    // ---- the groups part, part + parts, ... of the tokens' codes and of A, a few of them ahead
    const uint16_t* A = static_cast<const uint16_t*>(P.A) + size_t(a) * P.rank * p.K;
    const int8_t* qsrc = p.q + size_t(n0 + min(tid >> 3, live - 1)) * p.K + part * DN_GROUP + 16 * (tid & 7);
    const uint16_t* asrc = A + size_t(tid >> 4) * p.K + part * DN_GROUP + 8 * (tid & 15);
    const float* ssrc = p.s + size_t(n0 + min(tid, live - 1)) * groups + part;
    const uint32_t qdst = area_s + C::Q + (tid >> 3) * C::LDQ + 16 * (tid & 7), adst = area_s + (tid >> 4) * C::LDA + 16 * (tid & 15), sdst = area_s + C::SX + 4 * tid;
    uint32_t fst = 0;                          // the stage that is filled next
    auto fetch = [&](int i) {                  // one commit per call, so groups count uniformly
        if (i < mygroups) {
            cp_async16(qdst + fst, qsrc, (tid >> 3) < live);
            qsrc += parts * DN_GROUP;
#pragma unroll
            for (int m = 0; m < RT; ++m) {     // behind the pool's ranks: zeros
                const bool there = 16 * m + (tid >> 4) < P.rank;
                cp_async16(adst + fst + 16 * m * C::LDA, there ? asrc + size_t(16 * m) * p.K : A, there);
            }
            asrc += parts * DN_GROUP;
            if (tid < AD_TOK) cp_async4(sdst + fst, ssrc, tid < live);
            ssrc += parts;
            fst = fst + C::STAGE == C::STAGES * C::STAGE ? 0 : fst + C::STAGE;
        }
        cp_async_commit();
    };
    for (int i = 0; i < C::STAGES - 1; ++i) fetch(i);
    if constexpr (C::WIDE)
        if (warp == 0) { ptx::tmem_alloc(ptx::smem_u32(ad_smem + 28), 256); ptx::tmem_relinquish(); }
    const int rank_there = P.ranks ? __ldg(P.ranks + a) : P.rank;  // looked at when the sums are there: a wait for it here would hold up what follows
    const float scale = P.scale ? __ldg(P.scale + a) : 1.f;
    // ---- this CTA's rows of B are wanted when H is done: into L2, and a small rank's first ones into registers
    constexpr int ROWS = C::WIDE ? 128 : 32;   // of a step of the second product
    const int steps = (P.rows + ROWS - 1) / ROWS, per = (steps + parts - 1) / parts, first = part * per, end = min(steps, first + per);
    const uint16_t* B = static_cast<const uint16_t*>(P.B) + size_t(a) * P.rows * P.rank;
    constexpr bool EARLY = RT == 1;
    uint2 braw[4];
    auto load_b = [&](uint2 (&to)[4], int c, int rt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 32 * c + 4 * g + i, j = 16 * rt + 4 * t;
            to[i] = make_uint2(0u, 0u);
            if (row < P.rows && j < P.rank) to[i] = __ldg(reinterpret_cast<const uint2*>(B + size_t(row) * P.rank + j));
        }
    };
    const int c0 = first + warp;
    if constexpr (EARLY)
        if (c0 < end) load_b(braw, c0, 0);
    {
        const int from = ROWS * first, to = min(ROWS * end, P.rows);
        if (tid == 0 && to > from) l2_prefetch(B + size_t(from) * P.rank, (to - from) * P.rank * 2);
    }
    // ---- sums of H over these groups
    const int wr = warp % C::WR, wk = warp / C::WR;
    float h[C::RW][4][4] = {};
#pragma unroll 1
    for (int i = 0; i < mygroups; ++i) {
        cp_async_wait<C::STAGES - 2>();
        __syncthreads();                       // group i is in for everybody; group i - 1 is done with, its stage can be refilled
        fetch(i + C::STAGES - 1);
        const uint8_t* st = area + (i % C::STAGES) * C::STAGE;
        constexpr int KN = 8 / C::WK;          // runs of sixteen: KN wk .. KN wk + KN - 1
        float c[C::RW][4][4] = {};
        uint32_t w[4][KN];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            const uint8_t* src = st + C::Q + (8 * nt + g) * C::LDQ + 32 * t + 4 * KN * wk;
            if constexpr (KN == 1) w[nt][0] = *reinterpret_cast<const uint32_t*>(src);
            else if constexpr (KN == 2) *reinterpret_cast<uint2*>(w[nt]) = *reinterpret_cast<const uint2*>(src);
            else
#pragma unroll
                for (int k = 0; k < KN; k += 4) *reinterpret_cast<uint4*>(&w[nt][k]) = *reinterpret_cast<const uint4*>(src + 4 * k);
        }
#pragma unroll
        for (int k = 0; k < KN; ++k) {
            uint2 x[C::RW], z[C::RW];
#pragma unroll
            for (int r = 0; r < C::RW; ++r) {
                const uint8_t* src = st + (16 * (C::RW * wr + r) + g) * C::LDA + 32 * (KN * wk + k) + 8 * t;
                x[r] = *reinterpret_cast<const uint2*>(src);
                z[r] = *reinterpret_cast<const uint2*>(src + 8 * C::LDA);
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                uint32_t b0, b1;
                T::widen(w[nt][k], b0, b1);
#pragma unroll
                for (int r = 0; r < C::RW; ++r) T::mma(c[r][nt], x[r].x, z[r].x, x[r].y, z[r].y, b0, b1);
            }
        }
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            const float2 sx = *reinterpret_cast<const float2*>(st + C::SX + 4 * (8 * nt + 2 * t));
#pragma unroll
            for (int r = 0; r < C::RW; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) h[r][nt][e] = fmaf(e & 1 ? sx.y : sx.x, c[r][nt][e], h[r][nt][e]);
        }
    }
    cp_async_wait<0>();
    __syncthreads();                           // the stages are done with
    const int rank = min(max(rank_there, 0), P.rank);
    // 128 rows of B as the tensor cores read them: row 4 g + i of 32 is the tile's g + 8 i, a thread then gets four neighbouring rows from tensor memory.
    // Behind the rank, whatever B has there, and behind P's rows: zeros.
    auto fetch_b = [&](int c) {
        if (c < end)
#pragma unroll
            for (int m = 0; m < 128 * C::R / 8; m += AD_THREADS) {
                const int r = (m + tid) / (C::R / 8), j = (m + tid) % (C::R / 8) * 8, row = 128 * c + r, at = r / 32 * 32 + r / 4 % 8 + r % 4 * 8;
                const int bytes = row < P.rows ? min(max(rank - j, 0), 8) * 2 : 0;
                cp_async16_some(area_s + C::tile_at(c - first) + j / 64 * C::WBLOCK + at * 128 + ((j % 64 / 8 ^ (at & 7)) << 4),
                                bytes ? B + size_t(row) * P.rank + j : B, bytes);
            }
        cp_async_commit();
    };
    // The same of fp16, through registers: a thread's eight ranks of every 2048 / R-th row asked for, and put into the tile as fp32 numbers.
    constexpr int ASKED = C::WIDE && T::TF32 ? C::R / 16 : 1;
    uint4 raw[ASKED];
    auto ask_b = [&](int c) {
        const int j = tid % (C::R / 8) * 8;
#pragma unroll
        for (int m = 0; m < ASKED; ++m) {
            const int row = 128 * c + m * (AD_THREADS * 8 / C::R) + tid / (C::R / 8);
            raw[m] = c < end && row < P.rows && j < rank ? __ldg(reinterpret_cast<const uint4*>(B + size_t(row) * P.rank + j)) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto put_b = [&]() {
        // (every other block's lanes begin with their second four ranks: eight neighbouring lanes then store to all banks)
        const int j = tid % (C::R / 8) * 8, left = rank - j, swap = j / 32 & 1;
        uint32_t mask[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mask[k] = 2 * k + 1 < left ? 0xffffffffu : 2 * k < left ? 0xffffu : 0u;
#pragma unroll
        for (int m = 0; m < ASKED; ++m) {
            const int r = m * (AD_THREADS * 8 / C::R) + tid / (C::R / 8), at = r / 32 * 32 + r / 4 % 8 + r % 4 * 8;
            const uint32_t w[4] = {raw[m].x & mask[0], raw[m].y & mask[1], raw[m].z & mask[2], raw[m].w & mask[3]};
            uint8_t* to = area + C::block_at(j / 32) + at * 128;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 a = half2_floats(swap ? w[2 - 2 * k] : w[2 * k]), b = half2_floats(swap ? w[3 - 2 * k] : w[2 * k + 1]);
                *reinterpret_cast<float4*>(to + ((j % 32 / 4 + (k ^ swap) ^ (at & 7)) << 4)) = make_float4(a.x, a.y, b.x, b.y);
            }
        }
        ptx::fence_proxy_async_smem();
    };
    if constexpr (C::WIDE) {
        if constexpr (T::TF32) ask_b(first);
        else
            for (int c = first; c < first + C::WTILES - 1; ++c) fetch_b(c);
    }
    float* sums = reinterpret_cast<float*>(area);
#pragma unroll
    for (int r = 0; r < C::RW; ++r)
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sums[C::sum_at(wk * AD_TOK + 8 * nt + 2 * t + (e & 1), 16 * (C::RW * wr + r) + g + 8 * (e >> 1))] = h[r][nt][e];
    __syncthreads();
    // ---- four ranks of a token at a time: this CTA's sums, to a slot in every other CTA of the cluster, and all CTAs' in their order
    constexpr int QUADS = (C::R * AD_TOK / 4 + AD_THREADS - 1) / AD_THREADS;
    float4 own[QUADS];
    bool ok = true;
    if (parts > 1) cluster_wait();
#pragma unroll
    for (int m = 0; m < QUADS; ++m) {
        const int i = tid + m * AD_THREADS, n = 4 * i / C::R, j = 4 * i % C::R;
        own[m] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n < AD_TOK) {
#pragma unroll
            for (int k = 0; k < C::WK; ++k) {
                const float4 u = *reinterpret_cast<const float4*>(sums + C::sum_at(k * AD_TOK + n, j));
                own[m].x += u.x; own[m].y += u.y; own[m].z += u.z; own[m].w += u.w;
            }
            for (int k = 0; k < parts; ++k)
                if (k != part) cluster_store4(cluster_address(slots_s + (part - (part > k)) * C::SLOT + 16 * i, k), own[m], cluster_address(bar, k));
        }
    }
    if (parts > 1) {
        ok = ptx::mbar_wait(bar, 0, abort_flag);
        cluster_acquire(bar);
    }
    uint8_t* hs = area + C::H_AT;
    {
        const float4* slots = reinterpret_cast<const float4*>(ad_smem + C::HEAD);
#pragma unroll
        for (int m = 0; m < QUADS; ++m) {
            const int i = tid + m * AD_THREADS, n = 4 * i / C::R, j = 4 * i % C::R;
            if (n >= AD_TOK) break;
            float v[4] = {};
#pragma unroll 4
            for (int k = 0; k < parts; ++k) {
                const float4 u = k == part ? own[m] : slots[(k - (k > part)) * (C::SLOT / 16) + i];
                v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
            }
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = j + e < rank ? v[e] * scale : 0.f;      // what A has behind the rank, whatever it is, does not count
            if constexpr (T::TF32) {
                float4 w[2];
                w[0] = make_float4(to_tf32(x[0]), to_tf32(x[1]), to_tf32(x[2]), to_tf32(x[3]));
                w[1] = make_float4(to_tf32(x[0] - w[0].x), to_tf32(x[1] - w[0].y), to_tf32(x[2] - w[0].z), to_tf32(x[3] - w[0].w));
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (C::WIDE) *reinterpret_cast<float4*>(hs + j / 32 * C::HBLOCK + (AD_TOK * k + n) * 128 + ((j % 32 / 4 ^ (n & 7)) << 4)) = w[k];
                    else *reinterpret_cast<float4*>(hs + (AD_TOK * k + n) * C::LDH + 4 * j) = w[k];
                }
            } else {
                uint32_t w[3][2];
#pragma unroll
                for (int k = 0; k < 3; ++k) { w[k][0] = T::part(x[0], x[1]); w[k][1] = T::part(x[2], x[3]); }
                if constexpr (C::WIDE) {
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        *reinterpret_cast<uint2*>(hs + j / 64 * C::HBLOCK + (AD_TOK * k + n) * 128 + ((j % 64 / 8 ^ (n & 7)) << 4) + j % 8 * 2) = make_uint2(w[k][0], w[k][1]);
                } else {
                    *reinterpret_cast<uint4*>(hs + n * C::LDH + 4 * j) = make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
                    *reinterpret_cast<uint2*>(hs + AD_TOK * C::LDH + n * C::LDH3 + 2 * j) = make_uint2(w[2][0], w[2][1]);
                }
            }
        }
    }
    if constexpr (C::WIDE) ptx::fence_proxy_async_smem();
    ok = __syncthreads_and(ok);                // H is there
    // Where sums are missing this CTA leaves Y as it is, says so, and stays until the others' stores into its shared memory are in: whatever its rank and rows.
    if (!ok) {
        cp_async_wait<0>();
        if (tid == 0) {
            atomicOr(&g_dense_err, ERR_WAIT_FOLD);
            *abort_flag = 0;
            ptx::mbar_wait(bar, 0, abort_flag);
        }
        __syncthreads();
        if constexpr (C::WIDE)
            if (warp == 0) ptx::tmem_dealloc(*reinterpret_cast<volatile uint32_t*>(ad_smem + 28), 256);
        return;
    }
    if constexpr (C::WIDE) {
        // ---- Y, 128 rows at a time on tcgen05: a tile of B times all parts of H beside one another into tensor memory
        ptx::tc_fence_after();
        const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(ad_smem + 28);
        const uint32_t dhi = ptx::desc_hi(1024) | (2u << 29), idesc = ptx::idesc_f16(128, T::PARTS * AD_TOK, false, false) | (T::TF32 ? 2u << 7 | 2u << 10 : 1u << 7 | 1u << 10);      // tf32 or bf16
        constexpr int COLS = AD_TOK / 2;       // of a warp: a quarter of the rows, half of the tokens
        const int nw = COLS * (warp >> 2);
        int issued = 0;
        auto multiply = [&](int c) {           // by warp 0
            const uint32_t acc = tmem + ((c - first) & 1) * 128;
#pragma unroll
            for (int k = 0; k < C::BLOCKS; ++k) {
                const uint32_t tile = area_s + (T::TF32 ? C::block_at(k) : C::tile_at(c - first) + k * C::WBLOCK);
                mma_adapter_block_warp<T::TF32>(acc, ptx::desc_lo(tile, 16), ptx::desc_lo(ptx::smem_u32(hs) + k * C::HBLOCK, 16), dhi, idesc, k > 0);
            }
            ptx::mma_commit_warp(bar + 8 + 8 * ((c - first) & 1));
        };
        // (the sums have been passed on)
        if constexpr (T::TF32) {
            put_b();
            ask_b(first + 1);
        } else {
            fetch_b(first + C::WTILES - 1);
            cp_async_wait<C::WTILES - 1>();
            ptx::fence_proxy_async_smem();
        }
        __syncthreads();
        if (rank != 0 && first < end) {
            if (warp == 0) multiply(first);
            issued = 1;
        }
        // the products of the next rows run while these rows' are on their way to Y: two accumulators (8 segments of 128 tokens of rank 64 13.0 -> 12.2 us)
#pragma unroll 1
        for (int c = first; c < end && issued; ++c) {
            if constexpr (T::TF32) {
                ok = ptx::mbar_wait_warp(bar + 8 + 8 * ((c - first) & 1), ((c - first) >> 1) & 1, abort_flag);
                if (ok && c + 1 < end) put_b();              // the tile has been read
            } else if (c + 1 < end) {
                cp_async_wait<C::WTILES - 2>();
                ptx::fence_proxy_async_smem();
            }
            ptx::tc_fence_before();
            ok = __syncthreads_and(ok);        // B is there, the former rows have been read from tensor memory
            if (!ok) break;
            ptx::tc_fence_after();
            if (c + 1 < end) {
                if (warp == 0) multiply(c + 1);
                ++issued;
            }
            if constexpr (T::TF32) ask_b(c + 2);
            else {
                ok = ptx::mbar_wait_warp(bar + 8 + 8 * ((c - first) & 1), ((c - first) >> 1) & 1, abort_flag);
                ptx::tc_fence_after();
                fetch_b(c + C::WTILES);        // in the place of the tile just used
            }
            // rows 4 g and + 1 in the first, + 2 and + 3 in the second; tokens 8 i + 2 t and + 1; a part 32 columns behind the other
            uint32_t ra[T::PARTS][COLS / 2], rb[T::PARTS][COLS / 2];
            const int row = 128 * c + 32 * (warp & 3) + 4 * g;
            const uint32_t from = tmem + ((c - first) & 1) * 128 + (uint32_t(32 * (warp & 3)) << 16) + nw;
#pragma unroll
            for (int k = 0; k < T::PARTS; ++k) {
                ptx::tmem_ld16x256_cols(from + k * AD_TOK, ra[k]);
                ptx::tmem_ld16x256_cols(from + k * AD_TOK + (16u << 16), rb[k]);
            }
#pragma unroll
            for (int k = 0; k < T::PARTS; ++k) {
                ptx::tmem_wait_ld_tied(ra[k]);
                ptx::tmem_wait_ld_tied(rb[k]);
            }
            ptx::tc_fence_before();
            auto sum = [&](uint32_t (&r)[T::PARTS][COLS / 2], int i) {
                float v = __uint_as_float(r[T::PARTS - 1][i]);
#pragma unroll
                for (int k = T::PARTS - 2; k >= 0; --k) v += __uint_as_float(r[k][i]);
                return v;
            };
            float* yrow = p.Y + (n0 + nw) * p.ldy + P.row0 + row;
            if (ok && row < P.rows)
#pragma unroll
                for (int i = 0; i < COLS / 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int n = 8 * i + 2 * t + e;
                        if (nw + n < live) add_to4(yrow + n * p.ldy, sum(ra, 4 * i + e), sum(ra, 4 * i + 2 + e), sum(rb, 4 * i + e), sum(rb, 4 * i + 2 + e));
                    }
        }
        cp_async_wait<0>();
        ok = __syncthreads_and(ok);
        if (tid == 0 && !ok) {                 // products that are still on their way
            atomicOr(&g_dense_err, ERR_WAIT_FOLD);
            for (int k = max(0, issued - 2); k < issued; ++k) {
                *abort_flag = 0;
                ptx::mbar_wait(bar + 8 + 8 * (k & 1), (k >> 1) & 1, abort_flag);
            }
        }
        __syncthreads();
        if (warp == 0) ptx::tmem_dealloc(tmem, 256);
    } else {
        if (rank == 0) return;
        // ---- Y, a warp for 32 rows and 32 tokens
#pragma unroll 1
        for (int c = c0; c < end; c += AD_WARPS) {
            const int row = 32 * c + 4 * g;
            const bool mine = row < P.rows;
            if (!EARLY && c == c0) load_b(braw, c, 0);         // of the ranks that follow, and of the next rows, they are loaded one step ahead
            float acc[2][4][4] = {};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (16 * rt >= rank) break;
                const int j = 16 * rt + 4 * t;
                // B as it is: a lane's four ranks are its K slots, as in the first product. What B has behind the rank, whatever it is, does not count.
                const uint32_t m0 = j + 1 < rank ? 0xffffffffu : j < rank ? 0xffffu : 0u, m1 = j + 3 < rank ? 0xffffffffu : j + 2 < rank ? 0xffffu : 0u;
                uint32_t w[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) { w[i][0] = braw[i].x & m0; w[i][1] = braw[i].y & m1; }
                const bool last = 16 * rt + 16 >= rank;
                if (!last || c + AD_WARPS < end) load_b(braw, last ? c + AD_WARPS : c, last ? 0 : rt + 1);
                // the smallest part first; no product right behind another one into the same accumulator
                if constexpr (T::TF32) {
                    float2 f[4][2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) { f[i][0] = half2_floats(w[i][0]); f[i][1] = half2_floats(w[i][1]); }
#pragma unroll
                    for (int k = 1; k >= 0; --k) {
                        float4 x[4];
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt) x[nt] = *reinterpret_cast<const float4*>(hs + (AD_TOK * k + 8 * nt + g) * C::LDH + 4 * j);
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
                                    mma_tf32(acc[i][nt], f[2 * i][half].x, f[2 * i + 1][half].x, f[2 * i][half].y, f[2 * i + 1][half].y, half ? x[nt].z : x[nt].x, half ? x[nt].w : x[nt].y);
                    }
                } else {
                    uint4 x[4];
                    uint2 z[4];
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt) {
                        x[nt] = *reinterpret_cast<const uint4*>(hs + (8 * nt + g) * C::LDH + 4 * j);
                        z[nt] = *reinterpret_cast<const uint2*>(hs + AD_TOK * C::LDH + (8 * nt + g) * C::LDH3 + 2 * j);
                    }
#pragma unroll
                    for (int k = 2; k >= 0; --k)
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                T::mma(acc[i][nt], w[2 * i][0], w[2 * i + 1][0], w[2 * i][1], w[2 * i + 1][1], k == 2 ? z[nt].x : k ? x[nt].z : x[nt].x,
                                       k == 2 ? z[nt].y : k ? x[nt].w : x[nt].y);
                }
            }
            if (!mine) continue;
            float* yrow = p.Y + n0 * p.ldy + P.row0 + row;
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int n = 8 * nt + 2 * t + e;
                    if (n >= live) continue;
                    add_to4(yrow + n * p.ldy, acc[0][nt][e], acc[0][nt][2 + e], acc[1][nt][e], acc[1][nt][2 + e]);
                }
        }
    }
}

}  // namespace llattn

namespace {
// CTAs of a cluster, by the sizes alone (the segments are on the device): as many as are on the chip at once, two an SM where their shared memory lets
// them. How many clusters of 2, 4 and 8 there are with one CTA an SM is asked of the runtime (74, 33 and 15: groups of SMs are not multiples of eight).
// In a graph, with 2 / 4 / 8 CTAs: rank 16, 1 token 8.7 / 6.0 / 4.9 us, 32 tiles 11.0 / 8.7 / 8.9, 64 (segments of 32 tokens) 13.2 / 13.0 / 18.2, 128 20.5 / 26.4 /
// -; rank 64, 8 tiles 18.3 / 11.7 / 9.1, 18 11.5 / 8.5 / 14.6, 32 19.2 / 12.2 / 29.6, 128 28.5 / 32.9 / 86.
template <typename T, int RT>
int launch_adapters(llattn::AdapterParams& p, int npools, cudaStream_t stream) {
    using namespace llattn;
    using C = AdapterTile<RT, T::TF32>;
    constexpr int ONE_AN_SM = 200 * 1024, TWO_AN_SM = 113 * 1024;
    static std::mutex mu;
    static int clusters[64][3];                // by device; the first one 0: not asked yet
    auto* kernel = adapters_kernel<T, RT>;
    int dev = 0, fit[3];
    CU(cudaGetDevice(&dev));
    if (dev >= 64) return fail(LLATTN_EINVAL, "adapters_w4a8: device index %d not supported", dev);
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!clusters[dev][0]) {
            CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(C::bytes(C::MOST), ONE_AN_SM)));
            for (int i = 2; i >= 0; --i) {
                cudaLaunchConfig_t cfg{};
                cudaLaunchAttribute attr{};
                attr.id = cudaLaunchAttributeClusterDimension;
                attr.val.clusterDim.x = 2 << i; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
                cfg.gridDim = dim3(2 << i); cfg.blockDim = dim3(AD_THREADS); cfg.dynamicSmemBytes = ONE_AN_SM;
                cfg.attrs = &attr; cfg.numAttrs = 1;
                int n = 0;
                CU(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
                clusters[dev][i] = i ? n : std::max(n, 1);
            }
        }
        for (int i = 0; i < 3; ++i) fit[i] = 2 << i > C::MOST ? 0 : clusters[dev][i] * (C::bytes(2 << i) <= TWO_AN_SM ? 2 : 1);
    }
    const long long work = std::max<long long>(std::min(p.nseg, p.ntokens), (p.ntokens + AD_TOK - 1) / AD_TOK) * npools;       // tiles, in the mean
    p.parts = 1;
    for (int i = 0; i < 3; ++i)
        if (work <= fit[i]) p.parts = 2 << i;
    // no more tiles than this, however the segments cut the tokens: each has at most one that is not full
    const long long tiles = std::min<long long>(p.ntokens, (p.ntokens + (AD_TOK - 1ll) * p.nseg) / AD_TOK);
    CU(launch_dependent_cluster(kernel, dim3(unsigned(tiles * p.parts), npools), AD_THREADS, C::bytes(p.parts), p.parts, stream, p));
    return LLATTN_OK;
}
template <typename T>
int launch_adapters_rank(llattn::AdapterParams& p, int npools, int rank, cudaStream_t stream) {
    if (rank <= 16) return launch_adapters<T, 1>(p, npools, stream);
    if (rank <= 32) return launch_adapters<T, 2>(p, npools, stream);
    if (rank <= 64) return launch_adapters<T, 4>(p, npools, stream);
    return launch_adapters<T, 8>(p, npools, stream);
}
}  // namespace

extern "C" int llattn_adapters_w4a8(const llattn_adapter_pool* pools, int npools, const int8_t* q, const float* s, float* Y, int64_t ldy, int ntokens, int K,
                                    const int32_t* seg_first, const int32_t* seg_adapter, int nseg, void* stream) {
    using namespace llattn;
    if (!pools || !q || !s || !Y || !seg_first || !seg_adapter) return fail(LLATTN_EINVAL, "adapters_w4a8: null pointer");
    if (npools < 1 || npools > AD_MAX_POOLS) return fail(LLATTN_EINVAL, "adapters_w4a8: %d pools; 1 to %d", npools, AD_MAX_POOLS);
    if (ntokens < 0 || ntokens > 1 << 22) return fail(LLATTN_EINVAL, "adapters_w4a8: ntokens = %d", ntokens);
    if (K <= 0 || K % DN_GROUP || K > 1 << 20) return fail(LLATTN_EINVAL, "adapters_w4a8: K = %d (a multiple of 128)", K);
    if (nseg < 0 || nseg > 1 << 16) return fail(LLATTN_EINVAL, "adapters_w4a8: nseg = %d", nseg);
    if (ldy <= 0 || ldy % 4 || ldy > int64_t(1) << 32) return fail(LLATTN_EINVAL, "adapters_w4a8: ldy = %lld (a multiple of 4)", (long long)ldy);
    if (!aligned16(q) || !aligned16(Y)) return fail(LLATTN_EINVAL, "adapters_w4a8: q and Y must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(s) | reinterpret_cast<uintptr_t>(seg_first) | reinterpret_cast<uintptr_t>(seg_adapter)) % 4)
        return fail(LLATTN_EINVAL, "adapters_w4a8: s, seg_first and seg_adapter must be 4-byte aligned");
    AdapterParams p{};
    int rank = 0;
    const unsigned long long groups = K / DN_GROUP, T = ntokens, ybytes = T ? ((T - 1) * ldy + 1) * 4 : 0;
    for (int i = 0; i < npools; ++i) {
        const llattn_adapter_pool& a = pools[i];
        if (!a.A || !a.B) return fail(LLATTN_EINVAL, "adapters_w4a8: pool %d: null pointer", i);
        if (a.type != LLATTN_F16 && a.type != LLATTN_BF16) return fail(LLATTN_EINVAL, "adapters_w4a8: pool %d: type = %d", i, a.type);
        if (a.type != pools[0].type) return fail(LLATTN_EINVAL, "adapters_w4a8: the pools of a call have one type");
        if (a.n < 1 || a.n > 1 << 20 || a.rank < 8 || a.rank % 8 || a.rank > AD_MAX_RANK)
            return fail(LLATTN_EINVAL, "adapters_w4a8: pool %d: %d adapters of rank %d (a multiple of 8 up to %d)", i, a.n, a.rank, AD_MAX_RANK);
        if (a.rows < 4 || a.rows % 4 || a.rows > 1 << 20 || a.row0 < 0 || a.row0 % 4 || a.row0 > 1 << 24 || a.row0 + a.rows > ldy)
            return fail(LLATTN_EINVAL, "adapters_w4a8: pool %d: rows [%d, %d + %d) of %lld (multiples of 4)", i, a.row0, a.row0, a.rows, (long long)ldy);
        if (!aligned16(a.A) || !aligned16(a.B) || (reinterpret_cast<uintptr_t>(a.scale) | reinterpret_cast<uintptr_t>(a.ranks)) % 4)
            return fail(LLATTN_EINVAL, "adapters_w4a8: pool %d: A and B must be 16-byte aligned, scale and ranks 4-byte", i);
        for (int k = 0; k < i; ++k)
            if (a.row0 < pools[k].row0 + pools[k].rows && pools[k].row0 < a.row0 + a.rows) return fail(LLATTN_EINVAL, "adapters_w4a8: pools %d and %d share rows", k, i);
        const unsigned long long n = a.n;
        const float* y0 = Y + a.row0;
        const unsigned long long yb = ybytes ? ybytes + (a.rows - 1) * 4ull : 0;
        if (overlap(y0, yb, a.A, n * a.rank * K * 2) || overlap(y0, yb, a.B, n * a.rank * a.rows * 2) || overlap(y0, yb, a.scale, n * 4) || overlap(y0, yb, a.ranks, n * 4) ||
            overlap(y0, yb, q, T * K) || overlap(y0, yb, s, T * groups * 4) || overlap(y0, yb, seg_first, 4ull * nseg + 4) || overlap(y0, yb, seg_adapter, 4ull * nseg))
            return fail(LLATTN_EINVAL, "adapters_w4a8: Y overlaps an input");
        p.pool[i] = AdapterPoolDesc{a.A, a.B, a.scale, a.ranks, a.n, a.rank, a.rows, a.row0};
        rank = std::max(rank, a.rank);
    }
    if (ntokens == 0 || nseg == 0) return LLATTN_OK;
    p.q = q; p.s = s; p.Y = Y; p.first = seg_first; p.adapter = seg_adapter;
    p.ldy = ldy; p.ntokens = ntokens; p.K = K; p.nseg = nseg;
    return pools[0].type == LLATTN_F16 ? launch_adapters_rank<AdapterF16>(p, npools, rank, as_stream(stream))
                                       : launch_adapters_rank<AdapterBF16>(p, npools, rank, as_stream(stream));
}

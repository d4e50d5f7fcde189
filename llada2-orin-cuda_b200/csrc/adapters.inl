// Low-rank adapters of many requests beside a shared projection (llattn_adapters_w4a8).
//
// Tokens come in segments, each with an adapter of a pool or none:
//   H[n][j] = c_a * sum_g s[n][g] * (sum_{k in group g} q[n][k] * A_a[j][k])       j < rank of adapter a
//   Y[n][row0 + i] += sum_j H[n][j] * B_a[i][j]
// from the int8 activations that the projection itself reads (codes in fragment order, one scale for each group of 128).
//
// A CTA takes up to 32 tokens of one segment and a part of the rows. First product: the codes are exact in 16 bits, so mma.sync multiplies them
// with A as it is, and each group's sum takes its scale in fp32: nothing is rounded but the fp32 sums. A lane's word of the fragment order is
// four neighbouring values of a run of sixteen; the four K slots of a lane in an m16n8k16 are given to just these, and A is read to match, eight
// bytes a lane. Second product: H is two tf32 numbers, value and remainder (22 bits; one alone would leave 2^-11 of the adapter's
// part, and bf16 pairs 2^-17), B is exact in tf32. A warp takes 32 rows, four for each of its eight row lanes, so that a token's 32 values of
// Y are one 128-byte line and every access to Y is 16 bytes a lane.
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
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const half2*>(&w)); }
};
struct AdapterBF16 {
    // through fp32 (2^23 + v + 128, exact), whose upper halves are the bf16 numbers: eight bits are enough for them
    static __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
        const uint32_t u = w ^ 0x80808080u;
        uint32_t f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __float_as_uint(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + e)) - 8388736.f);
        lo = __byte_perm(f[0], f[1], 0x7632); hi = __byte_perm(f[2], f[3], 0x7632);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}

// Shared memory of a CTA: where its tokens are, H as value and remainder, and the partial sums of H: a slot for each half of the groups of each CTA
// of the cluster.
template <int RT> struct AdapterSmem {
    static constexpr int R = 16 * RT, LDH = R + 2;          // a row of (value, remainder) pairs is 16 bytes longer than its values: conflict-free reads
    static constexpr int LDP = AD_TOK + 8;                  // and eight rows of a slot are eight banks apart
    int scan[AD_WARPS], tile[4];
    __align__(16) float2 h[AD_TOK][LDH];
    float part[2][R][LDP];                                  // 2 x the cluster's CTAs of them
    static constexpr int bytes(int ctas) { return int(sizeof(AdapterSmem)) + 2 * (ctas - 1) * R * LDP * 4; }
};

// The shared-memory address `addr` of this CTA in CTA `rank` of its cluster.
__device__ __forceinline__ uint32_t cluster_address(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_store2(uint32_t addr, float a, float b) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The segment and tokens of tile `want`, the tiles of the segments being counted through in order: {adapter or -1, first token, tokens}. Bounds that
// are out of range or not in order give no tokens. Every thread calls.
__device__ __forceinline__ void adapter_tile(const AdapterParams& p, int want, int (&scan)[AD_WARPS], int (&tile)[4]) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) { tile[0] = -1; tile[2] = 0; }
    int before = 0;
    for (int base = 0; base < p.nseg; base += AD_THREADS) {
        const int i = base + tid;
        int t0 = 0, t1 = 0, a = -1;
        if (i < p.nseg) {
            t0 = min(max(__ldg(p.first + i), 0), p.ntokens);
            t1 = min(max(__ldg(p.first + i + 1), 0), p.ntokens);
            a = __ldg(p.adapter + i);
        }
        const int tiles = t1 > t0 ? (t1 - t0 + AD_TOK - 1) / AD_TOK : 0;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        __syncthreads();                       // the former round's sums are read, and tile is set
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int k = 0; k < AD_WARPS; ++k) {
            if (k < warp) upto += scan[k];
            total += scan[k];
        }
        const int k = want - before - (upto - tiles);        // the segment's tile, if it is one of its own
        if (k >= 0 && k < tiles) {
            tile[0] = a;
            tile[1] = t0 + AD_TOK * k;
            tile[2] = min(AD_TOK, t1 - t0 - AD_TOK * k);
        }
        before += total;
        if (before > want) break;
    }
    __syncthreads();
}

template <typename T, int RT>
__global__ void __launch_bounds__(AD_THREADS, RT <= 4 ? 2 : 1) adapters_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ __align__(16) uint8_t ad_smem[];
    using S = AdapterSmem<RT>;
    S& sm = *reinterpret_cast<S*>(ad_smem);
    ptx::grid_dependency_wait();               // nothing is read or written before the kernel ahead has completed
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const AdapterPoolDesc& P = p.pool[blockIdx.y];
    const int parts = p.parts, part = blockIdx.x % parts;          // a cluster is the parts of one tile
    if (parts > 1) cluster_arrive();           // the others may write here once this CTA is there
    adapter_tile(p, blockIdx.x / parts, sm.scan, sm.tile);
    const int a = sm.tile[0], n0 = sm.tile[1], live = sm.tile[2];
    const int rank = live == 0 || a < 0 || a >= P.n ? 0 : P.ranks ? min(max(__ldg(P.ranks + a), 0), P.rank) : P.rank;
    if (rank == 0) {                           // the same for the whole cluster
        if (parts > 1) cluster_wait();
        return;
    }
    const float scale = P.scale ? __ldg(P.scale + a) : 1.f;
    const int groups = p.K / DN_GROUP;
    const int chunks = (P.rows + 31) / 32, per = (chunks + parts - 1) / parts, end = min(chunks, (part + 1) * per);
    // ---- this warp's first 32 rows of Y are on their way from the start
    float4 y[4][2];
    auto load_y = [&](int c) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int n = 8 * nt + 2 * t + e, row = 32 * c + 4 * g;
                if (n < live && row < P.rows) y[nt][e] = *reinterpret_cast<const float4*>(p.Y + (long long)(n0 + n) * p.ldy + P.row0 + row);
            }
    };
    const int c0 = part * per + warp;
    if (c0 < end) load_y(c0);
    // ---- H over this CTA's groups (part, part + parts, ...), a warp for eight tokens and every second of them
    {
        const int nt = warp & 3, half_ = warp >> 2, n = 8 * nt + g;
        const uint16_t* A = static_cast<const uint16_t*>(P.A) + size_t(a) * P.rank * p.K + 4 * t;
        float h[RT][4] = {};
#pragma unroll 1
        for (int gi = part + half_ * parts; gi < groups && 8 * nt < live; gi += 2 * parts) {
            uint4 w[2] = {};
            if (n < live) {
                const uint4* src = reinterpret_cast<const uint4*>(p.q + size_t(n0 + n) * p.K + size_t(gi) * DN_GROUP + 32 * t);
                w[0] = __ldg(src); w[1] = __ldg(src + 1);
            }
            float sx[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) sx[e] = __ldg(p.s + size_t(n0 + min(8 * nt + 2 * t + e, live - 1)) * groups + gi);
            const uint32_t words[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (16 * rt >= rank) break;
                float c[4] = {};
                const bool lo = 16 * rt + g < rank, hi = 16 * rt + g + 8 < rank;      // rows behind the rank are not read
                const uint16_t* r0 = A + size_t(16 * rt + g) * p.K + size_t(gi) * DN_GROUP;
                uint2 x[8], z[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] = z[k] = make_uint2(0u, 0u);
                    if (lo) x[k] = __ldg(reinterpret_cast<const uint2*>(r0 + 16 * k));
                    if (hi) z[k] = __ldg(reinterpret_cast<const uint2*>(r0 + size_t(8) * p.K + 16 * k));
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    uint32_t b0, b1;
                    T::widen(words[k], b0, b1);
                    T::mma(c, x[k].x, z[k].x, x[k].y, z[k].y, b0, b1);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) h[rt][e] = fmaf(sx[e & 1], c[e], h[rt][e]);
            }
        }
        // to every CTA of the cluster: its slot 2 part + half there
        const uint32_t mine = ptx::smem_u32(&sm.part[0][0][0]) + uint32_t(((2 * part + half_) * S::R + g) * S::LDP + 8 * nt + 2 * t) * 4;
        if (parts > 1) cluster_wait();
        for (int k = 0; k < parts; ++k) {
            const uint32_t at = parts > 1 ? cluster_address(mine, k) : mine;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                cluster_store2(at + 16 * rt * S::LDP * 4, h[rt][0], h[rt][1]);
                cluster_store2(at + (16 * rt + 8) * S::LDP * 4, h[rt][2], h[rt][3]);
            }
        }
    }
    if (parts > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    for (int i = tid; i < AD_TOK * S::R; i += AD_THREADS) {
        const int n = i & 31, j = i >> 5;
        float v = 0.f;
        for (int k = 0; k < 2 * parts; ++k) v += sm.part[0][k * S::R + j][n];
        v *= scale;
        const float hi = __uint_as_float(to_tf32(v));
        sm.h[n][j] = make_float2(hi, __uint_as_float(to_tf32(v - hi)));
    }
    __syncthreads();
    // ---- Y, a warp for 32 rows
    const uint16_t* B = static_cast<const uint16_t*>(P.B) + size_t(a) * P.rows * P.rank;
#pragma unroll 1
    for (int c = c0; c < end; c += AD_WARPS) {
        const int row = 32 * c + 4 * g;
        const bool mine = row < P.rows;
        if (c != c0) load_y(c);
        float acc[2][4][4] = {};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (16 * rt >= rank) break;
            const int j = 16 * rt + 4 * t;
            uint32_t w[4][4];                  // [row][j]: exact in tf32
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint2 v = {};
                if (mine && j < rank) v = __ldg(reinterpret_cast<const uint2*>(B + size_t(row + i) * P.rank + j));
                const float2 u = T::unpack(v.x), z = T::unpack(v.y);
                w[i][0] = __float_as_uint(u.x); w[i][1] = __float_as_uint(u.y); w[i][2] = __float_as_uint(z.x); w[i][3] = __float_as_uint(z.y);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e >= rank) w[i][e] = 0u;          // what lies behind the rank, whatever it is, does not count
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const float4 u = *reinterpret_cast<const float4*>(&sm.h[8 * nt + g][j]), v = *reinterpret_cast<const float4*>(&sm.h[8 * nt + g][j + 2]);
                const uint32_t hi[4] = {__float_as_uint(u.x), __float_as_uint(u.z), __float_as_uint(v.x), __float_as_uint(v.z)};
                const uint32_t lo[4] = {__float_as_uint(u.y), __float_as_uint(u.w), __float_as_uint(v.y), __float_as_uint(v.w)};
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        mma_tf32(acc[i][nt], w[2 * i][k], w[2 * i + 1][k], w[2 * i][k + 1], w[2 * i + 1][k + 1], lo[k], lo[k + 1]);
                        mma_tf32(acc[i][nt], w[2 * i][k], w[2 * i + 1][k], w[2 * i][k + 1], w[2 * i + 1][k + 1], hi[k], hi[k + 1]);
                    }
            }
        }
        if (!mine) continue;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int n = 8 * nt + 2 * t + e;
                if (n >= live) continue;
                float4 v = y[nt][e];
                v.x += acc[0][nt][e]; v.y += acc[0][nt][2 + e]; v.z += acc[1][nt][e]; v.w += acc[1][nt][2 + e];
                *reinterpret_cast<float4*>(p.Y + (long long)(n0 + n) * p.ldy + P.row0 + row) = v;
            }
    }
}

}  // namespace llattn

namespace {
template <typename T, int RT>
int launch_adapters(llattn::AdapterParams& p, int npools, long long tiles, int sms, cudaStream_t stream) {
    using namespace llattn;
    // CTAs of a cluster: as many as it takes to fill the chip
    p.parts = 1;
    while (p.parts < 8 && p.parts * RT < 16 && 2 * p.parts * tiles * npools <= 4 * sms) p.parts *= 2;
    const int smem = AdapterSmem<RT>::bytes(p.parts);
    auto* kernel = adapters_kernel<T, RT>;
    if (smem > 48 * 1024) CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CU(launch_dependent_cluster(kernel, dim3(unsigned(tiles * p.parts), npools), AD_THREADS, smem, p.parts, stream, p));
    return LLATTN_OK;
}
template <typename T>
int launch_adapters_rank(llattn::AdapterParams& p, int npools, int rank, long long tiles, int sms, cudaStream_t stream) {
    if (rank <= 16) return launch_adapters<T, 1>(p, npools, tiles, sms, stream);
    if (rank <= 32) return launch_adapters<T, 2>(p, npools, tiles, sms, stream);
    if (rank <= 64) return launch_adapters<T, 4>(p, npools, tiles, sms, stream);
    return launch_adapters<T, 8>(p, npools, tiles, sms, stream);
}
}  // namespace

extern "C" int llattn_adapters_w4a8(const llattn_adapter_pool* pools, int npools, const int8_t* q, const float* s, float* Y, int64_t ldy, int ntokens, int K,
                                    const int32_t* seg_first, const int32_t* seg_adapter, int nseg, void* stream) {
    using namespace llattn;
    if (!pools || !q || !s || !Y || !seg_first || !seg_adapter) return fail(LLATTN_EINVAL, "adapters_w4a8: null pointer");
    if (npools < 1 || npools > AD_MAX_POOLS) return fail(LLATTN_EINVAL, "adapters_w4a8: %d pools; 1 to %d", npools, AD_MAX_POOLS);
    if (ntokens < 0 || ntokens > 1 << 22) return fail(LLATTN_EINVAL, "adapters_w4a8: ntokens = %d", ntokens);
    if (K <= 0 || K % DN_GROUP || K > 1 << 20) return fail(LLATTN_EINVAL, "adapters_w4a8: K = %d (a multiple of 128)", K);
    if (nseg < 0 || nseg > 1 << 20) return fail(LLATTN_EINVAL, "adapters_w4a8: nseg = %d", nseg);
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
    int dev = 0, sms = 0;
    CU(cudaGetDevice(&dev));
    CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // no more tiles than this, however the segments cut the tokens: each has at most one that is not full
    const long long tiles = std::min<long long>(ntokens, (ntokens + (AD_TOK - 1ll) * nseg) / AD_TOK);
    return pools[0].type == LLATTN_F16 ? launch_adapters_rank<AdapterF16>(p, npools, rank, tiles, sms, as_stream(stream))
                                       : launch_adapters_rank<AdapterBF16>(p, npools, rank, tiles, sms, as_stream(stream));
}

// Products of e4m3 codes with a scale for each block of 128 of the contracted dimension (hiptk_block_product):
//
//     D[m][n] = alpha sum_kb SA[kb][m] SB[kb][n / block_rows] P_kb[m][n] + beta C[m][n],   P_kb[m][n] = sum_{k in kb} A[m][k] B[n][k]
//
// v_mfma_f32_16x16x128_f8f6f4 contracts exactly one block: P_kb comes out of a zero accumulator, and the sum over blocks is
// an f32 fused multiply-add with the product of the two scales.  B feeds the first operand and A the second, so that a lane
// holds four consecutive n of one m (a 16 x 16 result has lane l hold rows 4 (l / 16) .. + 3 of column l % 16): the scale of
// A is one value a lane, and D is stored in runs along its rows.  How k is dealt to the lanes does not matter as long as
// both operands are dealt alike.
//
// The 8-bit matrix instructions (all four shapes alike) align the products that they add to the largest of a small group of
// neighbouring k and drop what lies 2^-13 below it: on gaussian codes a sum over a block is 1.5e-5 off (2-norm; at most 2e-4 of the sum of the terms'
// magnitudes), which a result rounded to f16 (2e-4) or bf16 (1.7e-3) does not show but in single elements whose terms cancel, and one in f32 does.  Results in f32 are
// therefore multiplied as f16: every e4m3 value is an f16 value, and v_mfma_f32_16x16x32_f16 sums exactly enough (8e-8), at half the rate.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "dma_lds.hpp"
#include "hd_addr.hpp"
#include "hiptk_kernels.h"
#include "tile_walk.hpp"

namespace
{
    using hiptk::each;

    typedef int   v8i __attribute__((ext_vector_type(8)));
    typedef float v4f __attribute__((ext_vector_type(4)));

    struct PArgs
    {
        const uint8_t *A, *B;
        const float *  SA, *SB;
        const void*    C;
        void*          D;
        int64_t        lda, ldb, ldsa, ldsb, ldd;
        int32_t        M, N, K;
        int32_t        tiles_m, tiles_n;
        int32_t        block_shift; // rows of B per scale: 2^block_shift
        float          alpha, beta;
        int32_t        vec;   // codes in 16-byte vectors
        int32_t        type;
        int32_t        per_slice; // blocks of K per slice of a split launch (grid y), 0: not split
        float*         partial;   // [slice][M][ld_partial]
        int64_t        ld_partial;
    };

    __device__ __forceinline__ v4f mfma128(const v8i& b, const v8i& a)
    {
        const v4f zero = {0.f, 0.f, 0.f, 0.f};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, zero, 0, 0, 0, 0, 0, 0); // no scales: the plain instruction
    }

    // The 32 codes of a lane as f16, which holds every one of them exactly (a NaN stays one)
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    struct Wide
    {
        h8 part[4];
    };
    __device__ __forceinline__ Wide widen(const v8i& x)
    {
        Wide w;
#pragma unroll
        for(int q = 0; q < 8; q++)
        {
            const h2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)x[q], 1.f, false);
            const h2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)x[q], 1.f, true);
            const int at = 4 * (q & 1);
            w.part[q / 2][at]     = lo[0];
            w.part[q / 2][at + 1] = lo[1];
            w.part[q / 2][at + 2] = hi[0];
            w.part[q / 2][at + 3] = hi[1];
        }
        return w;
    }
    __device__ __forceinline__ v4f mfma128(const Wide& b, const Wide& a)
    {
        v4f p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for(int q = 0; q < 4; q++)
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.part[q], a.part[q], p, 0, 0, 0);
        return p;
    }

    template <bool WIDE>
    struct Operand
    {
        typedef v8i type;
    };
    template <>
    struct Operand<true>
    {
        typedef Wide type;
    };
    template <typename F>
    __device__ __forceinline__ F operand(const v8i& x)
    {
        if constexpr(sizeof(F) == sizeof(v8i))
            return x;
        else
            return widen(x);
    }

    template <typename T>
    __device__ __forceinline__ void store_one(const PArgs& a, int m, int n, float v)
    {
        const int64_t at = (int64_t)m * a.ldd + n;
        v *= a.alpha;
        if(a.beta != 0.f)
            v = __builtin_fmaf(a.beta, (float)((const T*)a.C)[at], v);
        ((T*)a.D)[at] = (T)v;
    }

    // 16 rows of W results (a wavefront's, rows of W + 4 in LDS) from (m, n) on: D = alpha * result + beta * C, 16 bytes a lane at any
    // element (global memory wants no alignment on this target), the last columns element by element
    template <typename T, int W, bool ADD> // (ADD: beta is not 0)
    struct Rows
    {
        static constexpr int V = 16 / sizeof(T), LANES = W / V, ROWS = 64 / LANES;
        typedef T            vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        vec_t                y[16 / ROWS]; // C's
    };
    template <typename T, int W, bool ADD>
    __device__ __forceinline__ void fetch_rows(const PArgs& a, Rows<T, W, ADD>& rows, int m, int n, int lane)
    {
        typedef Rows<T, W, ADD> R;
#pragma unroll
        for(int i = 0; i < 16 / R::ROWS; i++)
        {
            const int r = i * R::ROWS + lane / R::LANES, c = R::V * (lane % R::LANES);
            rows.y[i]   = {};
            if(m + r < a.M && n + c + R::V <= a.N)
                rows.y[i] = *(const typename R::vec_t*)((const T*)a.C + (int64_t)(m + r) * a.ldd + n + c);
        }
    }
    template <typename T, int W, bool ADD>
    __device__ __forceinline__ void store_rows(const PArgs& a, const Rows<T, W, ADD>& rows, const float* stage, int m, int n, int lane)
    {
        typedef Rows<T, W, ADD>   R;
        typedef typename R::vec_t vec_t;
        constexpr int             V = R::V, LANES = R::LANES, ROWS = R::ROWS;
#pragma unroll
        for(int r0 = 0; r0 < 16; r0 += ROWS)
        {
            const int r = r0 + lane / LANES, c = V * (lane % LANES);
            if(m + r >= a.M)
                continue;
            if(n + c + V <= a.N)
            {
                const int64_t at = (int64_t)(m + r) * a.ldd + n + c;
                vec_t         x;
#pragma unroll
                for(int q = 0; q < V; q += 4)
                {
                    const v4f v = *(const v4f*)&stage[r * (W + 4) + c + q];
#pragma unroll
                    for(int e = 0; e < 4; e++)
                        x[q + e] = (T)(ADD ? __builtin_fmaf(a.beta, (float)rows.y[r0 / ROWS][q + e], a.alpha * v[e]) : a.alpha * v[e]);
                }
                *(vec_t*)((T*)a.D + at) = x;
            }
            else
            {
#pragma unroll 1
                for(int e = c; e < c + V && n + e < a.N; e++)
                    store_one<T>(a, m + r, n + e, stage[r * (W + 4) + e]);
            }
        }
    }

    // 16 codes of a row from k on; those beyond K, and rows beyond the last, are zero codes
    __device__ __forceinline__ uint4 load16(const uint8_t* base, int64_t ld, int row, int rows, int k, int K, bool vec)
    {
        uint4 x = {0, 0, 0, 0};
        if(row >= rows || k >= K)
            return x;
        const uint8_t* p = base + (int64_t)row * ld + k;
        if(vec && k + 16 <= K)
            return *(const uint4*)p;
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for(int i = 0; i < 16; i++)
            if(k + i < K)
                w[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
        return uint4{w[0], w[1], w[2], w[3]};
    }

    // Any alignment and leading dimension: a 64 x 64 tile on four wavefronts, staged through registers, one block of K at a time.  Bound by its
    // byte loads: 2048^3 with rows of 2049 bytes 418 us, 16 on the tiles below (operands on multiples of 16 are the caller's choice).
    template <typename T>
    __global__ void __launch_bounds__(256, 2) block_product_any_kernel(const PArgs a)
    {
        constexpr int PITCH = 144; // 128 codes and 16 bytes: rows start in different banks
        __shared__ __attribute__((aligned(16))) uint8_t sa[64 * PITCH], sb[64 * PITCH];
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int m0 = (int)(blockIdx.x % (uint32_t)a.tiles_m) * 64, n0 = (int)(blockIdx.x / (uint32_t)a.tiles_m) * 64;
        const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
        const int srow = tid >> 2, sk = (tid & 3) * 32;
        v4f       acc[2][2] = {};
        for(int k0 = 0; k0 < a.K; k0 += 128)
        {
            const int kb = k0 >> 7;
#pragma unroll
            for(int h = 0; h < 2; h++)
            {
                *(uint4*)&sa[srow * PITCH + sk + 16 * h] = load16(a.A, a.lda, m0 + srow, a.M, k0 + sk + 16 * h, a.K, a.vec);
                *(uint4*)&sb[srow * PITCH + sk + 16 * h] = load16(a.B, a.ldb, n0 + srow, a.N, k0 + sk + 16 * h, a.K, a.vec);
            }
            __syncthreads();
            // results in f32: the codes are widened, see above
            typedef typename Operand<sizeof(T) == 4>::type frag_t;
            frag_t fb[2], fa[2];
#pragma unroll
            for(int i = 0; i < 2; i++)
            {
                fb[i] = operand<frag_t>(*(const v8i*)&sb[(wn + 16 * i + (lane & 15)) * PITCH + 32 * (lane >> 4)]);
                fa[i] = operand<frag_t>(*(const v8i*)&sa[(wm + 16 * i + (lane & 15)) * PITCH + 32 * (lane >> 4)]);
            }
            __syncthreads();
#pragma unroll
            for(int j = 0; j < 2; j++)
            {
                const int   m  = m0 + wm + 16 * j + (lane & 15);
                const float fs = a.SA[(int64_t)kb * a.ldsa + (m < a.M ? m : a.M - 1)];
#pragma unroll
                for(int i = 0; i < 2; i++)
                {
                    const v4f p = mfma128(fb[i], fa[j]);
#pragma unroll
                    for(int r = 0; r < 4; r++)
                    {
                        int n        = n0 + wn + 16 * i + 4 * (lane >> 4) + r;
                        n            = n < a.N ? n : a.N - 1;
                        const float s = fs * a.SB[(int64_t)kb * a.ldsb + (n >> a.block_shift)];
                        acc[i][j][r]  = __builtin_fmaf(p[r], s, acc[i][j][r]);
                    }
                }
            }
        }
#pragma unroll
        for(int i = 0; i < 2; i++)
#pragma unroll
            for(int j = 0; j < 2; j++)
#pragma unroll
                for(int r = 0; r < 4; r++)
                {
                    const int m = m0 + wm + 16 * j + (lane & 15), n = n0 + wn + 16 * i + 4 * (lane >> 4) + r;
                    if(m < a.M && n < a.N)
                        store_one<T>(a, m, n, acc[i][j][r]);
                }
    }

    // ---- tiles loaded straight into LDS ------------------------------------------------------------------------------

    // The slice of K that a workgroup of a split launch takes: its blocks of the operands and scales, its part of the sums
    __device__ __forceinline__ void slice_of(PArgs& a, uint32_t slice)
    {
        const int64_t kb = (int64_t)slice * a.per_slice, k = kb * 128;
        a.A += k;
        a.B += k;
        a.SA += kb * a.ldsa;
        a.SB += kb * a.ldsb;
        const int64_t left = a.K - k, most = (int64_t)a.per_slice * 128;
        a.K                = (int32_t)(left < most ? left : most);
        a.D                = a.partial + (int64_t)slice * a.M * a.ld_partial;
        a.ldd              = a.ld_partial;
        a.alpha            = 1.f;
        a.beta             = 0.f;
        a.type             = HIPTK_F32;
    }

    // BM x BN on WM x WN wavefronts, a wavefront NJ x NI blocks of 16 x 16.  A ring of ST LDS stages of one block of K each; rows of 128 codes, the
    // 16-byte chunk at position c of a row holding chunk c ^ (row / 2) % 8 (16 lanes that read one chunk of 16 rows then touch
    // disjoint banks).  Bound by LDS and power in the large tiles: 256 x 256 reads 192 KB and receives 64 KB a stage, about the cycles
    // of its MFMAs, and 8192^3 takes 455 us (2420 TFLOP/s, MFMAs 66 % of the busy cycles; ring of 2 loaded without lookahead 545); widened to f16 the
    // vector unit (conversions and scales 51 % of the cycles, MFMAs 47 %): 4096 x 4096 x 8189 254 us, 1081 TFLOP/s.
    template <int BM, int BN, int WM, int WN, int ST, bool ROWS, bool WIDE>
    struct Tile
    {
        static constexpr int WAVES = WM * WN, NJ = BM / WM / 16, NI = BN / WN / 16;
        static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES; // loads of 8 rows per wavefront and stage
        static constexpr int SCALES = BM * 4, SCALES_B = ROWS ? BN * 4 : 256; // bytes per stage
        static constexpr int STAGE = (BM + BN) * 128;
        static constexpr int OFF_S = ST * STAGE;
        static constexpr int LDS   = ST * (STAGE + SCALES + SCALES_B);
        // scales: 64 of the tile's rows a load, A's and then B's (square blocks: one load, of which BN / 128 are used)
        static constexpr int SLA = BM / 64, SLB = ROWS ? BN / 64 : 1, SL = (SLA + SLB + WAVES - 1) / WAVES;
        static constexpr int LOADS = LA + LB + SL; // per wavefront and stage
        static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && LDS <= 160 * 1024, "");
    };

    template <int BM, int BN, int WM, int WN, int ST, bool ROWS, bool WIDE>
    __global__ void __launch_bounds__(64 * WM * WN, 2) block_product_kernel(const PArgs whole)
    {
        PArgs a = whole;
        if(whole.per_slice)
            slice_of(a, blockIdx.y);
        typedef Tile<BM, BN, WM, WN, ST, ROWS, WIDE> T;
        constexpr int NI = T::NI, NJ = T::NJ, WAVES = T::WAVES;
        extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
        typedef uint8_t __attribute__((address_space(3))) * lds_ptr;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;

        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave % WM, wn = wave / WM;
        int       tm, tn;
        hiptk::tile_of(hiptk::place_of(blockIdx.x, (uint32_t)a.tiles_m * (uint32_t)a.tiles_n), a.tiles_m, a.tiles_n, tm, tn);
        const int m0 = tm * BM, n0 = tn * BN;

        // what each lane loads: rows beyond the last read the last one
        const uint8_t* abase = a.A + (int64_t)m0 * a.lda;
        const uint8_t* bbase = a.B + (int64_t)n0 * a.ldb;
        uint32_t       voff[T::LA + T::LB];
        const int      lrow = lane >> 3;
        each<T::LA + T::LB>([&](auto i_c) __attribute__((always_inline)) {
            constexpr int  i   = decltype(i_c)::value;
            constexpr bool isa = i < T::LA;
            const int      row = (isa ? wave * T::LA + i : wave * T::LB + i - T::LA) * 8 + lrow;
            const int      most = isa ? a.M - 1 - m0 : a.N - 1 - n0;
            voff[i] = (uint32_t)(row < most ? row : most) * (uint32_t)(isa ? a.lda : a.ldb) + 16u * (uint32_t)hiptk::hk_chunk_pos(row, lane & 7);
        });
        // Scales: every wavefront issues as many loads of 64, so that one count says what has landed (the surplus repeats the last).
        uint64_t sfrom[T::SL];
        int64_t  sstep[T::SL];
        uint32_t soff[T::SL], sdst[T::SL];
        each<T::SL>([&](auto q_c) __attribute__((always_inline)) {
            constexpr int q  = decltype(q_c)::value;
            int           u  = wave + q * WAVES;
            u                = u < T::SLA + T::SLB ? u : T::SLA + T::SLB - 1;
            const int n_most = ((a.N - 1) >> a.block_shift) - (n0 >> a.block_shift);
            if(u < T::SLA)
            {
                const int r = u * 64 + lane, most = a.M - 1 - m0;
                sfrom[q]    = (uint64_t)(a.SA + m0);
                sstep[q]    = 4 * a.ldsa;
                soff[q]     = 4u * (uint32_t)(r < most ? r : most);
                sdst[q]     = (uint32_t)u * 256u;
            }
            else
            {
                const int r = (u - T::SLA) * 64 + lane;
                sfrom[q]    = (uint64_t)(a.SB + (n0 >> a.block_shift));
                sstep[q]    = 4 * a.ldsb;
                soff[q]     = 4u * (uint32_t)(r < n_most ? r : n_most);
                sdst[q]     = (uint32_t)(T::SCALES + (u - T::SLA) * 256);
            }
        });

        const int nk   = (a.K + 127) >> 7;
        const int tail = a.K & 127;
        // load i of the wavefront's LOADS of stage t, into ring slot s
        auto load_part = [&](int t, int s, auto i_c) __attribute__((always_inline)) {
            constexpr int  i  = decltype(i_c)::value;
            const uint32_t st = lds0 + (uint32_t)s * T::STAGE;
            if constexpr(i < T::LA + T::LB)
            {
                constexpr bool isa = i < T::LA;
                const int  q   = isa ? wave * T::LA + i : wave * T::LB + i - T::LA;
                hiptk::dma_dst_at(st, (uint32_t)((isa ? 0 : BM * 128) + q * 1024));
                hiptk::dma_load(voff[i], (isa ? abase : bbase) + (int64_t)t * 128);
            }
            else
            {
                constexpr int q = i - T::LA - T::LB;
                hiptk::dma_dst_at(lds0 + T::OFF_S + (uint32_t)s * (T::SCALES + T::SCALES_B), sdst[q]);
                hiptk::dma_load1(soff[q], (const void*)(sfrom[q] + (uint64_t)(t * sstep[q])));
            }
        };

        // Before the loads of a last block that K ends in: chunks that begin beyond K are not in the row; they read the
        // block's first one, and are cleared before use.
        auto shorten = [&]() __attribute__((always_inline)) {
            int l = lane;
            asm volatile("" : "+v"(l)); // (nothing of this is kept in registers through the main loop)
            each<T::LA + T::LB>([&](auto i_c) __attribute__((always_inline)) {
                constexpr int i = decltype(i_c)::value;
                const int     q = i < T::LA ? wave * T::LA + i : wave * T::LB + i - T::LA;
                const int     c = hiptk::hk_chunk_pos(q * 8 + (l >> 3), l & 7);
                voff[i] -= 16 * c >= tail ? 16u * (uint32_t)c : 0u;
            });
        };

        v4f acc[NI][NJ];
#pragma unroll
        for(int i = 0; i < NI; i++)
#pragma unroll
            for(int j = 0; j < NJ; j++)
                acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

        // operand fetch: lane l holds row l % 16 and the chunks l / 16 and l / 16 + 4 of the block
        const int frow  = lane & 15;
        const int fa0   = (wm * NJ * 16 + frow) * 128 + 16 * hiptk::hk_chunk_pos(frow, lane >> 4);
        const int fa1   = (wm * NJ * 16 + frow) * 128 + 16 * hiptk::hk_chunk_pos(frow, (lane >> 4) + 4);
        const int fb0   = (BM + wn * NI * 16 + frow) * 128 + 16 * hiptk::hk_chunk_pos(frow, lane >> 4);
        const int fb1   = (BM + wn * NI * 16 + frow) * 128 + 16 * hiptk::hk_chunk_pos(frow, (lane >> 4) + 4);
        auto      fetch = [&](const uint8_t* at0, const uint8_t* at1) __attribute__((always_inline)) {
            const int4 x = *(const int4*)at0, y = *(const int4*)at1;
            return v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        };

        // One step multiplies one stage.  Its first operands are in registers when it begins; the rest is fetched one block of 16
        // tokens ahead.  When the last fetch of stage t has been issued, one barrier says both that stage t + 1 has landed
        // (every wavefront has waited for its own loads) and that the slot of stage t is free: under the MFMAs that are
        // left the first operands of stage t + 1 are fetched, and the loads of stage t + ST begin, which go on in step t + 1.
        constexpr int NB = NI * NJ, LAG = 2; // sums come LAG blocks behind their MFMA, whose result takes longer than the next one to come
        constexpr int MEET = (NJ - 1) * NI; // blocks in front of the barrier
        constexpr int LEFT = NI < T::LOADS ? NI : T::LOADS; // loads behind it in the same step
        static_assert(NJ % 2 == 0 && NI >= 2 && ST >= 2, "");
        typedef typename Operand<WIDE>::type frag_t;
        v8i    ra[2], rb[NI]; // codes as they come
        frag_t fa[2], fb[NI]; // what the MFMAs take
        v4f    sb[NI], p[LAG + 1];
        float  sa[4], s1[4], sb1 = 0.f;
        auto   fetch_a = [&](const uint8_t* st, auto j_c) __attribute__((always_inline)) {
            constexpr int j = decltype(j_c)::value;
            ra[j & 1]       = fetch(st + fa0 + j * 2048, st + fa1 + j * 2048);
        };
        auto fetch_b = [&](const uint8_t* st, auto i_c) __attribute__((always_inline)) {
            constexpr int i = decltype(i_c)::value;
            rb[i]           = fetch(st + fb0 + i * 2048, st + fb1 + i * 2048);
        };
        auto fetch_sa = [&](const uint8_t* ss, auto j_c) __attribute__((always_inline)) {
            sa[decltype(j_c)::value & 3] = *(const float*)(ss + 4 * (wm * NJ * 16 + 16 * decltype(j_c)::value + frow));
        };
        auto fetch_sb = [&](const uint8_t* ss) __attribute__((always_inline)) {
            if constexpr(ROWS)
            {
#pragma unroll
                for(int i = 0; i < NI; i++)
                    sb[i] = *(const v4f*)(ss + T::SCALES + 4 * (wn * NI * 16 + 16 * i + 4 * (lane >> 4)));
            }
            else
                sb1 = *(const float*)(ss + T::SCALES + 4 * ((wn * NI * 16) >> 7));
        };
        auto stage_at  = [&](int slot) __attribute__((always_inline)) { return (const uint8_t*)lds + slot * T::STAGE; };
        auto scales_at = [&](int slot) __attribute__((always_inline)) { return (const uint8_t*)lds + T::OFF_S + slot * (T::SCALES + T::SCALES_B); };
        // codes beyond K in the last stage: zeros (a row may hold anything there, NaN codes too)
        auto clear_tail = [&](int slot) __attribute__((always_inline)) {
            uint8_t* st = lds + slot * T::STAGE;
            for(int row = tid; row < BM + BN; row += 64 * WAVES)
                for(int c = tail >> 4; c < 8; c++)
                {
                    uint4*    q    = (uint4*)(st + row * 128 + 16 * hiptk::hk_chunk_pos(row, c));
                    const int keep = tail - 16 * c; // codes of this chunk that are K's (none: 0 or less)
                    uint4     x    = {0, 0, 0, 0};
                    if(keep > 0)
                    {
                        x             = *q;
                        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for(int i = 0; i < 4; i++)
                        {
                            const int left = keep - 4 * i;
                            w[i] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                        }
                        x = uint4{w[0], w[1], w[2], w[3]};
                    }
                    *q = x;
                }
            __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_lgkm0);
            hiptk::lds_barrier();
        };
        // loads FROM .. TO - 1 of stage t into slot s, all at once
        auto load_all = [&](int t, int s, auto from_c, auto to_c) __attribute__((always_inline)) {
            if(tail && t == nk - 1 && decltype(from_c)::value == 0)
                shorten();
            each<T::LOADS>([&](auto l_c) __attribute__((always_inline)) {
                if constexpr(decltype(l_c)::value >= decltype(from_c)::value && decltype(l_c)::value < decltype(to_c)::value)
                    load_part(t, s, l_c);
            });
        };
        typedef std::integral_constant<int, 0>        First;
        typedef std::integral_constant<int, LEFT>     Left;
        typedef std::integral_constant<int, T::LOADS> All;

        int  slot = 0; // of stage t
        auto step = [&](int t, auto more_c, auto rest_c, auto follows_c) __attribute__((always_inline)) {
            constexpr bool MORE = decltype(more_c)::value, REST = decltype(rest_c)::value, FOLLOWS = decltype(follows_c)::value; // stages t + ST, t + ST - 1, t + 1 exist
            const int      before = slot == 0 ? ST - 1 : slot - 1, next = slot == ST - 1 ? 0 : slot + 1; // slots of stages t + ST - 1 and t + 1
            const uint8_t *st = stage_at(slot), *nst = stage_at(next), *ss = scales_at(slot);
            each<NB + LAG>([&](auto b_c) __attribute__((always_inline)) {
                constexpr int b = decltype(b_c)::value;
                if constexpr(b < NB)
                {
                    constexpr int j = b / NI, i = b % NI;
                    if constexpr(FOLLOWS && b == MEET)
                    {
                        // (loads complete in order: those of the stages behind t + 1 may be under way)
                        __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_vm_lgkm0(REST ? (ST - 2) * T::LOADS : 0));
                        hiptk::lds_barrier();
                        if(!MORE && tail && t + 1 == nk - 1)
                            clear_tail(next);
                        if(MORE && tail && t + ST == nk - 1)
                            shorten();
                    }
                    if constexpr(WIDE && i == 0)
                        fa[j & 1] = operand<frag_t>(ra[j & 1]);
                    if constexpr(WIDE && j == 0)
                        fb[i] = operand<frag_t>(rb[i]);
                    if constexpr(WIDE)
                        p[b % (LAG + 1)] = mfma128(fb[i], fa[j & 1]);
                    else
                        p[b % (LAG + 1)] = mfma128(rb[i], ra[j & 1]);
                    asm volatile("" : "+v"(p[b % (LAG + 1)])); // (neither the product nor the sum may be moved from where it stands)
                    if constexpr(i == 0 && j + 1 < NJ)
                    {
                        fetch_a(st, std::integral_constant<int, j + 1>{});
                        fetch_sa(ss, std::integral_constant<int, j + 1>{});
                    }
                    if constexpr(REST && b < MEET)
                        each<T::LOADS>([&](auto l_c) __attribute__((always_inline)) {
                            if constexpr(decltype(l_c)::value >= LEFT && (decltype(l_c)::value - LEFT) % MEET == b)
                                load_part(t + ST - 1, before, l_c);
                        });
                    if constexpr(FOLLOWS && b >= MEET)
                    {
                        if constexpr(i == 0)
                            fetch_a(nst, First{});
                        fetch_b(nst, std::integral_constant<int, i>{});
                    }
                    if constexpr(MORE && b >= MEET && b - MEET < LEFT)
                        load_part(t + ST, slot, std::integral_constant<int, b - MEET>{});
                }
                if constexpr(b >= LAG)
                {
                    constexpr int c = b - LAG, j = c / NI, i = c % NI;
                    if constexpr(i == 0)
                        s1[j & 3] = sa[j & 3] * sb1;
#pragma unroll
                    for(int r = 0; r < 4; r++)
                        acc[i][j][r] = __builtin_fmaf(p[c % (LAG + 1)][r], ROWS ? sa[j & 3] * sb[i][r] : s1[j & 3], acc[i][j][r]);
                    asm volatile("" : "+v"(acc[i][j]));
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr(FOLLOWS)
            {
                fetch_sa(scales_at(next), First{});
                fetch_sb(scales_at(next));
            }
            slot = next;
        };

        each<ST - 1>([&](auto q_c) __attribute__((always_inline)) {
            constexpr int q = decltype(q_c)::value;
            if(q < nk)
                load_all(q, q, First{}, All{});
        });
        if(ST - 1 < nk)
        {
            load_all(ST - 1, ST - 1, First{}, Left{});
            __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_vm_lgkm0((ST - 2) * T::LOADS + LEFT));
        }
        else
            __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_vm_lgkm0(0));
        hiptk::lds_barrier();
        if(tail && nk == 1)
            clear_tail(0);
        fetch_a(stage_at(0), First{});
        each<NI>([&](auto i_c) __attribute__((always_inline)) { fetch_b(stage_at(0), i_c); });
        fetch_sa(scales_at(0), First{});
        fetch_sb(scales_at(0));
        int t = 0;
        for(; t + ST < nk; t++)
            step(t, std::true_type{}, std::true_type{}, std::true_type{});
        if(t + ST - 1 < nk)
        {
            step(t, std::false_type{}, std::true_type{}, std::true_type{});
            t++;
        }
        if constexpr(ST > 2)
            for(; t + 1 < nk; t++)
                step(t, std::false_type{}, std::false_type{}, std::true_type{});
        step(t, std::false_type{}, std::false_type{}, std::false_type{});
        // Results pass through LDS, 16 rows at a time and within the wavefront, so that D is written (and C read) in whole lines:
        // stored as the accumulators lie, 32 bytes in each of 16 rows, a compute unit wrote 8 bytes a cycle.  C's rows are asked for a group
        // ahead: D may be C, so no load passes a store, and asked for where they are added each would be waited for.
        hiptk::lds_barrier(); // (every wavefront is done with the last stage)
        float* stage = (float*)lds + wave * 16 * (NI * 16 + 4);
        auto   store = [&](auto type, auto add_c) __attribute__((always_inline)) {
            constexpr bool                     ADD = decltype(add_c)::value;
            Rows<decltype(type), NI * 16, ADD> rows[2];
            const int                          m = m0 + wm * NJ * 16, n = n0 + wn * NI * 16;
            if constexpr(ADD)
                fetch_rows(a, rows[0], m, n, lane);
            each<NJ>([&](auto j_c) __attribute__((always_inline)) {
                constexpr int j = decltype(j_c)::value;
                if constexpr(ADD && j + 1 < NJ)
                    fetch_rows(a, rows[(j + 1) % 2], m + (j + 1) * 16, n, lane);
#pragma unroll
                for(int i = 0; i < NI; i++)
                    *(v4f*)&stage[frow * (NI * 16 + 4) + 16 * i + 4 * (lane >> 4)] = acc[i][j];
                store_rows(a, rows[j % 2], stage, m + j * 16, n, lane);
            });
        };
        auto store_as = [&](auto type) __attribute__((always_inline)) {
            if(a.beta != 0.f)
                store(type, std::true_type{});
            else
                store(type, std::false_type{});
        };
        if(WIDE || a.type == HIPTK_F32)
            store_as(0.f);
        else if(a.type == HIPTK_F16)
            store_as((_Float16)0);
        else
            store_as((__bf16)0.f);
    }

    // ---- few tokens: the weight is read once, straight into registers --------------------------------------------------

    // 16 rows of B against up to 16 TM tokens, on eight wavefronts that take the blocks of K in turn, U at a time with all
    // their loads under way together, and add their sums up in LDS in a fixed order.  Bound by memory: 8192 x 4096 codes take a call
    // 8.4 us for one token and 10.5 for 16, 4096 x 8192 13.3 for 23 (a call that reads next to nothing 5.5).  Workgroups begin at different blocks: rows lie a power of
    // two apart, so that the same block of all rows is in a few of the memory's channels (10.4 and 11.5 us where all begin at
    // the first).  More or fewer loads under way change nothing (U = 2 or 8, 16 wavefronts), loads past the caches cost 1 us.  Both operands come from memory in the
    // lanes that multiply them: lane l holds the chunks l / 16 and l / 16 + 4 of row l % 16.
    template <int TM, bool ROWS, bool WIDE>
    __global__ void __launch_bounds__(512) block_product_few_kernel(const PArgs a)
    {
        constexpr int WAVES = 8, U = 4;
        __shared__ v4f part[WAVES][TM][64];
        const int      lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        const int      row = lane & 15, g = lane >> 4;
        const int      n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * TM, nk = (a.K + 127) >> 7, tail = a.K & 127;
        const uint8_t* brow = a.B + (int64_t)(n0 + row < a.N ? n0 + row : a.N - 1) * a.ldb;
        const uint8_t* arow[TM];
        int            am[TM];
#pragma unroll
        for(int i = 0; i < TM; i++)
        {
            am[i]   = m0 + 16 * i + row < a.M ? m0 + 16 * i + row : a.M - 1;
            arow[i] = a.A + (int64_t)am[i] * a.lda;
        }
        int64_t bs[4]; // the scales of the four rows of B that the lane has results for
#pragma unroll
        for(int r = 0; r < 4; r++)
        {
            const int n = n0 + 4 * g + r;
            bs[r]       = (n < a.N ? n : a.N - 1) >> a.block_shift;
        }
        typedef typename Operand<WIDE>::type frag_t;
        // codes beyond K: chunks that begin there read the block's first one instead, and all of them count as zeros
        auto load = [&](const uint8_t* at, int kb) __attribute__((always_inline)) {
            const bool last = tail && kb == nk - 1;
            const int  c0 = 16 * g, c1 = 16 * g + 64;
            at += (int64_t)kb * 128;
            const int4 x = *(const int4*)(at + (last && c0 >= tail ? 0 : c0)), y = *(const int4*)(at + (last && c1 >= tail ? 0 : c1));
            v8i        v = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            if(last)
            {
#pragma unroll
                for(int q = 0; q < 8; q++)
                {
                    const int left = tail - (q < 4 ? c0 : c1) - 4 * (q & 3); // codes of this word
                    v[q] &= left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
                }
            }
            return v;
        };
        const int rot = (int)(blockIdx.x % (uint32_t)nk);
        v4f acc[TM] = {};
        for(int k0 = wave; k0 < nk; k0 += WAVES * U)
        {
            v8i   b[U], x[U][TM];
            float sa[U][TM];
            v4f   sb[U];
#pragma unroll
            for(int u = 0; u < U; u++)
            {
                int kb = k0 + WAVES * u;
                if(kb < nk)
                {
                    kb += rot;
                    kb -= kb >= nk ? nk : 0;
                    b[u] = load(brow, kb);
#pragma unroll
                    for(int i = 0; i < TM; i++)
                    {
                        x[u][i]  = load(arow[i], kb);
                        sa[u][i] = a.SA[(int64_t)kb * a.ldsa + am[i]];
                    }
#pragma unroll
                    for(int r = 0; r < (ROWS ? 4 : 1); r++)
                        sb[u][r] = a.SB[(int64_t)kb * a.ldsb + bs[r]];
                }
            }
#pragma unroll
            for(int u = 0; u < U; u++)
                if(k0 + WAVES * u < nk)
                {
                    const frag_t fb = operand<frag_t>(b[u]);
#pragma unroll
                    for(int i = 0; i < TM; i++)
                    {
                        const v4f p = mfma128(fb, operand<frag_t>(x[u][i]));
#pragma unroll
                        for(int r = 0; r < 4; r++)
                            acc[i][r] = __builtin_fmaf(p[r], sa[u][i] * sb[u][ROWS ? r : 0], acc[i][r]);
                    }
                }
        }
#pragma unroll
        for(int i = 0; i < TM; i++)
            part[wave][i][lane] = acc[i];
        __syncthreads();
        // (one thread a result: 16 consecutive n of a token are neighbouring threads)
        for(int o = threadIdx.x; o < 256 * TM; o += 64 * WAVES)
        {
            const int i = o >> 8, m = (o >> 4) & 15, n = o & 15;
            float     v = 0.f;
#pragma unroll
            for(int w = 0; w < WAVES; w++)
                v += part[w][i][16 * (n >> 2) + m][n & 3];
            if(m0 + 16 * i + m < a.M && n0 + n < a.N)
            {
                if(WIDE)
                    store_one<float>(a, m0 + 16 * i + m, n0 + n, v);
                else if(a.type == HIPTK_F16)
                    store_one<_Float16>(a, m0 + 16 * i + m, n0 + n, v);
                else
                    store_one<__bf16>(a, m0 + 16 * i + m, n0 + n, v);
            }
        }
    }

    // The slices' sums, added in their order: four columns a thread
    template <typename T>
    __global__ void __launch_bounds__(256) block_product_join_kernel(const PArgs a, int slices)
    {
        const int64_t quads = a.ld_partial / 4, q = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if(q >= quads * a.M)
            return;
        const int m = (int)(q / quads), n = 4 * (int)(q % quads);
        v4f       v = {0.f, 0.f, 0.f, 0.f};
        for(int s = 0; s < slices; s++)
            v += *(const v4f*)&a.partial[((int64_t)s * a.M + m) * a.ld_partial + n];
#pragma unroll
        for(int r = 0; r < 4; r++)
            if(n + r < a.N)
                store_one<T>(a, m, n + r, v[r]);
    }

    bool well_formed(const hiptk_block_product_t* p)
    {
        constexpr int64_t MOST = 0x7fffff00; // (tile ends stay below 2^31)
        if(!p || p->M < 0 || p->N < 0 || p->K < 0 || p->M > MOST || p->N > MOST || p->K > MOST || (p->block_rows != 1 && p->block_rows != 128))
            return false;
        if(p->type != HIPTK_F16 && p->type != HIPTK_BF16 && p->type != HIPTK_F32)
            return false;
        if(p->M == 0 || p->N == 0)
            return true;
        return p->D && (p->beta == 0.f || p->C) && (p->K == 0 || (p->A && p->B && p->SA && p->SB));
    }

    // ---- selection ------------------------------------------------------------------------------------------------------

    // A tile, how many of its workgroups a compute unit holds, and what one block of K costs a compute unit that holds one
    // of them and one that holds all (us, measured on launches of 16 to 64 blocks of K that leave the unit alone / fill the device; what the
    // rule takes is within 3 % of the best of all tiles and slices on 14 shapes of 64 x 4096 x 8192 to 4096 x 1024 x 4096).
    // A smaller tile costs more per flop: what it loads grows against what it multiplies (64 bytes a cycle arrive in
    // a unit; 256 x 256 takes 1024 cycles of them for 2048 of MFMAs, 64 x 64 256 for 128).
    struct Choice
    {
        int         bm, bn, slots;
        float       one, all, around; // around: before and behind its main loop
        const char* name;
    };
    constexpr Choice NARROW[] = {{256, 256, 1, 1.25f, 1.78f, 2.f, "block_product_256x256"}, {256, 128, 1, 0.68f, 1.00f, 2.f, "block_product_256x128"},
                                 {128, 128, 2, 0.64f, 1.05f, 2.f, "block_product_128x128"}, {64, 128, 2, 0.29f, 0.55f, 2.f, "block_product_64x128"},
                                 {64, 64, 2, 0.19f, 0.33f, 2.f, "block_product_64x64"}};
    // ... and with the operands widened to f16 (results in f32: their tiles end with 64 or 128 KB written and, where they are added to C, read, beside
    // another's main loop in the smaller: 4096 x 8192 x 200 onto C 95 us in tiles of 256 x 128, 76 of 128 x 128; with many blocks of K the larger's stages cost less)
    constexpr Choice WIDENED[] = {{256, 128, 1, 1.70f, 1.93f, 6.f, "block_product_256x128_f16"}, {128, 128, 2, 1.22f, 2.00f, 4.f, "block_product_128x128_f16"},
                                  {64, 64, 2, 0.53f, 0.63f, 2.f, "block_product_64x64_f16"}};
    constexpr int UNITS = 256;
    // Rows of A up to which B may be streamed through registers, and what that costs: us for each block of K that a compute unit with `beside`
    // workgroups of 16 tm rows takes.  (Measured against the tiles on 126 shapes of 1 to 128 rows, us through registers and in tiles: 16 x 4096 x 4096
    // 6.7 and 12.2, 16 x 8192 x 8192 17.6 and 16.4, 32 x 8192 x 8192 27.6 and 17.3, 128 x 512 x 4096 6.5 and 10.6, 96 x 1024 x 8192 14.6 and 11.8.
    // Workgroups that share a unit read A anew, fewer rows of it less.)
    constexpr int64_t FEW = 128;
    double            few_cost(int64_t M, int tm, int64_t beside, bool wide)
    {
        const double each = tm == 2 ? (beside == 1 ? 0.15 : 0.18) : beside == 1 ? 0.08 : beside == 2 ? 0.10 : 0.14;
        return (double)beside * each * (M < 16 ? 0.65 + 0.35 * (double)M / 16 : 1.0) * (wide ? 1.1 : 1.0);
    }
    constexpr uint64_t MOST_WORKSPACE = 256ull << 20;

    struct Plan
    {
        int         kind; // 0: any, 1: few tokens, 2: a tile
        int         tile, slices;
        int64_t     per_slice;
        uint64_t    bytes; // of workspace
        const char* name;
    };

    Plan plan_of(const hiptk_block_product_t* p, uint64_t workspace)
    {
        Plan       plan = {0, 0, 1, 0, 0, p->type == HIPTK_F32 ? "block_product_64x64_any_f16" : "block_product_64x64_any"};
        const bool wide = p->type == HIPTK_F32;
        if(p->K == 0 || (((uintptr_t)p->A | (uintptr_t)p->B | (uint64_t)p->lda | (uint64_t)p->ldb) & 15) || p->lda >= (1 << 23) || p->ldb >= (1 << 23))
            return plan; // (a lane's offset into a tile is 32 bits)
        const int64_t nk    = (p->K + 127) / 128;
        const Choice* tiles = wide ? WIDENED : NARROW;
        const int     count = wide ? (int)(sizeof(WIDENED) / sizeof(Choice)) : (int)(sizeof(NARROW) / sizeof(Choice));
        const int64_t ldp   = (p->N + 3) / 4 * 4;
        double        best  = 1e30;
        for(int i = 0; i < count; i++)
        {
            const Choice& c     = tiles[i];
            const int64_t tiles_ = ((p->M + c.bm - 1) / c.bm) * ((p->N + c.bn - 1) / c.bn);
            for(int slices = 1; slices <= 16; slices *= 2)
            {
                const int64_t per = (nk + slices - 1) / slices, used = (nk + per - 1) / per; // (no slice is empty)
                const uint64_t bytes = slices == 1 ? 0 : 4ull * (uint64_t)used * (uint64_t)p->M * (uint64_t)ldp;
                if(slices > 1 && (per < 4 || bytes > workspace || bytes > MOST_WORKSPACE))
                    break;
                // rounds of full units, and what is left over; each round begins and ends with latency that nothing covers
                const int64_t work = tiles_ * used, full = work / (UNITS * c.slots), left = work - full * UNITS * c.slots;
                double        us   = 5.0 + (double)full * (c.around + per * c.all) + (left > UNITS ? c.around + per * c.all : left ? c.around + per * c.one : 0.0);
                if(slices > 1)
                    us += 4.0 + (double)bytes / 3e6; // the partial sums written and read, and a launch
                if(us < best)
                {
                    best           = us;
                    plan.kind      = 2;
                    plan.tile      = i;
                    plan.slices    = (int)used;
                    plan.per_slice = used > 1 ? per : 0;
                    plan.bytes     = used > 1 ? bytes : 0;
                    plan.name      = c.name;
                }
            }
        }
        // (neither is faster than B comes from memory, and where both are as fast as that the registers are)
        const double floor = 5.0 + (double)p->N * (double)p->K / 4.8e6;
        best               = best < floor ? floor : best;
        const bool fits    = (p->N + 15) / 16 * 512 < (1ll << 31); // (threads of the grid in x)
        for(int tm = 1; tm <= 2 && p->M <= FEW && fits; tm++)
        {
            const int64_t beside = (((p->M + 16 * tm - 1) / (16 * tm)) * ((p->N + 15) / 16) + UNITS - 1) / UNITS;
            double        us     = 6.5 + (double)nk * few_cost(p->M, tm, beside, wide);
            us                   = us < floor ? floor : us;
            if(us < best || (us == best && plan.kind == 2))
            {
                best = us;
                plan = {1, tm, 1, 0, 0, wide ? "block_product_few_f16" : "block_product_few"};
            }
        }
        return plan;
    }

    template <int BM, int BN, int WM, int WN, int ST, bool ROWS, bool WIDE>
    hipError_t launch_tile(PArgs a, uint32_t slices, hipStream_t stream)
    {
        typedef Tile<BM, BN, WM, WN, ST, ROWS, WIDE> T;
        auto                               kern = block_product_kernel<BM, BN, WM, WN, ST, ROWS, WIDE>;
        static const hipError_t            attr = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if(attr != hipSuccess)
            return attr;
        a.tiles_m = (a.M + BM - 1) / BM;
        a.tiles_n = (a.N + BN - 1) / BN;
        kern<<<dim3((uint32_t)a.tiles_m * (uint32_t)a.tiles_n, slices), dim3(64 * WM * WN), T::LDS, stream>>>(a);
        return hipGetLastError();
    }

    template <bool ROWS>
    hipError_t launch_choice(const PArgs& a, const Plan& plan, hipStream_t stream)
    {
        const uint32_t slices = (uint32_t)plan.slices;
        if(a.type == HIPTK_F32)
            switch(plan.tile)
            {
            case 0: return launch_tile<256, 128, 4, 2, 2, ROWS, true>(a, slices, stream);
            case 1: return launch_tile<128, 128, 2, 2, 2, ROWS, true>(a, slices, stream);
            default: return launch_tile<64, 64, 2, 2, 4, ROWS, true>(a, slices, stream);
            }
        switch(plan.tile)
        {
        case 0: return launch_tile<256, 256, 2, 4, 2, ROWS, false>(a, slices, stream);
        case 1: return launch_tile<256, 128, 4, 2, 3, ROWS, false>(a, slices, stream);
        case 2: return launch_tile<128, 128, 2, 2, 2, ROWS, false>(a, slices, stream);
        case 3: return launch_tile<64, 128, 2, 2, 3, ROWS, false>(a, slices, stream);
        default: return launch_tile<64, 64, 2, 2, 4, ROWS, false>(a, slices, stream);
        }
    }

    template <int TM, bool WIDE>
    hipError_t launch_few(const PArgs& a, hipStream_t stream)
    {
        const dim3 grid((uint32_t)((a.N + 15) / 16), (uint32_t)((a.M + 16 * TM - 1) / (16 * TM)));
        if(a.block_shift)
            block_product_few_kernel<TM, false, WIDE><<<grid, dim3(512), 0, stream>>>(a);
        else
            block_product_few_kernel<TM, true, WIDE><<<grid, dim3(512), 0, stream>>>(a);
        return hipGetLastError();
    }

    template <typename T>
    hipError_t launch_join(const PArgs& a, int slices, hipStream_t stream)
    {
        const int64_t threads = a.ld_partial / 4 * a.M;
        block_product_join_kernel<T><<<dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, stream>>>(a, slices);
        return hipGetLastError();
    }

    template <typename T>
    hipError_t launch_any(PArgs a, hipStream_t stream)
    {
        a.tiles_m = (a.M + 63) / 64;
        a.tiles_n = (a.N + 63) / 64;
        block_product_any_kernel<T><<<dim3((uint32_t)a.tiles_m * (uint32_t)a.tiles_n), dim3(256), 0, stream>>>(a);
        return hipGetLastError();
    }
}

extern "C" const char* hiptk_block_product_kernel_name(const hiptk_block_product_t* p)
{
    return well_formed(p) ? plan_of(p, MOST_WORKSPACE).name : "";
}

extern "C" uint64_t hiptk_block_product_workspace_bytes(const hiptk_block_product_t* p)
{
    if(!p || p->M <= 0 || p->N <= 0 || p->K <= 0)
        return 0;
    hiptk_block_product_t q = *p; // (as for operands on multiples of 16)
    q.A = q.B = nullptr;
    q.lda = q.ldb = 0;
    return plan_of(&q, MOST_WORKSPACE).bytes;
}

extern "C" int hiptk_block_product(const hiptk_block_product_t* p, void* workspace, uint64_t workspace_bytes, void* stream_, int* hip_error)
{
    if(hip_error)
        *hip_error = 0;
    if(!well_formed(p))
        return HIPTK_ERR_ARG;
    if(p->M == 0 || p->N == 0)
        return HIPTK_OK;
    if(((p->M + 63) / 64) * ((p->N + 63) / 64) > 0x7fffffff / 256)
        return HIPTK_ERR_ARG;
    PArgs a       = {};
    a.A           = (const uint8_t*)p->A;
    a.B           = (const uint8_t*)p->B;
    a.SA          = p->SA;
    a.SB          = p->SB;
    a.C           = p->C;
    a.D           = p->D;
    a.lda         = p->lda;
    a.ldb         = p->ldb;
    a.ldsa        = p->ldsa;
    a.ldsb        = p->ldsb;
    a.ldd         = p->ldd;
    a.M           = (int32_t)p->M;
    a.N           = (int32_t)p->N;
    a.K           = (int32_t)p->K;
    a.block_shift = p->block_rows == 128 ? 7 : 0;
    a.alpha       = p->alpha;
    a.beta        = p->beta;
    a.vec         = (((uintptr_t)p->A | (uintptr_t)p->B | (uint64_t)p->lda | (uint64_t)p->ldb) & 15) == 0;
    a.type        = p->type;
    const bool  usable = workspace && ((uintptr_t)workspace & 15) == 0;
    const Plan  plan   = plan_of(p, usable ? workspace_bytes : 0);
    hipStream_t stream = (hipStream_t)stream_;
    a.per_slice        = (int32_t)plan.per_slice;
    a.partial          = (float*)workspace;
    a.ld_partial       = (p->N + 3) / 4 * 4;
    hipError_t e;
    if(plan.kind == 0)
        e = p->type == HIPTK_F32 ? launch_any<float>(a, stream) : p->type == HIPTK_F16 ? launch_any<_Float16>(a, stream) : launch_any<__bf16>(a, stream);
    else if(plan.kind == 1)
    {
        if(p->type == HIPTK_F32)
            e = plan.tile == 1 ? launch_few<1, true>(a, stream) : launch_few<2, true>(a, stream);
        else
            e = plan.tile == 1 ? launch_few<1, false>(a, stream) : launch_few<2, false>(a, stream);
    }
    else
    {
        e = p->block_rows == 1 ? launch_choice<true>(a, plan, stream) : launch_choice<false>(a, plan, stream);
        if(e == hipSuccess && plan.slices > 1)
            e = p->type == HIPTK_F32   ? launch_join<float>(a, plan.slices, stream)
                : p->type == HIPTK_F16 ? launch_join<_Float16>(a, plan.slices, stream)
                                       : launch_join<__bf16>(a, plan.slices, stream);
    }
    if(hip_error)
        *hip_error = (int)e;
    return e == hipSuccess ? HIPTK_OK : HIPTK_ERR_LAUNCH;
}

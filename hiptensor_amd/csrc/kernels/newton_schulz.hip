// Newton-Schulz orthogonalisation (hiptk_orthogonalize):
//
//     X <- X / (|X|_F + epsilon);   `steps` times:  A = X X^T,  B = b A + c A A,  X <- a X + B X      (X: m x n, m <= n)
//
// What is held in which type, and why.  The products run on v_mfma_f32_16x16x32_f16 (f16 operands, f32 sums; bf16 operands
// would lose a factor of 8).  Two roundings would otherwise dominate the result:
//   * X itself.  A rounding of X is noise in all directions, and the iteration amplifies what lies in directions of small
//     singular values by up to a per step (485 over five steps).  X is therefore held as hi + lo, two f16 (22 bits): A is of hi, and
//     the term a X sees both.  So must B X, or none of it: in a direction of small singular value B is small as a whole, but its diagonal
//     part is not.  Where all of B X is of hi, what is missing (B lo) lies in directions of large singular values only, where nothing
//     amplifies it, and is four times the rounding of X there; where the diagonal's part sees lo and B' X does not, it is a third of that for
//     matrices whose A is near the identity, and diag(e) lo, noise in all directions, for those of few directions (rank 1: 5e-2 off at
//     2 x 2, 6e-3 at 64 x 64 after five steps).  A matrix of one workgroup multiplies lo too, which costs it little; on tiles, where lo in the product would
//     be half of the update again, the diagonal's part sees lo in the last two steps, behind which no noise grows by more than a.
//   * The diagonals of A and B.  Near the end A is close to the identity, and b A + c A A, a X + B X cancel to a
//     fraction of their terms.  A = diag(d) + A', B = diag(e) + B' with d, e in f32 and only A', B' rounded to f16:
//         A A = A' A' + (d_i + d_j) A'_ij + delta_ij d_i^2,      a X + B X = a X + e_i X + B' X,
//     elementwise terms that the epilogues of the products add in f32.
// On gaussian matrices the result is 5e-4 .. 1.1e-3 off (2-norm, five steps; 1e-3 .. 2e-3 with plain f16, 1e-2 with bf16), on low rank plus
// 1 % noise 3e-4 .. 1e-3 (4e-2 with plain f16, 0.3 with bf16): below the rounding of a bf16 result, 1.7e-3.
// X is held times 2^10, A' and B' times the power of two up to 2^10 that what a call's coefficients can make of them leaves (Scales): the default ones leave
// 2^10, entries stay below 64 and keep full precision down to 2^-24.
//
// A' and B' are symmetric: tiles above the diagonal are mirrored, not multiplied.  B' X contracts the rows of
// X_hi: its tiles go into LDS as they lie, row by row, and the reads from there transpose.  All dimensions are padded to multiples of 64 with zeros,
// which every step keeps zero.
#include <hip/hip_runtime.h>

#include <array>
#include <string>
#include <type_traits>

#include "dma_lds.hpp"
#include "hd_addr.hpp"
#include "hiptk_kernels.h"
#include "tile_walk.hpp"

namespace
{
    using hiptk::each;

    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typedef float    f4 __attribute__((ext_vector_type(4)));

    // the quintic whose slope at 0 is largest among those that keep [0, 1] within 0.7 .. 1.2 after a few steps (these numbers: K. Jordan et al.,
    // "Muon: An optimizer for hidden layers in neural networks", 2024)
    constexpr float DEFAULT_COEFFICIENTS[3] = {3.4445f, -4.7750f, 2.0315f};
    constexpr float UP = 1024.f, DOWN = 1.f / 1024.f;

    // What the f16 A' and B' of all steps are held times.  No entry of a matrix is larger than its largest singular value: with those of X up to `most`
    // (1 at first: X / |X|_F), A's are t = s^2 up to most^2, B's |b t + c t^2|, and those of the next X s |a + b t + c t^2|, largest at the end of
    // the range or where the derivative is zero.  (The iterates of a call's coefficients stay below MOST_X by the interface, which X's own scale needs,
    // whatever this bound for any matrix says.  One pair for all steps: read anew in each, it cost a 64 x 64 matrix 0.8 of 10.8 us.)
    struct Scales
    {
        float up_a, down_a, up_b, down_b;
    };
    constexpr double MOST_X = 16.0;
    Scales           scales_of(const float* coefficients, int steps)
    {
        if(!coefficients)
            return Scales{UP, DOWN, UP, DOWN}; // (from [0, 1.21] back into it, B up to 2.81)
        double most = 1.0, most_a = 0.0, most_b = 0.0;
        for(int s = 0; s < steps; s++)
        {
            const double a = coefficients[3 * s], b = coefficients[3 * s + 1], c = coefficients[3 * s + 2], end = most * most;
            double       peak_b = 0.0, peak_x = 0.0;
            auto         at     = [&](double t) { // (a t that is not a number is not in the range)
                if(t > 0.0 && t <= end)
                {
                    const double v = t * (b + c * t);
                    peak_b         = __builtin_fmax(peak_b, __builtin_fabs(v));
                    peak_x         = __builtin_fmax(peak_x, __builtin_sqrt(t) * __builtin_fabs(a + v));
                }
            };
            const double root = __builtin_sqrt(9.0 * b * b - 20.0 * a * c); // of a + 3 b t + 5 c t^2
            at(end);
            at(-b / (2.0 * c));
            at((-3.0 * b - root) / (10.0 * c));
            at((-3.0 * b + root) / (10.0 * c));
            at(-a / (3.0 * b)); // (c = 0)
            most_a = __builtin_fmax(most_a, end);
            most_b = __builtin_fmax(most_b, peak_b);
            most   = peak_x < MOST_X ? peak_x : MOST_X;
        }
        auto up = [](double peak) { // the largest power of two that keeps peak, and its roundings, within f16 (of a peak that is not finite the smallest)
            double u = UP;
            while(!(peak * u <= 60000.0) && u > 0x1p-100)
                u *= 0.5;
            return (float)u;
        };
        const float ua = up(most_a), ub = up(most_b);
        return Scales{ua, 1.f / ua, ub, 1.f / ub};
    }

    struct NsArgs
    {
        _Float16 *hi, *lo;     // X, [m][n]
        _Float16* hi_out;      // X_hi of the next step (its tiles are operands of other workgroups until the step ends)
        _Float16 *A, *B;       // A', B' [m][m]
        float *   d, *e;       // [m]
        double*   partial;     // [parts]
        float*    sums;        // [slice][tile of all matrices][4096], of a square in slices
        int32_t   slices;
        const void* X;
        void*       O;
        int64_t     ldx, stride_x, ldo, stride_o;
        int64_t     per; // bytes of workspace per matrix: all of the above of the next matrix lie that much further on
        int32_t     m, n; // padded
        int32_t     rows, cols; // of X
        int32_t     tall;       // rows > cols: X is read and O written transposed
        int32_t     parts, lanes_log; // of the norm
        int32_t     type_x, type_o;
        float       a, b, c, epsilon;
        Scales      scales;
        float       e_lo; // how much of X_lo the diagonal of B multiplies: 1 in the last two steps, 0 before
    };

    template <typename T>
    __device__ __forceinline__ T* of_matrix(T* p, const NsArgs& a, uint32_t z)
    {
        return (T*)((char*)p + (int64_t)z * a.per);
    }

    __device__ __forceinline__ float element(const void* base, int64_t at, int type)
    {
        return type == HIPTK_F32 ? ((const float*)base)[at] : type == HIPTK_F16 ? (float)((const _Float16*)base)[at] : (float)((const __bf16*)base)[at];
    }

    // (vector loads and stores at any element: global memory wants no alignment on this target)
    typedef float    any_f4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t any_u4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint16_t any_h4 __attribute__((ext_vector_type(4), aligned(2)));

    __device__ __forceinline__ float bits16(uint16_t b, int type)
    {
        return type == HIPTK_F16 ? (float)__builtin_bit_cast(_Float16, b) : __builtin_bit_cast(float, (uint32_t)b << 16);
    }

    // eight elements of a row of X from column c on, as f32; beyond the row zeros
    __device__ __forceinline__ void eight(const NsArgs& a, int64_t row_at, int c, float (&v)[8])
    {
        if(c + 8 <= a.cols)
        {
            if(a.type_x == HIPTK_F32)
            {
                const any_f4 x = *(const any_f4*)((const float*)a.X + row_at + c), y = *(const any_f4*)((const float*)a.X + row_at + c + 4);
#pragma unroll
                for(int h = 0; h < 4; h++)
                {
                    v[h]     = x[h];
                    v[h + 4] = y[h];
                }
            }
            else
            {
                const any_u4 x = *(const any_u4*)((const uint16_t*)a.X + row_at + c);
#pragma unroll
                for(int h = 0; h < 8; h++)
                    v[h] = bits16((uint16_t)(h & 1 ? x[h / 2] >> 16 : x[h / 2] & 0xffffu), a.type_x);
            }
        }
        else
        {
#pragma unroll
            for(int h = 0; h < 8; h++)
                v[h] = c + h < a.cols ? element(a.X, row_at + c + h, a.type_x) : 0.f;
        }
    }

    // sum over a workgroup of 256, in all of its threads
    __device__ __forceinline__ double sum_256(double s)
    {
        __shared__ double part[4];
#pragma unroll
        for(int o = 32; o; o >>= 1)
            s += __shfl_xor(s, o);
        if((threadIdx.x & 63) == 0)
            part[threadIdx.x >> 6] = s;
        __syncthreads();
        return part[0] + part[1] + part[2] + part[3];
    }

    // Sums of squares, in f64 (the square of an f32 or bf16 value may not be one), one per workgroup: block (part, matrix).  2^lanes_log
    // threads take a row, eight columns each at a time (no division: one per chunk, in 64 bits, was 6 of the 9 us of a 300 x 300 matrix).
    __global__ void __launch_bounds__(256) ns_norm_kernel(const NsArgs a)
    {
        const int64_t base = (int64_t)blockIdx.y * a.stride_x;
        const int     lanes = 1 << a.lanes_log, rows = 256 >> a.lanes_log;
        double        s    = 0.0;
        for(int r = (int)blockIdx.x * rows + ((int)threadIdx.x >> a.lanes_log); r < a.rows; r += a.parts * rows)
            for(int c = 8 * ((int)threadIdx.x & (lanes - 1)); c < a.cols; c += 8 * lanes)
            {
                float v[8];
                eight(a, base + (int64_t)r * a.ldx, c, v);
#pragma unroll
                for(int h = 0; h < 8; h++)
                    s = __builtin_fma((double)v[h], (double)v[h], s);
            }
        s = sum_256(s);
        if(threadIdx.x == 0)
            of_matrix(a.partial, a, blockIdx.y)[blockIdx.x] = s;
    }

    // hi and lo of the normalised matrix: one 64 x 64 tile (bound by memory: 8192 x 4096 bf16 34 us, 6 TB/s)
    __global__ void __launch_bounds__(256) ns_begin_kernel(const NsArgs a)
    {
        __shared__ float tile[64][65];
        const uint32_t   z  = blockIdx.z;
        const int        m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, t = threadIdx.x;
        const double*    p  = of_matrix(a.partial, a, z);
        double           s  = 0.0;
        for(int i = t; i < a.parts; i += 256)
            s += p[i];
        s = sum_256(s);
        const double     factor = (double)UP / (sqrt(s) + (double)a.epsilon); // (f64: a tiny norm's reciprocal may not be an f32)
#pragma unroll
        for(int i = 0; i < 2; i++)
        {
            const int r = i * 32 + t / 8, c = 8 * (t % 8); // along X's rows
            const int row = (a.tall ? n0 : m0) + r, col = (a.tall ? m0 : n0) + c;
            float     v[8] = {};
            if(row < a.rows && col < a.cols)
            {
                eight(a, (int64_t)z * a.stride_x + (int64_t)row * a.ldx, col, v);
#pragma unroll
                for(int h = 0; h < 8; h++)
                    v[h] = col + h < a.cols ? (float)((double)v[h] * factor) : 0.f;
            }
#pragma unroll
            for(int h = 0; h < 8; h++)
                (a.tall ? tile[c + h][r] : tile[r][c + h]) = v[h];
        }
        __syncthreads();
        _Float16 *hi = of_matrix(a.hi, a, z), *lo = of_matrix(a.lo, a, z);
#pragma unroll
        for(int i = 0; i < 2; i++)
        {
            const int r = i * 32 + t / 8, c = 8 * (t % 8);
            h8        h, l;
#pragma unroll
            for(int q = 0; q < 8; q++)
            {
                const float v = tile[r][c + q];
                h[q]          = (_Float16)v;
                l[q]          = (_Float16)(v - (float)h[q]);
            }
            *(h8*)&hi[(int64_t)(m0 + r) * a.n + n0 + c] = h;
            *(h8*)&lo[(int64_t)(m0 + r) * a.n + n0 + c] = l;
        }
    }

    enum
    {
        NS_SQUARE = 0, // A', d   from X X^T
        NS_MIX    = 1, // B', e   from A' A'
        NS_UPDATE = 2, // X       from B' X (rows: n, columns: m), X_hi read along n
        NS_LAST   = 3, // ... of the last step, to O
        // X X^T of few tiles and long n in slices of n: the sums of a slice, as they lie in the registers, and the square from all slices' sums
        NS_SLICE = 4,
        NS_JOIN  = 5
    };

    // Tile t of a triangle of `tiles` rows (row >= column): bands of four rows, column by column in a band, so that neighbours share panels.  The
    // bands before band g hold 8 g^2 + 2 g tiles.
    __device__ __forceinline__ void triangle(int t, int tiles, int& ti, int& tj)
    {
        int g = (int)((sqrtf(4.f + 32.f * (float)t) - 2.f) * 0.0625f);
        while(8 * (g + 1) * (g + 1) + 2 * (g + 1) <= t)
            g++;
        while(8 * g * g + 2 * g > t)
            g--;
        int       u    = t - (8 * g * g + 2 * g);
        const int rows = tiles - 4 * g < 4 ? tiles - 4 * g : 4, whole = rows * (4 * g + 1); // columns that all rows of the band have
        if(u < whole)
        {
            ti = 4 * g + u % rows;
            tj = u / rows;
            return;
        }
        u -= whole;
        int c = 1; // column 4 g + c has the rows 4 g + c and on
        while(u >= rows - c)
        {
            u -= rows - c;
            c++;
        }
        ti = 4 * g + c + u;
        tj = 4 * g + c;
    }

    // One product P Q^T of a step, BP x BQ outputs a workgroup on WP x WQ wavefronts, NI x NJ blocks of 16 x 16 each, k in stages of 64 through a ring
    // of ST in LDS (rows of 128 bytes; the 16-byte chunk at position c of a row holds chunk c ^ (row / 2) % 8).
    // 8192 x 4096: square 120 us on tiles of 192 (MFMAs 76 % of the busy cycles), mix 71, update 239 on tiles of 256 (63 %, and 670 MB that it
    // moves); 12 x 1024 x 1024 on tiles of 128: 21, 23 and 39 us (45, 40 and 36 %: LDS, and what a workgroup spends before and behind its
    // main loop).  A transposed copy of X beside X, for an update that reads along m, took it 267 and 43 us.
    template <int BP, int BQ, int WP, int WQ, int ST>
    struct Tile
    {
        static constexpr int WAVES = WP * WQ, NI = BP / WP / 16, NJ = BQ / WQ / 16;
        static constexpr int LP = BP / 8 / WAVES, LQ = BQ / 8 / WAVES, LOADS = LP + LQ; // loads of 8 rows per wavefront and stage
        static constexpr int STAGE = (BP + BQ) * 128;
        static constexpr int LDS   = ST * STAGE;
        static constexpr bool BIG  = NI * NJ >= 36; // sums in AGPRs, one wavefront per SIMD
        static_assert(BP % (8 * WAVES) == 0 && BQ % (8 * WAVES) == 0 && NI % 2 == 0 && NJ % 2 == 0 && ST >= 2 && LDS <= 160 * 1024, "");
        // Which pair of 16-byte chunks of row k of an operand that lies k by k is kept at position 0 (position x holds pair x ^ turned(k)): the four rows
        // that 16 lanes read 32 bytes of, and in rows of whole 256 bytes the eight of 32 lanes, touch disjoint banks
        static __device__ __forceinline__ int turned(int k) { return (k & 3) | (BP % 128 ? 0 : (k >> 1) & 4); }
        // what the results pass through: 16 rows of f32 and 32 of 16 bits, of W + 4 and W + 8
        static constexpr int W = NI * 16, PR = W + 4, PT = W + 8, PASS = 16 * PR * 4 + 32 * PT * 2;
        static_assert(WAVES * PASS <= LDS && PASS % 16 == 0, "");
    };

    // Which block of a wavefront's tile the b-th MFMA of a k-step multiplies: squares of 2 x 2, the squares row by row in alternating
    // directions, so that neighbours share an operand (the clock that the device holds depends on it)
    template <int NI, int NJ>
    constexpr int block_i(int b)
    {
        return 2 * ((b / 4) / (NJ / 2)) + (b % 4) / 2;
    }
    template <int NI, int NJ>
    constexpr int block_j(int b)
    {
        const int row = (b / 4) / (NJ / 2), col = (b / 4) % (NJ / 2), inner = b % 4;
        return 2 * (row % 2 ? NJ / 2 - 1 - col : col) + (inner == 1 || inner == 2);
    }

    template <int MODE, int BP, int BQ, int WP, int WQ, int ST>
    __global__ void __launch_bounds__(64 * WP * WQ, (Tile<BP, BQ, WP, WQ, ST>::BIG ? 1 : 2)) ns_product_kernel(const NsArgs a)
    {
        typedef Tile<BP, BQ, WP, WQ, ST> T;
        constexpr int  NI = T::NI, NJ = T::NJ;
        constexpr bool UPDATE = MODE == NS_UPDATE || MODE == NS_LAST, SQUARE = MODE == NS_SQUARE || MODE == NS_SLICE || MODE == NS_JOIN;
        extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
        typedef uint8_t __attribute__((address_space(3))) * lds_ptr;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;
        const int      tid = threadIdx.x, lane = tid & 63;
        const int      wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int      wp = wave % WP, wq = wave / WP;
        int            ti, tj;
        const uint32_t tiles_q = (uint32_t)((a.m + BQ - 1) / BQ), tiles_p = (uint32_t)((a.n + BP - 1) / BP);
        const uint32_t tiles = UPDATE ? tiles_p * tiles_q : tiles_q * (tiles_q + 1) / 2, place = hiptk::place_of(blockIdx.x, gridDim.x); // (the tiles of all matrices are one list, matrix after matrix)
        const uint32_t z = place / tiles;
        if(UPDATE)
            hiptk::tile_of(place - z * tiles, (int)tiles_p, (int)tiles_q, ti, tj);
        else
            triangle((int)(place - z * tiles), (int)tiles_q, ti, tj);
        const int rows_p = UPDATE ? a.n : a.m, K = SQUARE ? a.n : a.m;
        const int p0 = ti * BP, q0 = tj * BQ;
        const int first_k = MODE == NS_SLICE ? (int)blockIdx.y * ((K / 64 + a.slices - 1) / a.slices) * 64 : 0;
        // (in scalar registers from here on: the loads of the main loop carry no wait states, so nothing may move an address into them there)
        const uint8_t* pbase = (const uint8_t*)hiptk::hd_scalar(of_matrix(MODE == NS_MIX ? a.A : a.hi, a, z) + (UPDATE ? (int64_t)p0 : (int64_t)p0 * K + first_k));
        const int64_t  pstep = UPDATE ? (int64_t)a.n * 128 : 128; // bytes from a stage to the next
        const uint8_t* qbase = (const uint8_t*)hiptk::hd_scalar(of_matrix(SQUARE ? a.hi : MODE == NS_MIX ? a.A : a.B, a, z) + (int64_t)q0 * K + first_k);

        // what each lane loads (rows beyond the last read the last one; K is a multiple of 64)
        uint32_t  voff[T::LOADS];
        const int lrow = lane >> 3;
        each<T::LOADS>([&](auto l_c) __attribute__((always_inline)) {
            constexpr int  l    = decltype(l_c)::value;
            constexpr bool isp  = l < T::LP;
            if constexpr(UPDATE && isp)
            {
                const int at = (wave * T::LP + l) * 64 + lane, k = at / (BP / 8), col = 8 * ((at % (BP / 8)) ^ 2 * T::turned(k)), most = rows_p - 8 - p0;
                voff[l]      = (uint32_t)k * (uint32_t)(2 * a.n) + 2u * (uint32_t)(col < most ? col : most);
                return;
            }
            const int      row  = (isp ? wave * T::LP + l : wave * T::LQ + l - T::LP) * 8 + lrow;
            const int      most = isp ? rows_p - 1 - p0 : a.m - 1 - q0;
            voff[l]             = (uint32_t)(row < most ? row : most) * (uint32_t)(2 * K) + 16u * (uint32_t)hiptk::hk_chunk_pos(row, lane & 7);
        });
        auto load_part = [&](int t, int slot, auto l_c) __attribute__((always_inline)) {
            constexpr int  l   = decltype(l_c)::value;
            constexpr bool isp = l < T::LP;
            const int      q   = isp ? wave * T::LP + l : wave * T::LQ + l - T::LP;
            hiptk::dma_dst_at(lds0 + (uint32_t)slot * T::STAGE, (uint32_t)((isp ? 0 : BP * 128) + q * 1024));
            hiptk::dma_load(voff[l], isp ? pbase + t * pstep : qbase + (int64_t)t * 128);
        };
        // ... and its two halves, for either side of an MFMA (dma_lds.hpp)
        auto load_dst = [&](int slot, auto l_c) __attribute__((always_inline)) {
            constexpr int  l   = decltype(l_c)::value;
            constexpr bool isp = l < T::LP;
            const int      q   = isp ? wave * T::LP + l : wave * T::LQ + l - T::LP;
            hiptk::dma_dst_at(lds0 + (uint32_t)slot * T::STAGE, (uint32_t)((isp ? 0 : BP * 128) + q * 1024));
        };
        auto load_src = [&](int t, auto l_c) __attribute__((always_inline)) {
            constexpr int l = decltype(l_c)::value;
            hiptk::dma_load_in_loop(voff[l], l < T::LP ? pbase + t * pstep : qbase + (int64_t)t * 128);
        };

        // The elementwise terms of the epilogue: chunks of eight p of one q.
        constexpr int W = T::W, PR = T::PR, PT = T::PT, IT = (2 * W + 63) / 64; // chunks of eight p a lane takes of 16 rows
        float *       d = of_matrix(a.d, a, z), *e = of_matrix(a.e, a, z);
        const int     p = p0 + wp * W;
        _Float16 *    A_ = of_matrix(a.A, a, z), *hi = of_matrix(a.hi, a, z), *lo = of_matrix(a.lo, a, z);
        // (loads return in order with the stores issued between them: the terms of the epilogue are asked for DEEP column groups of 16 ahead, so that no load waits for a store
        // that has only just gone out, and what does not depend on the group once; with each group's terms loaded where they are used a
        // workgroup of 256 x 256 spent 23 us behind its main loop)
        constexpr int DEEP = NJ < 4 ? NJ : 4;
        h8            one[DEEP][IT], two[DEEP][IT];
        float         of_q[DEEP][IT];
        f4            dp[IT][2];
        // (rows of 16 q and, with W a multiple of 32 and the matrix of 64, runs of 32 p are inside or outside as a whole)
        auto chunk = [&](int it, int& r, int& c) __attribute__((always_inline)) {
            const int u = it * 64 + lane;
            r           = u / (W / 8);
            c           = 8 * (u % (W / 8));
            return (2 * W % 64 == 0 || u < 2 * W) && p + c < rows_p;
        };
        auto fetch_terms = [&](auto j_c) __attribute__((always_inline)) {
            constexpr int j = decltype(j_c)::value, s = j % DEEP;
            const int     qb = q0 + (wq * NJ + j) * 16;
            if(SQUARE || qb >= a.m)
                return;
#pragma unroll
            for(int it = 0; it < IT; it++)
            {
                int r, c;
                if(chunk(it, r, c))
                {
                    const int64_t at = (int64_t)(qb + r) * rows_p + p + c;
                    one[s][it]       = *(const h8*)((MODE == NS_MIX ? A_ : hi) + at); // (A' is symmetric)
                    if constexpr(UPDATE)
                        two[s][it] = *(const h8*)(lo + at);
                    of_q[s][it] = (MODE == NS_MIX ? d : e)[qb + r];
                }
            }
        };
        auto fetch_first = [&]() __attribute__((always_inline)) {
            if constexpr(MODE == NS_MIX)
            {
#pragma unroll
                for(int it = 0; it < IT; it++)
                {
                    int r, c;
                    if(chunk(it, r, c))
                    {
                        dp[it][0] = *(const f4*)&d[p + c];
                        dp[it][1] = *(const f4*)&d[p + c + 4];
                    }
                }
            }
            each<DEEP>([&](auto j_c) __attribute__((always_inline)) { fetch_terms(j_c); });
        };
        // ... the first of them before the main loop in small tiles, whose registers they fit
        constexpr bool EARLY = NI * NJ <= 4;
        if constexpr(EARLY)
            fetch_first();

        // Block (i, j): lane l holds rows p 4 (l / 16) .. + 3 of column q l % 16.  A stage is two k-steps of 32; the operands of k-step h of a
        // block of 16 rows: lane l holds row l % 16, chunk l / 16 + 4 h.
        f4 acc[NI][NJ];
        each<NI * NJ>([&](auto b_c) __attribute__((always_inline)) { acc[decltype(b_c)::value / NJ][decltype(b_c)::value % NJ] = f4{0.f, 0.f, 0.f, 0.f}; });
        const int frow = lane & 15;
        int       pat[2], qat[2];
#pragma unroll
        for(int h = 0; h < 2; h++)
        {
            if constexpr(!UPDATE)
                pat[h] = (wp * NI * 16 + frow) * 128 + 16 * hiptk::hk_chunk_pos(frow, (lane >> 4) + 4 * h);
            qat[h] = (BP + wq * NJ * 16 + frow) * 128 + 16 * hiptk::hk_chunk_pos(frow, (lane >> 4) + 4 * h);
        }
        // (P of the update lies k by k: lanes 4 r .. 4 r + 3 of 16 read 32 bytes of row r, of which the read hands each lane its p)
        int turned[NI];
        if constexpr(UPDATE)
        {
            const int k = 8 * (lane >> 4) + (frow >> 2);
#pragma unroll
            for(int i = 0; i < NI; i++)
                turned[i] = k * (2 * BP) + 32 * ((wp * NI + i) ^ T::turned(k)) + 8 * (frow & 3);
        }
        h8   fp[2][NI], fq[2][NJ];
        // operand block u of a k-step: P's, then Q's
        auto fetch = [&](const uint8_t* st, auto h_c, auto u_c) __attribute__((always_inline)) {
            constexpr int h = decltype(h_c)::value, u = decltype(u_c)::value;
            if constexpr(u < NI && UPDATE)
            {
                typedef short s4 __attribute__((ext_vector_type(4)));
                typedef s4 __attribute__((address_space(3))) * s4_ptr;
                typedef const uint8_t __attribute__((address_space(3))) * at_ptr;
                const at_ptr at = (at_ptr)st + turned[u];
                const uint2  x  = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_ptr)(at + h * (64 * BP))));
                const uint2  y  = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_ptr)(at + h * (64 * BP) + 8 * BP)));
                fp[h][u]        = __builtin_bit_cast(h8, uint4{x.x, x.y, y.x, y.y});
            }
            else if constexpr(u < NI)
                fp[h][u] = *(const h8*)(st + pat[h] + u * 2048);
            else
                fq[h][u - NI] = *(const h8*)(st + qat[h] + (u - NI) * 2048);
        };

        // While a k-step is multiplied the operands of the next one are read, evenly spread (a read of 1 KiB takes the LDS 8 cycles; those of all
        // wavefronts together take half of its time): in the first k-step of a stage those of its second, in the second
        // those of the next stage's first.  Between the two one barrier says both that stage t + 1 has landed and that all reads of stage t are done:
        // the loads of stage t + ST go into its slot under the second k-step.
        constexpr int NB = NI * NJ, NF = NI + NJ;
        static_assert(T::LOADS <= NB && NF <= NB, "");
        auto mfma = [&](f4& c, const h8& x, const h8& y) __attribute__((always_inline)) {
            if constexpr(T::BIG)
                asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(x), "v"(y));
            else
            {
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
                asm volatile("" : "+v"(c)); // (it stays where it is written, and in its registers)
            }
        };
        auto kstep = [&](auto h_c, const uint8_t* from, auto reads_c, int t, int slot, auto loads_c) __attribute__((always_inline)) {
            constexpr int  h     = decltype(h_c)::value;
            constexpr bool READS = decltype(reads_c)::value, LOADS = decltype(loads_c)::value;
            each<NB>([&](auto b_c) __attribute__((always_inline)) {
                constexpr int b = decltype(b_c)::value, i = block_i<NI, NJ>(b), j = block_j<NI, NJ>(b);
                constexpr int gap = NB / T::LOADS, l = b / gap; // this block's load, if any: LDS address in front of the MFMA, the load behind it
                if constexpr(READS)
                    each<NF>([&](auto u_c) __attribute__((always_inline)) {
                        // (done in the first three quarters: the wait in front of the barrier is for them too)
                        if constexpr(decltype(u_c)::value * (3 * NB / 4) / NF == b)
                            fetch(from, std::integral_constant<int, 1 - h>{}, u_c);
                    });
                if constexpr(LOADS && b % gap == 0 && l < T::LOADS)
                    load_dst(slot, std::integral_constant<int, l>{});
                mfma(acc[i][j], fp[h][i], fq[h][j]);
                if constexpr(LOADS && b % gap == 0 && l < T::LOADS)
                    load_src(t, std::integral_constant<int, l>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        typedef std::integral_constant<int, 0> First;
        typedef std::integral_constant<int, 1> Second;
        // (a slice takes the stages from `first` on)
        const int per = MODE == NS_SLICE ? (K / 64 + a.slices - 1) / a.slices : 0, first = MODE == NS_SLICE ? (int)blockIdx.y * per : 0;
        const int nk  = (int)hiptk::hd_scalar((uint32_t)(MODE != NS_SLICE || K / 64 - first < per ? K / 64 - first : per));
        int       slot = 0;
        auto      step = [&](int t, auto more_c, auto follows_c) __attribute__((always_inline)) {
            constexpr bool MORE = decltype(more_c)::value, FOLLOWS = decltype(follows_c)::value; // stages t + ST and t + 1 exist
            const int      next = slot == ST - 1 ? 0 : slot + 1;
            kstep(First{}, lds + slot * T::STAGE, std::true_type{}, 0, 0, std::false_type{});
            if constexpr(FOLLOWS)
            {
                __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_vm_lgkm0(MORE ? (ST - 2) * T::LOADS : 0));
                hiptk::lds_barrier();
            }
            kstep(Second{}, lds + next * T::STAGE, follows_c, t + ST, slot, more_c);
            slot = next;
        };
        // where a slice's sums of this tile lie: a wavefront's blocks one after the other, a lane's four sums together
        float* const sums = a.sums + ((int64_t)place * (BP * BQ) + wave * (NB * 256)) + 4 * lane;
        const int64_t slice_ld = (int64_t)gridDim.x * (BP * BQ);
        if constexpr(MODE == NS_JOIN)
        {
            for(int sl = 0; sl < a.slices; sl++)
                each<NB>([&](auto b_c) __attribute__((always_inline)) {
                    constexpr int b = decltype(b_c)::value;
                    acc[b / NJ][b % NJ] += *(const f4*)(sums + sl * slice_ld + b * 256);
                });
        }
        else
        {
            each<ST>([&](auto q_c) __attribute__((always_inline)) {
                constexpr int q = decltype(q_c)::value;
                if(q < nk)
                    each<T::LOADS>([&](auto l_c) __attribute__((always_inline)) { load_part(q, q, l_c); });
            });
            if(ST <= nk)
                __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_vm_lgkm0((ST - 1) * T::LOADS));
            else
                __builtin_amdgcn_s_waitcnt(hiptk::waitcnt_vm_lgkm0(0));
            hiptk::lds_barrier();
            each<NF>([&](auto u_c) __attribute__((always_inline)) { fetch(lds, First{}, u_c); });
            int t = 0;
            for(; t + ST < nk; t++)
                step(t, std::true_type{}, std::true_type{});
            for(; t + 1 < nk; t++)
                step(t, std::false_type{}, std::true_type{});
            step(t, std::false_type{}, std::false_type{});
        }
        if constexpr(MODE == NS_SLICE)
        {
            each<NB>([&](auto b_c) __attribute__((always_inline)) {
                constexpr int b = decltype(b_c)::value;
                *(f4*)(sums + blockIdx.y * slice_ld + b * 256) = acc[b / NJ][b % NJ];
            });
            return;
        }
        if constexpr(T::BIG)
            asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); // (the compiler does not know these for MFMAs: more wait states than any needs before its result may be read)

        // Results pass through LDS within the wavefront, so that everything outside is read and written in runs of 64 bytes or more (pieces
        // of 32 bytes, as the accumulators lie, cost twice the time: they were 40 us of 140 at 4096 x 4096).  16 columns q at a time
        // go through `rows` as f32 rows of W consecutive p; a lane then holds eight p of one q, reads the elementwise terms (a column group
        // ahead), and stores along p.  The other orientation (the mirrored half of a symmetric matrix, O of a tall X) is stored
        // every 32 q from `turn`, by transposing reads that hand a lane four consecutive q of one p.
        hiptk::lds_barrier(); // (every wavefront is done with the last stage)
        float*    rows = (float*)(lds + wave * T::PASS);
        uint16_t* turn = (uint16_t*)(lds + wave * T::PASS + 16 * PR * 4);
        if constexpr(!EARLY)
            fetch_first();
        // where rows q along p, and rows p along q, go
        uint16_t* along_p = (uint16_t*)(SQUARE ? A_ : of_matrix(MODE == NS_MIX ? a.B : a.hi_out, a, z));
        uint16_t* along_q = along_p;
        // the last step's to O, within its bounds
        if constexpr(MODE == NS_LAST)
            along_p = along_q = (uint16_t*)a.O + (int64_t)z * a.stride_o;
        const int64_t ld_p = MODE == NS_LAST ? a.ldo : rows_p, ld_q = MODE == NS_LAST ? a.ldo : a.m;
        const bool    do_p = MODE != NS_LAST || !a.tall, do_q = MODE == NS_LAST ? (bool)a.tall : !UPDATE && ti != tj;
        const int     end_p = MODE != NS_LAST ? rows_p : a.tall ? a.rows : a.cols, end_q = MODE != NS_LAST ? a.m : a.tall ? a.cols : a.rows;
        each<NJ>([&](auto j_c) __attribute__((always_inline)) {
            constexpr int j = decltype(j_c)::value, s = j % DEEP;
            const int     qb = q0 + (wq * NJ + j) * 16;
            if(qb < a.m)
            {
#pragma unroll
                for(int i = 0; i < NI; i++)
                    *(f4*)&rows[frow * PR + 16 * i + 4 * (lane >> 4)] = acc[i][j];
#pragma unroll
                for(int it = 0; it < IT; it++)
                {
                    int r, c;
                    if(!chunk(it, r, c))
                        continue;
                    const int q = qb + r, pc = p + c;
                    float     v[8];
                    *(f4*)&v[0] = *(const f4*)&rows[r * PR + c];
                    *(f4*)&v[4] = *(const f4*)&rows[r * PR + c + 4];
                    uint16_t bits[8];
                    if constexpr(!UPDATE)
                    {
                        const float    down_a = a.scales.down_a, up = SQUARE ? a.scales.up_a : a.scales.up_b;
                        const float    dq   = MODE == NS_MIX ? of_q[s][it] : 0.f;
                        const uint32_t diag = (uint32_t)(q - pc); // the chunk's element on the diagonal, if less than 8
#pragma unroll
                        for(int h = 0; h < 8; h++)
                        {
                            v[h] *= SQUARE ? DOWN * DOWN : down_a * down_a;
                            if constexpr(MODE == NS_MIX)
                            {
                                // (on the diagonal A' is zero, and d_i^2 is added to A A, d_i to A below)
                                const float off = (float)one[s][it][h] * down_a;
                                v[h]            = a.b * off + a.c * (v[h] + (dp[it][h / 4][h % 4] + dq) * off);
                            }
                        }
                        if(diag < 8)
                        {
                            float x = 0.f;
#pragma unroll
                            for(int h = 0; h < 8; h++)
                                if(diag == (uint32_t)h)
                                {
                                    x    = v[h];
                                    v[h] = 0.f;
                                }
                            (SQUARE ? d : e)[q] = SQUARE ? x : x + a.b * dq + a.c * dq * dq;
                        }
#pragma unroll
                        for(int h = 0; h < 8; h++)
                            bits[h] = __builtin_bit_cast(uint16_t, (_Float16)(v[h] * up));
                    }
                    else
                    {
                        const float f = a.a + of_q[s][it], g = a.a + a.e_lo * of_q[s][it];
#pragma unroll
                        for(int h = 0; h < 8; h++)
                            v[h] = f * (float)one[s][it][h] + (g * (float)two[s][it][h] + v[h] * a.scales.down_b);
                        if constexpr(MODE == NS_UPDATE)
                        {
                            h8 low;
#pragma unroll
                            for(int h = 0; h < 8; h++)
                            {
                                const _Float16 top = (_Float16)v[h];
                                bits[h]            = __builtin_bit_cast(uint16_t, top);
                                low[h]             = (_Float16)(v[h] - (float)top);
                            }
                            *(h8*)(lo + (int64_t)q * rows_p + pc) = low;
                        }
                        else
                        {
#pragma unroll
                            for(int h = 0; h < 8; h++)
                            {
                                const float x = v[h] * DOWN;
                                bits[h]       = a.type_o == HIPTK_F16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : __builtin_bit_cast(uint16_t, (__bf16)x);
                            }
                        }
                    }
                    const uint4 out = {bits[0] | (uint32_t)bits[1] << 16, bits[2] | (uint32_t)bits[3] << 16, bits[4] | (uint32_t)bits[5] << 16,
                                       bits[6] | (uint32_t)bits[7] << 16};
                    uint16_t* const here = &turn[((j & 1) * 16 + r) * PT + c];
                    if(do_q || MODE == NS_LAST)
                        *(uint4*)here = out;
                    if(do_p)
                    {
                        uint16_t* at = along_p + (int64_t)q * ld_p + pc;
                        if(MODE != NS_LAST)
                            *(uint4*)at = out;
                        else if(q < end_q && pc + 8 <= end_p)
                            *(any_u4*)at = any_u4{out.x, out.y, out.z, out.w};
                        else if(q < end_q)
                        {
#pragma unroll 1
                            for(int h = 0; h < 8 && pc + h < end_p; h++)
                                at[h] = here[h];
                        }
                    }
                }
            }
            if constexpr(j + DEEP < NJ)
                fetch_terms(std::integral_constant<int, j + DEEP>{});
            if constexpr(j & 1)
                if(do_q && qb - 16 < a.m)
                {
                    typedef short s4 __attribute__((ext_vector_type(4)));
                    typedef s4 __attribute__((address_space(3))) * s4_ptr;
                    typedef uint16_t __attribute__((address_space(3))) * u16_ptr;
                    const u16_ptr t0 = (u16_ptr)turn + (8 * (lane >> 4) + (frow >> 2)) * PT + 4 * (frow & 3);
                    const int     col = qb - 16 + 8 * (lane >> 4); // (the matrix is a multiple of 64: 32 q are inside or outside as a whole)
#pragma unroll
                    for(int i = 0; i < NI; i++)
                    {
                        if(p + 16 * i >= rows_p)
                            break;
                        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_ptr)(t0 + 16 * i)));
                        const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_ptr)(t0 + 4 * PT + 16 * i)));
                        const int   row = p + 16 * i + frow;
                        uint16_t*   at = along_q + (int64_t)row * ld_q + col;
                        if(MODE != NS_LAST)
                            *(uint4*)at = uint4{x.x, x.y, y.x, y.y};
                        else if(row < end_p && col + 8 <= end_q)
                            *(any_u4*)at = any_u4{x.x, x.y, y.x, y.y};
                        else if(row < end_p)
                        {
#pragma unroll 1
                            for(int r = 0; r < 8 && col + r < end_q; r++)
                                at[r] = turn[(8 * (lane >> 4) + r) * PT + 16 * i + frow];
                        }
                    }
                }
        });
    }

    // ---- matrices that one compute unit holds --------------------------------------------------------------------------

    // The whole iteration of one matrix (padded to MP x NP) in one workgroup of eight wavefronts: X_hi, X_lo and A' (then B') in LDS, X in f32 in the registers
    // of the lanes that update it, so that there is one launch instead of three a step (64 x 256: 65 us in 17 launches,
    // 21 us so, 300 of them 36 us; most of it is the latency of LDS and barriers).  X_hi is read along n for X X^T and, by transposing reads, along m for
    // B X, as X_lo is.
    struct Coefficients
    {
        static constexpr int MOST = 16; // steps
        float                abc[3 * MOST];
    };

    template <int MP, int NP>
    struct Small
    {
        static constexpr int WAVES = 8, MB = MP / 16, NBL = NP / 16;
        static constexpr int PX = NP + 8, PA = MP + 8;           // rows of X_hi and of A', in f16
        static constexpr int SQ = MB * MB / WAVES;               // blocks of A a wavefront: SI rows' blocks by SJ
        static constexpr int SJ = SQ < 4 ? SQ : 4, SI = SQ / SJ; // (MB 4: 1 x 2; MB 8: 2 x 4)
        static constexpr int XB = MB * NBL / WAVES;             // blocks of X a wavefront: UI along n by UJ along m
        static constexpr int UJ = XB < MB ? XB : MB, UI = XB / UJ;
        static constexpr int  LEAST  = 2 * (MP * PX + MP * PA) + 4 * 2 * MP + 64;
        static constexpr bool BESIDE = LEAST + 2 * MP * PX <= 160 * 1024; // X_lo has a place of its own (else X_hi's, when that has been read)
        static constexpr int  LDS    = LEAST + (BESIDE ? 2 * MP * PX : 0);
        static_assert(MB * MB % WAVES == 0 && UI * UJ * WAVES == MB * NBL && MB % UJ == 0 && LDS <= 160 * 1024, "");
    };

    template <int MP, int NP>
    __global__ void __launch_bounds__(512) ns_small_kernel(const NsArgs a, const Coefficients coefficients, int steps)
    {
        typedef Small<MP, NP> T;
        constexpr int PX = T::PX, PA = T::PA, SI = T::SI, SJ = T::SJ, UI = T::UI, UJ = T::UJ;
        extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
        _Float16 *      X = (_Float16*)lds, *lower = T::BESIDE ? X + MP * PX : X, *A = lower + MP * PX;
        float *         d = (float*)(A + MP * PA), *e = d + MP;
        double*         part = (double*)(e + MP);
        const int       tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, g = lane >> 4;
        const uint32_t  z = blockIdx.x;
        // this wavefront's blocks: of A and B rows si .. and columns sj .. ; of X columns ui .. (along n) and rows uj .. (along m)
        const int si = wave / (T::MB / SJ) * SI, sj = wave % (T::MB / SJ) * SJ;
        const int ui = wave / (T::MB / UJ) * UI, uj = wave % (T::MB / UJ) * UJ;

        // X: block (i, j): lane l holds four n of row m l % 16
        f4     x[UI][UJ];
        double s = 0.0;
#pragma unroll
        for(int i = 0; i < UI; i++)
#pragma unroll
            for(int j = 0; j < UJ; j++)
            {
                const int     m = 16 * (uj + j) + fr, n = 16 * (ui + i) + 4 * g;
                const int64_t at = (int64_t)z * a.stride_x + (a.tall ? (int64_t)n * a.ldx + m : (int64_t)m * a.ldx + n);
                if(!a.tall && m < a.rows && n + 4 <= a.cols)
                {
                    if(a.type_x == HIPTK_F32)
                        x[i][j] = *(const any_f4*)((const float*)a.X + at);
                    else
                    {
                        const any_h4 h = *(const any_h4*)((const uint16_t*)a.X + at);
#pragma unroll
                        for(int r = 0; r < 4; r++)
                            x[i][j][r] = bits16(h[r], a.type_x);
                    }
                }
                else
                {
#pragma unroll
                    for(int r = 0; r < 4; r++)
                    {
                        const bool in = a.tall ? n + r < a.rows && m < a.cols : m < a.rows && n + r < a.cols;
                        x[i][j][r]    = in ? element(a.X, at + (a.tall ? (int64_t)r * a.ldx : r), a.type_x) : 0.f;
                    }
                }
#pragma unroll
                for(int r = 0; r < 4; r++)
                    s = __builtin_fma((double)x[i][j][r], (double)x[i][j][r], s);
            }
#pragma unroll
        for(int o = 32; o; o >>= 1)
            s += __shfl_xor(s, o);
        if(lane == 0)
            part[wave] = s;
        __syncthreads();
        s = 0.0;
#pragma unroll
        for(int w = 0; w < T::WAVES; w++)
            s += part[w];
        const double factor = (double)UP / (sqrt(s) + (double)a.epsilon);
        auto low_of = [&](const f4& v) __attribute__((always_inline)) {
            h4 h;
#pragma unroll
            for(int r = 0; r < 4; r++)
                h[r] = (_Float16)(v[r] - (float)(_Float16)v[r]);
            return h;
        };
        auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
            for(int i = 0; i < UI; i++)
#pragma unroll
                for(int j = 0; j < UJ; j++)
                {
                    const int at = (16 * (uj + j) + fr) * PX + 16 * (ui + i) + 4 * g;
                    h4        h;
#pragma unroll
                    for(int r = 0; r < 4; r++)
                        h[r] = (_Float16)x[i][j][r];
                    *(h4*)&X[at] = h;
                    if constexpr(T::BESIDE)
                        *(h4*)&lower[at] = low_of(x[i][j]);
                }
        };
#pragma unroll
        for(int i = 0; i < UI; i++)
#pragma unroll
            for(int j = 0; j < UJ; j++)
            {
#pragma unroll
                for(int r = 0; r < 4; r++)
                    x[i][j][r] = (float)((double)x[i][j][r] * factor); // (the padding's zeros too: a factor that is not finite makes the matrix NaN as it is)
                // (X_hi is of this f32, as X_lo is: left to itself the compiler rounds the f64 product to X_hi in one step, which is
                // another f16 where the f32 lies halfway between two, and X_hi + X_lo would not be X there)
                asm volatile("" : "+v"(x[i][j]));
            }
        put();
        __syncthreads();

        for(int step = 0; step < steps; step++)
        {
            const float ca = coefficients.abc[3 * step], cb = coefficients.abc[3 * step + 1], cc = coefficients.abc[3 * step + 2];
            // A = X X^T
            f4 acc[SI][SJ];
#pragma unroll
            for(int i = 0; i < SI; i++)
#pragma unroll
                for(int j = 0; j < SJ; j++)
                    acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for(int k = 0; k < NP; k += 32)
            {
                h8 fp[SI], fq[SJ];
#pragma unroll
                for(int i = 0; i < SI; i++)
                    fp[i] = *(const h8*)&X[(16 * (si + i) + fr) * PX + k + 8 * g];
#pragma unroll
                for(int j = 0; j < SJ; j++)
                    fq[j] = *(const h8*)&X[(16 * (sj + j) + fr) * PX + k + 8 * g];
#pragma unroll
                for(int i = 0; i < SI; i++)
#pragma unroll
                    for(int j = 0; j < SJ; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[i], fq[j], acc[i][j], 0, 0, 0);
            }
            h4 mine[SI][SJ]; // this lane's elements of A'
#pragma unroll
            for(int i = 0; i < SI; i++)
#pragma unroll
                for(int j = 0; j < SJ; j++)
                {
                    const int p = 16 * (si + i) + 4 * g, q = 16 * (sj + j) + fr;
#pragma unroll
                    for(int r = 0; r < 4; r++)
                    {
                        float v = acc[i][j][r] * (DOWN * DOWN);
                        if(p + r == q)
                        {
                            d[q] = v;
                            v    = 0.f;
                        }
                        mine[i][j][r] = (_Float16)(v * a.scales.up_a);
                    }
                    *(h4*)&A[q * PA + p] = mine[i][j]; // (symmetric)
                }
            __syncthreads();
            // B = b A + c A A
#pragma unroll
            for(int i = 0; i < SI; i++)
#pragma unroll
                for(int j = 0; j < SJ; j++)
                    acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for(int k = 0; k < MP; k += 32)
            {
                h8 fp[SI], fq[SJ];
#pragma unroll
                for(int i = 0; i < SI; i++)
                    fp[i] = *(const h8*)&A[(16 * (si + i) + fr) * PA + k + 8 * g];
#pragma unroll
                for(int j = 0; j < SJ; j++)
                    fq[j] = *(const h8*)&A[(16 * (sj + j) + fr) * PA + k + 8 * g];
#pragma unroll
                for(int i = 0; i < SI; i++)
#pragma unroll
                    for(int j = 0; j < SJ; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[i], fq[j], acc[i][j], 0, 0, 0);
            }
            __syncthreads(); // (A' has been read: B' takes its place)
#pragma unroll
            for(int i = 0; i < SI; i++)
#pragma unroll
                for(int j = 0; j < SJ; j++)
                {
                    const int p = 16 * (si + i) + 4 * g, q = 16 * (sj + j) + fr;
                    const f4  dp = *(const f4*)&d[p];
                    const float dq = d[q];
                    h4        out;
#pragma unroll
                    for(int r = 0; r < 4; r++)
                    {
                        const float off = (float)mine[i][j][r] * a.scales.down_a;
                        float       v = cb * off + cc * (acc[i][j][r] * (a.scales.down_a * a.scales.down_a) + (dp[r] + dq) * off);
                        if(p + r == q)
                        {
                            e[q] = v + cb * dq + cc * dq * dq;
                            v    = 0.f;
                        }
                        out[r] = (_Float16)(v * a.scales.up_b);
                    }
                    *(h4*)&A[q * PA + p] = out;
                }
            __syncthreads();
            // X <- a X + B X
            // (in place: (a + e) X scaled as the products are, and back)
            h4 low[T::BESIDE ? 1 : UI][T::BESIDE ? 1 : UJ];
#pragma unroll
            for(int j = 0; j < UJ; j++)
            {
                const float f = (ca + e[16 * (uj + j) + fr]) * a.scales.up_b;
#pragma unroll
                for(int i = 0; i < UI; i++)
                {
                    if constexpr(!T::BESIDE)
                        low[i][j] = low_of(x[i][j]);
                    x[i][j] *= f;
                }
            }
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef s4 __attribute__((address_space(3))) * s4_ptr;
            typedef _Float16 __attribute__((address_space(3))) * h_ptr;
            auto turned = [&](const _Float16* from, int k, int i) __attribute__((always_inline)) {
                const h_ptr at = (h_ptr)from + (k + 8 * g + (fr >> 2)) * PX + 16 * (ui + i) + 4 * (fr & 3);
                const uint2 u = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_ptr)at));
                const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_ptr)(at + 4 * PX)));
                return __builtin_bit_cast(h8, uint4{u.x, u.y, v.x, v.y});
            };
            auto product = [&](auto both_c) __attribute__((always_inline)) { // B' X_hi, or B' (X_hi + X_lo)
                constexpr bool BOTH = decltype(both_c)::value;
#pragma unroll 2
                for(int k = 0; k < MP; k += 32)
                {
                    h8 fp[UI], fl[UI], fq[UJ];
#pragma unroll
                    for(int i = 0; i < UI; i++)
                    {
                        fp[i] = turned(X, k, i);
                        if constexpr(BOTH)
                            fl[i] = turned(lower, k, i);
                    }
#pragma unroll
                    for(int j = 0; j < UJ; j++)
                        fq[j] = *(const h8*)&A[(16 * (uj + j) + fr) * PA + k + 8 * g];
#pragma unroll
                    for(int i = 0; i < UI; i++)
#pragma unroll
                        for(int j = 0; j < UJ; j++)
                            x[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[i], fq[j], x[i][j], 0, 0, 0);
                    if constexpr(BOTH)
                    {
#pragma unroll
                        for(int i = 0; i < UI; i++)
#pragma unroll
                            for(int j = 0; j < UJ; j++)
                                x[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[i], fq[j], x[i][j], 0, 0, 0);
                    }
                }
            };
            if constexpr(T::BESIDE)
                product(std::true_type{});
            else
            {
                // (a wavefront holds all of m here: the columns of X_hi that it reads are its own, and LDS serves a wavefront in order)
                static_assert(UJ == T::MB, "");
                auto in_order = [&]() __attribute__((always_inline)) {
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                };
                product(std::false_type{});
                in_order();
#pragma unroll
                for(int i = 0; i < UI; i++)
#pragma unroll
                    for(int j = 0; j < UJ; j++)
                        *(h4*)&X[(16 * (uj + j) + fr) * PX + 16 * (ui + i) + 4 * g] = low[i][j];
                in_order();
                product(std::false_type{});
            }
#pragma unroll
            for(int i = 0; i < UI; i++)
#pragma unroll
                for(int j = 0; j < UJ; j++)
                    x[i][j] *= a.scales.down_b;
            __syncthreads(); // (X_hi, X_lo, B' and e have been read)
            if(step + 1 < steps)
            {
                put();
                __syncthreads();
            }
        }
        int last_fr = fr, last_g = g;
        asm volatile("" : "+v"(last_fr), "+v"(last_g)); // (what O's addresses share with X's is not kept in registers through the steps)
#pragma unroll
        for(int i = 0; i < UI; i++)
#pragma unroll
            for(int j = 0; j < UJ; j++)
            {
                const int     m = 16 * (uj + j) + last_fr, n = 16 * (ui + i) + 4 * last_g;
                const int64_t at = (int64_t)z * a.stride_o + (a.tall ? (int64_t)n * a.ldo + m : (int64_t)m * a.ldo + n);
                any_h4        h;
#pragma unroll
                for(int r = 0; r < 4; r++)
                {
                    const float v = x[i][j][r] * DOWN;
                    h[r]          = a.type_o == HIPTK_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v);
                }
                if(!a.tall && m < a.rows && n + 4 <= a.cols)
                    *(any_h4*)((uint16_t*)a.O + at) = h;
                else
                {
#pragma unroll
                    for(int r = 0; r < 4; r++)
                        if(a.tall ? n + r < a.rows && m < a.cols : m < a.rows && n + r < a.cols)
                            ((uint16_t*)a.O)[at + (a.tall ? (int64_t)r * a.ldo : r)] = h[r];
                }
            }
    }

    template <int MODE, int BP, int BQ, int WP, int WQ, int ST>
    hipError_t launch_tile(const NsArgs& a, uint32_t batch, hipStream_t stream)
    {
        typedef Tile<BP, BQ, WP, WQ, ST> T;
        auto                             kern = ns_product_kernel<MODE, BP, BQ, WP, WQ, ST>;
        static const hipError_t          attr = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if(attr != hipSuccess)
            return attr;
        const uint32_t tm = (uint32_t)((a.m + BQ - 1) / BQ), tn = (uint32_t)((a.n + BP - 1) / BP);
        kern<<<dim3((MODE == NS_UPDATE || MODE == NS_LAST ? tm * tn : tm * (tm + 1) / 2) * batch, MODE == NS_SLICE ? (uint32_t)a.slices : 1), dim3(64 * WP * WQ), T::LDS, stream>>>(a);
        return hipGetLastError();
    }

    // A tile, its ring of stages, how many of its workgroups a compute unit holds, what a stage of 64 k costs a unit that holds one of them and one
    // that holds all (us), and what a workgroup spends before and behind its main loop, for the square, the mix and the update.
    struct Choice
    {
        int   edge, stages, slots;
        float one, all, around[3];
    };
    // (Tiles of 64 with two stages wait for their loads where a unit holds one: 1000 x 2731 257 us with them in the products of m x m, 189 with
    // four.  With two or three a unit they do without a second round of few tiles: 2048 x 2048 359 us with four stages, 344 so.  With more
    // the units' loads no longer meet in the L2s: 3000 x 4500 1108 us against 907 on larger tiles, so they are taken up to three a unit.)
    constexpr Choice CHOICES[] = {{256, 2, 1, 1.15f, 1.45f, {13.f, 18.f, 20.f}},
                                  {192, 3, 1, 0.92f, 0.93f, {10.f, 13.f, 15.f}},
                                  {128, 2, 2, 0.54f, 0.88f, {6.f, 7.f, 8.f}},
                                  {64, 4, 2, 0.18f, 0.35f, {3.5f, 4.f, 4.5f}},
                                  {64, 2, 3, 0.42f, 0.50f, {3.5f, 4.f, 4.5f}}};
    constexpr int     TILES     = sizeof(CHOICES) / sizeof(CHOICES[0]);
    constexpr int64_t UNITS     = 256;
    constexpr int     ONE_ROUND = 4; // (of the choices: the last)

    // us of `work` workgroups of a tile, `steps` stages each: rounds that fill the units, and one of what is left
    double rounds(const Choice& c, int mode, int64_t work, int64_t steps)
    {
        const int64_t full = work / (UNITS * c.slots), left = work - full * UNITS * c.slots, beside = (left + UNITS - 1) / UNITS;
        double        stage = (double)beside * c.all / c.slots;
        if(c.slots == 1 && 2 * left <= UNITS) // (the clock is higher with half of the units at rest)
            stage = 0.0;
        if(stage < c.one)
            stage = c.one;
        return (double)full * (c.around[mode] + steps * c.all) + (left ? c.around[mode] + steps * stage : 0.0);
    }

    // The tile whose rounds over the compute units cost least: large ones load least for what they multiply (64 bytes a cycle arrive in a unit;
    // 256 x 256 takes 1024 cycles of them for 2048 of MFMAs, 64 x 64 256 for 128), small ones fill the device and end soon.
    int choice_of(int mode, int64_t m, int64_t n, int64_t batch, double* us = nullptr)
    {
        int    best  = 0;
        double least = 1e30;
        for(int i = 0; i < TILES; i++)
        {
            const Choice& c = CHOICES[i];
            const int64_t tm = (m + c.edge - 1) / c.edge, tn = (n + c.edge - 1) / c.edge;
            const int64_t work = batch * (mode == NS_UPDATE ? tm * tn : tm * (tm + 1) / 2);
            const double  t    = rounds(c, mode, work, (mode == NS_SQUARE ? n : m) / 64);
            if(t < least && (i != ONE_ROUND || work <= UNITS * c.slots))
            {
                least = t;
                best  = i;
            }
        }
        if(us)
            *us = least;
        return best;
    }

    // How many slices of n the square is cut into (1: none), where its tiles are few and n is long: tiles of 64, a second launch that adds the slices up
    // (4 x 40 x 6047, one tile a matrix and 95 stages: a call of five steps takes 143 us, in slices 104; 500 x 8000 226
    // and 178).
    constexpr int64_t MOST_SUMS = 16 << 20;
    int64_t slices_of(int64_t m, int64_t n, int64_t batch)
    {
        double least = 0.0;
        (void)choice_of(NS_SQUARE, m, n, batch, &least);
        const int64_t tm = m / 64, tiles = batch * (tm * (tm + 1) / 2), steps = n / 64;
        int64_t       best = 1;
        for(int64_t want = 2; want <= 16; want *= 2)
        {
            const int64_t per = (steps + want - 1) / want, slices = (steps + per - 1) / per; // (no slice is empty)
            if(per < 4 || slices * tiles * 4096 * 4 > MOST_SUMS)
                break;
            const double us = rounds(CHOICES[3], NS_SQUARE, tiles * slices, per) + 4.0 + 0.15 * (double)slices;
            if(us < least)
            {
                least = us;
                best  = slices;
            }
        }
        return best;
    }

    template <int MODE>
    hipError_t launch(const NsArgs& a, int choice, uint32_t batch, hipStream_t stream)
    {
        switch(choice)
        {
        case 0: return launch_tile<MODE, 256, 256, 2, 2, CHOICES[0].stages>(a, batch, stream);
        case 1: return launch_tile<MODE, 192, 192, 2, 2, CHOICES[1].stages>(a, batch, stream);
        case 2: return launch_tile<MODE, 128, 128, 2, 2, CHOICES[2].stages>(a, batch, stream);
        case 3: return launch_tile<MODE, 64, 64, 2, 2, CHOICES[3].stages>(a, batch, stream);
        default: return launch_tile<MODE, 64, 64, 2, 2, CHOICES[4].stages>(a, batch, stream);
        }
    }

    struct Layout
    {
        int64_t m, n, parts, lanes_log;
        int64_t hi, next, lo, A, B, d, e, partial, per; // byte offsets
        int64_t slices, sums; // of the square: their number, and the bytes of their sums behind all matrices
    };

    Layout layout_of(const hiptk_orthogonalize_t* p)
    {
        Layout        l;
        const int64_t s = p->rows < p->cols ? p->rows : p->cols, t = p->rows < p->cols ? p->cols : p->rows;
        l.m             = (s + 63) / 64 * 64;
        l.n             = (t + 63) / 64 * 64;
        // the norm: a row of X to as many threads as it has eights of columns (a power of two, 256 at most), and a partial sum of squares for every
        // 4 Ki elements, 1024 at most (the next kernel's workgroups add them up, four a thread; 256 left 8192 x 4096 at 1.4 TB/s)
        for(l.lanes_log = 0; l.lanes_log < 8 && (8 << l.lanes_log) < p->cols; l.lanes_log++)
            ;
        l.parts = (s * t + 4095) / 4096;
        l.parts = l.parts > 1024 ? 1024 : l.parts;
        int64_t at = 0;
        auto    take = [&](int64_t bytes) {
            const int64_t here = at;
            at += (bytes + 255) / 256 * 256;
            return here;
        };
        l.hi      = take(2 * l.m * l.n);
        l.lo      = take(2 * l.m * l.n);
        l.next    = take(2 * l.m * l.n);
        l.A       = take(2 * l.m * l.m);
        l.B       = take(2 * l.m * l.m);
        l.d       = take(4 * l.m);
        l.e       = take(4 * l.m);
        l.partial = take(8 * l.parts);
        l.per     = at;
        l.slices  = slices_of(l.m, l.n, p->batch);
        l.sums    = l.slices == 1 ? 0 : l.slices * p->batch * (l.m / 64 * (l.m / 64 + 1) / 2) * 4096 * 4;
        return l;
    }

    template <int MP, int NP>
    hipError_t launch_small(const NsArgs& a, const Coefficients& c, int steps, uint32_t batch, hipStream_t stream)
    {
        auto                    kern = ns_small_kernel<MP, NP>;
        static const hipError_t attr = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, Small<MP, NP>::LDS);
        if(attr != hipSuccess)
            return attr;
        kern<<<dim3(batch), dim3(512), Small<MP, NP>::LDS, stream>>>(a, c, steps);
        return hipGetLastError();
    }

    // Whether one compute unit holds a matrix: 64 x 512 or 128 x 256 after padding, and the coefficients fit a launch
    bool is_small(const hiptk_orthogonalize_t* p)
    {
        const int64_t s = p->rows < p->cols ? p->rows : p->cols, t = p->rows < p->cols ? p->cols : p->rows;
        return p->steps <= Coefficients::MOST && ((s <= 64 && t <= 512) || (s <= 128 && t <= 256));
    }

    bool well_formed(const hiptk_orthogonalize_t* p)
    {
        if(!p || p->batch < 0 || p->rows < 0 || p->cols < 0 || p->steps < 1)
            return false;
        // (tiles of the grids: 65535 in y and z)
        if(p->batch > 65535 || p->rows > (1 << 20) || p->cols > (1 << 20) || (p->rows < p->cols ? p->rows : p->cols) > (1 << 16))
            return false;
        if((p->type_x != HIPTK_F16 && p->type_x != HIPTK_BF16 && p->type_x != HIPTK_F32) || (p->type_o != HIPTK_F16 && p->type_o != HIPTK_BF16))
            return false;
        return true;
    }
}

// newton_schulz_products and the tiles of square (or "sliced"), mix and update; "64r2" is the tile of 64 with two stages
extern "C" const char* hiptk_orthogonalize_kernel_name(const hiptk_orthogonalize_t* p)
{
    if(!well_formed(p) || p->batch == 0 || p->rows == 0 || p->cols == 0)
        return "";
    if(is_small(p))
        return "newton_schulz_small";
    static const auto names = [] {
        const char*                                              tile[TILES + 1] = {"256", "192", "128", "64", "64r2", "sliced"};
        std::array<std::string, (TILES + 1) * TILES * TILES> all;
        for(int i = 0; i < (int)all.size(); i++)
            all[i] = std::string("newton_schulz_products_") + tile[i / (TILES * TILES)] + "_" + tile[i / TILES % TILES] + "_" + tile[i % TILES];
        return all;
    }();
    const Layout l = layout_of(p);
    const int    square = l.slices > 1 ? TILES : choice_of(NS_SQUARE, l.m, l.n, p->batch);
    return names[(square * TILES + choice_of(NS_MIX, l.m, l.n, p->batch)) * TILES + choice_of(NS_UPDATE, l.m, l.n, p->batch)].c_str();
}

extern "C" uint64_t hiptk_orthogonalize_workspace_bytes(const hiptk_orthogonalize_t* p)
{
    if(!well_formed(p) || p->batch == 0 || p->rows == 0 || p->cols == 0 || is_small(p))
        return 0;
    const Layout l = layout_of(p);
    return (uint64_t)(l.per * p->batch + l.sums);
}

extern "C" int hiptk_orthogonalize(const hiptk_orthogonalize_t* p, void* workspace, uint64_t workspace_bytes, void* stream_, int* hip_error)
{
    if(hip_error)
        *hip_error = 0;
    if(!well_formed(p))
        return HIPTK_ERR_ARG;
    if(p->batch == 0 || p->rows == 0 || p->cols == 0)
        return HIPTK_OK;
    if(!p->X || !p->O)
        return HIPTK_ERR_ARG;
    const uint64_t need = hiptk_orthogonalize_workspace_bytes(p);
    if(need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)))
        return HIPTK_ERR_WORKSPACE;
    const Layout l      = layout_of(p);
    char*        ws     = (char*)workspace;
    hipStream_t  stream = (hipStream_t)stream_;
    NsArgs       a      = {};
    a.hi                = (_Float16*)(ws + l.hi);
    a.lo                = (_Float16*)(ws + l.lo);
    a.A                 = (_Float16*)(ws + l.A);
    a.B                 = (_Float16*)(ws + l.B);
    a.d                 = (float*)(ws + l.d);
    a.e                 = (float*)(ws + l.e);
    a.partial           = (double*)(ws + l.partial);
    a.X                 = p->X;
    a.O                 = p->O;
    a.ldx               = p->ldx;
    a.stride_x          = p->stride_x;
    a.ldo               = p->ldo;
    a.stride_o          = p->stride_o;
    a.per               = l.per;
    a.m                 = (int32_t)l.m;
    a.n                 = (int32_t)l.n;
    a.rows              = (int32_t)p->rows;
    a.cols              = (int32_t)p->cols;
    a.tall              = p->rows > p->cols;
    a.parts             = (int32_t)l.parts;
    a.lanes_log         = (int32_t)l.lanes_log;
    a.slices            = (int32_t)l.slices;
    a.sums              = (float*)(ws + l.per * p->batch);
    a.type_x            = p->type_x;
    a.type_o            = p->type_o;
    a.epsilon           = p->epsilon;
    a.scales            = scales_of(p->coefficients, p->steps);
    if(is_small(p))
    {
        Coefficients c;
        for(int i = 0; i < 3 * p->steps; i++)
            c.abc[i] = p->coefficients ? p->coefficients[i] : DEFAULT_COEFFICIENTS[i % 3];
        const uint32_t   b = (uint32_t)p->batch;
        const hipError_t e = l.m > 64    ? (l.n > 128 ? launch_small<128, 256>(a, c, p->steps, b, stream) : launch_small<128, 128>(a, c, p->steps, b, stream))
                             : l.n > 256 ? launch_small<64, 512>(a, c, p->steps, b, stream)
                             : l.n > 128 ? launch_small<64, 256>(a, c, p->steps, b, stream)
                             : l.n > 64  ? launch_small<64, 128>(a, c, p->steps, b, stream)
                                         : launch_small<64, 64>(a, c, p->steps, b, stream);
        if(hip_error)
            *hip_error = (int)e;
        return e == hipSuccess ? HIPTK_OK : HIPTK_ERR_LAUNCH;
    }
    const uint32_t batch = (uint32_t)p->batch, tm = (uint32_t)(l.m / 64), tn = (uint32_t)(l.n / 64);
    const int      square = choice_of(NS_SQUARE, l.m, l.n, batch), mix = choice_of(NS_MIX, l.m, l.n, batch), update = choice_of(NS_UPDATE, l.m, l.n, batch);
    ns_norm_kernel<<<dim3((uint32_t)l.parts, batch), dim3(256), 0, stream>>>(a);
    ns_begin_kernel<<<dim3(tn, tm, batch), dim3(256), 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    for(int s = 0; s < p->steps && e == hipSuccess; s++)
    {
        const float* abc = p->coefficients ? p->coefficients + 3 * s : DEFAULT_COEFFICIENTS;
        a.a              = abc[0];
        a.b              = abc[1];
        a.c              = abc[2];
        a.e_lo           = s + 2 >= p->steps ? 1.f : 0.f;
        a.hi             = (_Float16*)(ws + (s & 1 ? l.next : l.hi));
        a.hi_out         = (_Float16*)(ws + (s & 1 ? l.hi : l.next));
        if(l.slices > 1)
        {
            e = launch_tile<NS_SLICE, 64, 64, 2, 2, 4>(a, batch, stream);
            if(e == hipSuccess)
                e = launch_tile<NS_JOIN, 64, 64, 2, 2, 4>(a, batch, stream);
        }
        else
            e = launch<NS_SQUARE>(a, square, batch, stream);
        if(e == hipSuccess)
            e = launch<NS_MIX>(a, mix, batch, stream);
        if(e == hipSuccess)
            e = s + 1 < p->steps ? launch<NS_UPDATE>(a, update, batch, stream) : launch<NS_LAST>(a, update, batch, stream);
    }
    if(hip_error)
        *hip_error = (int)e;
    return e == hipSuccess ? HIPTK_OK : HIPTK_ERR_LAUNCH;
}

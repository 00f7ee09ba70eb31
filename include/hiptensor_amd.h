/*
 * Flat C ABI of the contraction path and of the tensor permutation (extern "C", plain
 * pointers and sizes).
 *
 * The reference's public functions take C++ structs with std::vector members
 * (library/include/hiptensor/hiptensor_types.hpp:177-227), so they cannot be bound
 * from C, ctypes, cgo or JNI.  Each function below is the same call with those
 * structs held behind opaque pointers that the library allocates; argument meaning,
 * check order and status codes are those of the function cited beside it, because
 * each one forwards to that function's implementation in this library.
 *
 * Status codes are hiptensorStatus_t values (0 = success).  Data types are
 * hipDataType values (0 f32, 1 f64, 2 f16, 4 c32, 5 c64, 14 bf16), compute types
 * hiptensorComputeType_t values (1 f16, 4 f32, 16 f64, 1024 bf16, 2048 c32, 4096 c64).
 */
#ifndef HIPTENSOR_AMD_H
#define HIPTENSOR_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* hiptensorCreate / hiptensorDestroy            (library/include/hiptensor/hiptensor.hpp:41,46) */
int hiptensorAmdCreate(void** handle);
int hiptensorAmdDestroy(void* handle);
/* A handle without a device: descriptors, workspace queries and planning work (for
 * inspection and host-side tests); hiptensorAmdContraction refuses it with
 * HIPTENSOR_STATUS_ARCH_MISMATCH.  No counterpart in the reference. */
int hiptensorAmdCreateHostOnly(void** handle);

/* hiptensorInitTensorDescriptor                                        (hiptensor.hpp:60-66) */
int hiptensorAmdInitTensorDescriptor(const void*    handle,
                                     void**         desc,
                                     uint32_t       numModes,
                                     const int64_t* lens,
                                     const int64_t* strides,
                                     int            dataType,
                                     int            unaryOp);
int hiptensorAmdDestroyTensorDescriptor(void* desc);

/* hiptensorGetErrorString                                                 (hiptensor.hpp:71) */
const char* hiptensorAmdGetErrorString(int status);

/* hiptensorGetAlignmentRequirement                                   (hiptensor.hpp:108-111) */
int hiptensorAmdGetAlignmentRequirement(const void* handle,
                                        const void* ptr,
                                        const void* desc,
                                        uint32_t*   alignmentRequirement);

/* hiptensorInitContractionDescriptor                                 (hiptensor.hpp:131-145) */
int hiptensorAmdInitContractionDescriptor(const void*    handle,
                                          void**         desc,
                                          const void*    descA,
                                          const int32_t* modeA,
                                          uint32_t       alignmentRequirementA,
                                          const void*    descB,
                                          const int32_t* modeB,
                                          uint32_t       alignmentRequirementB,
                                          const void*    descC,
                                          const int32_t* modeC,
                                          uint32_t       alignmentRequirementC,
                                          const void*    descD,
                                          const int32_t* modeD,
                                          uint32_t       alignmentRequirementD,
                                          int            typeCompute);
int hiptensorAmdDestroyContractionDescriptor(void* desc);

/* hiptensorInitContractionFind                                       (hiptensor.hpp:157-159) */
int hiptensorAmdInitContractionFind(const void* handle, void** find, int algo);
int hiptensorAmdDestroyContractionFind(void* find);

/* hiptensorContractionGetWorkspaceSize                               (hiptensor.hpp:170-174) */
int hiptensorAmdContractionGetWorkspaceSize(
    const void* handle, const void* desc, const void* find, int pref, uint64_t* workspaceSize);

/* hiptensorInitContractionPlan                                       (hiptensor.hpp:191-195) */
int hiptensorAmdInitContractionPlan(
    const void* handle, void** plan, const void* desc, const void* find, uint64_t workspaceSize);
int hiptensorAmdDestroyContractionPlan(void* plan);

/* hiptensorContraction; stream is a hipStream_t                      (hiptensor.hpp:218-228) */
int hiptensorAmdContraction(const void* handle,
                            const void* plan,
                            const void* alpha,
                            const void* A,
                            const void* B,
                            const void* beta,
                            const void* C,
                            void*       D,
                            void*       workspace,
                            uint64_t    workspaceSize,
                            void*       stream);

/* hiptensorAmdContraction for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  No counterpart in the
 * reference.  Same arguments and results as hiptensorAmdContraction, minus the workspace: whatever
 * workspace the plan needs (split-K partials, packed operand copies) is taken from a device array
 * of HIPTK_STATIC_WORKSPACE_BYTES (32 MiB) that the library itself holds on every device until the
 * process ends.  The call allocates nothing and frees nothing (and skips the PERF_TRACE timing,
 * which would create events).  A plan that needs more than the array holds is refused with
 * HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE: plan with a smaller workspaceSize.  Every call on one
 * device uses the same array: calls that overlap in time on one device (different streams, or
 * threads) race on it and must be serialised by the caller; calls in one stream are safe. */
int hiptensorAmdContractionNoAlloc(const void* handle,
                                   const void* plan,
                                   const void* alpha,
                                   const void* A,
                                   const void* B,
                                   const void* beta,
                                   const void* C,
                                   void*       D,
                                   void*       stream);

/* hiptensorPermutation; typeScalar is a hipDataType, stream a hipStream_t  (hiptensor.hpp:89-98) */
int hiptensorAmdPermutation(const void*    handle,
                            const void*    alpha,
                            const void*    A,
                            const void*    descA,
                            const int32_t* modeA,
                            void*          B,
                            const void*    descB,
                            const int32_t* modeB,
                            int            typeScalar,
                            void*          stream);

/* What hiptensorAmdPermutation would launch for these descriptors, mode lists and addresses
 * (only the alignment of A and B is looked at; nothing is read or launched, no device is
 * needed).  Returns the status the call would return before launching.  No counterpart in
 * the reference. */
typedef struct hiptensorAmdPermutationInfo
{
    int32_t fused_rank;   /* modes left after extent-1 modes are dropped and neighbours fused */
    int32_t extent[6];    /* fused extents in A's order, fastest first                        */
    int32_t a_stride[6], b_stride[6];
    int32_t kernel;       /* HIPTK_PERM_COPY / TILED / ROWS / GATHER / STRIP / GROUPED / SHARED */
    int32_t mode_i, mode_j, tile, vec_r, vec_w;
    int32_t empty;        /* 1: an extent is zero, nothing would be launched                  */
    char    kernel_name[96];
} hiptensorAmdPermutationInfo_t;
int hiptensorAmdPermutationInfo(const void*                    descA,
                                const int32_t*                 modeA,
                                const void*                    descB,
                                const int32_t*                 modeB,
                                const void*                    A,
                                const void*                    B,
                                hiptensorAmdPermutationInfo_t* out);

/* logger control                                                     (hiptensor.hpp:308-343) */
typedef void (*hiptensorAmdLoggerCallback_t)(int32_t logContext, const char* funcName, const char* msg);
int hiptensorAmdLoggerSetCallback(hiptensorAmdLoggerCallback_t callback);
int hiptensorAmdLoggerOpenFile(const char* logFile);
int hiptensorAmdLoggerSetLevel(int level);
int hiptensorAmdLoggerSetMask(int32_t mask);
int hiptensorAmdLoggerForceDisable(void);
int hiptensorAmdGetHiprtVersion(void);

/* What a plan decided; for tests, benchmarks and logs.  No counterpart in the reference
 * (its plan exposes only a kernel pointer). */
typedef struct hiptensorAmdPlanInfo
{
    int64_t  P, Q, K;        /* folded GEMM view: rows, columns, reduction            */
    int32_t  swapped;        /* 1: rows come from B and columns from A                */
    int32_t  kernel_class;   /* HIPTK_* element class                                 */
    int32_t  tile_p, tile_q, tile_k, threads, lds_bytes;
    int32_t  split_k;
    int32_t  x_kfast, y_kfast, x_vec, y_vec, cd_vec;
    int32_t  n_pdims, n_qdims, n_kdims; /* dims left after fusion                     */
    uint64_t workspace_bytes;
    uint64_t kernel_uid;
    double   estimate_us;
    char     kernel_name[96];
    /* operands the plan first moves into a packed copy in the workspace (interleaved layouts
     * that would otherwise be gathered element by element); the view above is that of the copies */
    int32_t  pack_a, pack_b;
    uint64_t pack_bytes;     /* leading part of workspace_bytes that holds the copies  */
    char     pack_a_kernel[96], pack_b_kernel[96];
} hiptensorAmdPlanInfo_t;
int hiptensorAmdPlanInfo(const void* plan, hiptensorAmdPlanInfo_t* out);
/* Size of a handle's plan cache: `states` = plan states it holds (each owns its offset tables on the
 * device; one per distinct planning decision; beyond 4096 the least recently planned one that was never
 * executed is retired), `requests` = distinct planning requests (problem x workspace size ...) that map onto them.
 * No counterpart in the reference, whose plans point into process-wide singletons. */
int hiptensorAmdPlanCacheInfo(const void* handle, int64_t* states, int64_t* requests);
/* Keeps the plan's state (and its offset tables on the device) until hiptensorDestroy: the cache never
 * retires it.  The first execution of a plan does the same by itself, since from then on a captured
 * graph or a launch in another thread may read the tables; this call is for a caller that holds a
 * plan for later without having executed it.  Returns HIPTENSOR_STATUS_INTERNAL_ERROR for a plan whose
 * state was retired already.  No counterpart in the reference (its plans never expire). */
int hiptensorAmdPlanRetain(const void* plan);

/* Copies offset table `which` (0 xp, 1 xk, 2 yq, 3 yk, 4 cp, 5 cq, 6 dp, 7 dq; logical
 * length only, without padding) into out[0..cap); returns the logical length. */
int64_t hiptensorAmdPlanTable(const void* plan, int which, int32_t* out, int64_t cap);

/* ------------------------------------------------------------------------------------------
 * Operators of a linear layer that is trained and served in 8-bit floating point.  No counterpart in the reference.
 * Matrices are device addresses with sizes and leading dimensions (elements); nothing is planned or kept between
 * calls, nothing is allocated, every kernel goes to `stream`, and the calls may be captured into a graph.
 *
 * Codes: OCP e4m3 (hipDataType HIP_R_8F_E4M3), one byte each, the contracted dimension contiguous.  Scales: f32, one
 * for 128 consecutive codes of one row, or of 128 rows ("square" blocks), stored block by block of the contracted
 * dimension: the scale of code (r, k) is S[(k / 128) * ldS + r / blockRows], so ldS >= ceil(rows / blockRows).  A leading
 * dimension that separates nothing (one row, one block) is not looked at.
 * A code stands for code * scale.
 *
 * Status codes: NOT_INITIALIZED (a handle or needed pointer is null), INVALID_VALUE (a
 * negative or too large extent, a leading dimension below its row, an address that is no multiple of its element),
 * NOT_SUPPORTED (a data type or block shape there is no kernel for, or too many tiles), INSUFFICIENT_WORKSPACE, ARCH_MISMATCH (a handle
 * without a device, or another current device), EXECUTION_FAILED (the launch failed).
 * Limits: extents of the quantisation and of the product at most 2^31 - 256, the former's matrix fewer than 2^23 tiles of 128 x 128, the latter's
 * result fewer than 2^23 of 64 x 64; the orthogonalisation's batch at most 65535, its matrices' shorter side 2^16, the longer one 2^20.
 * An empty result returns SUCCESS without a launch.
 * ------------------------------------------------------------------------------------------ */

/* Codes and scales of X [rows, cols] (HIP_R_16F, HIP_R_16BF or HIP_R_32F).  For each block, in f32:
 *     amax = max |x|,  r = min(448 / amax, 2^126),  scale = 1 / r,  code = e4m3(x * r), rounded to nearest even.
 * A block that holds a NaN or an infinity has NaN codes (a NaN: and a NaN scale); a block of zeros has zero codes.
 *   Q [rows, cols],  S: blocks of 128 columns         - for products that contract the columns
 *   QT [cols, rows], ST: blocks of 128 rows of X      - for products that contract the rows (a weight gradient)
 * blockRows 1: one row of Q (of QT) per scale.  blockRows 128: square blocks; Q and QT hold the same values.
 * Either form may be left out (null codes and scales); bytes beyond a row's codes are not written. */
int hiptensorAmdBlockQuantize(const void* handle,
                              int64_t     rows,
                              int64_t     cols,
                              const void* X,
                              int         typeX,
                              int64_t     ldX,
                              int         blockRows,
                              void*       Q,
                              int64_t     ldQ,
                              float*      S,
                              int64_t     ldS,
                              void*       QT,
                              int64_t     ldQT,
                              float*      ST,
                              int64_t     ldST,
                              void*       stream);

/* D = alpha * A' B'^T + beta * C for A' [M, K] and B' [N, K], the values of codes A with one row per scale and of codes B
 * with blockRowsB (1 or 128) rows per scale.  C and D [M, N]: typeD (HIP_R_16F, HIP_R_16BF or HIP_R_32F) and ldD; D may be
 * C; with beta 0 C is not read and may be null.  alpha, beta: host f32.  Sums are in f32 for a D in
 * f32; for a D of 16 bits a block of 128 is summed by the 8-bit matrix instructions, which drop what lies 13 bits below the largest of neighbouring
 * terms: 2e-5 of the result in 2-norm, far below D's rounding, and less than 2^-11 of the sum of the terms' magnitudes in any element, which is more than
 * its rounding where they cancel to a small part of that sum (ask for a D in f32 where single elements count).  Blocks are summed in f32, D is rounded once.  Kernels load 16 bytes at a time where both operands' addresses and
 * leading dimensions are multiples of 16 (a slower kernel runs otherwise); they may read up to the end of the aligned 16
 * bytes that a row of codes ends in, and what lies there does not change the result.
 * workspace: GetWorkspaceSize says with how much the call is fastest (16-byte aligned); with less, 0 included, it
 * computes the same product without splitting K. */
int hiptensorAmdBlockScaledProductGetWorkspaceSize(
    const void* handle, int64_t M, int64_t N, int64_t K, int blockRowsB, int typeD, uint64_t* workspaceSize);
int hiptensorAmdBlockScaledProduct(const void*  handle,
                                   int64_t      M,
                                   int64_t      N,
                                   int64_t      K,
                                   const float* alpha,
                                   const void*  A,
                                   int64_t      ldA,
                                   const float* SA,
                                   int64_t      ldSA,
                                   const void*  B,
                                   int64_t      ldB,
                                   const float* SB,
                                   int64_t      ldSB,
                                   int          blockRowsB,
                                   const float* beta,
                                   const void*  C,
                                   void*        D,
                                   int          typeD,
                                   int64_t      ldD,
                                   void*        workspace,
                                   uint64_t     workspaceSize,
                                   void*        stream);

/* O = X orthogonalised by Newton-Schulz products, for each of `batch` matrices [rows, cols] (strideX, strideO elements
 * apart):  X <- X / (|X|_F + epsilon), then `steps` times  A = X X^T,  B = b A + c A A,  X <- a X + B X  on the shorter side.
 * coefficients: host f32 a, b, c for each step, or null for 3.4445, -4.7750, 2.0315 in every step.  typeX: HIP_R_16F,
 * HIP_R_16BF or HIP_R_32F; typeO: HIP_R_16F or HIP_R_16BF.  The products are of f16 with f32 sums; the iterate is held in
 * 22 bits and the diagonals of A and B in f32.  With the default coefficients and before O's rounding, that keeps the result within 3e-3 (2-norm) of
 * the exact iteration's for up to 6 steps and 6e-3 for up to 12; four times that where the shorter side is below 16 or entries or rows repeat, so that
 * roundings do not average out; and 2^-22 * 3.4445^steps more where X lacks directions (4e-4 after 6 steps, 6e-2 after 10), since each step multiplies
 * what rounding leaves there.  The iterates' singular values must stay below 16, which the default coefficients guarantee (A and B have whatever size follows).  O may be X where the types' sizes
 * and the layouts agree.  The workspace (256-byte aligned) is required in full; GetWorkspaceSize says how much is enough for
 * any number of steps.  Matrices of up to 64 x 512 or 128 x 256 (or turned) with up to 16 steps need none: null is accepted there. */
int hiptensorAmdOrthogonalizeGetWorkspaceSize(
    const void* handle, int64_t batch, int64_t rows, int64_t cols, int typeX, int typeO, uint64_t* workspaceSize);
int hiptensorAmdOrthogonalize(const void*  handle,
                              int64_t      batch,
                              int64_t      rows,
                              int64_t      cols,
                              const void*  X,
                              int          typeX,
                              int64_t      ldX,
                              int64_t      strideX,
                              int          steps,
                              const float* coefficients,
                              float        epsilon,
                              void*        O,
                              int          typeO,
                              int64_t      ldO,
                              int64_t      strideO,
                              void*        workspace,
                              uint64_t     workspaceSize,
                              void*        stream);

#ifdef __cplusplus
}
#endif
#endif /* HIPTENSOR_AMD_H */

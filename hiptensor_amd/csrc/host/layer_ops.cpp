// hiptensorAmdBlockQuantize, hiptensorAmdBlockScaledProduct, hiptensorAmdOrthogonalize: argument checks, device check,
// the call into the kernel layer and its status.  No counterpart in the reference.
#include <cstdio>
#include <initializer_list>

#include <hip/hip_runtime_api.h>

#include <hiptensor/hiptensor.hpp>
#include <hiptensor_amd.h>

#include "handle.hpp"
#include "logger.hpp"

using hipta::Handle;
using hipta::Logger;

namespace
{
    constexpr int64_t MOST = 0x7fffff00; // extents (tile ends stay below 2^31)

    struct Param
    {
        const void* p;
        const char* name;
    };

    hiptensorStatus_t refuse(const char* fn, hiptensorStatus_t st, const char* why)
    {
        Logger::get().errorf(fn, "%s (%s)", why, hiptensorGetErrorString(st));
        return st;
    }

    hiptensorStatus_t needed(const char* fn, std::initializer_list<Param> params)
    {
        hiptensorStatus_t st = HIPTENSOR_STATUS_SUCCESS;
        for(const auto& q : params)
            if(!q.p)
            {
                st = HIPTENSOR_STATUS_NOT_INITIALIZED;
                Logger::get().errorf(fn, "Initialization Error : %s = nullptr (%s)", q.name, hiptensorGetErrorString(st));
            }
        return st;
    }

    // the kernel layer's element class of a hipDataType, or -1
    int class_of(int type)
    {
        return type == HIP_R_16F ? HIPTK_F16 : type == HIP_R_16BF ? HIPTK_BF16 : type == HIP_R_32F ? HIPTK_F32 : -1;
    }

    int64_t bytes_of(int type)
    {
        return type == HIP_R_32F ? 4 : 2;
    }

    int64_t blocks(int64_t n, int64_t b)
    {
        return (n + b - 1) / b;
    }

    // Whether a leading dimension is smaller than the rows of `span` elements that it separates; of a single row it is not used.
    bool short_of(int64_t ld, int64_t span, int64_t rows)
    {
        return rows > 1 && ld < span;
    }

    bool off(const void* p, int64_t bytes)
    {
        return (uintptr_t)p % (uint64_t)bytes != 0;
    }

    hiptensorStatus_t device_of(const char* fn, const void* handle, Handle*& h)
    {
        h = Handle::from(((const hiptensorHandle_t*)handle)->fields);
        if(!h)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        if(h->hostOnly())
            return refuse(fn, HIPTENSOR_STATUS_ARCH_MISMATCH, "This handle has no device; it cannot execute");
        int cur = -1;
        if(hipGetDevice(&cur) != hipSuccess || cur != h->device())
        {
            Logger::get().errorf(fn, "Device mismatch error: current device id: %d, handle device id: %d (%s)", cur, h->device(),
                                 hiptensorGetErrorString(HIPTENSOR_STATUS_ARCH_MISMATCH));
            return HIPTENSOR_STATUS_ARCH_MISMATCH;
        }
        return HIPTENSOR_STATUS_SUCCESS;
    }

    // Launches, with HIPTENSOR_LOG_LEVEL_PERF_TRACE between two events (whose line names the kernel; not while a capture is in progress, which the
    // synchronisation would invalidate), and turns the kernel layer's code into a status.
    template <typename N, typename F>
    hiptensorStatus_t execute(const char* fn, N&& name, double flops, double bytes, hipStream_t stream, F&& launch)
    {
        Logger&    log   = Logger::get();
        bool       timed = (log.mask() & HIPTENSOR_LOG_LEVEL_PERF_TRACE) != 0;
        hipEvent_t e0 = nullptr, e1 = nullptr;
        if(timed)
        {
            hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
            if(hipStreamIsCapturing(stream, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone)
                timed = false;
        }
        if(timed)
        {
            if(hipEventCreate(&e0) != hipSuccess)
                return HIPTENSOR_STATUS_HIP_ERROR;
            if(hipEventCreate(&e1) != hipSuccess)
            {
                (void)hipEventDestroy(e0);
                return HIPTENSOR_STATUS_HIP_ERROR;
            }
            (void)hipEventRecord(e0, stream);
        }
        int hipErr = 0;
        int rc     = launch(&hipErr);
        if(timed)
        {
            (void)hipEventRecord(e1, stream);
            (void)hipEventSynchronize(e1);
            float ms = 0.f;
            (void)hipEventElapsedTime(&ms, e0, e1);
            (void)hipEventDestroy(e0);
            (void)hipEventDestroy(e1);
            if(rc == HIPTK_OK)
            {
                const char* kernel = name();
                uint64_t    uid    = 1469598103934665603ull;
                for(const char* c = kernel; *c; ++c)
                    uid = (uid ^ (unsigned char)*c) * 1099511628211ull;
                char msg[512];
                snprintf(msg, sizeof(msg), "KernelId: %lu KernelName: %s, %0.3f ms, %0.3f TFlops, %0.3f GB/s", (unsigned long)uid, kernel, ms,
                         flops / 1e9 / ms, bytes / 1e6 / ms);
                log.perf(fn, msg);
            }
        }
        switch(rc)
        {
        case HIPTK_OK: return HIPTENSOR_STATUS_SUCCESS;
        case HIPTK_ERR_WORKSPACE: return refuse(fn, HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE, "The workspace is too small or not aligned");
        case HIPTK_ERR_LAUNCH:
            log.errorf(fn, "Kernel launch failed: %s (%s)", hipGetErrorString((hipError_t)hipErr), hiptensorGetErrorString(HIPTENSOR_STATUS_EXECUTION_FAILED));
            return HIPTENSOR_STATUS_EXECUTION_FAILED;
        default: return refuse(fn, HIPTENSOR_STATUS_INTERNAL_ERROR, "Selected kernel is unable to solve the problem");
        }
    }

    // Nothing that happens below a C entry may leave it as an exception (the log sink may allocate).
    template <typename F>
    int entry(F&& body)
    {
        try
        {
            return (int)body();
        }
        catch(...)
        {
            return (int)HIPTENSOR_STATUS_INTERNAL_ERROR;
        }
    }

    hiptensorStatus_t check_product(const char* fn, int64_t M, int64_t N, int64_t K, int blockRowsB, int typeD)
    {
        if(M < 0 || N < 0 || K < 0 || M > MOST || N > MOST || K > MOST)
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : an extent is negative or 2^31 - 256 or more");
        if(class_of(typeD) < 0)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "Unsupported Data Type Error : D is HIP_R_16F, HIP_R_16BF or HIP_R_32F");
        if(blockRowsB != 1 && blockRowsB != 128)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "A scale of B stands for 1 or 128 rows");
        return HIPTENSOR_STATUS_SUCCESS;
    }

    hiptensorStatus_t check_orthogonalize(const char* fn, int64_t batch, int64_t rows, int64_t cols, int typeX, int typeO)
    {
        const int64_t s = rows < cols ? rows : cols, t = rows < cols ? cols : rows;
        if(batch < 0 || s < 0 || batch > 65535 || s > (1 << 16) || t > (1 << 20))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE,
                          "Input Parameter Error : batch is 0 .. 65535, the shorter side at most 2^16, the longer one at most 2^20");
        if(class_of(typeX) < 0 || class_of(typeO) < 0 || typeO == HIP_R_32F)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "Unsupported Data Type Error : X is HIP_R_16F, HIP_R_16BF or HIP_R_32F, O HIP_R_16F or HIP_R_16BF");
        return HIPTENSOR_STATUS_SUCCESS;
    }
}

extern "C" int hiptensorAmdBlockQuantize(const void* handle,
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
                                         void*       stream)
{
    return entry([&]() -> hiptensorStatus_t {
        const char* fn = "hiptensorBlockQuantize";
        Logger::get().apif(fn,
                           "handle=%p, rows=%lld, cols=%lld, X=%p, typeX=0x%02X, ldX=%lld, blockRows=%d, Q=%p, ldQ=%lld, S=%p, ldS=%lld, QT=%p, "
                           "ldQT=%lld, ST=%p, ldST=%lld, stream=%p",
                           handle, (long long)rows, (long long)cols, X, (unsigned)typeX, (long long)ldX, blockRows, Q, (long long)ldQ, (void*)S,
                           (long long)ldS, QT, (long long)ldQT, (void*)ST, (long long)ldST, stream);
        if(auto st = needed(fn, {{handle, "handle"}}); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        const bool empty = rows == 0 || cols == 0;
        if(!empty)
        {
            if(auto st = needed(fn, {{X, "X"}}); st != HIPTENSOR_STATUS_SUCCESS)
                return st;
            if((Q != nullptr) != (S != nullptr) || (QT != nullptr) != (ST != nullptr) || (!Q && !QT))
                return refuse(fn, HIPTENSOR_STATUS_NOT_INITIALIZED, "Initialization Error : codes and scales of at least one form are needed, and of both or neither");
        }
        if(rows < 0 || cols < 0 || rows > MOST || cols > MOST)
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : an extent is negative or 2^31 - 256 or more");
        if(class_of(typeX) < 0)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "Unsupported Data Type Error : X is HIP_R_16F, HIP_R_16BF or HIP_R_32F");
        if(blockRows != 1 && blockRows != 128)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "A scale stands for 1 or 128 rows");
        if(short_of(ldX, cols, rows) || (Q && (short_of(ldQ, cols, rows) || short_of(ldS, blocks(rows, blockRows), blocks(cols, 128))))
           || (QT && (short_of(ldQT, rows, cols) || short_of(ldST, blocks(cols, blockRows), blocks(rows, 128)))))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : a leading dimension is smaller than what it spans");
        if(off(X, bytes_of(typeX)) || off(S, 4) || off(ST, 4))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : an address is no multiple of its element's size");
        if(blocks(rows, 128) * blocks(cols, 128) > MOST / 256)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "A matrix of 2^23 tiles of 128 x 128 or more is not supported");
        Handle* h = nullptr;
        if(auto st = device_of(fn, handle, h); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        if(empty)
            return HIPTENSOR_STATUS_SUCCESS;
        hiptk_block_quantize_t p = {};
        p.rows                   = rows;
        p.cols                   = cols;
        p.X                      = X;
        p.type                   = class_of(typeX);
        p.block_rows             = blockRows;
        p.ldx                    = ldX;
        p.Q                      = Q;
        p.S                      = S;
        p.ldq                    = ldQ;
        p.lds                    = ldS;
        p.QT                     = QT;
        p.ST                     = ST;
        p.ldqt                   = ldQT;
        p.ldst                   = ldST;
        const double n           = (double)rows * (double)cols;
        return execute(fn, [&] { return hiptk_block_quantize_kernel_name(&p); }, n, n * (double)(bytes_of(typeX) + (Q != nullptr) + (QT != nullptr)), (hipStream_t)stream,
                       [&](int* e) { return hiptk_block_quantize(&p, stream, e); });
    });
}

extern "C" int hiptensorAmdBlockScaledProductGetWorkspaceSize(
    const void* handle, int64_t M, int64_t N, int64_t K, int blockRowsB, int typeD, uint64_t* workspaceSize)
{
    return entry([&]() -> hiptensorStatus_t {
        const char* fn = "hiptensorBlockScaledProductGetWorkspaceSize";
        Logger::get().apif(fn, "handle=%p, M=%lld, N=%lld, K=%lld, blockRowsB=%d, typeD=0x%02X, workspaceSize=%p", handle, (long long)M, (long long)N,
                           (long long)K, blockRowsB, (unsigned)typeD, (void*)workspaceSize);
        if(auto st = needed(fn, {{handle, "handle"}, {workspaceSize, "workspaceSize"}}); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        *workspaceSize = 0;
        if(auto st = check_product(fn, M, N, K, blockRowsB, typeD); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        hiptk_block_product_t p = {};
        p.M                     = M;
        p.N                     = N;
        p.K                     = K;
        p.block_rows            = blockRowsB;
        p.type                  = class_of(typeD);
        *workspaceSize          = hiptk_block_product_workspace_bytes(&p);
        return HIPTENSOR_STATUS_SUCCESS;
    });
}

extern "C" int hiptensorAmdBlockScaledProduct(const void*  handle,
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
                                              void*        stream)
{
    return entry([&]() -> hiptensorStatus_t {
        const char* fn = "hiptensorBlockScaledProduct";
        Logger::get().apif(fn,
                           "handle=%p, M=%lld, N=%lld, K=%lld, alpha=%p, A=%p, ldA=%lld, SA=%p, ldSA=%lld, B=%p, ldB=%lld, SB=%p, ldSB=%lld, "
                           "blockRowsB=%d, beta=%p, C=%p, D=%p, typeD=0x%02X, ldD=%lld, workspace=%p, workspaceSize=%llu, stream=%p",
                           handle, (long long)M, (long long)N, (long long)K, (const void*)alpha, A, (long long)ldA, (const void*)SA, (long long)ldSA, B,
                           (long long)ldB, (const void*)SB, (long long)ldSB, blockRowsB, (const void*)beta, C, D, (unsigned)typeD, (long long)ldD,
                           workspace, (unsigned long long)workspaceSize, stream);
        if(auto st = needed(fn, {{handle, "handle"}, {alpha, "alpha"}, {beta, "beta"}}); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        const bool empty = M == 0 || N == 0;
        if(!empty)
        {
            if(auto st = needed(fn, {{D, "D"}}); st != HIPTENSOR_STATUS_SUCCESS)
                return st;
            if(K != 0)
                if(auto st = needed(fn, {{A, "A"}, {SA, "SA"}, {B, "B"}, {SB, "SB"}}); st != HIPTENSOR_STATUS_SUCCESS)
                    return st;
            if(*beta != 0.f)
                if(auto st = needed(fn, {{C, "C"}}); st != HIPTENSOR_STATUS_SUCCESS)
                    return st;
        }
        if(auto st = check_product(fn, M, N, K, blockRowsB, typeD); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        if(short_of(ldD, N, M)
           || (K != 0 && (short_of(ldA, K, M) || short_of(ldB, K, N) || short_of(ldSA, M, blocks(K, 128)) || short_of(ldSB, blocks(N, blockRowsB), blocks(K, 128)))))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : a leading dimension is smaller than what it spans");
        if(off(SA, 4) || off(SB, 4) || off(D, bytes_of(typeD)) || (*beta != 0.f && off(C, bytes_of(typeD))))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : an address is no multiple of its element's size");
        if(blocks(M, 64) * blocks(N, 64) > MOST / 256)
            return refuse(fn, HIPTENSOR_STATUS_NOT_SUPPORTED, "A result of 2^23 tiles of 64 x 64 or more is not supported");
        Handle* h = nullptr;
        if(auto st = device_of(fn, handle, h); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        if(empty)
            return HIPTENSOR_STATUS_SUCCESS;
        hiptk_block_product_t p = {};
        p.M                     = M;
        p.N                     = N;
        p.K                     = K;
        p.A                     = A;
        p.B                     = B;
        p.SA                    = SA;
        p.SB                    = SB;
        // (of a single row: as if the rows were padded to the loads' 16 bytes)
        p.lda                   = M > 1 ? ldA : blocks(K, 16) * 16;
        p.ldb                   = N > 1 ? ldB : blocks(K, 16) * 16;
        p.ldsa                  = ldSA;
        p.ldsb                  = ldSB;
        p.block_rows            = blockRowsB;
        p.type                  = class_of(typeD);
        p.alpha                 = *alpha;
        p.beta                  = *beta;
        p.C                     = C;
        p.D                     = D;
        p.ldd                   = ldD;
        const double m = (double)M, n = (double)N, k = (double)K;
        return execute(fn, [&] { return hiptk_block_product_kernel_name(&p); }, 2.0 * m * n * k, (m + n) * k + m * n * (double)bytes_of(typeD) * (*beta != 0.f ? 2.0 : 1.0),
                       (hipStream_t)stream, [&](int* e) { return hiptk_block_product(&p, workspace, workspaceSize, stream, e); });
    });
}

extern "C" int hiptensorAmdOrthogonalizeGetWorkspaceSize(
    const void* handle, int64_t batch, int64_t rows, int64_t cols, int typeX, int typeO, uint64_t* workspaceSize)
{
    return entry([&]() -> hiptensorStatus_t {
        const char* fn = "hiptensorOrthogonalizeGetWorkspaceSize";
        Logger::get().apif(fn, "handle=%p, batch=%lld, rows=%lld, cols=%lld, typeX=0x%02X, typeO=0x%02X, workspaceSize=%p", handle, (long long)batch,
                           (long long)rows, (long long)cols, (unsigned)typeX, (unsigned)typeO, (void*)workspaceSize);
        if(auto st = needed(fn, {{handle, "handle"}, {workspaceSize, "workspaceSize"}}); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        *workspaceSize = 0;
        if(auto st = check_orthogonalize(fn, batch, rows, cols, typeX, typeO); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        hiptk_orthogonalize_t p = {};
        p.batch                 = batch;
        p.rows                  = rows;
        p.cols                  = cols;
        p.type_x                = class_of(typeX);
        p.type_o                = class_of(typeO);
        p.steps                 = INT32_MAX; // (enough for any number)
        *workspaceSize          = hiptk_orthogonalize_workspace_bytes(&p);
        return HIPTENSOR_STATUS_SUCCESS;
    });
}

extern "C" int hiptensorAmdOrthogonalize(const void*  handle,
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
                                         void*        stream)
{
    return entry([&]() -> hiptensorStatus_t {
        const char* fn = "hiptensorOrthogonalize";
        Logger::get().apif(fn,
                           "handle=%p, batch=%lld, rows=%lld, cols=%lld, X=%p, typeX=0x%02X, ldX=%lld, strideX=%lld, steps=%d, coefficients=%p, "
                           "epsilon=%g, O=%p, typeO=0x%02X, ldO=%lld, strideO=%lld, workspace=%p, workspaceSize=%llu, stream=%p",
                           handle, (long long)batch, (long long)rows, (long long)cols, X, (unsigned)typeX, (long long)ldX, (long long)strideX, steps,
                           (const void*)coefficients, (double)epsilon, O, (unsigned)typeO, (long long)ldO, (long long)strideO, workspace,
                           (unsigned long long)workspaceSize, stream);
        if(auto st = needed(fn, {{handle, "handle"}}); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        const bool empty = batch == 0 || rows == 0 || cols == 0;
        if(!empty)
            if(auto st = needed(fn, {{X, "X"}, {O, "O"}}); st != HIPTENSOR_STATUS_SUCCESS)
                return st;
        if(auto st = check_orthogonalize(fn, batch, rows, cols, typeX, typeO); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        if(steps < 1 || !(epsilon >= 0.f))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : at least one step, and an epsilon that is not negative");
        if(short_of(ldX, cols, rows) || short_of(ldO, cols, rows) || (batch > 1 && (strideX < 0 || strideO < (rows - 1) * ldO + cols)))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : a leading dimension or a stride is smaller than what it spans");
        if(off(X, bytes_of(typeX)) || off(O, bytes_of(typeO)))
            return refuse(fn, HIPTENSOR_STATUS_INVALID_VALUE, "Input Parameter Error : an address is no multiple of its element's size");
        hiptk_orthogonalize_t p = {};
        p.batch                 = batch;
        p.rows                  = rows;
        p.cols                  = cols;
        p.X                     = X;
        p.type_x                = class_of(typeX);
        p.type_o                = class_of(typeO);
        p.ldx                   = ldX;
        p.stride_x              = strideX;
        p.O                     = O;
        p.ldo                   = ldO;
        p.stride_o              = strideO;
        p.steps                 = steps;
        p.epsilon               = epsilon;
        const uint64_t need     = hiptk_orthogonalize_workspace_bytes(&p);
        if(need && (!workspace || workspaceSize < need || off(workspace, 256)))
        {
            Logger::get().errorf(fn, "Insufficient workspace: given %llu bytes, needed %llu, on a multiple of 256 (%s)", (unsigned long long)workspaceSize,
                                 (unsigned long long)need, hiptensorGetErrorString(HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE));
            return HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE;
        }
        Handle* h = nullptr;
        if(auto st = device_of(fn, handle, h); st != HIPTENSOR_STATUS_SUCCESS)
            return st;
        if(empty)
            return HIPTENSOR_STATUS_SUCCESS;
        const double s = (double)(rows < cols ? rows : cols), t = (double)(rows < cols ? cols : rows), b = (double)batch;
        p.coefficients = coefficients;
        return execute(fn, [&] { return hiptk_orthogonalize_kernel_name(&p); }, b * steps * (3.0 * s * s * t + s * s * s), b * s * t * (double)(bytes_of(typeX) + bytes_of(typeO)),
                       (hipStream_t)stream, [&](int* e) { return hiptk_orthogonalize(&p, workspace, workspaceSize, stream, e); });
    });
}

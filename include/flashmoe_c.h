/* Flat C ABI of libflashMoe.so: the same operations as iMoeKernelLauncher.h for
 * callers that cannot bind a C++ vtable (ctypes, cgo, JNI, ...).  Plain
 * pointers and sizes only.  Every function returns a cudaError_t value as int
 * (0 == success) unless stated otherwise.
 *
 * Each entry names the reference interface it stands for (paths relative to the
 * reference project).
 */
#ifndef FLASHMOE_C_H_
#define FLASHMOE_C_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct FlashMoeHandle_t* FlashMoeHandle;

typedef struct {
  int32_t hiddenSize;
  int32_t expertIntermediateSize;
  int32_t expertsNum;
  int32_t topk;
  int32_t dtype; /* 0 bf16, 1 fp32 I/O */
  int32_t reserved[3];
} FlashMoeConfig;

/* GetDistributedUniqueId (include/iMoeKernelLauncher.h:26): fills 128 bytes. */
int FlashMoeGetUniqueId(int empty, uint8_t out[128]);

/* CreateLauncher / CreateLauncherEx (include/iMoeKernelLauncher.h:29-35,
 * python/pyMoeLauncherTorch.cpp:71-107).  config == NULL selects the
 * Qwen3-30B-A3B shape in bf16.  `stream` is a cudaStream_t. */
int FlashMoeCreate(FlashMoeHandle* out, const void* gateWeights, const void* ffn1ExpertWeights,
                   const void* ffn2ExpertWeights, int maxTokens, void* stream,
                   const uint8_t uid[128], int rank, int worldSize, const FlashMoeConfig* config);

/* IMoeKernelLauncher::Launch (include/iMoeKernelLauncher.h:12-13,
 * python/pyMoeLauncherTorch.cpp:44-61): device pointers, asynchronous. */
int FlashMoeLaunch(FlashMoeHandle h, const void* tokens, void* output, int tokensNum, void* stream);

/* Launch with HOST buffers: copies `tokens` to the device, runs the layer and
 * copies the result back.  The input must be complete in host memory when the
 * call is made; the result is complete once `stream` has reached this point.
 * Returns after enqueueing (pinned host memory).  The three steps run on
 * internal streams with two sets of staging buffers, so back-to-back calls
 * overlap the copies of one call with the kernel of the other.  The reference's
 * tests do the same three steps by hand (test/singleGPU/cpp/moe/moeTest.cpp:38-56). */
int FlashMoeLaunchHost(FlashMoeHandle h, const void* hostTokens, void* hostOutput, int tokensNum,
                       void* stream);

/* DestroyLauncher (include/iMoeKernelLauncher.h:38-39). */
int FlashMoeDestroy(FlashMoeHandle h, void* stream);

/* First device-side error of the launcher since creation (0 == none) and its
 * detail word; does not synchronise.  The reference has no counterpart: its
 * device waits are unbounded (src/hip/taskSystem/taskManager.h:208-215). */
int FlashMoeGetLastStatus(FlashMoeHandle h, uint32_t* code, uint32_t* info);

/* Stage buffers of the last launch, for parity tests (the reference checks the
 * same stages with purpose-built kernels, test/singleGPU/cpp/moe/internal/).
 * `which`: 0 top-k indices int32 [T,K]; 1 routing weights fp32 [T,K];
 * 2 rows per local expert uint32 [E_local]; 3 packed rows bf16 [E_local*cap,H];
 * 4 row sideband 16 B [E_local*cap]; 5 activations bf16 [E_local*cap,I];
 * 6 weighted expert outputs bf16 [maxTokens,K,H]; 7 {cap_rows, E_local, grid, smem} int32[4];
 * 8 event trace of the last launch (only with FLASHMOE_PROFILE=1 at create): per CTA 512 records of
 * {kind, t0, t1, t2} uint32 ns, record 0 = {count,...}.
 * Copies min(bytes, size) bytes starting at `offset` to host memory `dst`
 * after synchronising the device. */
int FlashMoeDebugRead(FlashMoeHandle h, int which, void* dst, size_t offset, size_t bytes);

/* Task-system self test (reference: test/singleGPU/cpp/taskSystem/
 * saxpyCoherenceTest.hip:43-143): every element of `data` (device, int32,
 * n a multiple of 256) goes through two dependent tasks, x*2 then +1, the
 * second pushed by the first through the global queue. */
int FlashMoeTestTaskSystem(FlashMoeHandle h, int32_t* data, int n, void* stream);

/* Runs pre-built FFN2-style tile tasks through the queue as a plain grouped
 * GEMM: out[r, :] = A[r, :] * W2[expert]^T for rows written into the expert
 * buffers by the caller (reference: test/singleGPU/cpp/taskSystem/gemmTest/
 * gemmTest.cpp:69-73).  `rowsPerExpert[E_local]`, `A` bf16 [sum rows, I] host
 * order by expert, `out` bf16 [sum rows, H]; device pointers. */
int FlashMoeTestQueueGemm(FlashMoeHandle h, const uint32_t* rowsPerExpertHost, const void* A,
                          void* out, void* stream);

/* Test hook for the device-side time-outs (the reference has no counterpart: its device waits are
 * unbounded, src/hip/taskSystem/taskManager.h:208-215): a launch that expects one task nobody ever
 * publishes.  Every worker's wait for work runs out after FLASHMOE_TIMEOUT_MS, the kernel records
 * status 1 (a worker found no work for too long) and returns; the context stays usable, the launcher
 * refuses further launches until it is destroyed and created again.  Nothing faults or hangs. */
int FlashMoeTestStall(FlashMoeHandle h, void* stream);

/* The whole layer in one call that allocates nothing (no counterpart in the reference, whose
 * launcher always allocates its scratch in Init, src/hip/launcher/moeKernelLauncher.hip:139-165).
 * For callers that may not touch the device allocator: an engine that has frozen its memory pool,
 * a callback that must not call allocating runtime functions, a process whose memory belongs to
 * another allocator.  All scratch comes from a fixed 32 MiB array inside the library image (held
 * on every GPU that loads the library); a call whose scratch does not fit is rejected with
 * cudaErrorInvalidValue.  Single rank, bf16, device pointers.  config == NULL means the
 * Qwen3-30B-A3B shape, whose 128 expert buffers alone exceed the array, so that call is always
 * rejected: pass the (smaller) layer you run.  The first call on a device does one-time set-up (it
 * may be the moment the 32 MiB become resident there): make it before any stream capture and before
 * the host freezes its memory budget.  Calls share the array: do not let two of them overlap on a
 * GPU.  Every call synchronises `stream` and returns after the layer has finished; a device-side
 * error is reported as cudaErrorUnknown. */
int FlashMoeLaunchNoAlloc(const void* gateWeights, const void* ffn1ExpertWeights,
                          const void* ffn2ExpertWeights, const void* tokens, void* output, int tokensNum,
                          const FlashMoeConfig* config, void* stream);

/* ---------------------------------------------------------------- dense operators
 * The gated feed-forward block of a dense layer or of a shared expert, its gradient, and 4-bit
 * microscaled weights for it (the reference has no counterpart; its experts' FFN is
 * src/hip/kernel/moeKernel.h).  These entries need no handle: every call enqueues its work on `stream`,
 * takes scratch from the caller and can be captured into a CUDA graph; calls with different workspaces
 * may overlap.  Matrices are contiguous, row-major, on the current device, and start on 16 bytes.  Results,
 * scratch and what is kept lie on no other memory of the call (cudaErrorInvalidValue), but for `y`, which may be
 * `x`, in the two forward calls.
 * Results are deterministic: the same call gives the same bits.  Another number of tokens, or a forward
 * call that keeps what the backward pass needs instead of one that does not, may use another kernel, whose
 * sums have another order. */
typedef struct {
  int32_t hiddenSize;       /* H, a multiple of 8 (4-bit weights: 32) */
  int32_t intermediateSize; /* I, a multiple of 8 (4-bit weights: 32) */
  int32_t dtype;            /* 0 bf16, 2 fp16 */
  int32_t reserved[5];      /* zero */
} FlashMoeFfnConfig;

/* Bytes of scratch for a forward (backward == 0) or backward call, and of what a forward call keeps for
 * the backward pass; 0 for an unsupported config. */
size_t FlashMoeFfnWorkspaceBytes(const FlashMoeFfnConfig* config, int64_t tokensNum, int backward);
size_t FlashMoeFfnSavedBytes(const FlashMoeFfnConfig* config, int64_t tokensNum);

/* y[T,H] = (silu(x Wg^T) * (x Wu^T)) W2^T with w13 = [Wg; Wu] [2I,H], w2 [H,I].  `saved`, if not NULL,
 * receives what FlashMoeFfnBackward needs (the projections in 24 bits, and h), and no workspace is needed then.  `y`
 * may be `x`.  The projections, the activation and both products are accumulated in fp32; h = silu(g) * u
 * is rounded to the dtype. */
int FlashMoeFfnForward(const FlashMoeFfnConfig* config, const void* x, const void* w13, const void* w2,
                       void* y, void* saved, void* workspace, size_t workspaceBytes, int64_t tokensNum,
                       void* stream);

/* Gradients of x [T,H], w13 [2I,H] and w2 [H,I] from that of y; each of the three may be NULL.  With no
 * tokens the gradients of the weights are zero.  The gradients of the projections are rounded to the dtype
 * (fp16: infinite beyond 65504, zero below 3e-8) before the last products. */
int FlashMoeFfnBackward(const FlashMoeFfnConfig* config, const void* dy, const void* x, const void* w13,
                        const void* w2, const void* saved, void* dx, void* dw13, void* dw2,
                        void* workspace, size_t workspaceBytes, int64_t tokensNum, void* stream);

/* 4-bit microscaled matrices: E2M1 values, two to a byte (even element low), [batch, rows, cols / 2], and
 * one E8M0 scale per 32 elements of a row in blocks of 512 bytes for 128 rows and 128 columns (the scale of
 * row r and column block c is byte (r % 32) * 16 + (r / 32) * 4 + c), an even number of blocks per 128
 * rows.  cols is a multiple of 32.  FlashMoeMx4ScaleBytes gives the size of the scales, 0 if unsupported. */
size_t FlashMoeMx4ScaleBytes(int64_t batch, int64_t rows, int64_t cols);

/* x (dtype 0 bf16, 1 fp32, 2 fp16; strides in elements, multiples of 16 bytes) to values and scales: the
 * scale is 2^(floor(log2(largest magnitude)) - 2), elements are rounded to nearest even and saturate at 6.
 * A block with a NaN or an infinity stands for NaN. */
int FlashMoeMx4Quantize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols,
                        int64_t batchStride, int64_t rowStride, void* values, void* scales, void* stream);

/* The values that a 4-bit matrix stands for, contiguous. */
int FlashMoeMx4Dequantize(const void* values, const void* scales, int64_t batch, int64_t rows, int64_t cols,
                          int dtype, void* out, void* stream);

/* out[m,n] = a[m,k] b[n,k]^T, accumulated in fp32.  gated != 0: b is a batch of two matrices [2,n,k], gate
 * and up projection, and out = silu(a b0^T) * (a b1^T).  dtype of out: 0 bf16, 1 fp32, 2 fp16.  With m or n
 * above 8388480, n is a multiple of 8 (fp32 results: 4). */
int FlashMoeMx4Matmul(const void* aValues, const void* aScales, const void* bValues, const void* bScales,
                      void* out, int dtype, int64_t m, int64_t n, int64_t k, int gated, void* stream);

/* The block with 4-bit weights (w13 as a batch of two [2,I,H], w2 [H,I]): x and h are quantised on the way. */
size_t FlashMoeMx4FfnWorkspaceBytes(const FlashMoeFfnConfig* config, int64_t tokensNum);
int FlashMoeMx4FfnForward(const FlashMoeFfnConfig* config, const void* x, const void* w13Values,
                          const void* w13Scales, const void* w2Values, const void* w2Scales, void* y,
                          void* workspace, size_t workspaceBytes, int64_t tokensNum, void* stream);

/* First device-side error of the dense operators in this process (0 == none; a bounded wait that ran out,
 * FLASHMOE_TIMEOUT_MS); does not synchronise.  After one, dense calls are refused with cudaErrorUnknown
 * until `reset` != 0 clears it. */
int FlashMoeDenseStatus(uint32_t* code, int reset);

/* Test hooks: products whose loads are left out, so that their waits run out after FLASHMOE_TIMEOUT_MS.
 * Nothing faults or hangs.  FlashMoeTestDenseStall: those of the calling thread's dense calls, until it is
 * turned off; FlashMoeTestFfnStall: those of one forward call. */
int FlashMoeTestDenseStall(int on);
int FlashMoeTestFfnStall(const FlashMoeFfnConfig* config, const void* x, const void* w13, const void* w2,
                         void* y, void* workspace, size_t workspaceBytes, int64_t tokensNum, void* stream);

const char* FlashMoeErrorString(int code);

#ifdef __cplusplus
}
#endif
#endif /* FLASHMOE_C_H_ */

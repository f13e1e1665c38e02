/*
 * Avocado/cuda_backend_ext.h -- additive entry points of the B200 convolution backend.
 *
 * None of these has a counterpart in the reference's include/Avocado/cuda_backend.h; they add what the fixed
 * signatures of that header cannot carry.  No existing signature changes, so a caller that ignores this
 * header keeps working.
 */
#ifndef AVOCADO_CUDA_BACKEND_EXT_H_
#define AVOCADO_CUDA_BACKEND_EXT_H_

#include <Avocado/backend_defs.h>

#ifdef __cplusplus
namespace avocado
{
	namespace backend
	{
		extern "C"
		{
#endif

/* Attaches per-output-channel requantisation scales (float32[K], device memory) to a convolution descriptor.
 * cudaConvolutionImplicitGemmForward uses them when x and w are INT8 and y is INT8:
 *   q[k] = saturate_int8(round_to_nearest_even(activation(alpha1 * float(acc + bias[k]) * scale[k] + alpha2 * z)))
 * Pass AVOCADO_INVALID_DESCRIPTOR to detach.  No counterpart in the reference: its int8 kernel
 * (src/conv2d_implicit_gemm.cu:330-339) has a single scalar alpha and an int32 output only. */
DLL_PUBLIC avStatus_t cudaSetConvolutionQuantization(avConvolutionDescriptor_t desc, const avMemoryDescriptor_t scalesMem);

/* Raw device pointer behind a memory handle, for interoperation with a communication library (the dW
 * all-reduce of the training step).  No counterpart in the reference. */
DLL_PUBLIC avStatus_t cudaGetMemoryPointer(const avMemoryDescriptor_t desc, void **result);

/* cudaStream_t of a context (null for a default context), so a caller can order its own work after the
 * library's.  No counterpart in the reference. */
DLL_PUBLIC avStatus_t cudaGetContextStream(avContextDescriptor_t context, void **result);

/* Waits for the context's stream, then returns and clears the error word that tensor-core kernels set when one
 * of their bounded waits (TMA arrival, MMA completion) gave up: 0 = none.  No counterpart in the reference,
 * whose kernels have no device-side waits. */
DLL_PUBLIC avStatus_t cudaGetLastDeviceStatus(avContextDescriptor_t context, int *result);

/* Failure-detection self test: launches one small kernel that waits, with a limit of `limitMicroseconds`, on a barrier
 * nobody will ever signal.  The wait must run out, the kernel must return normally, bit 5 of the context's device status
 * word must be set (read it with cudaGetLastDeviceStatus) and the context must stay usable.  This exercises, without
 * faulting or hanging the GPU, the path every tensor-core kernel takes when one of its waits gives up.
 * No counterpart in the reference. */
DLL_PUBLIC avStatus_t cudaRunBoundedWaitSelfTest(avContextDescriptor_t context, int limitMicroseconds);

/* The same self test with the kernel pointed at the error word of cudaConvolutionWinogradFusedForwardNoAlloc's fixed
 * array on the context's device (shared by all contexts of that device) instead of the context's own word: the report
 * must surface through cudaGetLastDeviceStatus all the same.  Returns AVOCADO_STATUS_BAD_PARAM while no call of that
 * entry point has been made on the device.  No counterpart in the reference. */
DLL_PUBLIC avStatus_t cudaRunBoundedWaitSelfTestNoAlloc(avContextDescriptor_t context, int limitMicroseconds);

/* Switches fusion inside the non-fused Winograd pipeline on or off for one context; `flags` is 0 or a combination of the
 * two values below.  The call sequence of the reference stays as it is (ref app/CudaBackend.cu:401-420: weight transform,
 * input transform, cudaGemmBatched, cudaWinogradOutputTransform); what changes is how many kernels it becomes.
 *
 * AVOCADO_WINOGRAD_FUSE_WEIGHTS: a cudaWinogradWeightTransform of a 3x3 kernel is held back and rides along in the launch
 *   of the cudaWinogradInputTransform that follows it (a few blocks at the front of that grid).  Its result is written as
 *   usual, bit for bit; only the separate launch, a few microseconds of latency for 74 KB of weights, disappears.
 * AVOCADO_WINOGRAD_FUSE_OUTPUT: a cudaGemmBatched call that is the contraction of an F(4x4,3x3) pipeline (36 planes, (N, T),
 *   float16 / bfloat16, alpha 1, beta 0) is held back; if the next call on the context is the cudaWinogradOutputTransform
 *   of exactly the tensor it was to write, ONE kernel contracts and transforms and the transform-domain products are
 *   NEVER WRITTEN to the caller's workspace -- the workspace keeps whatever it held.  That is the one observable
 *   difference, and the reason fusion is opt-in.
 *
 * Any other call on the context (another operator, a copy, a synchronisation, the end of a capture, destruction of the
 * context or of any memory descriptor) launches what was held back first, in the order it was asked for, so nothing
 * else can tell that it was deferred.  Default contexts cannot fuse.  No counterpart in the reference, whose calls always
 * run as one kernel each (src/winograd_nonfused.cu:608-651, src/gemm.cpp:126-209, src/winograd_nonfused.cu:703-777). */
#define AVOCADO_WINOGRAD_FUSE_WEIGHTS 1
#define AVOCADO_WINOGRAD_FUSE_OUTPUT 2
DLL_PUBLIC avStatus_t cudaContextSetWinogradFusion(avContextDescriptor_t context, int flags);

/* Orders two contexts on the device without blocking the host: everything enqueued on `waiting` after this call runs
 * after everything enqueued on `signalling` before it.  The reference has only cudaSynchronizeWithContext, which blocks
 * the calling thread; with this a caller can run independent steps on two contexts (for instance the weight transform
 * next to the input transform of the same layer) and join them.  Inside a capture (below) the second context's work
 * becomes a parallel branch of the captured graph: let it wait for the capturing context first, and let the capturing
 * context wait for it before the capture ends.  No counterpart in the reference. */
DLL_PUBLIC avStatus_t cudaContextWaitForContext(avContextDescriptor_t waiting, avContextDescriptor_t signalling);

/* Records the work that API calls enqueue on a context instead of running it, and replays it later with one launch.
 * Between Begin and End every call on `context` is captured into a CUDA graph; host scalars (alpha, beta) are read at
 * capture time and baked in; the memory handles used must stay alive while the graph exists.  Run the same call
 * sequence once before capturing, so that one-time set-up (kernel attributes, scratch allocation) is already done.
 * The default context cannot capture.  No counterpart in the reference, which launches kernel by kernel. */
DLL_PUBLIC avStatus_t cudaContextBeginCapture(avContextDescriptor_t context);
DLL_PUBLIC avStatus_t cudaContextEndCapture(avContextDescriptor_t context, av_int64 *graph);
DLL_PUBLIC avStatus_t cudaContextLaunchGraph(avContextDescriptor_t context, av_int64 graph);
DLL_PUBLIC avStatus_t cudaDestroyCapturedGraph(av_int64 graph);

/* Size of the fixed scratch array behind cudaConvolutionWinogradFusedForwardNoAlloc.  Every GPU on which the library's
 * device code is loaded holds this much device memory (plus 256 bytes) until the process exits. */
#define AVOCADO_NO_ALLOC_SCRATCH_BYTES (8u * 1024u * 1024u)

/* cudaConvolutionWinogradFusedForward for callers that may not cause a device allocation -- a host that has given
 * all GPU memory to its own pool, a latency-bound loop that cannot absorb the synchronisation cudaMalloc implies, a
 * process under a no-allocation-after-start-up rule.  Same arguments and same result, but the transform-domain
 * tensors live in a fixed array inside the library image instead of the context's cudaMalloc'ed scratch, and nothing
 * on this path allocates or frees.  It has no counterpart in the reference (whose fused entry point takes no
 * workspace and allocates none because it was never finished).
 *  - float16 / bfloat16 tensors, 3x3 kernel, unit stride and dilation, C and K multiples of 8, y the size of x;
 *    anything else returns UNSUPPORTED_DATATYPE / NOT_SUPPORTED.
 *  - 32 * (K*C + tiles*C) bytes, tiles = N*ceil(H/2)*ceil(W/2), must fit AVOCADO_NO_ALLOC_SCRATCH_BYTES (plus
 *    32 * tiles*K when y, z or the bias is not 16 / 16 / 4-byte aligned, because the products are then written out);
 *    a larger problem returns AVOCADO_STATUS_BAD_PARAM and launches nothing.
 *  - The first call on a device resolves the array's device address and, with the runtime's lazy loading, is when the
 *    driver places the array and the kernels on the device: make it at start-up, before the host's own pool takes the
 *    remaining memory and before any stream capture.
 *  - All calls on one device share the array: calls that overlap on the GPU race.  It keeps the last call's contents;
 *    the only part that must start at zero, the kernels' 256-byte error word, starts as zero and is cleared when
 *    cudaGetLastDeviceStatus (of any context on the device) reads it, so a report is never lost. */
DLL_PUBLIC avStatus_t cudaConvolutionWinogradFusedForwardNoAlloc(avContextDescriptor_t context, const avConvolutionDescriptor_t config, const void *alpha1,
		const avTensorDescriptor_t xDesc, const avMemoryDescriptor_t xMem, const avTensorDescriptor_t wDesc, const avMemoryDescriptor_t wMem,
		const avTensorDescriptor_t bDesc, const avMemoryDescriptor_t bMem, const void *alpha2, const avTensorDescriptor_t zDesc,
		const avMemoryDescriptor_t zMem, const void *beta, const avTensorDescriptor_t yDesc, avMemoryDescriptor_t yMem, avActivationType_t activation);

/* ------------------------------------------------------------------------------------------------------------
 * 8-bit floating point with block scales: the quantised-inference path beside cudaGemm.  No counterpart in the reference.
 *
 * A quantised tensor is a pair: codes (AVOCADO_DTYPE_FLOAT8_E4M3) and float32 scales; a code q of a block with scale s stands
 * for q * s.  Blocks lie along the last dimension, 128 elements each, the last one shorter when the extent is not a multiple
 * of 128; the other dimensions are taken together as rows.  Two forms, told apart by the shape of the scales:
 *   1 x 128    scales [rows..., ceil(C / 128)]              activations
 *   128 x 128  scales [ceil(rows / 128), ceil(C / 128)]     weights
 * With a = max(amax, 2^-100), amax being the largest magnitude in the block, the scale is a / 448 and the codes are
 * round_to_nearest_even(x * (448 / a)), all in float32.  A block of zeros gets the scale of 2^-100 and zero codes.  A NaN
 * makes its whole block NaN (scale and codes); an infinity gives an infinite scale, its own code NaN and zeros beside it.
 *
 * All three calls: memory blocks must hold at least what their descriptor says and lie on the context's device, and an output
 * must not overlap an input or another output except where stated (AVOCADO_STATUS_BAD_PARAM otherwise).  No scratch memory is
 * used and results do not depend on the order in which blocks run.  Tensors without elements succeed and write nothing.
 * ------------------------------------------------------------------------------------------------------------ */

/* x (float16, bfloat16, float32; any rank, rows of at most 2^30 elements) -> codes y (float8_e4m3, the shape of x) and scales,
 * in the form that the shape of scaleDesc asks for. */
DLL_PUBLIC avStatus_t cudaQuantizeBlocks(avContextDescriptor_t context, const avTensorDescriptor_t xDesc, const avMemoryDescriptor_t xMem,
		const avTensorDescriptor_t yDesc, avMemoryDescriptor_t yMem, const avTensorDescriptor_t scaleDesc, avMemoryDescriptor_t scaleMem);

/* Root-mean-square norm over the last dimension, with the residual's addition in front and the quantiser behind it, in one call:
 *   h = x + z;   y = h / sqrt(mean(h^2) + epsilon) * gamma;   (codes, scales) = quantise(y) in 1 x 128 blocks
 * x, z, h: float16, bfloat16 or float32, all of xDesc's type and shape, rows of at most 2^20 elements; gamma: float32 [C].  z is
 * optional (AVOCADO_INVALID_DESCRIPTOR: h = x); h is rounded once into hMem when that is given, and may be stored over x or
 * over z (the same memory, not a part of it).  Arithmetic is float32 and y is quantised without having been rounded before;
 * so is the sum of squares, which should stay below 2^128: a finite row that reaches it (from a root-mean-square of 1.8e19 / sqrt(C) on)
 * counts as infinitely long, its y is 0 (zero codes, the scale of 2^-100) and its h as ever.  Squares below 2^-126 lose bits, which
 * shows where C * epsilon is as small.  epsilon must be positive and finite as a float32. */
DLL_PUBLIC avStatus_t cudaRmsNormQuantize(avContextDescriptor_t context, const avTensorDescriptor_t xDesc, const avMemoryDescriptor_t xMem,
		const avMemoryDescriptor_t zMem, avMemoryDescriptor_t hMem, const avTensorDescriptor_t gammaDesc, const avMemoryDescriptor_t gammaMem, double epsilon,
		const avTensorDescriptor_t yDesc, avMemoryDescriptor_t yMem, const avTensorDescriptor_t scaleDesc, avMemoryDescriptor_t scaleMem);

/* C = alpha * A * B^T + beta * C for quantised A [M, K] in 1 x 128 blocks and B [N, K] in 128 x 128 blocks:
 *   C[m, n] = alpha * sum over g of aScale[m, g] * bScale[n / 128, g] * (sum over k in block g of A[m, k] * B[n, k]) + beta * C[m, n]
 * aDesc, bDesc: float8_e4m3; scales float32 [M, ceil(K / 128)] and [ceil(N / 128), ceil(K / 128)]; C float16, bfloat16 or
 * float32 [M, N]; extents up to 2^30; alpha and beta float.  aOp must be N and bOp T (AVOCADO_STATUS_NOT_SUPPORTED otherwise).  Sums are float32,
 * rounded once into C.  C is not read when beta is 0.  The product aScale * bScale of a block is formed first, in float32: it should be 0 or a
 * normal number (2^-126 to 2^128).  A smaller one costs up to 2^-150 * 128 * 448^2 < 2^-125 of absolute error for its block; a larger
 * one is infinite, and so is what it adds, or NaN where the block's sum is 0.  Row pitches of 16 bytes (K a multiple of 16, A and B on 16-byte
 * boundaries) are copied by the tensor memory accelerator; other pitches are correct and slower. */
DLL_PUBLIC avStatus_t cudaGemmBlockScaled(avContextDescriptor_t context, avGemmOperation_t aOp, avGemmOperation_t bOp, const void *alpha,
		const avTensorDescriptor_t aDesc, const avMemoryDescriptor_t aMem, const avTensorDescriptor_t aScaleDesc, const avMemoryDescriptor_t aScaleMem,
		const avTensorDescriptor_t bDesc, const avMemoryDescriptor_t bMem, const avTensorDescriptor_t bScaleDesc, const avMemoryDescriptor_t bScaleMem,
		const void *beta, const avTensorDescriptor_t cDesc, avMemoryDescriptor_t cMem);

#ifdef __cplusplus
		} /* extern "C" */
	} /* namespace backend */
} /* namespace avocado */
#endif

#endif /* AVOCADO_CUDA_BACKEND_EXT_H_ */

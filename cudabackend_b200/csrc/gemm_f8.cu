/*
 * gemm_f8.cu -- cudaGemmBlockScaled: C[M, N] = alpha * A * B^T + beta * C for e4m3 operands with float32 scales, A[M, K] in
 * 1 x 128 blocks and B[N, K] in 128 x 128 blocks.  No counterpart in the reference (its only 8-bit product is int8 -> int32,
 * src/gemm.cpp:42-57).
 *
 *   C[m, n] = alpha * sum_g aScale[m, g] * bScale[n / 128, g] * P_g[m, n] + beta * C[m, n],   P_g = sum over block g of A * B
 */
#include <Avocado/cuda_backend_ext.h>

#include "block_scaled.hpp"
#include "device_utils.cuh"
#include "objects.hpp"
#include "umma.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace
{
	using namespace avocado::backend;
	using namespace avocado::backend::b200;
	using namespace bk;

	struct ScaledGemm
	{
			int M, N, K;
			int blocks; /* blocks of 128 along K */
			const uint8_t *a, *b;
			const float *a_scale, *b_scale;
			void *c;
			float alpha, beta;
	};

	/* Plain form on the CUDA cores: a block computes 64 x 64 results, 16 per thread, from 32 elements of K at a time. */
	template<typename T>
	__global__ void __launch_bounds__(256) kernel_gemm_f8_simt(ScaledGemm p)
	{
		constexpr int kTile = 64, kStep = 32;
		__shared__ float a_s[kStep][kTile + 1], b_s[kStep][kTile + 1];
		chain_release();
		chain_wait();
		const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
		const long long tiles_n = (p.N + kTile - 1) / kTile;
		const long long m0 = blockIdx.x / tiles_n * kTile, n0 = blockIdx.x % tiles_n * kTile;
		float acc[4][4] = { };
		for (int g = 0; g < p.blocks; g++)
		{
			float part[4][4] = { };
			for (int k0 = g * kScaleBlock; k0 < min(p.K, (g + 1) * kScaleBlock); k0 += kStep)
			{
				for (int i = threadIdx.x; i < kTile * kStep; i += 256)
				{
					const int r = i / kStep, k = i % kStep;
					__nv_fp8_e4m3 va, vb;
					va.__x = (m0 + r < p.M and k0 + k < p.K) ? p.a[(m0 + r) * p.K + k0 + k] : 0;
					vb.__x = (n0 + r < p.N and k0 + k < p.K) ? p.b[(n0 + r) * p.K + k0 + k] : 0;
					a_s[k][r] = static_cast<float>(va);
					b_s[k][r] = static_cast<float>(vb);
				}
				__syncthreads();
				for (int k = 0; k < kStep; k++)
					for (int i = 0; i < 4; i++)
						for (int j = 0; j < 4; j++)
							part[i][j] = fmaf(a_s[k][ty * 4 + i], b_s[k][tx + j * 16], part[i][j]);
				__syncthreads();
			}
			for (int i = 0; i < 4; i++)
			{
				const long long m = m0 + ty * 4 + i;
				const float sa = m < p.M ? p.a_scale[m * p.blocks + g] : 0.0f;
				const float s = sa * p.b_scale[n0 / kScaleBlock * p.blocks + g];
				for (int j = 0; j < 4; j++)
					acc[i][j] = fmaf(part[i][j], s, acc[i][j]);
			}
		}
		T *c = reinterpret_cast<T*>(p.c);
		for (int i = 0; i < 4; i++)
			for (int j = 0; j < 4; j++)
			{
				const long long m = m0 + ty * 4 + i, n = n0 + tx + j * 16;
				if (m < p.M and n < p.N)
				{
					const float old = p.beta != 0.0f ? p.beta * to_compute(c[m * p.N + n]) : 0.0f;
					c[m * p.N + n] = from_compute<T>(fmaf(p.alpha, acc[i][j], old));
				}
			}
	}

	template<typename T>
	avStatus_t launch(ContextObject &ctx, const ScaledGemm &p)
	{
		const long long grid = static_cast<long long>((p.M + 63) / 64) * ((p.N + 63) / 64);
		if (grid > 0x7FFFFFFFll)
			return AVOCADO_STATUS_NOT_SUPPORTED;
		const cudaError_t launched = launch_chained(kernel_gemm_f8_simt<T>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, ctx.getStream(), p);
		return launched != cudaSuccess ? convertStatus(launched) : checkForErrors();
	}
}

namespace avocado
{
	namespace backend
	{
		avStatus_t cudaGemmBlockScaled(avContextDescriptor_t context, avGemmOperation_t aOp, avGemmOperation_t bOp, const void *alpha,
				const avTensorDescriptor_t aDesc, const avMemoryDescriptor_t aMem, const avTensorDescriptor_t aScaleDesc, const avMemoryDescriptor_t aScaleMem,
				const avTensorDescriptor_t bDesc, const avMemoryDescriptor_t bMem, const avTensorDescriptor_t bScaleDesc, const avMemoryDescriptor_t bScaleMem,
				const void *beta, const avTensorDescriptor_t cDesc, avMemoryDescriptor_t cMem)
		{
			AVOCADO_API_BEGIN
				ContextObject &ctx = getContext(context);
				const TensorObject &a = getTensor(aDesc);
				const TensorObject &b = getTensor(bDesc);
				const TensorObject &c = getTensor(cDesc);
				const TensorObject &a_scale = getTensor(aScaleDesc);
				const TensorObject &b_scale = getTensor(bScaleDesc);
				if (is_transpose(aOp) or not is_transpose(bOp))
					return AVOCADO_STATUS_NOT_SUPPORTED;
				if (a.dtype != AVOCADO_DTYPE_FLOAT8_E4M3 or b.dtype != AVOCADO_DTYPE_FLOAT8_E4M3 or a_scale.dtype != AVOCADO_DTYPE_FLOAT32
						or b_scale.dtype != AVOCADO_DTYPE_FLOAT32)
					return AVOCADO_STATUS_UNSUPPORTED_DATATYPE;
				if (c.dtype != AVOCADO_DTYPE_FLOAT16 and c.dtype != AVOCADO_DTYPE_BFLOAT16 and c.dtype != AVOCADO_DTYPE_FLOAT32)
					return AVOCADO_STATUS_UNSUPPORTED_DATATYPE;
				for (const TensorObject *t : { &a, &b, &c, &a_scale, &b_scale })
					if (t->nb_dims != 2 or not valid_extents(*t))
						return AVOCADO_STATUS_BAD_PARAM;
				ScaledGemm p;
				p.M = a.dims[0];
				p.N = b.dims[0];
				p.K = a.dims[1];
				p.blocks = scale_blocks(p.K);
				if (b.dims[1] != p.K or c.dims[0] != p.M or c.dims[1] != p.N or a_scale.dims[0] != p.M or a_scale.dims[1] != p.blocks
						or b_scale.dims[0] != scale_blocks(p.N) or b_scale.dims[1] != p.blocks)
					return AVOCADO_STATUS_BAD_PARAM;
				if (p.M == 0 or p.N == 0)
					return AVOCADO_STATUS_SUCCESS;
				Operand ao, bo, co, as, bs;
				if (not get_operand(ao, ctx, aMem, a) or not get_operand(bo, ctx, bMem, b) or not get_operand(co, ctx, cMem, c)
						or not get_operand(as, ctx, aScaleMem, a_scale) or not get_operand(bs, ctx, bScaleMem, b_scale))
					return AVOCADO_STATUS_BAD_PARAM;
				if (co.overlaps(ao) or co.overlaps(bo) or co.overlaps(as) or co.overlaps(bs))
					return AVOCADO_STATUS_BAD_PARAM;
				p.a = ao.ptr;
				p.b = bo.ptr;
				p.c = co.ptr;
				p.a_scale = reinterpret_cast<const float*>(as.ptr);
				p.b_scale = reinterpret_cast<const float*>(bs.ptr);
				p.alpha = getAlphaValue<float>(alpha);
				p.beta = getBetaValue<float>(beta);
				ctx.setDevice();
				switch (c.dtype)
				{
					case AVOCADO_DTYPE_FLOAT16:
						return launch<half>(ctx, p);
					case AVOCADO_DTYPE_BFLOAT16:
						return launch<__nv_bfloat16>(ctx, p);
					default:
						return launch<float>(ctx, p);
				}
			AVOCADO_API_END
		}
	} /* namespace backend */
} /* namespace avocado */

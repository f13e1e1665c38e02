/*
 * quantize.cu -- cudaQuantizeBlocks and cudaRmsNormQuantize: what turns 16-bit or float32 tensors into the e4m3 codes and
 * float32 block scales that cudaGemmBlockScaled reads.  No counterpart in the reference.
 *
 *   block of 128 elements:  amax = max |x|,  a = max(amax, 2^-100),  scale = a / 448,  code = e4m3_rne(x * (448 / a))
 *   norm:                   h = x + z,  y = h * (1 / sqrt(mean(h^2) + eps)) * gamma,  then the same on y
 *
 * Both move every element once: the inputs are read into registers, reduced, scaled and written from there.  A block of 128
 * elements belongs to 16 neighbouring lanes (half a warp) with eight elements each: 16 bytes of a 16-bit tensor per load, 8
 * bytes of codes per store; up to four blocks of a half-warp share the shuffles of their maxima and the divisions.  Magnitudes
 * are compared as integers (the bit pattern without its sign grows with the magnitude and puts NaN above infinity), so one
 * NaN reaches its block's scale.  The product x * (448 / a) is at most 448 * (1 + 2^-23), which rounds to 448, so nothing
 * saturates.  All arithmetic is float32; the only other roundings are those of the codes and of the stored sum h.
 *
 * Bound: HBM.  Measured in graphs (of 6566 GB/s copied): 4096 x 8192 bfloat16 to 1 x 128 blocks 20.0 us (102 MB, 0.77), 8192 x 8192 to 128
 * x 128 blocks 33.6 us (201 MB, 0.91), norm of 8192 x 8192 with residual 81 us (470 MB, 0.88), norm of 50176 x 264 float16 13.7 us (40 MB,
 * 0.44: instructions, over 200 per row; a block's work does not shrink with its 8 of 128 columns).
 * Not bound by HBM: rows that cannot be moved in 16-byte pieces, whose elements and codes go one by one (8192 x 8191 bfloat16 to 1 x 128
 * blocks 150 us, 0.20, float32 62 us, 0.82; norm with residual 169 us, 0.42), and norms of more than 8192 columns, whose blocks of 512 or
 * 1024 threads leave a thread 64 registers for four blocks (4096 x 16384 bfloat16 with residual 126 us, 0.57; float32 160 us, 0.83).
 */
#include <Avocado/cuda_backend_ext.h>

#include "block_scaled.hpp"
#include "device_utils.cuh"
#include "objects.hpp"

#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

namespace
{
	using namespace avocado::backend;
	using namespace avocado::backend::b200;
	using namespace bk;

	constexpr int kLanes = 16;   /* lanes that share one block of 128 elements */
	constexpr int kPerLane = 8;  /* elements of it per lane */
	constexpr int kThreads = 256;
	constexpr int kMaxQuantizedRow = 1 << 30; /* column indices, rounded up to whole blocks, stay in 32 bits */
	constexpr int kMaxNormedRow = 1 << 20;    /* a thread adds up at most 1024 squares: the sum keeps about 20 of its 24 bits */
	constexpr unsigned kFullWarp = 0xFFFFFFFFu;

	__device__ __forceinline__ uint32_t magnitude_bits(float x)
	{
		return __float_as_uint(x) & 0x7FFFFFFFu;
	}
	/* the clamped maximum as a float; NaN passes (its bit pattern is above that of 2^-100) */
	__device__ __forceinline__ float clamped_amax(uint32_t bits)
	{
		return __uint_as_float(max(bits, __float_as_uint(kSmallestAmax)));
	}
	/* The maxima of up to four blocks, each held in parts by the 16 lanes of a half-warp, reduced together: every exchange halves
	 * what a lane is responsible for (five shuffles for four blocks instead of sixteen), so that lane l ends with block
	 * item_of(l)'s maximum and the two divisions are done once for all of them. */
	template<int ITEMS>
	struct BlockFactors
	{
			static_assert(ITEMS >= 1 and ITEMS <= 4, "blocks of one half-warp");
			float factor; /* 448 / max(amax, 2^-100) of block item_of(lane) */
			float scale;  /* max(amax, 2^-100) / 448 */

			__device__ __forceinline__ explicit BlockFactors(const uint32_t (&bits)[ITEMS])
			{
				const int l = threadIdx.x % kLanes;
				uint32_t own = bits[0];
				if constexpr (ITEMS == 1)
					own = max(own, __shfl_xor_sync(kFullWarp, own, 8));
				else if constexpr (ITEMS == 2)
				{
					const uint32_t other = (l & 8) ? bits[0] : bits[1];
					own = (l & 8) ? bits[1] : bits[0];
					own = max(own, __shfl_xor_sync(kFullWarp, other, 8));
				}
				else
				{
					const uint32_t last = ITEMS == 4 ? bits[ITEMS - 1] : 0u;
					const uint32_t other0 = (l & 8) ? bits[0] : bits[2], other1 = (l & 8) ? bits[1] : last;
					uint32_t own0 = (l & 8) ? bits[2] : bits[0], own1 = (l & 8) ? last : bits[1];
					own0 = max(own0, __shfl_xor_sync(kFullWarp, other0, 8));
					own1 = max(own1, __shfl_xor_sync(kFullWarp, other1, 8));
					const uint32_t other = (l & 4) ? own0 : own1;
					own = (l & 4) ? own1 : own0;
					own = max(own, __shfl_xor_sync(kFullWarp, other, 4));
				}
				if constexpr (ITEMS <= 2)
					own = max(own, __shfl_xor_sync(kFullWarp, own, 4));
				own = max(own, __shfl_xor_sync(kFullWarp, own, 2));
				own = max(own, __shfl_xor_sync(kFullWarp, own, 1));
				const float amax = clamped_amax(own);
				factor = kLargestE4m3 / amax;
				scale = amax / kLargestE4m3;
			}
			/* the block whose values a lane holds, and the lane that stores them */
			__device__ __forceinline__ static int item_of(int l)
			{
				return ITEMS == 1 ? 0 : ITEMS == 2 ? l / 8 : l / 4;
			}
			__device__ __forceinline__ static bool stores(int l)
			{
				return l % (ITEMS == 1 ? 16 : ITEMS == 2 ? 8 : 4) == 0 and item_of(l) < ITEMS;
			}
			__device__ __forceinline__ float factor_of(int item) const
			{
				return __shfl_sync(kFullWarp, factor, item * (ITEMS == 2 ? 8 : 4), kLanes);
			}
	};
	__device__ __forceinline__ uint32_t four_codes(const float *x, float r)
	{
		const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[0], r), __fmul_rn(x[1], r)), __NV_SATFINITE, __NV_E4M3);
		const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[2], r), __fmul_rn(x[3], r)), __NV_SATFINITE, __NV_E4M3);
		return low | (high << 16);
	}

	/* The eight elements of lane `l` of the block that starts at column `first`: consecutive ones where rows can be moved in
	 * 16-byte pieces (VEC), every 16th otherwise, so that neighbouring lanes touch neighbouring elements either way. */
	template<bool VEC>
	__device__ __forceinline__ int column_of(int first, int l, int i)
	{
		return VEC ? first + l * kPerLane + i : first + l + i * kLanes;
	}
	/* the same as they are stored, for kernels that hold many at once; positions past the end hold zeros */
	template<bool VEC, typename T>
	__device__ __forceinline__ void load_eight(Vec<T, kPerLane> &v, const T *row, int first, int l, int columns)
	{
#pragma unroll
		for (int i = 0; i < kPerLane; i++)
			v.v[i] = from_compute<T>(0.0f);
		if constexpr (VEC)
		{
			const int column = first + l * kPerLane;
			if (column < columns)
			{
				constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
#pragma unroll
				for (int j = 0; j < kPerLane; j += kPiece)
					*reinterpret_cast<Vec<T, kPiece>*>(&v.v[j]) = load_vec<T, kPiece>(row + column + j);
			}
		}
		else
		{
#pragma unroll
			for (int i = 0; i < kPerLane; i++)
			{
				const int column = column_of<VEC>(first, l, i);
				if (column < columns)
					v.v[i] = row[column];
			}
		}
	}
	template<bool VEC, typename T>
	__device__ __forceinline__ void load_eight(float (&v)[kPerLane], const T *row, int first, int l, int columns)
	{
		if constexpr (VEC)
		{
			const int column = first + l * kPerLane;
			if (column < columns) /* VEC: columns is a multiple of eight */
			{
				constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
#pragma unroll
				for (int j = 0; j < kPerLane; j += kPiece)
				{
					const Vec<T, kPiece> piece = load_vec<T, kPiece>(row + column + j);
#pragma unroll
					for (int i = 0; i < kPiece; i++)
						v[j + i] = to_compute(piece.v[i]);
				}
			}
			else
			{
#pragma unroll
				for (int i = 0; i < kPerLane; i++)
					v[i] = 0.0f;
			}
		}
		else
		{
#pragma unroll
			for (int i = 0; i < kPerLane; i++)
			{
				const int column = column_of<VEC>(first, l, i);
				v[i] = column < columns ? to_compute(row[column]) : 0.0f;
			}
		}
	}
	template<bool VEC, typename T>
	__device__ __forceinline__ void store_eight(T *row, const float (&v)[kPerLane], int first, int l, int columns)
	{
		if constexpr (VEC)
		{
			const int column = first + l * kPerLane;
			if (column < columns)
			{
				constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
#pragma unroll
				for (int j = 0; j < kPerLane; j += kPiece)
				{
					Vec<T, kPiece> piece;
#pragma unroll
					for (int i = 0; i < kPiece; i++)
						piece.v[i] = from_compute<T>(v[j + i]);
					store_vec<T, kPiece>(row + column + j, piece);
				}
			}
		}
		else
		{
#pragma unroll
			for (int i = 0; i < kPerLane; i++)
			{
				const int column = column_of<VEC>(first, l, i);
				if (column < columns)
					row[column] = from_compute<T>(v[i]);
			}
		}
	}
	template<bool VEC>
	__device__ __forceinline__ void store_codes(uint8_t *row, const float (&v)[kPerLane], float r, int first, int l, int columns)
	{
		const uint2 codes = make_uint2(four_codes(v, r), four_codes(v + 4, r));
		if constexpr (VEC)
		{
			const int column = first + l * kPerLane;
			if (column < columns)
				*reinterpret_cast<uint2*>(row + column) = codes;
		}
		else
		{
#pragma unroll
			for (int i = 0; i < kPerLane; i++)
			{
				const int column = column_of<VEC>(first, l, i);
				if (column < columns)
					row[column] = static_cast<uint8_t>((i < 4 ? codes.x : codes.y) >> (8 * (i % 4)));
			}
		}
	}
	/* the largest magnitude as an integer; max.NaN keeps a NaN, whose positive pattern is above every number's */
	template<bool PACKED>
	__device__ __forceinline__ uint32_t largest_magnitude(const float (&v)[kPerLane])
	{
		if constexpr (not PACKED)
		{
			uint32_t bits = 0;
#pragma unroll
			for (int i = 0; i < kPerLane; i++)
				bits = max(bits, magnitude_bits(v[i]));
			return bits;
		}
		float largest = fabsf(v[0]);
#pragma unroll
		for (int i = 1; i < kPerLane; i++)
			asm("max.NaN.f32 %0, %0, %1;" : "+f"(largest) : "f"(fabsf(v[i])));
		return __float_as_uint(largest) & 0x7FFFFFFFu;
	}
	/* two products, each rounded like a product of its own, in one instruction */
	__device__ __forceinline__ void multiply_pair(float &x0, float &x1, float y0, float y1)
	{
		asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(x0), "+f"(x1) : "f"(y0), "f"(y1));
	}
	__device__ __forceinline__ void square_pair(float &sum0, float &sum1, float x0, float x1)
	{
		asm("{\n\t.reg .b64 s, x;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 x, {%2, %3};\n\tfma.rn.f32x2 s, x, x, s;\n\tmov.b64 {%0, %1}, s;\n\t}" : "+f"(sum0), "+f"(sum1) : "f"(x0), "f"(x1));
	}

	/* The largest magnitude of raw elements as an integer; two 16-bit patterns are compared at once. */
	__device__ __forceinline__ uint32_t raw_max(const Vec<float, kPerLane> &v, uint32_t bits)
	{
#pragma unroll
		for (int i = 0; i < kPerLane; i++)
			bits = max(bits, magnitude_bits(v.v[i]));
		return bits;
	}
	template<typename T>
	__device__ __forceinline__ uint32_t raw_max(const Vec<T, kPerLane> &v, uint32_t bits)
	{
		const uint32_t *pairs = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
		for (int i = 0; i < kPerLane / 2; i++)
			bits = __vmaxu2(bits, pairs[i] & 0x7FFF7FFFu);
		return bits;
	}
	template<typename T>
	__device__ __forceinline__ uint32_t float_bits(uint32_t bits) /* of the larger half */
	{
		if constexpr (sizeof(T) == 4)
			return bits;
		else
		{
			const uint16_t largest = static_cast<uint16_t>(max(bits & 0xFFFFu, bits >> 16));
			return __float_as_uint(to_compute(*reinterpret_cast<const T*>(&largest)));
		}
	}
	template<bool VEC, typename T>
	__device__ __forceinline__ void store_codes(uint8_t *row, const Vec<T, kPerLane> &v, float r, int first, int l, int columns)
	{
		float x[kPerLane];
#pragma unroll
		for (int i = 0; i < kPerLane; i++)
			x[i] = to_compute(v.v[i]);
		store_codes<VEC>(row, x, r, first, l, columns);
	}

	/* ---- 1 x 128 blocks: half a warp per block, no block-wide step ------------------------------------------------
	 * A half-warp takes kAtOnce blocks, one after every sixteenth, and requests all of them before it works on the first, so that
	 * an SM has 64 KB (16-bit) on the way; positions advance by addition, the only division is the first. */
	constexpr int kAtOnce = 4;
	constexpr int kHalfWarps = kThreads / kLanes;

	struct BlockAt
	{
			long long row;
			int block;

			__device__ __forceinline__ void advance(long long rows, int step, int blocks)
			{
				row += rows;
				block += step;
				if (block >= blocks)
				{
					block -= blocks;
					row++;
				}
			}
	};

	template<typename T, bool VEC>
	__global__ void __launch_bounds__(kThreads) kernel_quantize_rows(const T *__restrict__ x, uint8_t *__restrict__ y, float *__restrict__ scales,
			long long total, int columns, int blocks, long long strideRows, int strideBlocks)
	{
		chain_release();
		chain_wait();
		const int l = threadIdx.x % kLanes;
		long long b = static_cast<long long>(blockIdx.x) * (kHalfWarps * kAtOnce) + threadIdx.x / kLanes;
		BlockAt at;
		at.row = b / blocks;
		at.block = static_cast<int>(b - at.row * blocks);
		const int next_rows = kHalfWarps / blocks, next_blocks = kHalfWarps % blocks;
		for (long long first = b - threadIdx.x / kLanes; first < total; first += static_cast<long long>(gridDim.x) * (kHalfWarps * kAtOnce))
		{
			Vec<T, kPerLane> v[kAtOnce];
			long long offset[kAtOnce];
			int column[kAtOnce];
			BlockAt a = at;
#pragma unroll
			for (int i = 0; i < kAtOnce; i++)
			{
				const bool inside = b + i * kHalfWarps < total;
				offset[i] = inside ? a.row * columns : 0;
				column[i] = inside ? a.block * kScaleBlock : columns;
				load_eight<VEC>(v[i], x + offset[i], column[i], l, columns);
				a.advance(next_rows, next_blocks, blocks);
			}
			uint32_t bits[kAtOnce];
#pragma unroll
			for (int i = 0; i < kAtOnce; i++)
				bits[i] = float_bits<T>(raw_max(v[i], 0u));
			const BlockFactors<kAtOnce> f(bits);
#pragma unroll
			for (int i = 0; i < kAtOnce; i++)
				store_codes<VEC>(y + offset[i], v[i], f.factor_of(i), column[i], l, columns);
			const long long own = b + f.item_of(l) * kHalfWarps;
			if (f.stores(l) and own < total)
				scales[own] = f.scale;
			b += static_cast<long long>(gridDim.x) * (kHalfWarps * kAtOnce);
			at.advance(strideRows, strideBlocks, blocks);
		}
	}

	/* ---- 128 x 128 blocks: one thread block each, held in registers between the maximum and the codes ------------------
	 * as stored, not as float32: 80 registers instead of 106, 32 KB per block on the way (8192 x 8192 bfloat16: 72 -> 35 us) */
	template<typename T, bool VEC>
	__global__ void __launch_bounds__(kThreads) kernel_quantize_squares(const T *__restrict__ x, uint8_t *__restrict__ y, float *__restrict__ scales,
			long long total, long long rows, int columns, int blocks)
	{
		constexpr int kRowsPerPass = kThreads / kLanes;
		constexpr int kPasses = kScaleBlock / kRowsPerPass;
		__shared__ uint32_t warp_max[2][kThreads / 32];
		chain_release();
		chain_wait();
		const int l = threadIdx.x % kLanes;
		int turn = 0;
		for (long long b = blockIdx.x; b < total; b += gridDim.x, turn ^= 1)
		{
			const long long block_row = b / blocks;
			const int column = static_cast<int>(b - block_row * blocks) * kScaleBlock;
			const long long row0 = block_row * kScaleBlock + threadIdx.x / kLanes;
			Vec<T, kPerLane> v[kPasses];
			uint32_t bits = 0;
#pragma unroll
			for (int p = 0; p < kPasses; p++)
			{
				const long long row = row0 + p * kRowsPerPass;
				load_eight<VEC>(v[p], x + (row < rows ? row : 0) * columns, row < rows ? column : columns, l, columns);
			}
#pragma unroll
			for (int p = 0; p < kPasses; p++)
				bits = raw_max(v[p], bits);
			bits = __reduce_max_sync(kFullWarp, float_bits<T>(bits));
			if (threadIdx.x % 32 == 0)
				warp_max[turn][threadIdx.x / 32] = bits;
			__syncthreads(); /* two sets of slots: the next turn's writes cannot meet this turn's reads */
#pragma unroll
			for (int w = 0; w < kThreads / 32; w++)
				bits = max(bits, warp_max[turn][w]);
			const float amax = clamped_amax(bits);
			const float r = kLargestE4m3 / amax;
#pragma unroll
			for (int p = 0; p < kPasses; p++)
			{
				const long long row = row0 + p * kRowsPerPass;
				if (row < rows)
					store_codes<VEC>(y + row * columns, v[p], r, column, l, columns);
			}
			if (threadIdx.x == 0)
				scales[b] = amax / kLargestE4m3;
		}
	}

	/* ---- norm + quantise ------------------------------------------------------------------------------------------------
	 * `halves` half-warps (a power of two) share a row; number i of them owns the blocks i, i + halves, ... .  ITEMS > 0: at most
	 * ITEMS blocks each, kept in registers between the sum of squares and the codes.  ITEMS = 0: rows of any length, read twice. */
	template<typename T, int ITEMS, bool VEC, int THREADS>
	__global__ void __launch_bounds__(THREADS) kernel_rms_norm_quantize(const T *x, const T *z, T *h, const float *__restrict__ gamma, uint8_t *__restrict__ y,
			float *__restrict__ scales, long long rows, int columns, int blocks, int halves, float epsilon)
	{
		/* Pairs in one instruction where instructions are what bounds (short rows: 50176 x 264 float16 15.3 -> 14.3 us); with four
		 * blocks per half-warp their registers cost a resident thread block (8192 x 8192: 80 -> 89 us). */
		constexpr bool kPacked = ITEMS != 4;
		__shared__ float warp_sum[32];
		chain_release();
		chain_wait();
		const int l = threadIdx.x % kLanes;
		const int half = (threadIdx.x / kLanes) & (halves - 1);
		const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / kLanes / halves) + threadIdx.x / kLanes / halves;
		const bool inside = row < rows;
		const int limit = inside ? columns : 0; /* a row past the end has no columns: nothing is read or written for it */
		const long long offset = inside ? row * columns : 0;

		auto load_sum = [&](float (&v)[kPerLane], int column)
		{
			load_eight<VEC>(v, x + offset, column, l, limit);
			if (z != nullptr)
			{
				float other[kPerLane];
				load_eight<VEC>(other, z + offset, column, l, limit);
#pragma unroll
				for (int i = 0; i < kPerLane; i++)
					v[i] += other[i];
			}
		};
		auto scaled = [&](float (&v)[kPerLane], const float (&g)[kPerLane], int b, float rstd)
		{
			if (h != nullptr)
				store_eight<VEC>(h + offset, v, b * kScaleBlock, l, limit);
			if constexpr (kPacked)
			{
#pragma unroll
				for (int i = 0; i < kPerLane; i += 2)
				{
					multiply_pair(v[i], v[i + 1], rstd, rstd);
					multiply_pair(v[i], v[i + 1], g[i], g[i + 1]);
				}
			}
			else
			{
#pragma unroll
				for (int i = 0; i < kPerLane; i++)
					v[i] = __fmul_rn(__fmul_rn(v[i], rstd), g[i]);
			}
			return largest_magnitude<kPacked>(v);
		};
		float sum = 0.0f, odd_sum = 0.0f;
		auto add_squares = [&](const float (&v)[kPerLane])
		{
#pragma unroll
			for (int i = 0; i < kPerLane; i++)
			{
				if constexpr (not kPacked)
					sum = fmaf(v[i], v[i], sum);
				else if (i % 2 == 0)
					square_pair(sum, odd_sum, v[i], v[i + 1]);
			}
		};

		constexpr int kHeld = ITEMS > 0 ? ITEMS : 1;
		constexpr bool kGammaFirst = ITEMS == 1; /* a row per block: gamma's latency is hidden behind the row's, not added to it */
		float v[kHeld][kPerLane], g[kPerLane];
		if constexpr (ITEMS > 0)
		{
			{
				/* every load is requested before the first is used */
				Vec<T, kPerLane> rx[kHeld], rz[kHeld];
#pragma unroll
				for (int i = 0; i < kHeld; i++)
				{
					load_eight<VEC>(rx[i], x + offset, (half + i * halves) * kScaleBlock, l, limit);
					if (z != nullptr)
						load_eight<VEC>(rz[i], z + offset, (half + i * halves) * kScaleBlock, l, limit);
				}
#pragma unroll
				for (int i = 0; i < kHeld; i++)
#pragma unroll
					for (int k = 0; k < kPerLane; k++)
						v[i][k] = z != nullptr ? to_compute(rx[i].v[k]) + to_compute(rz[i].v[k]) : to_compute(rx[i].v[k]);
			}
			if constexpr (kGammaFirst)
				load_eight<VEC>(g, gamma, half * kScaleBlock, l, limit);
#pragma unroll
			for (int i = 0; i < kHeld; i++)
				add_squares(v[i]);
		}
		else
		{
			for (int b = half; b < blocks; b += halves)
			{
				load_sum(v[0], b * kScaleBlock);
				add_squares(v[0]);
			}
			__syncwarp();
		}
		if constexpr (kPacked)
			sum += odd_sum;
#pragma unroll
		for (int i = kLanes / 2; i > 0; i /= 2)
			sum += __shfl_xor_sync(kFullWarp, sum, i);
		if (halves > 1)
			sum += __shfl_xor_sync(kFullWarp, sum, kLanes);
		if (halves > 2)
		{
			const int warp = threadIdx.x / 32, warps = halves / 2;
			if (threadIdx.x % 32 == 0)
				warp_sum[warp] = sum;
			__syncthreads();
			sum = 0.0f;
			for (int w = 0; w < warps; w++) /* the same order in every thread of the row */
				sum += warp_sum[(warp & ~(warps - 1)) + w];
		}
		const float rstd = 1.0f / sqrtf(sum / static_cast<float>(columns) + epsilon);
		if constexpr (ITEMS > 0)
		{
			uint32_t bits[kHeld];
#pragma unroll
			for (int i = 0; i < kHeld; i++)
			{
				if constexpr (not kGammaFirst)
					load_eight<VEC>(g, gamma, (half + i * halves) * kScaleBlock, l, limit);
				bits[i] = scaled(v[i], g, half + i * halves, rstd);
			}
			const BlockFactors<kHeld> f(bits);
#pragma unroll
			for (int i = 0; i < kHeld; i++)
				store_codes<VEC>(y + offset, v[i], f.factor_of(i), (half + i * halves) * kScaleBlock, l, limit);
			const int own = half + f.item_of(l) * halves;
			if (f.stores(l) and own < blocks and inside)
				scales[row * blocks + own] = f.scale;
		}
		else
		{
			/* both half-warps of a warp go round equally often: the maximum is taken with all lanes present */
			for (int b = half; b - (half & 1) < blocks; b += halves)
			{
				load_sum(v[0], b * kScaleBlock);
				load_eight<VEC>(g, gamma, b * kScaleBlock, l, limit);
				const uint32_t bits[1] = { scaled(v[0], g, b, rstd) };
				const BlockFactors<1> f(bits);
				store_codes<VEC>(y + offset, v[0], f.factor, b * kScaleBlock, l, limit);
				if (l == 0 and b < blocks and inside)
					scales[row * blocks + b] = f.scale;
			}
		}
	}

	int sm_count(const ContextObject &ctx)
	{
		int sms = 148;
		cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, ctx.device);
		return sms;
	}

	template<typename T>
	avStatus_t launch_quantize(ContextObject &ctx, const Operand &x, const Operand &y, const Operand &scales, long long rows, int columns, bool squares)
	{
		const int blocks = scale_blocks(columns);
		const bool vec = columns % kPerLane == 0 and x.aligned(16) and y.aligned(8);
		const T *xp = reinterpret_cast<const T*>(x.ptr);
		float *sp = reinterpret_cast<float*>(scales.ptr);
		cudaError_t launched;
		if (squares)
		{
			const long long total = (rows + kScaleBlock - 1) / kScaleBlock * blocks;
			const dim3 grid(static_cast<unsigned>(std::min<long long>(total, 1 << 30)));
			auto kernel = vec ? kernel_quantize_squares<T, true> : kernel_quantize_squares<T, false>;
			launched = launch_chained(kernel, grid, dim3(kThreads), 0, ctx.getStream(), xp, y.ptr, sp, total, rows, columns, blocks);
		}
		else
		{
			const long long total = rows * blocks;
			constexpr int kPerBlock = kHalfWarps * kAtOnce;
			const long long wanted = (total + kPerBlock - 1) / kPerBlock;
			const dim3 grid(static_cast<unsigned>(std::min<long long>(wanted, 1 << 30)));
			const long long stride = static_cast<long long>(grid.x) * kPerBlock;
			auto kernel = vec ? kernel_quantize_rows<T, true> : kernel_quantize_rows<T, false>;
			launched = launch_chained(kernel, grid, dim3(kThreads), 0, ctx.getStream(), xp, y.ptr, sp, total, columns, blocks, stride / blocks,
					static_cast<int>(stride % blocks));
		}
		return launched != cudaSuccess ? convertStatus(launched) : checkForErrors();
	}

	struct NormArgs
	{
			Operand x, z, h, gamma, y, scales;
			long long rows;
			int columns;
			float epsilon;
	};
	template<typename T, bool VEC, int THREADS>
	auto norm_kernel(int items)
	{
		if (items > 4) /* more than 64 half-warps of four: blocks of 1024 threads only */
			return kernel_rms_norm_quantize<T, 0, VEC, 1024>;
		return items <= 1 ? kernel_rms_norm_quantize<T, 1, VEC, THREADS> : items <= 2 ? kernel_rms_norm_quantize<T, 2, VEC, THREADS> :
				items <= 3 ? kernel_rms_norm_quantize<T, 3, VEC, THREADS> : kernel_rms_norm_quantize<T, 4, VEC, THREADS>;
	}
	template<typename T, bool VEC>
	avStatus_t launch_norm(ContextObject &ctx, const NormArgs &a)
	{
		const int blocks = scale_blocks(a.columns);
		/* Half-warps per row: enough that each holds at most four blocks, or two where that makes 64 to 256 threads of a row.  bfloat16 with
		 * residual, us in a graph with at most two / four: 8192 x 2048 21.7 / 23.8, 4096 x 4096 22.8 / 22.5, 16384 x 1024 22.8 / 22.0, 8192 x 4096
		 * 41.7 / 39.9, 16384 x 640 19.7 / 16.2: two gains from 9 to 16 blocks only.  Outside that range 4096 x 5120 46.8 / 32.2, 8192 x 8192 101 /
		 * 80, 50176 x 264 float16 19.4 / 13.6.  While the rows do not fill the machine, as many half-warps as there are blocks, because then
		 * the time of one row is the time of the call. */
		const int most_items = (blocks > 4 and blocks <= 32) ? 2 : 4;
		int halves = 1;
		const long long room = static_cast<long long>(sm_count(ctx)) * (1024 / kLanes);
		while (halves < 64 and halves < blocks and ((blocks + halves - 1) / halves > most_items or a.rows * halves * 2 <= room))
			halves *= 2;
		const int per_half = (blocks + halves - 1) / halves;
		const int threads = halves >= 8 ? kLanes * halves : kThreads; /* rows that meet at a barrier have a thread block to themselves */
		const long long rows_per_block = threads / (kLanes * halves);
		const long long grid = (a.rows + rows_per_block - 1) / rows_per_block;
		if (grid > 0x7FFFFFFFll)
			return AVOCADO_STATUS_NOT_SUPPORTED;
		auto kernel = threads <= kThreads ? norm_kernel<T, VEC, kThreads>(per_half) : norm_kernel<T, VEC, 1024>(per_half);
		const cudaError_t launched = launch_chained(kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, ctx.getStream(),
				reinterpret_cast<const T*>(a.x.ptr), reinterpret_cast<const T*>(a.z.ptr), reinterpret_cast<T*>(a.h.ptr), reinterpret_cast<const float*>(a.gamma.ptr),
				a.y.ptr, reinterpret_cast<float*>(a.scales.ptr), a.rows, a.columns, blocks, halves, a.epsilon);
		return launched != cudaSuccess ? convertStatus(launched) : checkForErrors();
	}
	template<typename T>
	avStatus_t launch_norm(ContextObject &ctx, const NormArgs &a)
	{
		const bool vec = a.columns % kPerLane == 0 and a.x.aligned(16) and a.z.aligned(16) and a.h.aligned(16) and a.gamma.aligned(16) and a.y.aligned(8);
		return vec ? launch_norm<T, true>(ctx, a) : launch_norm<T, false>(ctx, a);
	}

	bool quantizable(avDataType_t dtype)
	{
		return dtype == AVOCADO_DTYPE_FLOAT16 or dtype == AVOCADO_DTYPE_BFLOAT16 or dtype == AVOCADO_DTYPE_FLOAT32;
	}
	bool same_shape(const TensorObject &a, const TensorObject &b)
	{
		if (a.nb_dims != b.nb_dims)
			return false;
		for (int i = 0; i < a.nb_dims; i++)
			if (a.dims[i] != b.dims[i])
				return false;
		return true;
	}
}

namespace avocado
{
	namespace backend
	{
		avStatus_t cudaQuantizeBlocks(avContextDescriptor_t context, const avTensorDescriptor_t xDesc, const avMemoryDescriptor_t xMem,
				const avTensorDescriptor_t yDesc, avMemoryDescriptor_t yMem, const avTensorDescriptor_t scaleDesc, avMemoryDescriptor_t scaleMem)
		{
			AVOCADO_API_BEGIN
				ContextObject &ctx = getContext(context);
				const TensorObject &x = getTensor(xDesc);
				const TensorObject &y = getTensor(yDesc);
				const TensorObject &scale = getTensor(scaleDesc);
				if (not quantizable(x.dtype) or y.dtype != AVOCADO_DTYPE_FLOAT8_E4M3 or scale.dtype != AVOCADO_DTYPE_FLOAT32)
					return AVOCADO_STATUS_UNSUPPORTED_DATATYPE;
				if (not valid_extents(x) or not valid_extents(scale) or not same_shape(x, y))
					return AVOCADO_STATUS_BAD_PARAM;
				const long long rows = row_count(x);
				const int columns = x.lastDim();
				const bool by_row = row_count(scale) == rows;
				const bool squares = not by_row and row_count(scale) == (rows + kScaleBlock - 1) / kScaleBlock;
				if (scale.lastDim() != scale_blocks(columns) or (not by_row and not squares))
					return AVOCADO_STATUS_BAD_PARAM;
				if (rows == 0 or columns == 0)
					return AVOCADO_STATUS_SUCCESS;
				if (columns > kMaxQuantizedRow)
					return AVOCADO_STATUS_NOT_SUPPORTED;
				Operand xo, yo, so;
				if (not get_operand(xo, ctx, xMem, x) or not get_operand(yo, ctx, yMem, y) or not get_operand(so, ctx, scaleMem, scale))
					return AVOCADO_STATUS_BAD_PARAM;
				if (yo.overlaps(xo) or so.overlaps(xo) or so.overlaps(yo))
					return AVOCADO_STATUS_BAD_PARAM;
				ctx.setDevice();
				switch (x.dtype)
				{
					case AVOCADO_DTYPE_FLOAT16:
						return launch_quantize<half>(ctx, xo, yo, so, rows, columns, squares);
					case AVOCADO_DTYPE_BFLOAT16:
						return launch_quantize<__nv_bfloat16>(ctx, xo, yo, so, rows, columns, squares);
					default:
						return launch_quantize<float>(ctx, xo, yo, so, rows, columns, squares);
				}
			AVOCADO_API_END
		}

		avStatus_t cudaRmsNormQuantize(avContextDescriptor_t context, const avTensorDescriptor_t xDesc, const avMemoryDescriptor_t xMem,
				const avMemoryDescriptor_t zMem, avMemoryDescriptor_t hMem, const avTensorDescriptor_t gammaDesc, const avMemoryDescriptor_t gammaMem,
				double epsilon, const avTensorDescriptor_t yDesc, avMemoryDescriptor_t yMem, const avTensorDescriptor_t scaleDesc, avMemoryDescriptor_t scaleMem)
		{
			AVOCADO_API_BEGIN
				ContextObject &ctx = getContext(context);
				const TensorObject &x = getTensor(xDesc);
				const TensorObject &gamma = getTensor(gammaDesc);
				const TensorObject &y = getTensor(yDesc);
				const TensorObject &scale = getTensor(scaleDesc);
				if (not quantizable(x.dtype) or gamma.dtype != AVOCADO_DTYPE_FLOAT32 or y.dtype != AVOCADO_DTYPE_FLOAT8_E4M3 or scale.dtype != AVOCADO_DTYPE_FLOAT32)
					return AVOCADO_STATUS_UNSUPPORTED_DATATYPE;
				if (not valid_extents(x) or not valid_extents(scale) or not same_shape(x, y))
					return AVOCADO_STATUS_BAD_PARAM;
				NormArgs a;
				a.rows = row_count(x);
				a.columns = x.lastDim();
				a.epsilon = static_cast<float>(epsilon);
				if (gamma.nb_dims != 1 or gamma.dims[0] != a.columns or row_count(scale) != a.rows or scale.lastDim() != scale_blocks(a.columns))
					return AVOCADO_STATUS_BAD_PARAM;
				if (not (a.epsilon > 0.0f) or std::isinf(a.epsilon))
					return AVOCADO_STATUS_BAD_PARAM;
				if (a.rows == 0 or a.columns == 0)
					return AVOCADO_STATUS_SUCCESS;
				if (a.columns > kMaxNormedRow)
					return AVOCADO_STATUS_NOT_SUPPORTED;
				const bool has_z = zMem != AVOCADO_INVALID_DESCRIPTOR, has_h = hMem != AVOCADO_INVALID_DESCRIPTOR;
				if (not get_operand(a.x, ctx, xMem, x) or (has_z and not get_operand(a.z, ctx, zMem, x)) or (has_h and not get_operand(a.h, ctx, hMem, x))
						or not get_operand(a.gamma, ctx, gammaMem, gamma) or not get_operand(a.y, ctx, yMem, y)
						or not get_operand(a.scales, ctx, scaleMem, scale))
					return AVOCADO_STATUS_BAD_PARAM;
				/* every thread writes h only where it has read x and z, so h may replace either of them, but not a shifted one */
				if ((a.h.overlaps(a.x) and not a.h.same_as(a.x)) or (a.h.overlaps(a.z) and not a.h.same_as(a.z)) or a.h.overlaps(a.gamma))
					return AVOCADO_STATUS_BAD_PARAM;
				for (const Operand *out : { &a.y, &a.scales })
					for (const Operand *other : { &a.x, &a.z, &a.h, &a.gamma })
						if (out->overlaps(*other))
							return AVOCADO_STATUS_BAD_PARAM;
				if (a.y.overlaps(a.scales))
					return AVOCADO_STATUS_BAD_PARAM;
				ctx.setDevice();
				switch (x.dtype)
				{
					case AVOCADO_DTYPE_FLOAT16:
						return launch_norm<half>(ctx, a);
					case AVOCADO_DTYPE_BFLOAT16:
						return launch_norm<__nv_bfloat16>(ctx, a);
					default:
						return launch_norm<float>(ctx, a);
				}
			AVOCADO_API_END
		}
	} /* namespace backend */
} /* namespace avocado */

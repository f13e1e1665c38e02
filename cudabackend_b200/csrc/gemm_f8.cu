/*
 * gemm_f8.cu -- cudaGemmBlockScaled: C[M, N] = alpha * A * B^T + beta * C for e4m3 operands with float32 scales, A[M, K] in
 * 1 x 128 blocks and B[N, K] in 128 x 128 blocks.  No counterpart in the reference (its only 8-bit product is int8 -> int32,
 * src/gemm.cpp:42-57).
 *
 *   C[m, n] = alpha * sum_g aScale[m, g] * bScale[n / 128, g] * P_g[m, n] + beta * C[m, n],   P_g = sum over block g of A * B
 *
 * P_g comes from tcgen05.mma kind::f8f6f4 (products exact, float32 accumulators in TMEM).  The scales are arbitrary float32
 * numbers, which the tensor core cannot apply, so every block of 128 gets an accumulator of its own and a "promotion" in
 * float32 registers, acc += scale * P_g: one read of the accumulator and one fused multiply-add per result and block, on the CUDA
 * cores, beside the MMAs of the next block.  An element is off by at most (min(K, 128) + blocks + 4) * 2^-23 of the sum of its terms'
 * magnitudes (what the tests allow); the root mean square of the error over that of the result was 6e-8 for float32 C of 333 x 2056 x
 * 1616.
 *
 * scale = aScale * bScale is formed first and has float32's range; scales from 2^-63 to 2^63 never meet its ends.  Two steps, (P_g *
 * aScale) * bScale with exact powers of two in between, for the blocks that need them would widen it, but looking for such blocks in
 * the promotion costs 3 to 17% (8192^3: 581 us, 597 to 687 us in six forms).
 *
 * Two kernels: kernel_gemm_f8_split (few rows of A, unaligned rows, few tiles; K split over a cluster) and kernel_gemm_f8_pair (256 x
 * 256 tiles on CTA pairs).  The choice is in launch(), with both sides measured.
 */
#include <Avocado/cuda_backend_ext.h>

#include "block_scaled.hpp"
#include "device_utils.cuh"
#include "objects.hpp"
#include "umma.cuh"

#include <algorithm>

namespace
{
	using namespace avocado::backend;
	using namespace avocado::backend::b200;
	using namespace bk;

	constexpr int kBlockBytes = 128 * kScaleBlock; /* one operand tile: 128 rows of one block of K */
	constexpr int kMaxSplits = 8;                  /* CTAs of a cluster, the portable limit */

	struct ScaledGemm
	{
			int M, N, K;
			int blocks; /* blocks of 128 along K */
			const uint8_t *a, *b;
			const float *a_scale, *b_scale;
			void *c;
			float alpha, beta;
			int c_type; /* avDataType_t of C */
			int c_vector; /* four neighbouring elements of C can be moved at once */
	};

	/* ---- C in any of its three types ------------------------------------------------------------------------------ */
	__device__ __forceinline__ float load_c(const ScaledGemm &p, long long i)
	{
		if (p.c_type == AVOCADO_DTYPE_FLOAT32)
			return reinterpret_cast<const float*>(p.c)[i];
		if (p.c_type == AVOCADO_DTYPE_FLOAT16)
			return to_compute(reinterpret_cast<const half*>(p.c)[i]);
		return to_compute(reinterpret_cast<const __nv_bfloat16*>(p.c)[i]);
	}
	__device__ __forceinline__ void store_c(const ScaledGemm &p, long long i, float v)
	{
		if (p.c_type == AVOCADO_DTYPE_FLOAT32)
			reinterpret_cast<float*>(p.c)[i] = v;
		else if (p.c_type == AVOCADO_DTYPE_FLOAT16)
			reinterpret_cast<half*>(p.c)[i] = from_compute<half>(v);
		else
			reinterpret_cast<__nv_bfloat16*>(p.c)[i] = from_compute<__nv_bfloat16>(v);
	}
	__device__ __forceinline__ uint32_t pack_two(int c_type, float x, float y)
	{
		if (c_type == AVOCADO_DTYPE_FLOAT16)
		{
			const half2 v = __floats2half2_rn(x, y);
			return *reinterpret_cast<const uint32_t*>(&v);
		}
		const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
		return *reinterpret_cast<const uint32_t*>(&v);
	}
	/* alpha * v + beta * C for four neighbouring elements of a row, of which `count` exist */
	__device__ __forceinline__ void finish_four(const ScaledGemm &p, long long i, float4 v, int count)
	{
		float x[4] = { p.alpha * v.x, p.alpha * v.y, p.alpha * v.z, p.alpha * v.w };
		if (p.beta != 0.0f)
		{
#pragma unroll
			for (int j = 0; j < 4; j++)
				if (j < count)
					x[j] = fmaf(p.beta, load_c(p, i + j), x[j]);
		}
		if (p.c_vector)
		{
			if (p.c_type == AVOCADO_DTYPE_FLOAT32)
				*reinterpret_cast<float4*>(reinterpret_cast<float*>(p.c) + i) = make_float4(x[0], x[1], x[2], x[3]);
			else
				*reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.c) + i) = make_uint2(pack_two(p.c_type, x[0], x[1]), pack_two(p.c_type, x[2], x[3]));
		}
		else
		{
#pragma unroll
			for (int j = 0; j < 4; j++)
				if (j < count)
					store_c(p, i + j, x[j]);
		}
	}

	/* K = 0: the sum is empty */
	__global__ void __launch_bounds__(256) kernel_scale_c(ScaledGemm p)
	{
		chain_release();
		chain_wait();
		const long long total = static_cast<long long>(p.M) * p.N;
		for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * 256)
			store_c(p, i, p.beta != 0.0f ? p.beta * load_c(p, i) : 0.0f);
	}

	/*
	 * Few rows of A ("tokens"), and any row pitch: 128 rows of B are the M side of the MMA and TOKENS rows of A its N side, so
	 * that a handful of tokens does not waste 128-row tiles; the result is transposed on the way out.
	 *
	 * Bound: the bytes of B in principle; at these sizes the set-up (1000 cycles), the first copy (1200) and the end (1500) of a CTA
	 * that lives 8000 cycles.  Measured in a graph, with more than 330 MB of weights in rotation (from HBM, as a decoding step finds
	 * them) / with two sets (from L2 where both fit): 1 x 4096 x 4096 6.0 / 4.7 us (2.8 TB/s from HBM), 13 x 8192 x 4096 9.1 / 6.3 us (3.7
	 * TB/s), 1 x 8192 x 8192 13.2 / 13.2 us (5.1 TB/s).  With two sets: 129 x 2048 x 4096 9.7 us, 333 x 2056 x 1616 10.0 us.
	 * One tile of 128 rows of B per CTA leaves most SMs without work at the usual sizes, so the blocks of
	 * K are split over the CTAs of a cluster.  Each CTA finishes a share of the tokens and adds everybody's partial sums for these in
	 * the order of the ranks: no scratch memory, no atomics, the same bits every time.
	 *
	 * full[s] (copy -> MMA) and done[s] (MMA and scales -> promotion, and back to the copies: the slot may be filled again) go round
	 * over the slots of shared memory, drained[b] (promotion -> MMA and scales) over the accumulators in TMEM.  Each block of K has
	 * an accumulator of its own, because its scales are applied outside the tensor core: acc[t] += scale[t] * part[t] in float32
	 * registers, lane = row of B.  Two blocks share a slot, so that every role waits once per eight MMAs, and two threads issue the
	 * MMAs of every other slot each (one takes 1150 cycles per slot, twice what the MMAs need).  A warp of its own loads
	 * the scales, slots ahead of their use, and hands them to all promotion warps through shared memory.
	 *
	 * LOADERS: eight warps fill the slots with plain loads instead of the TMA copies, for row pitches or addresses that are no
	 * multiple of 16 bytes; at most 64 tokens, because of their registers.  Bound by the latency of the loads that those registers
	 * hold (24 KB per SM): 1 x 4096 x 4095 13 us, 500 x 3000 x 1001 33 us, 4096 x 4096 x 4095 740 us.
	 */
	template<int TOKENS, bool LOADERS>
	struct SplitConfig
	{
			static constexpr int kPerStage = 2;
			static constexpr int kStages = TOKENS <= 64 ? 4 : 3;
			static constexpr int kBuffers = kStages * kPerStage * TOKENS <= 512 ? kStages : 512 / (kPerStage * TOKENS); /* accumulator slots in TMEM */
			static constexpr int kPairBytes = kBlockBytes + TOKENS * kScaleBlock;
			static constexpr int kStageBytes = kPerStage * kPairBytes;
			/* Two CTAs of different clusters never share an SM: each could wait for the TMEM of the other's neighbour. */
			static constexpr int kSmemBytes = kStages * kStageBytes + 1024;
			static_assert(kSmemBytes > 116 * 1024 and kSmemBytes <= 228 * 1024, "one CTA per SM");
			/* How partial sums meet: where they are few, every CTA sends its own, float by float, to the CTA that finishes the token;
			 * where they are many, they stay where they are and are read from there.  Graph of 1 x 4096 x 4096: 4.9 us sent, 5.6
			 * read; 128 x 4096 x 4096: 11.2 us sent, 11.3 copied in bulk, 10.0 read. */
			static constexpr bool kSendSums = TOKENS <= 32;
			static_assert((TOKENS + kMaxSplits) * 512 <= kStages * kStageBytes, "the partial sums reuse the slots");
			static constexpr int kWantedColumns = kBuffers * kPerStage * TOKENS;
			static constexpr int kTmemColumns = kWantedColumns <= 128 ? 128 : kWantedColumns <= 256 ? 256 : 512;
			/* promotion warps: four for the 128 lanes of TMEM, twice that where each would hold more than 32 tokens */
			static constexpr int kPromoteWarps = TOKENS > 32 ? 8 : 4;
			static constexpr int kPromoteThreads = kPromoteWarps * 32;
			static constexpr int kTokensPerWarp = TOKENS / (kPromoteWarps / 4);
			static constexpr int kMmaWarp = kPromoteWarps, kScaleWarp = kPromoteWarps + 2; /* two issuers */
			static constexpr int kLoaderWarps = LOADERS ? 8 : 1, kLoaderThreads = kLoaderWarps * 32;
			static constexpr int kThreads = kPromoteThreads + 96 + kLoaderThreads;
	};

	/* Plain loads into a slot: one row of at most 256 bytes (its two blocks) per warp and turn.  Rows start at any address, so lane
	 * l loads the aligned words l and l + 32 that cover it and shifts neighbours together.  Word l of a block's row lies in piece
	 * (l / 4) ^ (row % 8), the 128-byte swizzle that the descriptors name. */
	__device__ __forceinline__ uint32_t* slot_word(uint8_t *slot, int row, int lane)
	{
		return reinterpret_cast<uint32_t*>(slot + row * 128 + ((lane / 4) ^ (row & 7)) * 16 + lane % 4 * 4);
	}
	/* The aligned words reach up to three bytes outside the row: rows within four bytes of an end of the tensor go byte by byte. */
	__device__ __noinline__ void store_edge_row(uint8_t *slot, int row, int pairBytes, const uint8_t *from, int valid, int lane)
	{
		for (int block = 0; block < 2; block++)
		{
			uint32_t word = 0;
			for (int i = 0; i < 4; i++)
				if (block * 128 + 4 * lane + i < valid)
					word |= static_cast<uint32_t>(from[block * 128 + 4 * lane + i]) << (8 * i);
			slot_word(slot, row, lane)[block * pairBytes / 4] = word;
		}
	}
	/* ROWS rows of an operand, kLoaderWarps apart: all requested before the first is stored.  `rows`: how many of the tensor's rows
	 * there are from the first one on; start: its offset in the tensor of `total` bytes. */
	template<int ROWS, int STEP>
	__device__ __forceinline__ void load_rows(uint8_t *slot, int row0, int pairBytes, const uint8_t *tensor, long long start, long long total, int rows, int pitch,
			int columns, int lane)
	{
		uint32_t low[ROWS], high[ROWS], next[ROWS];
		bool any_edge = false;
		const long long step = static_cast<long long>(STEP) * pitch;
		auto end_of = [&](int i, long long at)
		{
			const bool edge = at < 4 or at + columns + 4 > total;
			return i * STEP < rows and not edge ? static_cast<int>(reinterpret_cast<uintptr_t>(tensor + at) & 3) + columns : 0;
		};
#pragma unroll
		for (int i = 0; i < ROWS; i++)
		{
			const long long at = start + i * step;
			const int end = end_of(i, at);
			any_edge = any_edge or (end == 0 and i * STEP < rows);
			const uint32_t *words = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(tensor + at) & ~static_cast<uintptr_t>(3));
			low[i] = 4 * lane < end ? words[lane] : 0u;
			high[i] = 4 * lane + 128 < end ? words[lane + 32] : 0u;
			next[i] = (lane == 31 and 256 < end) ? words[64] : 0u;
		}
#pragma unroll
		for (int i = 0; i < ROWS; i++)
		{
			const int shift = 8 * static_cast<int>(reinterpret_cast<uintptr_t>(tensor + start + i * step) & 3);
			uint32_t after_low = __shfl_down_sync(0xFFFFFFFFu, low[i], 1), after_high = __shfl_down_sync(0xFFFFFFFFu, high[i], 1);
			const uint32_t high_first = __shfl_sync(0xFFFFFFFFu, high[i], 0);
			if (lane == 31)
			{
				after_low = high_first;
				after_high = next[i];
			}
			/* bytes past the last column are zeros: of this lane's word at byte c, columns - c are kept */
			const int keep_low = min(max(columns - 4 * lane, 0), 4), keep_high = min(max(columns - 4 * lane - 128, 0), 4);
			const uint32_t mask_low = keep_low == 4 ? 0xFFFFFFFFu : (1u << (8 * keep_low)) - 1u, mask_high = keep_high == 4 ? 0xFFFFFFFFu : (1u << (8 * keep_high)) - 1u;
			uint32_t *to = slot_word(slot, row0 + i * STEP, lane);
			to[0] = __funnelshift_r(low[i], after_low, shift) & mask_low;
			to[pairBytes / 4] = __funnelshift_r(high[i], after_high, shift) & mask_high;
		}
		if (any_edge)
#pragma unroll 1
			for (int i = 0; i < ROWS; i++)
			{
				const long long at = start + i * step;
				if (i * STEP < rows and end_of(i, at) == 0)
					store_edge_row(slot, row0 + i * STEP, pairBytes, tensor + at, columns, lane);
			}
	}

	template<int TOKENS, bool LOADERS>
	__global__ void __launch_bounds__(SplitConfig<TOKENS, LOADERS>::kThreads, 1) kernel_gemm_f8_split(const __grid_constant__ CUtensorMap mapA,
			const __grid_constant__ CUtensorMap mapB, ScaledGemm p, int tokenTiles, int splits, int blocksPerSplit, int *deviceStatus)
	{
		using Cfg = SplitConfig<TOKENS, LOADERS>;
		constexpr int kStages = Cfg::kStages, kPerStage = Cfg::kPerStage;
		extern __shared__ uint8_t smem_raw[];
		uint8_t *smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));

		__shared__ __align__(8) uint64_t full_bar[kStages];
		__shared__ __align__(8) uint64_t done_bar[kStages];
		__shared__ __align__(8) uint64_t drained_bar[Cfg::kBuffers];
		__shared__ __align__(8) uint64_t sums_bar; /* the other CTAs' partial sums for this CTA's tokens have arrived */
		__shared__ uint32_t tmem_base_slot;
		__shared__ int abort_flag;
		__shared__ __align__(16) float scale_s[Cfg::kBuffers][kPerStage * TOKENS];

		const int warp = threadIdx.x / 32;
		const int lane = threadIdx.x % 32;
		const int rank = splits > 1 ? static_cast<int>(umma::cluster_cta_rank()) : 0;
		const int tile = blockIdx.x / splits;
		const int m0 = tile % tokenTiles * TOKENS;
		const int n_block = tile / tokenTiles;
		const int n0 = n_block * 128;
		const int first = min(p.blocks, rank * blocksPerSplit);
		const int last = min(p.blocks, first + blocksPerSplit);
		const int tokens = min(TOKENS, p.M - m0);
		const int share = (tokens + splits - 1) / splits; /* CTA r finishes tokens r * share .. */
		const int own_tokens = max(0, min(share, tokens - rank * share));

		if (threadIdx.x == 0)
		{
			abort_flag = 0;
			for (int s = 0; s < kStages; s++)
			{
				umma::mbar_init(&full_bar[s], LOADERS ? Cfg::kLoaderThreads : 1);
				umma::mbar_init(&done_bar[s], 2);
			}
			for (int b = 0; b < Cfg::kBuffers; b++)
				umma::mbar_init(&drained_bar[b], Cfg::kPromoteWarps);
			umma::mbar_init(&sums_bar, 1);
			umma::mbar_fence_init();
			umma::mbar_arrive_expect_tx(&sums_bar, static_cast<uint32_t>((splits - 1) * own_tokens * 512));
			if (not LOADERS)
			{
				umma::prefetch_tensormap(&mapA);
				umma::prefetch_tensormap(&mapB);
			}
		}
		if (warp == Cfg::kMmaWarp)
		{
			umma::tmem_alloc(&tmem_base_slot, Cfg::kTmemColumns);
			umma::tmem_relinquish();
		}
		umma::tcgen05_fence_before();
		__syncthreads();
		umma::tcgen05_fence_after();
		const uint32_t tmem_base = tmem_base_slot;
		volatile int *abort_ptr = &abort_flag;
		chain_release();
		chain_wait();

		if (warp == Cfg::kMmaWarp or warp == Cfg::kMmaWarp + 1)
		{
			if (lane == 0)
			{
				constexpr uint32_t idesc = umma::make_instr_desc(umma::kAccumF32, umma::kFormatE4M3, umma::kFormatE4M3, false, false, 128, TOKENS);
				const uint64_t desc0 = umma::make_smem_desc(umma::smem_u32(smem), 16, 1024, umma::kSwizzle128B);
				static_assert(kStages >= 2 and Cfg::kBuffers >= 2, "two slots further wraps round at most once");
				int stage = warp - Cfg::kMmaWarp, buffer = stage;
				uint32_t phase = 0, buffer_phase = 0;
				for (int kb = first + stage * kPerStage; kb < last; kb += 2 * kPerStage)
				{
					if (not umma::mbar_wait(&drained_bar[buffer], buffer_phase ^ 1u, abort_ptr))
					{
						umma::raise_error(abort_ptr, deviceStatus, umma::kErrorMmaWait);
						break;
					}
					if (not umma::mbar_wait(&full_bar[stage], phase, abort_ptr))
					{
						umma::raise_error(abort_ptr, deviceStatus, umma::kErrorTmaWait);
						break;
					}
					umma::tcgen05_fence_after();
#pragma unroll
					for (int j = 0; j < kPerStage; j++)
						if (kb + j < last)
						{
							const uint64_t desc = desc0 + static_cast<uint64_t>((stage * Cfg::kStageBytes + j * Cfg::kPairBytes) / 16);
							umma::mma_f8_k4(tmem_base + static_cast<uint32_t>((buffer * kPerStage + j) * TOKENS), desc, desc + kBlockBytes / 16, idesc, false);
						}
					umma::mma_commit(&done_bar[stage]);
					buffer += 2;
					if (buffer >= Cfg::kBuffers)
					{
						buffer -= Cfg::kBuffers;
						buffer_phase ^= 1u;
					}
					stage += 2;
					if (stage >= kStages)
					{
						stage -= kStages;
						phase ^= 1u;
					}
				}
			}
		}
		else if (warp == Cfg::kScaleWarp)
		{
			/* scale i * 32 + lane of a slot belongs to token (i * 32 + lane) % TOKENS of block kb + (i * 32 + lane) / TOKENS; the factors
			 * of the next kAhead slots are on their way while this warp waits for a buffer */
			constexpr int kScales = kPerStage * TOKENS / 32, kAhead = 2;
			float next_a[kAhead][kScales], next_b[kAhead][kScales];
			auto fetch = [&](float (&va)[kScales], float (&vb)[kScales], int kb)
			{
#pragma unroll
				for (int i = 0; i < kScales; i++)
				{
					const int t = m0 + (i * 32 + lane) % TOKENS, g = kb + (i * 32 + lane) / TOKENS;
					const bool inside = g < last and t < p.M;
					va[i] = inside ? p.a_scale[static_cast<long long>(t) * p.blocks + g] : 0.0f;
					vb[i] = inside ? p.b_scale[static_cast<long long>(n_block) * p.blocks + g] : 0.0f;
				}
			};
#pragma unroll
			for (int u = 0; u < kAhead; u++)
				fetch(next_a[u], next_b[u], first + u * kPerStage);
			int stage = 0, buffer = 0;
			uint32_t buffer_phase = 0;
			bool ok = true;
			for (int kb0 = first; kb0 < last and ok; kb0 += kAhead * kPerStage)
			{
#pragma unroll
				for (int u = 0; u < kAhead; u++)
				{
					const int kb = kb0 + u * kPerStage;
					if (kb >= last)
						break;
					ok = __all_sync(0xFFFFFFFFu, lane != 0 or umma::mbar_wait(&drained_bar[buffer], buffer_phase ^ 1u, abort_ptr));
					if (not ok)
					{
						if (lane == 0)
							umma::raise_error(abort_ptr, deviceStatus, umma::kErrorEpilogueWait);
						break;
					}
					__syncwarp(); /* a vote orders no memory: what lane 0 has waited for is ordered before the other lanes' writes here */
#pragma unroll
					for (int i = 0; i < kScales; i++)
						scale_s[buffer][i * 32 + lane] = next_a[u][i] * next_b[u][i];
					__syncwarp();
					if (lane == 0)
						umma::mbar_arrive(&done_bar[stage]);
					fetch(next_a[u], next_b[u], kb + kAhead * kPerStage);
					if (++stage == kStages)
						stage = 0;
					if (++buffer == Cfg::kBuffers)
					{
						buffer = 0;
						buffer_phase ^= 1u;
					}
				}
			}
		}
		else if (warp > Cfg::kScaleWarp)
		{
			if (LOADERS or lane == 0)
			{
				const int thread = threadIdx.x - Cfg::kPromoteThreads - 96;
				int stage = 0;
				uint32_t phase = 0;
				for (int kb = first; kb < last; kb += kPerStage)
				{
					const int count = min(kPerStage, last - kb);
					bool ready = umma::mbar_wait(&done_bar[stage], phase ^ 1u, abort_ptr);
					if constexpr (LOADERS)
						ready = __all_sync(0xFFFFFFFFu, ready); /* a warp's lanes exchange words below */
					if (not ready)
					{
						umma::raise_error(abort_ptr, deviceStatus, umma::kErrorStageWait);
						break;
					}
					uint8_t *slot = smem + stage * Cfg::kStageBytes;
					if constexpr (LOADERS)
					{
						static_assert(kPerStage == 2, "a row of the slot is two blocks");
						constexpr int kStep = Cfg::kLoaderWarps;
						const int k = kb * kScaleBlock, loader = thread / 32;
						const int columns = min(count * kScaleBlock, p.K - k);
#pragma unroll 1
						for (int part = 0; part < 128; part += 8 * kStep)
							load_rows<8, kStep>(slot, part + loader, Cfg::kPairBytes, p.b, (static_cast<long long>(n0) + part + loader) * p.K + k,
									static_cast<long long>(p.N) * p.K, p.N - n0 - part - loader, p.K, columns, lane);
						load_rows<TOKENS / kStep, kStep>(slot + kBlockBytes, loader, Cfg::kPairBytes, p.a, (static_cast<long long>(m0) + loader) * p.K + k,
								static_cast<long long>(p.M) * p.K, p.M - m0 - loader, p.K, columns, lane);
						umma::fence_proxy_async_smem();
						umma::mbar_arrive(&full_bar[stage]);
					}
					else
					{
						umma::mbar_arrive_expect_tx(&full_bar[stage], static_cast<uint32_t>(count * Cfg::kPairBytes));
						for (int j = 0; j < count; j++)
						{
							umma::tma_load_2d(slot + j * Cfg::kPairBytes, &mapB, &full_bar[stage], (kb + j) * kScaleBlock, n0);
							umma::tma_load_2d(slot + j * Cfg::kPairBytes + kBlockBytes, &mapA, &full_bar[stage], (kb + j) * kScaleBlock, m0);
						}
					}
					if (++stage == kStages)
					{
						stage = 0;
						phase ^= 1u;
					}
				}
			}
		}
		constexpr int kTokens = Cfg::kTokensPerWarp;
		const int row = warp % 4 * 32 + lane;
		const int token0 = warp / 4 * kTokens;
		float acc[kTokens];
		if (warp < Cfg::kPromoteWarps)
		{
			/* promotion: lane = row n0 + row of B, one accumulator per token of the warp's share */
#pragma unroll
			for (int t = 0; t < kTokens; t++)
				acc[t] = 0.0f;
			const uint32_t lanes = tmem_base + (static_cast<uint32_t>(warp % 4 * 32) << 16) + static_cast<uint32_t>(token0);
			int stage = 0, buffer = 0;
			uint32_t phase = 0;
			bool ok = true;
			for (int kb = first; kb < last; kb += kPerStage)
			{
				ok = __all_sync(0xFFFFFFFFu, umma::mbar_wait(&done_bar[stage], phase, abort_ptr));
				if (not ok)
				{
					if (lane == 0)
						umma::raise_error(abort_ptr, deviceStatus, umma::kErrorEpilogueWait);
					break;
				}
				umma::tcgen05_fence_after();
				/* The slot's accumulators of this warp, block after block, 32 columns per load and at most two loads at once; the
				 * buffer, with its scales, is handed back at the end. */
				constexpr int kLoads = kPerStage * kTokens / 32, kAtOnce = LOADERS or kLoads < 2 ? 1 : 2;
#pragma unroll
				for (int l0 = 0; l0 < kLoads; l0 += kAtOnce)
				{
					uint32_t r[kAtOnce][32];
#pragma unroll
					for (int l = 0; l < kAtOnce; l++)
					{
						const int f = (l0 + l) * 32, column = f / kTokens * TOKENS + f % kTokens;
						umma::tmem_load_32x32(lanes + static_cast<uint32_t>(buffer * kPerStage * TOKENS + column), r[l]);
					}
#pragma unroll
					for (int l = 0; l < kAtOnce; l++)
						umma::tmem_load_wait(r[l]);
#pragma unroll
					for (int l = 0; l < kAtOnce; l++)
					{
						const int f = (l0 + l) * 32;
						const float *scale = &scale_s[buffer][f / kTokens * TOKENS + token0 + f % kTokens];
#pragma unroll
						for (int e = 0; e < 32; e += 4)
						{
							if (kb + (f + e) / kTokens >= last)
								break; /* the slot's second block does not exist */
							const float4 s = *reinterpret_cast<const float4*>(scale + e);
							const int t = (f + e) % kTokens;
							acc[t] = fmaf(__uint_as_float(r[l][e]), s.x, acc[t]);
							acc[t + 1] = fmaf(__uint_as_float(r[l][e + 1]), s.y, acc[t + 1]);
							acc[t + 2] = fmaf(__uint_as_float(r[l][e + 2]), s.z, acc[t + 2]);
							acc[t + 3] = fmaf(__uint_as_float(r[l][e + 3]), s.w, acc[t + 3]);
						}
					}
				}
				umma::tcgen05_fence_before();
				__syncwarp();
				if (lane == 0)
					umma::mbar_arrive(&drained_bar[buffer]); /* this warp has read the accumulators and the scales */
				if (++buffer == Cfg::kBuffers)
					buffer = 0;
				if (++stage == kStages)
				{
					stage = 0;
					phase ^= 1u;
				}
			}
		}

		__syncthreads();
		if (abort_flag != 0)
			umma::drain_after_abort();
		/* Every MMA of a CTA that has come here has run (its promotion warps waited for the last one), and each had waited for its
		 * copies: its slots are free to take partial sums. */
		if (Cfg::kSendSums and splits > 1)
			umma::cluster_sync_all_relaxed();
		/* rows of 128 floats; sent: part of CTA q for token i of this CTA's share at row q * share + i; read: own part for token i of
		 * the tile at row i */
		float *sums = reinterpret_cast<float*>(smem);
		const uint32_t bar = umma::smem_u32(&sums_bar);
		if (warp < Cfg::kPromoteWarps)
		{
			int owner = token0 / share, place = token0 - owner * share;
#pragma unroll
			for (int t = 0; t < kTokens; t++)
			{
				if (token0 + t < tokens)
				{
					float *to = sums + (Cfg::kSendSums ? rank * share + place : token0 + t) * 128 + row;
					if (not Cfg::kSendSums or owner == rank)
						*to = acc[t];
					else
						umma::store_async_cluster(umma::map_to_cta(umma::smem_u32(to), static_cast<uint32_t>(owner)), acc[t],
								umma::map_to_cta(bar, static_cast<uint32_t>(owner)));
				}
				if (++place == share)
				{
					place = 0;
					owner++;
				}
			}
		}
		umma::tcgen05_fence_before();
		__syncthreads(); /* this CTA's own part is written */
		if (not Cfg::kSendSums and splits > 1)
			umma::cluster_sync_all(); /* and so is everybody's */
		if (threadIdx.x < Cfg::kPromoteThreads and own_tokens > 0)
		{
			bool arrived = true;
			if (Cfg::kSendSums)
			{
				/* the CTA may leave only when everything that is sent to it has arrived, whether or not a wait ran out before */
				volatile int ignored = 0;
				arrived = umma::mbar_wait(&sums_bar, 0, &ignored) and umma::mbar_try_wait_cluster(&sums_bar, 0);
				if (not arrived)
					umma::raise_error(abort_ptr, deviceStatus, umma::kErrorEpilogueWait);
			}
			for (int i = threadIdx.x; arrived and i < own_tokens * 32; i += Cfg::kPromoteThreads)
			{
				const int n = i % 32 * 4;
				if (n0 + n >= p.N)
					continue; /* before its loads: none may be on the way when the cluster's CTAs leave */
				float4 part[kMaxSplits];
#pragma unroll
				for (int q = 0; q < kMaxSplits; q++)
					if (q < splits)
					{
						if (Cfg::kSendSums)
							part[q] = reinterpret_cast<const float4*>(sums)[q * share * 32 + i];
						else if (splits > 1)
							asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(part[q].x), "=f"(part[q].y), "=f"(part[q].z), "=f"(part[q].w)
									: "r"(umma::map_to_cta(umma::smem_u32(sums) + static_cast<uint32_t>(rank * share * 32 + i) * 16u, static_cast<uint32_t>(q))));
						else
							part[q] = reinterpret_cast<const float4*>(sums)[i];
					}
				float4 sum = part[0];
#pragma unroll
				for (int q = 1; q < kMaxSplits; q++)
					if (q < splits)
						sum = make_float4(sum.x + part[q].x, sum.y + part[q].y, sum.z + part[q].z, sum.w + part[q].w);
				finish_four(p, static_cast<long long>(m0 + rank * share + i / 32) * p.N + n0 + n, sum, min(4, p.N - n0 - n));
			}
		}
		if (not Cfg::kSendSums)
		{
			__syncthreads();
			if (splits > 1)
				umma::cluster_sync_all_relaxed(); /* nobody leaves while its sums may still be read; what was read has been used */
		}
		if (warp == Cfg::kMmaWarp)
		{
			umma::tcgen05_fence_after();
			umma::tmem_dealloc(tmem_base, Cfg::kTmemColumns);
		}
	}

	/*
	 * Many rows on both sides: pairs of CTAs (cta_group::2) on tiles of 256 x 256.  Each CTA copies its 128 rows of A and its half of
	 * the rows of B, holds 128 x 256 accumulators in float32 registers (128 per thread of eight warps) and the two newest blocks
	 * of K in TMEM.
	 *
	 * Why 256 x 256: per block of K a CTA pulls 32 KB from L2 for 524 cycles of MMAs (four of N = 256, 131 cycles each), 62
	 * bytes per cycle, about what L2 delivers; 128 x 128 tiles on single CTAs pull the same 32 KB for 280 cycles.  The promotion
	 * reads 128 x 256 floats of TMEM per block of K and issues 256 fused multiply-adds per scheduler (packed pairs were slower:
	 * 690 cycles of promotion per block against 500).
	 *
	 * What bounds it: the round trip of an accumulator (MMAs 524 cycles, commit to wake-up 200, promotion 500, arrival to the next
	 * MMA 250) over the two that fit in TMEM: 890 cycles per block where the MMAs alone take 524, and, over long runs, the
	 * power limit (8192^3: 517 us for tens of milliseconds, 600 us at the clocks of seconds).  Measured and not kept: accumulators of
	 * 128 columns (twice the MMAs to issue, 1020 cycles per block), sixteen promotion warps (621 us against 511), loads of 32
	 * columns (the same).
	 * Why two issuing threads: a block of K costs its issuer two waits, four MMAs and two commits, about 680 cycles, more
	 * than the MMAs take; even and odd blocks have an issuer (and an accumulator) each.
	 *
	 * Measured (bfloat16 C): 8192^3 517 us, 2130 TFLOP/s; 4096 x 8192 x 4096 134 us; 50176 x 256 x 2304 38 us (2.65 waves of tiles).
	 *
	 *   full[s]        first CTA only: its producer posts the bytes of both CTAs' copies
	 *   empty[s]       both CTAs: the commit after a slot's MMAs
	 *   part_full[b]   both CTAs: the same, for the accumulator, and one arrival of the CTA's own warp that brings the scales
	 *   part_empty[b]  first CTA only: one arrival per promotion warp of both CTAs
	 */
	constexpr int kPairStages = 5;
	constexpr int kPairSlotBytes = 2 * kBlockBytes; /* 128 rows of A, 128 rows of B */
	constexpr int kPairControlThreads = 128;        /* producer, two issuers, one warp for the scales (and TMEM) */
	constexpr int kPairThreads = kPairControlThreads + 256;
	constexpr int kPairControlRegisters = 56;
	constexpr int kPairPromoteRegisters = 224;
	constexpr int kScaleSlots = 3, kScaleAhead = 3; /* blocks of K whose scales are in shared memory, and in flight to it */
	constexpr int kSubBytes = 32 * 128;             /* a warp's 32 rows, 128 bytes of C each */
	constexpr int kPairSmemBytes = kPairStages * kPairSlotBytes + 8 * 2 * kSubBytes + 1024;
	static_assert(kPairSmemBytes <= 232448 - 256 - kScaleSlots * 130 * 4, "shared memory of an SM");
	static_assert(kPairControlThreads * kPairControlRegisters + 256 * kPairPromoteRegisters <= kPairThreads * 168, "registers of the launch");
	constexpr int kBandRows = 8; /* tiles are walked in bands of this many tile rows, column by column, so that neighbours in time share operands in L2 */

	struct PairTile
	{
			int m, n;
	};
	__device__ __forceinline__ PairTile pair_tile(int tile, int mBlocks, int nBlocks)
	{
		const int band = tile / (kBandRows * nBlocks);
		const int rows = min(kBandRows, mBlocks - band * kBandRows);
		const int r = tile - band * kBandRows * nBlocks;
		PairTile t;
		t.m = band * kBandRows + r % rows;
		t.n = r / rows;
		return t;
	}
	/* One 32-row sub-tile of C (64 16-bit or 32 float32 columns) from registers: staged in the swizzled order of the store's tensor
	 * map, then written by one bulk copy, or row by row where C's pitch or address rules the copy out.  first: of a tile; the copies
	 * of the tile before, which end with either buffer where its last columns are past N, have read both before it is overwritten. */
	template<typename T, bool ADD>
	__device__ __forceinline__ void store_sub_tile(const ScaledGemm &p, const CUtensorMap *mapC, uint8_t *buffer, const float *acc, int row0, int column0, int lane,
			bool bulk, bool first)
	{
		constexpr int kColumns = 128 / static_cast<int>(sizeof(T));
		constexpr int kPerPiece = 16 / static_cast<int>(sizeof(T));
		if (row0 >= p.M or column0 >= p.N)
			return;
		if (bulk)
		{
			if (lane == 0)
			{
				if (first)
					umma::tma_store_wait_read<0>();
				else
					umma::tma_store_wait_read<1>(); /* the copy before last has read this buffer */
			}
			__syncwarp();
		}
		const T *old = reinterpret_cast<const T*>(p.c) + static_cast<long long>(row0 + lane) * p.N + column0;
		const int old_columns = (ADD and row0 + lane < p.M) ? p.N - column0 : 0;
#pragma unroll
		for (int j = 0; j < kColumns / kPerPiece; j++)
		{
			float x[kPerPiece];
#pragma unroll
			for (int i = 0; i < kPerPiece; i++)
				x[i] = p.alpha * acc[j * kPerPiece + i];
			if (ADD and j * kPerPiece < old_columns)
			{
				if (bulk) /* rows and pieces on 16-byte boundaries, whole pieces only */
				{
					const Vec<T, kPerPiece> v = load_vec<T, kPerPiece>(old + j * kPerPiece);
#pragma unroll
					for (int i = 0; i < kPerPiece; i++)
						x[i] = fmaf(p.beta, to_compute(v.v[i]), x[i]);
				}
				else
				{
#pragma unroll
					for (int i = 0; i < kPerPiece; i++)
						if (j * kPerPiece + i < old_columns)
							x[i] = fmaf(p.beta, to_compute(old[j * kPerPiece + i]), x[i]);
				}
			}
			Vec<T, kPerPiece> piece;
#pragma unroll
			for (int i = 0; i < kPerPiece; i++)
				piece.v[i] = from_compute<T>(x[i]);
			store_vec<T, kPerPiece>(reinterpret_cast<T*>(buffer + lane * 128 + ((j ^ (lane & 7)) << 4)), piece);
		}
		if (bulk)
		{
			umma::fence_proxy_async_smem();
			__syncwarp();
			if (lane == 0)
			{
				umma::tma_store_2d(mapC, buffer, column0, row0);
				umma::tma_store_commit();
			}
		}
		else
		{
			__syncwarp();
			for (int r = 0; r < min(32, p.M - row0); r++)
#pragma unroll
				for (int i = 0; i < kColumns / 32; i++)
				{
					const int column = i * 32 + lane;
					if (column0 + column < p.N)
						reinterpret_cast<T*>(p.c)[static_cast<long long>(row0 + r) * p.N + column0 + column] =
								reinterpret_cast<const T*>(buffer + r * 128 + (((column / kPerPiece) ^ (r & 7)) << 4))[column % kPerPiece];
				}
			__syncwarp();
		}
	}
	/* a warp's 32 x 128 results through two buffers in turn */
	template<typename T, bool ADD>
	__device__ __forceinline__ void store_rows(const ScaledGemm &p, const CUtensorMap *mapC, uint8_t *buffers, const float (&acc)[128], int row0, int column0, int lane,
			bool bulk)
	{
		constexpr int kColumns = 128 / static_cast<int>(sizeof(T));
#pragma unroll
		for (int sub = 0; sub < 128 / kColumns; sub++)
			store_sub_tile<T, ADD>(p, mapC, buffers + (sub & 1) * kSubBytes, acc + sub * kColumns, row0, column0 + sub * kColumns, lane, bulk, sub == 0);
	}

	/* ADD: beta is not 0.  The type of C and this are template parameters because the store runs once per tile, out of a cold
	 * instruction cache: every path that is not there is one that is not fetched. */
	template<typename T, bool ADD>
	__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1) kernel_gemm_f8_pair(const __grid_constant__ CUtensorMap mapA,
			const __grid_constant__ CUtensorMap mapB, const __grid_constant__ CUtensorMap mapC, ScaledGemm p, int mBlocks, int nBlocks, int numTiles, int bulkStore,
			int *deviceStatus)
	{
		extern __shared__ uint8_t smem_raw[];
		uint8_t *smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));

		__shared__ __align__(8) uint64_t full_bar[kPairStages];
		__shared__ __align__(8) uint64_t empty_bar[kPairStages];
		__shared__ __align__(8) uint64_t part_full_bar[2];
		__shared__ __align__(8) uint64_t part_empty_bar[2];
		__shared__ __align__(8) uint64_t scale_free_bar[kScaleSlots];
		__shared__ uint32_t tmem_base_slot;
		__shared__ int abort_flag;
		__shared__ __align__(16) float a_scale_s[kScaleSlots][128];
		__shared__ __align__(16) float b_scale_s[kScaleSlots][2];

		const int warp = threadIdx.x / 32;
		const int lane = threadIdx.x % 32;
		const int rank = static_cast<int>(umma::cluster_cta_rank());
		const int pair = blockIdx.x / 2;
		const int pairs = gridDim.x / 2;

		if (threadIdx.x == 0)
		{
			abort_flag = 0;
			for (int s = 0; s < kPairStages; s++)
			{
				umma::mbar_init(&full_bar[s], 1);
				umma::mbar_init(&empty_bar[s], 1);
			}
			for (int b = 0; b < 2; b++)
			{
				umma::mbar_init(&part_full_bar[b], 2);
				umma::mbar_init(&part_empty_bar[b], 2 * 8);
			}
			for (int b = 0; b < kScaleSlots; b++)
				umma::mbar_init(&scale_free_bar[b], 8);
			umma::mbar_fence_init();
			umma::prefetch_tensormap(&mapA);
			umma::prefetch_tensormap(&mapB);
			if (bulkStore)
				umma::prefetch_tensormap(&mapC);
		}
		if (warp == 3)
		{
			umma::tmem_alloc_pair(&tmem_base_slot, 512);
			umma::tmem_relinquish_pair();
		}
		umma::tcgen05_fence_before();
		__syncthreads();
		umma::cluster_sync_all(); /* both CTAs' barriers exist before anything arrives on them */
		umma::tcgen05_fence_after();
		const uint32_t tmem_base = tmem_base_slot;
		volatile int *abort_ptr = &abort_flag;
		chain_release();
		chain_wait();

		if (warp < kPairControlThreads / 32)
		{
			asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairControlRegisters));
		}
		if (warp == 0)
		{
			if (lane == 0)
			{
				int stage = 0;
				uint32_t phase = 0;
				bool ok = true;
				for (int tile = pair; tile < numTiles and ok; tile += pairs)
				{
					const PairTile t = pair_tile(tile, mBlocks, nBlocks);
					const int m0 = t.m * 256 + rank * 128, n0 = t.n * 256 + rank * 128;
					for (int kb = 0; kb < p.blocks; kb++)
					{
						if (not umma::mbar_wait(&empty_bar[stage], phase ^ 1u, abort_ptr))
						{
							umma::raise_error(abort_ptr, deviceStatus, umma::kErrorStageWait);
							ok = false;
							break;
						}
						const uint32_t bar = umma::map_to_cta(umma::smem_u32(&full_bar[stage]), 0);
						if (rank == 0)
							umma::mbar_arrive_expect_tx(&full_bar[stage], 2 * kPairSlotBytes);
						uint8_t *slot = smem + stage * kPairSlotBytes;
						umma::tma_load_2d_pair(slot, &mapA, bar, kb * kScaleBlock, m0);
						umma::tma_load_2d_pair(slot + kBlockBytes, &mapB, bar, kb * kScaleBlock, n0);
						if (++stage == kPairStages)
						{
							stage = 0;
							phase ^= 1u;
						}
					}
				}
			}
		}
		else if (warp == 1 or warp == 2)
		{
			if (lane == 0 and rank == 0)
			{
				/* issuer b takes the blocks b, b + 2, ... of the whole sequence of tiles, whose slots are two apart */
				constexpr uint32_t idesc = umma::make_instr_desc(umma::kAccumF32, umma::kFormatE4M3, umma::kFormatE4M3, false, false, 256, 256);
				const uint64_t desc0 = umma::make_smem_desc(umma::smem_u32(smem), 16, 1024, umma::kSwizzle128B);
				const int b = warp - 1;
				const int tiles = (numTiles - pair + pairs - 1) / pairs;
				const long long total = static_cast<long long>(tiles) * p.blocks;
				int stage = b;
				uint32_t phase = 0, part_phase = 0;
				bool ok = true;
				for (long long i = b; i < total and ok; i += 2)
				{
					if (not umma::mbar_wait(&full_bar[stage], phase, abort_ptr))
					{
						umma::raise_error(abort_ptr, deviceStatus, umma::kErrorTmaWait);
						break;
					}
					const uint64_t desc = desc0 + static_cast<uint64_t>(stage * (kPairSlotBytes / 16));
					if (not umma::mbar_wait(&part_empty_bar[b], part_phase ^ 1u, abort_ptr))
					{
						umma::raise_error(abort_ptr, deviceStatus, umma::kErrorMmaWait);
						ok = false;
						break;
					}
					umma::tcgen05_fence_after();
					umma::mma_f8_pair_k4(tmem_base + static_cast<uint32_t>(b * 256), desc, desc + kBlockBytes / 16, idesc, false);
					umma::mma_commit_pair(&empty_bar[stage], 3);
					umma::mma_commit_pair(&part_full_bar[b], 3); /* last: who has seen it need not expect another arrival */
					part_phase ^= 1u;
					stage += 2;
					if (stage >= kPairStages)
					{
						stage -= kPairStages;
						phase ^= 1u;
					}
				}
			}
		}
		else if (warp == 3)
		{
			/* Scales of this CTA's 128 rows and of the two column halves, four rows per lane, loaded kScaleAhead blocks before they are
			 * handed over.  Block i may use slot i % 3 once every promotion warp has read block i - 3 (scale_free), and may arrive on
			 * its accumulator's barrier once the phase of block i - 2 is over; both lie a block's time back, so that this warp is never
			 * the one that is waited for. */
			float ahead_a[kScaleAhead][4], ahead_b[kScaleAhead];
			const int tiles = (numTiles - pair + pairs - 1) / pairs;
			const long long total = static_cast<long long>(tiles) * p.blocks;
			const float *from_a[4], *from_b;
			int next_tile = pair, left = 0;
			auto fetch = [&](float (&va)[4], float &vb)
			{
				if (left == 0)
				{
					/* rows and columns past the end have products of zeros: any scale will do, the last one's is there */
					const PairTile t = pair_tile(min(next_tile, numTiles - 1), mBlocks, nBlocks);
					const int row0 = t.m * 256 + rank * 128 + lane;
#pragma unroll
					for (int j = 0; j < 4; j++)
						from_a[j] = p.a_scale + static_cast<long long>(min(row0 + j * 32, p.M - 1)) * p.blocks;
					from_b = p.b_scale + static_cast<long long>(min(t.n * 2 + (lane & 1), (p.N - 1) / kScaleBlock)) * p.blocks;
					next_tile += pairs;
					left = p.blocks;
				}
#pragma unroll
				for (int j = 0; j < 4; j++)
					va[j] = *from_a[j]++;
				vb = *from_b++;
				left--;
			};
#pragma unroll
			for (int d = 0; d < kScaleAhead; d++)
				fetch(ahead_a[d], ahead_b[d]);
			uint32_t slot_phase = 1; /* of the block before in the same slot: nothing to wait for in the first round */
			bool ok = true;
			for (long long i0 = 0; i0 < total and ok; i0 += kScaleAhead, slot_phase ^= 1u)
			{
#pragma unroll
				for (int d = 0; d < kScaleAhead; d++)
				{
					static_assert(kScaleSlots == kScaleAhead, "slot of block i0 + d");
					const long long i = i0 + d;
					if (i >= total)
						break;
					uint64_t *bar = &part_full_bar[i & 1];
					const uint32_t phase = (static_cast<uint32_t>(i >> 1) & 1u) ^ 1u;
					ok = __all_sync(0xFFFFFFFFu, umma::mbar_wait(&scale_free_bar[d], slot_phase, abort_ptr)
							and (i < 2 or umma::mbar_wait(bar, phase, abort_ptr)));
					if (not ok)
					{
						if (lane == 0)
							umma::raise_error(abort_ptr, deviceStatus, umma::kErrorEpilogueWait);
						break;
					}
#pragma unroll
					for (int j = 0; j < 4; j++)
						a_scale_s[d][j * 32 + lane] = ahead_a[d][j];
					if (lane < 2)
						b_scale_s[d][lane] = ahead_b[d];
					__syncwarp();
					if (lane == 0)
						umma::mbar_arrive(bar);
					fetch(ahead_a[d], ahead_b[d]);
				}
			}
		}
		else if (warp >= kPairControlThreads / 32)
		{
			asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairPromoteRegisters));
			const int quarter = warp % 4;
			const int column_half = (warp - kPairControlThreads / 32) / 4;
			const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(column_half * 128);
			uint8_t *buffers = smem + kPairStages * kPairSlotBytes + (warp - kPairControlThreads / 32) * 2 * kSubBytes;
			uint32_t b = 0, phase = 0, slot = 0;
			bool ok = true;
			for (int tile = pair; tile < numTiles and ok; tile += pairs)
			{
				const PairTile t = pair_tile(tile, mBlocks, nBlocks);
				const int row0 = t.m * 256 + rank * 128 + quarter * 32;
				const int column0 = t.n * 256 + column_half * 128;
				float acc[128];
#pragma unroll
				for (int i = 0; i < 128; i++)
					acc[i] = 0.0f;
				for (int kb = 0; kb < p.blocks; kb++)
				{
					ok = __all_sync(0xFFFFFFFFu, lane != 0 or umma::mbar_wait(&part_full_bar[b], phase, abort_ptr)); /* one lane polls: 590 -> 540 us at 8192^3 */
					if (not ok)
					{
						if (lane == 0)
							umma::raise_error(abort_ptr, deviceStatus, umma::kErrorEpilogueWait);
						break;
					}
					__syncwarp(); /* a vote orders no memory: what lane 0 has waited for is ordered before the other lanes' reads here */
					umma::tcgen05_fence_after();
					const uint32_t from = lanes + b * 256u;
					uint32_t r[2][16];
					umma::tmem_load_32x16(from, r[0]);
					const float scale = a_scale_s[slot][quarter * 32 + lane] * b_scale_s[slot][column_half];
					__syncwarp();
					if (lane == 0)
						umma::mbar_arrive(&scale_free_bar[slot]);
					slot = slot == kScaleSlots - 1 ? 0 : slot + 1;
#pragma unroll
					for (int chunk = 0; chunk < 8; chunk++)
					{
						umma::tmem_load_wait(r[chunk & 1]);
						if (chunk < 7)
							umma::tmem_load_32x16(from + static_cast<uint32_t>((chunk + 1) * 16), r[(chunk + 1) & 1]);
						else
						{
							umma::tcgen05_fence_before();
							__syncwarp();
							if (lane == 0)
								umma::mbar_arrive_cluster_relaxed(umma::map_to_cta(umma::smem_u32(&part_empty_bar[b]), 0));
						}
#pragma unroll
						for (int i = 0; i < 16; i++)
							acc[chunk * 16 + i] = fmaf(__uint_as_float(r[chunk & 1][i]), scale, acc[chunk * 16 + i]);
					}
					if ((b ^= 1u) == 0)
						phase ^= 1u;
				}
				if (not ok)
					break;
				store_rows<T, ADD>(p, &mapC, buffers, acc, row0, column0, lane, bulkStore != 0);
			}
			if (lane == 0)
				umma::tma_store_wait_all<0>();
		}

		/* neither CTA may leave (or free TMEM) while the other can still touch its shared memory, barriers or TMEM */
		__syncthreads();
		if (abort_flag != 0)
			umma::drain_after_abort();
		umma::tcgen05_fence_before();
		umma::cluster_sync_all();
		if (warp == 3)
		{
			umma::tcgen05_fence_after();
			umma::tmem_dealloc_pair(tmem_base, 512);
		}
	}

	int sm_count(const ContextObject &ctx)
	{
		int sms = 148;
		cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, ctx.device);
		return sms;
	}
	bool make_operand_map(CUtensorMap *map, const uint8_t *base, int rows, int k, int boxRows)
	{
		const uint64_t dims[2] = { static_cast<uint64_t>(k), static_cast<uint64_t>(rows) };
		const uint64_t strides[1] = { static_cast<uint64_t>(k) };
		const uint32_t box[2] = { kScaleBlock, static_cast<uint32_t>(boxRows) };
		return umma::make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
	}

	/* how many clusters of each size run at once: a cluster stays within a group of SMs and a CTA fills an SM, so SMs are left over in
	 * each group (148 SMs hold 45 clusters of three, 33 of four, 15 of eight) */
	struct ClustersAtOnce
	{
			int of_size[kMaxSplits + 1];
	};
	/* CTAs per tile: the number that ends first, where a CTA's time is its blocks of K (about 350 cycles each) plus that of
	 * kOverhead blocks for set-up, first copy and reduction. */
	int choose_splits(long long tiles, int blocks, const ClustersAtOnce &clusters)
	{
		constexpr int kOverhead = 6;
		int best = 1;
		long long best_cost = 0;
		for (int s = 1; s <= std::min(kMaxSplits, blocks); s++)
		{
			if (clusters.of_size[s] < 1)
				continue;
			const long long waves = (tiles + clusters.of_size[s] - 1) / clusters.of_size[s];
			const long long cost = waves * ((blocks + s - 1) / s + kOverhead);
			if (s == 1 or cost < best_cost)
			{
				best = s;
				best_cost = cost;
			}
		}
		return best;
	}

	template<int TOKENS, bool LOADERS>
	avStatus_t launch_split(ContextObject &ctx, const ScaledGemm &p)
	{
		using Cfg = SplitConfig<TOKENS, LOADERS>;
		auto kernel = kernel_gemm_f8_split<TOKENS, LOADERS>;
		cudaLaunchConfig_t config = { };
		config.blockDim = dim3(Cfg::kThreads);
		config.dynamicSmemBytes = Cfg::kSmemBytes;
		cudaLaunchAttribute attributes[2];
		config.attrs = attributes;
		attributes[0].id = cudaLaunchAttributeClusterDimension;
		attributes[0].val.clusterDim.y = 1;
		attributes[0].val.clusterDim.z = 1;
		static PerDeviceOnce configured;
		static ClustersAtOnce clusters[kMaxDevices];
		const cudaError_t ready = configured.run(ctx.device, [&]() -> cudaError_t
		{
			const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
			clusters[ctx.device].of_size[1] = sm_count(ctx);
			for (int s = 2; status == cudaSuccess and s <= kMaxSplits; s++)
			{
				attributes[0].val.clusterDim.x = static_cast<unsigned>(s);
				config.gridDim = dim3(static_cast<unsigned>(s));
				config.numAttrs = 1;
				if (cudaOccupancyMaxActiveClusters(&clusters[ctx.device].of_size[s], kernel, &config) != cudaSuccess)
				{
					cudaGetLastError();
					clusters[ctx.device].of_size[s] = 0; /* such clusters are not used */
				}
			}
			return status;
		});
		if (ready != cudaSuccess)
		{
			cudaGetLastError();
			return AVOCADO_STATUS_EXECUTION_FAILED;
		}
		CUtensorMap mapA = { }, mapB = { };
		if (not LOADERS and (not make_operand_map(&mapA, p.a, p.M, p.K, TOKENS) or not make_operand_map(&mapB, p.b, p.N, p.K, 128)))
			return AVOCADO_STATUS_INTERNAL_ERROR;
		const long long token_tiles = (static_cast<long long>(p.M) + TOKENS - 1) / TOKENS;
		const long long tiles = token_tiles * scale_blocks(p.N);
		const int splits = choose_splits(tiles, p.blocks, clusters[ctx.device]);
		if (tiles * splits > 0x7FFFFFFFll)
			return AVOCADO_STATUS_NOT_SUPPORTED;
		config.gridDim = dim3(static_cast<unsigned>(tiles * splits));
		config.stream = ctx.getStream();
		attributes[0].val.clusterDim.x = static_cast<unsigned>(splits);
		cudaLaunchAttribute &chained = attributes[splits > 1 ? 1 : 0];
		chained.id = cudaLaunchAttributeProgrammaticStreamSerialization;
		chained.val.programmaticStreamSerializationAllowed = chained_launches_enabled() ? 1 : 0;
		config.numAttrs = splits > 1 ? 2 : 1;
		const cudaError_t launched = cudaLaunchKernelEx(&config, kernel, mapA, mapB, p, static_cast<int>(token_tiles), splits, (p.blocks + splits - 1) / splits,
				ctx.getDeviceStatus());
		return launched != cudaSuccess ? convertStatus(launched) : checkForErrors();
	}
	template<bool LOADERS>
	avStatus_t launch_split(ContextObject &ctx, const ScaledGemm &p)
	{
		if (p.M <= 16)
			return launch_split<16, LOADERS>(ctx, p);
		if (p.M <= 32)
			return launch_split<32, LOADERS>(ctx, p);
		if (LOADERS or p.M <= 64)
			return launch_split<64, LOADERS>(ctx, p);
		return launch_split<128, false>(ctx, p);
	}

	template<typename T, bool ADD>
	avStatus_t launch_pair(ContextObject &ctx, const ScaledGemm &p)
	{
		auto kernel = kernel_gemm_f8_pair<T, ADD>;
		static PerDeviceOnce configured;
		if (configured.run(ctx.device, [&]() -> cudaError_t { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmemBytes); }) != cudaSuccess)
		{
			cudaGetLastError();
			return AVOCADO_STATUS_EXECUTION_FAILED;
		}
		CUtensorMap mapA, mapB, mapC = { };
		if (not make_operand_map(&mapA, p.a, p.M, p.K, 128) or not make_operand_map(&mapB, p.b, p.N, p.K, 128))
			return AVOCADO_STATUS_INTERNAL_ERROR;
		constexpr int size = static_cast<int>(sizeof(T));
		const bool bulk = static_cast<long long>(p.N) * size % 16 == 0 and reinterpret_cast<uintptr_t>(p.c) % 16 == 0;
		if (bulk)
		{
			const CUtensorMapDataType type = p.c_type == AVOCADO_DTYPE_FLOAT32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 :
					p.c_type == AVOCADO_DTYPE_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
			const uint64_t dims[2] = { static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M) };
			const uint64_t strides[1] = { static_cast<uint64_t>(p.N) * size };
			const uint32_t box[2] = { static_cast<uint32_t>(128 / size), 32 };
			if (not umma::make_tensor_map(&mapC, type, 2, p.c, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
				return AVOCADO_STATUS_INTERNAL_ERROR;
		}
		const int m_blocks = (p.M + 255) / 256, n_blocks = (p.N + 255) / 256;
		const long long tiles = static_cast<long long>(m_blocks) * n_blocks;
		if (tiles > 0x3FFFFFFFll)
			return AVOCADO_STATUS_NOT_SUPPORTED;
		const int pairs = static_cast<int>(std::min<long long>(tiles, sm_count(ctx) / 2));
		const cudaError_t launched = launch_chained(kernel, dim3(2 * pairs), dim3(kPairThreads), kPairSmemBytes, ctx.getStream(), mapA, mapB, mapC, p, m_blocks,
				n_blocks, static_cast<int>(tiles), bulk ? 1 : 0, ctx.getDeviceStatus());
		return launched != cudaSuccess ? convertStatus(launched) : checkForErrors();
	}

	avStatus_t launch_pair(ContextObject &ctx, const ScaledGemm &p)
	{
		const bool add = p.beta != 0.0f;
		if (p.c_type == AVOCADO_DTYPE_FLOAT32)
			return add ? launch_pair<float, true>(ctx, p) : launch_pair<float, false>(ctx, p);
		if (p.c_type == AVOCADO_DTYPE_FLOAT16)
			return add ? launch_pair<half, true>(ctx, p) : launch_pair<half, false>(ctx, p);
		return add ? launch_pair<__nv_bfloat16, true>(ctx, p) : launch_pair<__nv_bfloat16, false>(ctx, p);
	}

	avStatus_t launch(ContextObject &ctx, const ScaledGemm &p)
	{
		if (p.K == 0)
		{
			const long long wanted = (static_cast<long long>(p.M) * p.N + 255) / 256;
			const dim3 grid(static_cast<unsigned>(std::min<long long>(wanted, static_cast<long long>(sm_count(ctx)) * 8)));
			const cudaError_t launched = launch_chained(kernel_scale_c, grid, dim3(256), 0, ctx.getStream(), p);
			return launched != cudaSuccess ? convertStatus(launched) : checkForErrors();
		}
		/* Few tiles leave most pairs idle, and 256-row tiles waste what few rows of A do not fill.  bfloat16 C, us in a graph, pairs / split:
		 * 129 x 2048 x 4096 (8 tiles) 19.2 / 9.7, 256 x 4096 x 4096 (16) 19.6 / 14.0, 1024^3 (16) 8.4 / 8.5, 333 x 2056 x 1616 (18) 11.1 / 10.0,
		 * 129 and 256 x 8192 x 4096 (32) 20.2 / 22.0 and 20.5 / 22.3, 512 x 4096 x 4096 (32) 20.0 / 22.0, 4096 x 512 x 4096 (32) 20.1 / 22.0,
		 * 2048^3 (64) 13.2 / 28.2. */
		const bool tma = p.K % 16 == 0 and (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16 == 0;
		if (tma and p.M > 128 and static_cast<long long>((p.M + 255) / 256) * ((p.N + 255) / 256) >= 32)
			return launch_pair(ctx, p);
		return tma ? launch_split<false>(ctx, p) : launch_split<true>(ctx, p);
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
				constexpr int kMaxExtent = 1 << 30; /* indices, rounded up to whole tiles, stay in 32 bits */
				if (p.M > kMaxExtent or p.N > kMaxExtent or p.K > kMaxExtent)
					return AVOCADO_STATUS_NOT_SUPPORTED;
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
				p.c_type = c.dtype;
				const int four = 4 * static_cast<int>(dtype_size(c.dtype));
				p.c_vector = (p.N % 4 == 0 and co.aligned(four)) ? 1 : 0;
				if (cuda_sm_version(ctx.device) != 100)
					return AVOCADO_STATUS_NOT_SUPPORTED;
				return launch(ctx, p);
			AVOCADO_API_END
		}
	} /* namespace backend */
} /* namespace avocado */

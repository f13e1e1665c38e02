/*
 * block_scaled.hpp -- what the operators on block-scaled 8-bit tensors (quantize.cu, gemm_f8.cu) share: the constants of the
 * format and the checks of their arguments.
 */
#ifndef B200_BLOCK_SCALED_HPP_
#define B200_BLOCK_SCALED_HPP_

#include "objects.hpp"

#include <cstdint>

namespace bk
{
	constexpr int kScaleBlock = 128;                          /* elements of the last dimension under one scale */
	constexpr float kLargestE4m3 = 448.0f;
	constexpr float kSmallestAmax = 7.888609052210118e-31f;   /* 2^-100: keeps the scale and its reciprocal normal numbers */

	inline int scale_blocks(int extent)
	{
		return extent / kScaleBlock + (extent % kScaleBlock != 0 ? 1 : 0);
	}

	/* Extents that no caller means (negative, no dimension, more than 2^40 elements) are refused before anything is computed
	 * from them, so that sizes in bytes stay far inside 64 bits. */
	inline bool valid_extents(const avocado::backend::b200::TensorObject &t)
	{
		if (t.nb_dims < 1)
			return false;
		bool empty = false;
		for (int i = 0; i < t.nb_dims; i++)
		{
			if (t.dims[i] < 0)
				return false;
			empty = empty or t.dims[i] == 0;
		}
		if (empty)
			return true;
		constexpr int64_t limit = static_cast<int64_t>(1) << 40;
		int64_t volume = 1;
		for (int i = 0; i < t.nb_dims; i++)
		{
			if (t.dims[i] > limit / volume)
				return false;
			volume *= t.dims[i];
		}
		return true;
	}
	inline int64_t row_count(const avocado::backend::b200::TensorObject &t) /* all dimensions but the last */
	{
		int64_t rows = 1;
		for (int i = 0; i + 1 < t.nb_dims; i++)
			rows *= t.dims[i];
		return rows;
	}

	/* A device operand: its address and how many bytes of it the call touches. */
	struct Operand
	{
			uint8_t *ptr = nullptr;
			int64_t bytes = 0;

			bool overlaps(const Operand &other) const
			{
				return bytes > 0 and other.bytes > 0 and ptr < other.ptr + other.bytes and other.ptr < ptr + bytes;
			}
			bool same_as(const Operand &other) const
			{
				return ptr == other.ptr and bytes == other.bytes;
			}
			bool aligned(int to) const
			{
				return reinterpret_cast<uintptr_t>(ptr) % to == 0;
			}
	};
	/* False when the memory block is too small for the tensor, lies on another device, or starts off the element's boundary. */
	inline bool get_operand(Operand &result, const avocado::backend::b200::ContextObject &ctx, avocado::backend::avMemoryDescriptor_t mem,
			const avocado::backend::b200::TensorObject &desc)
	{
		const avocado::backend::b200::MemoryObject &memory = avocado::backend::b200::getMemory(mem);
		result.ptr = reinterpret_cast<uint8_t*>(memory.ptr);
		result.bytes = desc.sizeInBytes();
		if (result.bytes == 0)
			return true;
		return result.ptr != nullptr and memory.size >= result.bytes and memory.device == ctx.device
				and result.aligned(static_cast<int>(avocado::backend::b200::dtype_size(desc.dtype)));
	}
} /* namespace bk */

#endif /* B200_BLOCK_SCALED_HPP_ */

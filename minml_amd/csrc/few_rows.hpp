/*
 * few_rows.hpp — products y = x W^T of at most 64 rows of x: single tokens and small batches, where every weight is read once and used a handful of times.
 *
 * The weights' bytes bound it, so they go from memory straight into MFMA operands, without LDS: a workgroup owns two blocks of 16 rows of W (of the two matrices of a pair, or neighbours), its 4 wavefronts
 * take every fourth 128-byte piece of k, and a lane loads 16 bytes of one row at a time: the 4 lanes of a row take a whole 128-byte line in two loads. x comes from the caches: the lanes that hold the
 * same row of x read the same addresses. The order of k inside a piece is whatever the loads give, the same for both operands. The partial sums meet in LDS.
 * Rows of any length and alignment: the last piece of k is put together element by element where it is not whole.
 */
#ifndef MINML_AMD_FEW_ROWS_HPP_
#define MINML_AMD_FEW_ROWS_HPP_

#include "gemm_core.hpp"
#include "training_utils.hpp"

#include <type_traits>

namespace mlhip
{
	/*
	 * Whether a product is taken here or on tiles. Up to 16 rows always (1 and 16 rows of 4096 -> 2 x 8192 fp16 26 and 31 us, tiles 30); up to 64 while rows times the weights' bytes are below 2^31 in fp16, where the rows
	 * of x cost more than the weights from there on (us here / tiles: 17 rows of 2048 -> 2 x 4096 10.6 / 15, of 4096 -> 2 x 8192 34 / 30, 64 rows 16.0 / 15.4 and 58 / 30; of 1024 -> 2 x 2048 9.8 / 13); in fp32, where the
	 * matrix cores bound both, up to 64 (64 rows of 4096 -> 2 x 8192 145 / 147).
	 */
	inline bool takes_few_rows(int rows, size_t weight_bytes, int element_size)
	{
		return rows <= 16 || (rows <= 64 && (element_size == 4 || rows * weight_bytes <= (size_t(1) << 31)));
	}

	template<typename T>
	__device__ __forceinline__ void mma_16x16(const uint4_t &a, const uint4_t &b, float4_t &c)
	{
		if constexpr (sizeof(T) == 2)
			c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
		else
		{
			const float4_t fa = __builtin_bit_cast(float4_t, a), fb = __builtin_bit_cast(float4_t, b);
#pragma unroll
			for (int e = 0; e < 4; e++)
				c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[e], fb[e], c, 0, 0, 0);
		}
	}
	/* 16 bytes of a row that may begin anywhere */
	template<typename T>
	__device__ __forceinline__ uint4_t load_piece(const T *p)
	{
		Elements<T, 16 / sizeof(T)> v;
		v.load(p);
		return __builtin_bit_cast(uint4_t, v.raw);
	}
	/* the same for what is read once: not meant to be kept in the caches */
	template<typename T>
	__device__ __forceinline__ uint4_t load_streaming(const T *p)
	{
		return __builtin_bit_cast(uint4_t, __builtin_nontemporal_load(reinterpret_cast<const typename Elements<T, 16 / sizeof(T)>::unaligned_t*>(p)));
	}
	/* the same where only `left` elements (perhaps none, or less) are the row's; the others are zero */
	template<typename T>
	__device__ __forceinline__ uint4_t load_piece(const T *p, int left)
	{
		constexpr int N = 16 / sizeof(T);
		if (left >= N)
			return load_piece(p);
		typename Elements<T, N>::vec_t v;
#pragma unroll
		for (int e = 0; e < N; e++)
			v[e] = e < left ? p[e] : static_cast<T>(0.0f);
		return __builtin_bit_cast(uint4_t, v);
	}

	/*
	 * sums[0][2][16 MB][16] (matrix or neighbour, row of x, row of W) in LDS when it returns, complete for all threads (the other WAVES - 1 are scratch). first: row of W of the first block, second: of the second; rows past the end are
	 * read as the last one, their sums are no one's.
	 */
	template<typename T, int MB, int WAVES>
	__device__ __forceinline__ void few_rows_sums(const T *x, int rows, const T *w_first, const T *w_second, int last_first, int last_second, int k, float (*sums)[2][16 * MB][16])
	{
		/* elements of a 128-byte piece and of a load; pieces of a batch: two batches of 16 KB of weights are on their way (8 KB where many rows of x take the registers) */
		constexpr int PIECE = 128 / sizeof(T), N = 16 / sizeof(T), STEPS = MB == 4 ? 1 : 2;
		const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
		const T *w[2] = { w_first + static_cast<size_t>(min(r, last_first)) * k, w_second + static_cast<size_t>(min(r, last_second)) * k };
		const T *xs[MB];
#pragma unroll
		for (int b = 0; b < MB; b++)
			xs[b] = x + static_cast<size_t>(min(b * 16 + r, rows - 1)) * k;
		float4_t acc[2][MB];
#pragma unroll
		for (int i = 0; i < 2; i++)
#pragma unroll
			for (int b = 0; b < MB; b++)
				acc[i][b] = float4_t { 0.0f, 0.0f, 0.0f, 0.0f };
		struct Batch
		{
				uint4_t weights[STEPS][2][2], rows[STEPS][MB][2];
		};
		const auto request = [&](Batch &batch, int piece) __attribute__((always_inline))
		{
#pragma unroll
			for (int s = 0; s < STEPS; s++)
#pragma unroll
				for (int h = 0; h < 2; h++)
				{
					const int at = (piece + WAVES * s) * PIECE + (2 * q + h) * N;
#pragma unroll
					for (int i = 0; i < 2; i++)
						batch.weights[s][i][h] = load_streaming(w[i] + at);
#pragma unroll
					for (int b = 0; b < MB; b++)
						batch.rows[s][b][h] = load_piece(xs[b] + at);
				}
		};
		const auto multiply = [&](const Batch &batch) __attribute__((always_inline))
		{
#pragma unroll
			for (int s = 0; s < STEPS; s++)
#pragma unroll
				for (int h = 0; h < 2; h++)
#pragma unroll
					for (int b = 0; b < MB; b++)
#pragma unroll
						for (int i = 0; i < 2; i++)
							mma_16x16<T>(batch.weights[s][i][h], batch.rows[s][b][h], acc[i][b]);
		};
		const int whole = k / PIECE;
		const int batches = max(0, (whole - wave + WAVES - 1) / WAVES) / STEPS; /* of this wavefront's pieces wave, wave + WAVES, ... */
		Batch even, odd;
		if (batches > 0)
			request(even, wave);
		for (int n = 0; n < batches; n += 2)
		{
			if (n + 1 < batches)
				request(odd, wave + (n + 1) * WAVES * STEPS);
			__builtin_amdgcn_sched_barrier(0); /* the next batch is on its way before this one is waited for */
			multiply(even);
			if (n + 1 < batches)
			{
				if (n + 2 < batches)
					request(even, wave + (n + 2) * WAVES * STEPS);
				__builtin_amdgcn_sched_barrier(0);
				multiply(odd);
			}
		}
		for (int piece = wave + batches * WAVES * STEPS; piece * PIECE < k; piece += WAVES)
#pragma unroll
			for (int h = 0; h < 2; h++)
			{
				const int at = piece * PIECE + (2 * q + h) * N;
				uint4_t weights[2];
#pragma unroll
				for (int i = 0; i < 2; i++)
					weights[i] = load_piece(w[i] + at, k - at);
#pragma unroll
				for (int b = 0; b < MB; b++)
				{
					const uint4_t v = load_piece(xs[b] + at, k - at);
#pragma unroll
					for (int i = 0; i < 2; i++)
						mma_16x16<T>(weights[i], v, acc[i][b]);
				}
			}
		/* lane: row of x r, rows 4 q .. 4 q + 3 of W. The wavefronts' sums are added up in order */
#pragma unroll
		for (int i = 0; i < 2; i++)
#pragma unroll
			for (int b = 0; b < MB; b++)
				*reinterpret_cast<float4_t*>(&sums[wave][i][b * 16 + r][4 * q]) = acc[i][b];
		__syncthreads();
		constexpr int COUNT = 2 * 16 * MB * 16;
		float *flat = &sums[0][0][0][0];
		for (int i = threadIdx.x; i < COUNT; i += 64 * WAVES)
		{
			float total = flat[i];
#pragma unroll
			for (int v = 1; v < WAVES; v++)
				total += flat[v * COUNT + i];
			flat[i] = total;
		}
		__syncthreads();
	}
	/*
	 * How many wavefronts share a row: as many as leave each four 128-byte pieces, so that a workgroup asks for whole rows at once and the chip for one dense stretch of the weights at a time. Up to 16 rows of x; more need
	 * the LDS for their sums.
	 */
	template<typename T>
	inline int few_rows_waves(int rows, int k)
	{
		const int pieces = k / (128 / static_cast<int>(sizeof(T)));
		return rows > 16 || pieces < 32 ? 4 : pieces < 64 ? 8 : 16;
	}
	/* f(MB, WAVES) as compile-time constants */
	template<typename T, typename F>
	inline void with_few_rows(int rows, int k, F &&f)
	{
		const int waves = few_rows_waves<T>(rows, k);
		typedef std::integral_constant<int, 4> four;
		if (rows > 32)
			f(four(), four());
		else if (rows > 16)
			f(std::integral_constant<int, 2>(), four());
		else if (waves == 4)
			f(std::integral_constant<int, 1>(), four());
		else if (waves == 8)
			f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
		else
			f(std::integral_constant<int, 1>(), std::integral_constant<int, 16>());
	}
} /* namespace mlhip */

#endif /* MINML_AMD_FEW_ROWS_HPP_ */

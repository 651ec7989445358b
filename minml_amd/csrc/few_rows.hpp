/*
 * few_rows.hpp — products y = x W^T of at most 64 rows of x: single tokens and small batches, where every weight is read once and used a handful of times.
 *
 * The weights' bytes bound it, so they go from memory straight into MFMA operands, without LDS: a workgroup owns two blocks of 16 rows of W (of the two matrices of a pair, or neighbours), its 4 wavefronts
 * take every fourth 128-byte piece of k, and a lane loads 16 bytes of one row at a time: the 4 lanes of a row take a whole 128-byte line in two loads. x comes from the caches: the lanes that hold the
 * same row of x read the same addresses. The order of k inside a piece is whatever the loads give, the same for both operands. The four partial sums meet in LDS.
 * Rows of any length and alignment: the last piece of k is put together element by element where it is not whole.
 */
#ifndef MINML_AMD_FEW_ROWS_HPP_
#define MINML_AMD_FEW_ROWS_HPP_

#include "gemm_core.hpp"
#include "training_utils.hpp"

namespace mlhip
{
	constexpr int MOST_FEW_ROWS = 64;

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
	 * sums[2][16 MB][16] (matrix or neighbour, row of x, row of W) in LDS when it returns, complete for all threads. first: row of W of the first block, second: of the second; rows past the end are
	 * read as the last one, their sums are no one's.
	 */
	template<typename T, int MB>
	__device__ __forceinline__ void few_rows_sums(const T *x, int rows, const T *w_first, const T *w_second, int last_first, int last_second, int k, float (*sums)[16 * MB][16])
	{
		/* elements of a 128-byte piece and of a load; pieces of a batch: two batches of 16 KB of weights are on their way (8 KB where many rows of x take the registers) */
		constexpr int PIECE = 128 / sizeof(T), N = 16 / sizeof(T), STEPS = MB == 1 ? 4 : 2;
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
					const int at = (piece + 4 * s) * PIECE + (2 * q + h) * N;
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
		const int batches = max(0, (whole - wave + 3) / 4) / STEPS; /* of this wavefront's pieces wave, wave + 4, ... */
		Batch even, odd;
		if (batches > 0)
			request(even, wave);
		for (int n = 0; n < batches; n += 2)
		{
			if (n + 1 < batches)
				request(odd, wave + (n + 1) * 4 * STEPS);
			__builtin_amdgcn_sched_barrier(0); /* the next batch is on its way before this one is waited for */
			multiply(even);
			if (n + 1 < batches)
			{
				if (n + 2 < batches)
					request(even, wave + (n + 2) * 4 * STEPS);
				__builtin_amdgcn_sched_barrier(0);
				multiply(odd);
			}
		}
		for (int piece = wave + batches * 4 * STEPS; piece * PIECE < k; piece += 4)
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
		/* lane: row of x r, rows 4 q .. 4 q + 3 of W. The wavefronts add theirs up in order */
		for (int turn = 0; turn < 4; turn++)
		{
			if (wave == turn)
#pragma unroll
				for (int i = 0; i < 2; i++)
#pragma unroll
					for (int b = 0; b < MB; b++)
					{
						float4_t *dst = reinterpret_cast<float4_t*>(&sums[i][b * 16 + r][4 * q]);
						*dst = turn == 0 ? acc[i][b] : *dst + acc[i][b];
					}
			__syncthreads();
		}
	}
} /* namespace mlhip */

#endif /* MINML_AMD_FEW_ROWS_HPP_ */

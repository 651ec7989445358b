/*
 * few_rows.hpp — products y = x W^T of at most 64 rows of x: single tokens and small batches, where every weight is read once and used a handful of times. The weights' bytes bound it.
 *
 * A workgroup of 4 wavefronts owns two blocks of 16 rows of W (of the two matrices of a pair, or neighbours) and leaves their sums with all rows of x in LDS. Every wavefront takes one 128-byte piece of every
 * 512 bytes of k; the partial sums meet in LDS.
 *   few_rows_stream: up to 32 rows of x whose rows are whole 16-byte pieces. W and x go through three slots of LDS by direct-to-LDS loads of 1 KB, each two whole runs of 512 bytes of a row, two
 *       slots on their way while one is multiplied: what the memory sees is long runs, and no register waits for it. 1 x 4096 -> 2 x 8192 fp16 23 us (5.8 TB/s).
 *   few_rows_sums: rows of any length, and up to 64 of them. The weights go from memory straight into MFMA operands: 16 bytes of one row per lane, the 4 lanes of a row take a 128-byte line in two loads;
 *       the lanes that hold the same row of x read the same addresses, from the caches. 29 us at the same size. The last piece of k is put together element by element.
 * The order of k inside a piece is whatever the loads give, the same for both operands.
 */
#ifndef MINML_AMD_FEW_ROWS_HPP_
#define MINML_AMD_FEW_ROWS_HPP_

#include "product_tiles.hpp"

#include <type_traits>

namespace mlhip
{
	/*
	 * Whether a product is taken here or on tiles: up to 32 rows, and up to 64 of weights up to 16 MB. Weights from memory, us here / tiles: 1, 16 and 32 rows of 4096 -> 2 x 8192 fp16 23 / 39, 23 / 40, 31 / 40, 64 rows
	 * 60 / 43, of 2048 -> 2 x 4096 18.0 / 17.5, of 1024 -> 2 x 2048 9.8 / 13; 1 row of 2048 x 65536 classes 49 / 71, of 1024 x 30000 17 / 23, 64 rows 36 / 24; fp32 64 rows of 1024 x 30000 88 / 75.
	 */
	inline bool takes_few_rows(int rows, size_t weight_bytes)
	{
		return rows <= 32 || (rows <= 64 && weight_bytes <= (size_t(1) << 24));
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

	constexpr int FEW_ROWS_WAVES = 4;
	/* the wavefronts' sums added up in order. Lane: row of x l % 16, rows 4 (l / 16) .. + 3 of W */
	template<int MB>
	__device__ __forceinline__ void join_few_rows(const float4_t (&acc)[2][MB], float (*sums)[2][16 * MB][16])
	{
		const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
		for (int i = 0; i < 2; i++)
#pragma unroll
			for (int b = 0; b < MB; b++)
				*reinterpret_cast<float4_t*>(&sums[wave][i][b * 16 + (lane & 15)][4 * (lane >> 4)]) = acc[i][b];
		__syncthreads();
		constexpr int COUNT = 2 * 16 * MB * 16;
		float *flat = &sums[0][0][0][0];
		for (int i = threadIdx.x; i < COUNT; i += 64 * FEW_ROWS_WAVES)
		{
			float total = flat[i];
#pragma unroll
			for (int v = 1; v < FEW_ROWS_WAVES; v++)
				total += flat[v * COUNT + i];
			flat[i] = total;
		}
		__syncthreads();
	}
	/*
	 * sums[0][2][16 MB][16] (matrix or neighbour, row of x, row of W) in LDS when it returns, complete for all threads (the other WAVES - 1 are scratch). first: row of W of the first block, second: of the second; rows past the end are
	 * read as the last one, their sums are no one's.
	 */
	template<typename T, int MB>
	__device__ __forceinline__ void few_rows_sums(const T *x, int rows, const T *w_first, const T *w_second, int last_first, int last_second, int k, float (*sums)[2][16 * MB][16])
	{
		/* elements of a 128-byte piece and of a load; pieces of a batch: two batches of 16 KB of weights are on their way (8 KB where many rows of x take the registers) */
		constexpr int PIECE = 128 / sizeof(T), N = 16 / sizeof(T), STEPS = MB == 4 ? 1 : 2, WAVES = FEW_ROWS_WAVES;
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
		join_few_rows<MB>(acc, sums);
	}
	/*
	 * The same for rows that are whole 16-byte pieces, aligned to 16 bytes. lds: FEW_ROWS_LDS<MB> bytes, where the sums lie in the end. A slot holds [32 rows of W][512 bytes] and [16 MB rows of x][512 bytes]; the 16-byte
	 * pieces of a row are permuted by row % 8 among eight, so that the lanes of a fragment read, which take the same piece of 16 rows, do not all meet the same banks. Rows of x that do not exist and what lies behind a row's end are
	 * zeros (loads behind the buffer's end).
	 */
	constexpr int FEW_ROWS_RUN = 512, FEW_ROWS_SLOTS = 3;
	template<int MB>
	constexpr int FEW_ROWS_SLOT = (32 + 16 * MB) * FEW_ROWS_RUN;
	template<int MB>
	constexpr int FEW_ROWS_LDS = FEW_ROWS_SLOTS * FEW_ROWS_SLOT<MB>;
	/* LDS of a workgroup: the slots, or the sums alone */
	template<int MB>
	constexpr int few_rows_lds(bool stream)
	{
		return stream ? FEW_ROWS_LDS<MB> : FEW_ROWS_WAVES * 2 * 16 * MB * 16 * 4;
	}
	template<typename T, int MB>
	__device__ __forceinline__ void few_rows_stream(const T *x, int rows, const T *w_first, const T *w_second, int last_first, int last_second, int k, uint8_t *lds)
	{
		constexpr int SLOT = FEW_ROWS_SLOT<MB>, X_LOADS = 2 * MB, LOADS = 4 + X_LOADS;
		const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
		const int row_bytes = k * static_cast<int>(sizeof(T)), runs = (row_bytes + FEW_ROWS_RUN - 1) / FEW_ROWS_RUN;
		constexpr int NOWHERE = static_cast<int>(0x80000000u);
		/* load u of this wavefront: rows 2 (wave + 4 u) + lane / 32 of the slot; their low three bits are the same for every u */
		const int in_run = ((lane & 31) ^ ((2 * wave + (lane >> 5)) & 7)) * 16;
		int w_offset[4], x_offset[X_LOADS];
#pragma unroll
		for (int u = 0; u < 4; u++)
		{
			const int row = (2 * (wave + 4 * u) + (lane >> 5)) & 15;
			w_offset[u] = row <= (u < 2 ? last_first : last_second) ? row * row_bytes + in_run : NOWHERE;
		}
#pragma unroll
		for (int u = 0; u < X_LOADS; u++)
		{
			const int row = 2 * (wave + 4 * u) + (lane >> 5);
			x_offset[u] = row < rows ? row * row_bytes + in_run : NOWHERE;
		}
		const uint8_t *first = reinterpret_cast<const uint8_t*>(w_first), *second = reinterpret_cast<const uint8_t*>(w_second), *x_bytes = reinterpret_cast<const uint8_t*>(x);
		/*
		 * Workgroups begin at different runs of their rows and go round: rows are often a power of two apart, and workgroups that all ask for the same run ask the same channels of memory. The workgroups of an XCD
		 * (block % 8) begin one run after another, the XCDs spread over the row (us, weights from memory, all from the front / so: 1 x 4096 -> 2 x 8192 fp16 26.9 / 23.1, 1 x 2048 x 65536 classes 55 / 49, fp32
		 * 105 / 88; rows of 4104 23.8 / 23.9).
		 */
		const int turn = static_cast<int>(((blockIdx.x >> 3) + (blockIdx.x & 7) * runs / 8) % runs);
		const auto request = [&](int run) __attribute__((always_inline))
		{
			uint8_t *slot = lds + run % FEW_ROWS_SLOTS * SLOT;
			const int actual = run + turn < runs ? run + turn : run + turn - runs;
			const int left = row_bytes - actual * FEW_ROWS_RUN;
			const size_t skip = static_cast<size_t>(actual) * FEW_ROWS_RUN;
			const bool there = in_run < left;
			const __amdgpu_buffer_rsrc_t buffers[2] = { buffer_of(const_cast<uint8_t*>(first + skip)), buffer_of(const_cast<uint8_t*>(second + skip)) };
#pragma unroll
			for (int u = 0; u < 4; u++)
				buffer_to_lds(buffers[u / 2], slot + (wave + 4 * u) * 1024, there ? w_offset[u] : NOWHERE);
			const __amdgpu_buffer_rsrc_t x_buffer = buffer_of(const_cast<uint8_t*>(x_bytes + skip));
#pragma unroll
			for (int u = 0; u < X_LOADS; u++)
				buffer_to_lds(x_buffer, slot + (16 + wave + 4 * u) * 1024, there ? x_offset[u] : NOWHERE);
		};
		const int fragment = r * FEW_ROWS_RUN + wave * 128 + (((2 * q) ^ (r & 7)) * 16);
		float4_t acc[2][MB];
#pragma unroll
		for (int i = 0; i < 2; i++)
#pragma unroll
			for (int b = 0; b < MB; b++)
				acc[i][b] = float4_t { 0.0f, 0.0f, 0.0f, 0.0f };
		request(0);
		if (runs > 1)
			request(1);
		for (int run = 0; run < runs; run++)
		{
			wait_lgkmcnt<0>(); /* this wavefront's reads of the run before are complete before anyone may overwrite its slot */
			if (run + 1 < runs)
				wait_vmcnt<LOADS>();
			else
				wait_vmcnt<0>();
			barrier_no_fence();
			if (run + 2 < runs)
				request(run + 2);
			const uint8_t *slot = lds + run % FEW_ROWS_SLOTS * SLOT;
#pragma unroll
			for (int h = 0; h < 2; h++)
			{
				uint4_t weights[2];
#pragma unroll
				for (int i = 0; i < 2; i++)
					weights[i] = *reinterpret_cast<const uint4_t*>(slot + i * 16 * FEW_ROWS_RUN + (fragment ^ (h * 16)));
#pragma unroll
				for (int b = 0; b < MB; b++)
				{
					const uint4_t v = *reinterpret_cast<const uint4_t*>(slot + (32 + 16 * b) * FEW_ROWS_RUN + (fragment ^ (h * 16)));
#pragma unroll
					for (int i = 0; i < 2; i++)
						mma_16x16<T>(weights[i], v, acc[i][b]);
				}
			}
		}
		__syncthreads();
		join_few_rows<MB>(acc, reinterpret_cast<float (*)[2][16 * MB][16]>(lds));
	}
	/* f(MB, whether the rows can be streamed) as compile-time constants */
	template<typename T, typename F>
	inline void with_few_rows(int rows, int k, F &&f)
	{
		const bool stream = (k * sizeof(T)) % 16 == 0 && k > 0;
		typedef std::integral_constant<int, 1> one;
		typedef std::integral_constant<int, 2> two;
		if (rows > 32)
			f(std::integral_constant<int, 4>(), std::false_type());
		else if (rows > 16)
			stream ? f(two(), std::true_type()) : f(two(), std::false_type());
		else
			stream ? f(one(), std::true_type()) : f(one(), std::false_type());
	}
} /* namespace mlhip */

#endif /* MINML_AMD_FEW_ROWS_HPP_ */

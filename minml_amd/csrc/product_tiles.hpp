/*
 * product_tiles.hpp — the products of a layer's forward and backward pass on tiles of 256x256 or 128x128: ACC[m][n] = sum_k A(m, k) B(n, k), where each operand lies in memory
 * either with its rows along k (ROWS) or with its rows across k (COLUMNS: element (m, k) at [k][m]). The three products of a layer y = x W^T need both:
 *     y  = x W^T       m = token, n = output, k = input     A = x ROWS,        B = W ROWS
 *     dx = d W         m = token, n = input,  k = output    A = d ROWS,        B = W COLUMNS
 *     dW = d^T x       m = output, n = input, k = token     A = d COLUMNS,     B = x COLUMNS
 * so no operand is transposed in memory.
 *
 * Operands move L2 -> LDS by direct-to-LDS loads in panels of 128 rows (of m or n) by 128 bytes of k, 16 KB each, which lie in LDS as they lie in memory:
 *   ROWS     [128 rows][128 bytes of k], the 16-byte pieces of a row permuted by (row / 2) % 8: an MFMA fragment is 16 bytes of one row, and the rows of a wavefront's read meet all banks;
 *   COLUMNS  [k][128 columns], the 32-column blocks of a row permuted by k: a fragment is gathered across k, in fp16 by the LDS's transposing read (a group of 16 lanes reads 4 rows of 16 columns, and each lane
 *            gets the 4 values of one column), in fp32 element by element.
 * Both kinds give a lane the same k, so they can be mixed. The loads go through a buffer descriptor whose base is a scalar that walks along k: a lane holds one 32-bit offset per load for the whole
 * product, whatever the size of the operand, and a lane that lies outside (a row past the end, k past the end) is sent behind the buffer's end, which reads as zero. So no element outside an operand
 * reaches an accumulator, and NaN or infinities beside it do not either.
 *
 * 256x256 (8 wavefronts, one workgroup per compute unit): two slots of four panels. A chunk of 64 k (fp32: 32) is multiplied in two phases, 64 x 64 of every wavefront each, with a barrier before each; a panel's
 * place takes the chunk after the next one as soon as it has been read, so a load has about one and a half chunks to arrive.
 * 128x128 (4 wavefronts): where 256x256 tiles would leave units without work, with two slots and two workgroups per compute unit; and where k is so short that a tile is mostly beginning and end, with one
 * slot and four workgroups per unit, which hide each other's waits. fp32, which the matrix cores bound by far, also has 64x128.
 * A product with a long k and few tiles is split along k (gridDim.y): each part leaves its sums in fp32, and a launch of its own adds them up in order.
 *
 * Epilogues work on the accumulators in registers, where a lane has 16 columns of every block (TilePlace), and what goes to memory passes through LDS, in the result's own type where nothing has to be added to it
 * there, so that neighbouring threads write whole rows, 16 bytes each.
 */
#ifndef MINML_AMD_PRODUCT_TILES_HPP_
#define MINML_AMD_PRODUCT_TILES_HPP_

#include "common.hpp"
#include "gemm_dma.hpp"
#include "training_utils.hpp"

#include <algorithm>
#include <cmath>

namespace mlhip
{
	enum class Side
	{
		ROWS, COLUMNS
	};
	/*
	 * One operand. Bytes between rows (of memory) and the base are multiples of 16. `depth` counts what lies along k: elements for ROWS (whole 16-byte pieces: what lies behind the last element of its piece
	 * has to be zero), rows for COLUMNS. extent: rows of m (n) that exist; for COLUMNS whole 16-byte pieces.
	 * PAIRED rows: the operand is two matrices of `extent` rows, `pair_bytes` apart, and a tile takes half its rows from each (first half of the tile: first matrix).
	 */
	struct Operand
	{
			const uint8_t *base;
			size_t row_bytes;
			int extent;
			int depth;
			size_t pair_bytes = 0;
	};
	constexpr int PANEL = 128; /* rows of a panel */
	constexpr int PANEL_BYTES = PANEL * 128;
	constexpr int OUTSIDE = static_cast<int>(0x80000000u); /* as an unsigned offset behind any buffer's end */

	/* in a scalar register, as the addresses made of it are then */
	__device__ __forceinline__ int wave_number()
	{
		return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	}
	/* 16 bytes per lane from the buffer to `place` + 16 * lane of LDS. The builtin is for the device pass alone: in the host pass every template that holds it loses its launch stub from the second
	 * instance on */
	__device__ __forceinline__ void buffer_to_lds(__amdgpu_buffer_rsrc_t buffer, uint8_t *place, int offset)
	{
#if defined(__HIP_DEVICE_COMPILE__)
		__builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_ptr_t) place, 16, offset, 0, 0, 0);
#endif
	}

	/* the loads of one panel (or of its first LOADED rows) by WAVES wavefronts, 1 KB each. SEGMENT: consecutive rows of the operand in a panel (64 where a panel holds both halves of a paired tile) */
	template<typename T, Side SIDE, int WAVES, int SEGMENT = PANEL, int LOADED = PANEL>
	struct PanelLoads
	{
			static_assert(LOADED == PANEL || SIDE == Side::ROWS, "columns come in whole panels");
			static constexpr int COUNT = LOADED / 8 / WAVES;
			static constexpr int CHUNK = 128 / sizeof(T); /* k of a chunk */
			static constexpr int K_PER_LOAD = 1024 / (PANEL * sizeof(T)); /* COLUMNS: rows of k that one load covers */
			int offset[COUNT];
			int k; /* ROWS: first byte of the lane's piece in its 128; COLUMNS: row of k of the lane's first load */

			/* `there`: rows of the operand from the panel's first on */
			__device__ __forceinline__ void begin(int there, size_t row_bytes, size_t pair_bytes)
			{
				const int lane = threadIdx.x & 63, wave = wave_number();
				if constexpr (SIDE == Side::ROWS)
				{
					/* the permutation (row / 2) % 8 is the same for all loads of a lane: their rows differ by multiples of 16 */
					k = ((lane & 7) ^ dma_swizzle(wave * 8 + (lane >> 3))) * 16;
#pragma unroll
					for (int u = 0; u < COUNT; u++)
					{
						const int place = (wave + WAVES * u) * 8 + (lane >> 3);
						const int row = place % SEGMENT;
						offset[u] = (row < there) ? static_cast<int>(row * row_bytes + (place / SEGMENT) * pair_bytes) + k : OUTSIDE;
					}
				}
				else
				{
					constexpr int PIECES = 32 * sizeof(T) / 16, LANES = 64 / K_PER_LOAD; /* 16-byte pieces of a block of 32 columns; lanes of a row */
					k = wave * K_PER_LOAD + lane / LANES;
#pragma unroll
					for (int u = 0; u < COUNT; u++)
					{
						const int row = k + u * WAVES * K_PER_LOAD, position = lane % LANES;
						const int permuted = (sizeof(T) == 2) ? (row & 3) : ((row >> 2) & 1);
						const int column = ((position / PIECES) ^ permuted) * 32 + (position % PIECES) * (16 / static_cast<int>(sizeof(T)));
						offset[u] = (column < there) ? static_cast<int>(row * row_bytes + column * sizeof(T)) : OUTSIDE;
					}
				}
			}
			/* `left`: bytes (ROWS) or rows (COLUMNS) of k from the chunk's first on */
			__device__ __forceinline__ void request(const uint8_t *base, int left, uint8_t *panel) const
			{
				const int wave = wave_number();
				const __amdgpu_buffer_rsrc_t buffer = buffer_of(const_cast<uint8_t*>(base));
#pragma unroll
				for (int u = 0; u < COUNT; u++)
				{
					const int at = (SIDE == Side::ROWS) ? k : k + u * WAVES * K_PER_LOAD;
					buffer_to_lds(buffer, panel + (wave + WAVES * u) * 1024, (at < left) ? offset[u] : OUTSIDE);
				}
			}
	};
	/* where the scalar base of an operand's panels walks */
	template<typename T, Side SIDE>
	struct PanelWalk
	{
			const uint8_t *base;
			size_t step;
			int left;

			__device__ __forceinline__ void begin(const Operand &o, int first_row, int first_chunk, int chunks)
			{
				constexpr int CHUNK = 128 / sizeof(T);
				step = (SIDE == Side::ROWS) ? 128 : CHUNK * o.row_bytes;
				base = o.base + (SIDE == Side::ROWS ? first_row * o.row_bytes : first_row * sizeof(T)) + first_chunk * step;
				const int per_chunk = (SIDE == Side::ROWS) ? 128 : CHUNK;
				const int depth = (SIDE == Side::ROWS) ? o.depth * static_cast<int>(sizeof(T)) : o.depth;
				left = min(depth - first_chunk * per_chunk, chunks * per_chunk);
			}
			__device__ __forceinline__ void advance()
			{
				base += step;
				left -= (SIDE == Side::ROWS) ? 128 : 128 / static_cast<int>(sizeof(T));
			}
	};
	/*
	 * The transposing read of LDS. The compiler would wait for every outstanding direct-to-LDS load before a read that says nothing about what it may alias, which is to wait for the panels two chunks
	 * ahead; a restricted pointer says that, as the type does for ordinary reads. What a read really depends on is counted by the kernels.
	 */
	typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
	typedef __attribute__((address_space(3))) fp16x4 *transposed_place_t;
	__device__ __forceinline__ uint2_t read_transposed(const transposed_place_t __restrict__ place)
	{
		return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16(place));
	}
	/* fragments of a panel: block b (32 rows of the panel), k step kk of 4. Lane l: row l % 32, k = 16 / sizeof(T) * (2 kk + l / 32) onwards */
	template<typename T, Side SIDE>
	struct PanelFragments
	{
			int first;

			__device__ __forceinline__ void begin(int block)
			{
				const int lane = threadIdx.x & 63;
				if constexpr (SIDE == Side::ROWS)
					first = (block * 32 + (lane & 31)) * 128 + (((lane >> 5) ^ dma_swizzle(lane & 31)) * 16);
				else if constexpr (sizeof(T) == 2)
				{
					const int t = lane & 15;
					first = ((lane >> 5) * 8 + (t >> 2)) * 256 + ((block ^ (t >> 2)) * 64) + ((lane >> 4) & 1) * 32 + (t & 3) * 8;
				}
				else
					first = (lane >> 5) * 2048 + ((block ^ (lane >> 5)) * 128) + (lane & 31) * 4;
			}
			__device__ __forceinline__ uint4_t read(const uint8_t *panel, int kk) const
			{
				if constexpr (SIDE == Side::ROWS)
					return *reinterpret_cast<const uint4_t*>(panel + (first ^ (kk * 32)));
				else if constexpr (sizeof(T) == 2)
				{
					const uint2_t lo = read_transposed((transposed_place_t) (panel + first + kk * 4096));
					const uint2_t hi = read_transposed((transposed_place_t) (panel + first + kk * 4096 + 1024));
					return uint4_t { lo[0], lo[1], hi[0], hi[1] };
				}
				else
				{
					uint4_t v;
#pragma unroll
					for (int e = 0; e < 4; e++)
						v[e] = *reinterpret_cast<const uint32_t*>(panel + first + kk * 4096 + e * 512);
					return v;
				}
			}
	};

	struct ProductArgs
	{
			Operand a, b;
			int rows; /* of the result */
			int first_tile_m, tiles_m, tiles_n; /* rows of tiles of this launch, columns */
			int chunks; /* of the whole product */
			int chunks_per_part; /* of one gridDim.y */
	};
	constexpr int TILE_GROUP = 8;
	/*
	 * Order of the tiles: every XCD has one contiguous eighth of them, walked in groups of 8 rows of tiles, down the rows first: the 32 tiles that an XCD has in hand at a time then need 8 panels' worth of
	 * rows and 4 of columns, near the least that 32 tiles can share.
	 */
	__device__ __forceinline__ void tile_of_block(const ProductArgs &p, int &tile_m, int &tile_n)
	{
		const unsigned int id = xcd_contiguous_block_id(blockIdx.x, gridDim.x);
		const unsigned int group_tiles = TILE_GROUP * p.tiles_n;
		const unsigned int group = id / group_tiles, within = id - group * group_tiles;
		const unsigned int rows = min(static_cast<unsigned int>(p.tiles_m) - group * TILE_GROUP, static_cast<unsigned int>(TILE_GROUP));
		tile_n = within / rows;
		tile_m = p.first_tile_m + group * TILE_GROUP + within - tile_n * rows;
	}

	/*
	 * Where a wavefront's accumulators lie in the tile, and how they leave it. Block (i, j) covers rows row(i) .. + 31 and columns column(j) .. + 31; lane l holds row l % 32 and, in registers 4 q .. 4 q + 3, columns
	 * 8 q + 4 (l / 32) .. + 3. In a paired product blocks (i, 0) and (i, 1) are the two matrices' sums of the same place.
	 */
	template<int BM, int BN>
	struct TilePlace
	{
			static constexpr int BLOCKS = BM / 64, THREADS = BM == 256 ? 512 : 256;
			int tile_m, tile_n, part, wave_m, wave_n;

			__device__ __forceinline__ int row(int i) const
			{
				return (BM == 256 ? (i >> 1) * 128 + wave_m * 64 + (i & 1) * 32 : i * 64 + wave_m * 32) + lane_row();
			}
			__device__ __forceinline__ int column(int j) const
			{
				return j * (BN / 2) + wave_n * 32;
			}
			__device__ __forceinline__ static int lane_row()
			{
				return threadIdx.x & 31;
			}
			__device__ __forceinline__ static int lane_column(int q)
			{
				return 8 * q + 4 * ((threadIdx.x >> 5) & 1);
			}
	};
	/* the bias of a lane's 16 columns of a block that begins at column n0 of the result; zeros where there is none, and behind the last column */
	template<typename T>
	__device__ __forceinline__ void load_lane_bias(float (&out)[16], const T *bias, int n0, int columns)
	{
#pragma unroll
		for (int r = 0; r < 16; r++)
			out[r] = 0.0f;
		if (bias == nullptr)
			return;
		const int lane_column = n0 + 4 * ((threadIdx.x >> 5) & 1);
		if (n0 + 32 <= columns)
		{
			Elements<T, 4> v[4];
#pragma unroll
			for (int q = 0; q < 4; q++)
				v[q].load(bias + lane_column + 8 * q);
#pragma unroll
			for (int q = 0; q < 4; q++)
#pragma unroll
				for (int e = 0; e < 4; e++)
					out[4 * q + e] = v[q][e];
		}
		else
#pragma unroll
			for (int q = 0; q < 4; q++)
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (lane_column + 8 * q + e < columns)
						out[4 * q + e] = static_cast<float>(bias[lane_column + 8 * q + e]);
	}
	/*
	 * A tile (or the rows of it that lie in LDS) to memory, 16 bytes per thread and whole rows by neighbouring threads. f(m, n, LDS place, elements): elements of the vector that exist, all of them or fewer at the
	 * matrix's edge.
	 */
	template<typename Out, int COLUMNS>
	struct Stage
	{
			static constexpr int VECTOR = 16 / sizeof(Out), STRIDE = COLUMNS + VECTOR; /* a row more than a whole number of banks' turns: the lanes of a block write 32 rows at a time */
			static constexpr int bytes(int rows)
			{
				return rows * STRIDE * static_cast<int>(sizeof(Out));
			}
			Out *place;

			typedef Out vec4_t __attribute__((ext_vector_type(4)));

			__device__ __forceinline__ void put(int row, int column, vec4_t v) const
			{
				*reinterpret_cast<vec4_t*>(place + row * STRIDE + column) = v;
			}
			__device__ __forceinline__ void put(int row, int column, float a, float b, float c, float d) const
			{
				put(row, column, vec4_t { static_cast<Out>(a), static_cast<Out>(b), static_cast<Out>(c), static_cast<Out>(d) });
			}
			template<int ROWS, int THREADS, typename F>
			__device__ __forceinline__ void for_vectors(int m0, int rows, int n0, int columns, F &&f) const
			{
				constexpr int LANES = COLUMNS / VECTOR, AT_A_TIME = THREADS / LANES;
				const int n = n0 + (threadIdx.x % LANES) * VECTOR;
				const int there = min(columns - n, VECTOR);
				if (there <= 0)
					return;
#pragma unroll 4
				for (int row = threadIdx.x / LANES; row < ROWS; row += AT_A_TIME)
					if (m0 + row < rows)
						f(m0 + row, n, place + row * STRIDE + (n - n0), there);
			}
			/* to rows `stride` elements apart */
			template<int ROWS, int THREADS>
			__device__ __forceinline__ void copy(Out *out, size_t stride, int m0, int rows, int n0, int columns) const
			{
				for_vectors<ROWS, THREADS>(m0, rows, n0, columns, [&](int m, int n, const Out *src, int there) __attribute__((always_inline))
				{
					Out *dst = out + m * stride + n;
					if (there == VECTOR)
					{
						typedef typename Elements<Out, VECTOR>::vec_t vec_t;
						*reinterpret_cast<typename Elements<Out, VECTOR>::unaligned_t*>(dst) = *reinterpret_cast<const vec_t*>(src);
					}
					else
						for (int e = 0; e < there; e++)
							dst[e] = src[e];
				});
			}
	};
	/* rows of a tile that lie in LDS at a time in fp32: half of them, of the smallest tile all */
	constexpr int rows_at_a_time(int rows)
	{
		return std::max(rows / 2, 64);
	}
	/* the sums of a tile through LDS in fp32: f(m, n, 4 sums in LDS, elements) */
	template<int BM, int BN, typename Acc, typename F>
	__device__ __forceinline__ void sums_in_rows(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows, int columns, F &&f)
	{
		constexpr int ROWS = rows_at_a_time(BM), BLOCKS = ROWS / 64;
		const Stage<float, BN> stage { reinterpret_cast<float*>(lds) };
		static_for<BM / ROWS>([&](auto half)
		{
			constexpr int h = decltype(half)::value;
			__syncthreads();
#pragma unroll
			for (int i = h * BLOCKS; i < (h + 1) * BLOCKS; i++)
#pragma unroll
				for (int j = 0; j < 2; j++)
#pragma unroll
					for (int q = 0; q < 4; q++)
					{
						const Acc &v = acc[i][j];
						stage.put(at.row(i) - h * ROWS, at.column(j) + at.lane_column(q), v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
					}
			__syncthreads();
			stage.template for_vectors<ROWS, TilePlace<BM, BN>::THREADS>(at.tile_m * BM + h * ROWS, rows, at.tile_n * BN, columns, f);
		});
	}

	template<typename T, Side SA, Side SB, bool PAIRED, typename Epilogue>
	__global__ __launch_bounds__(512, 1) void kernel_product_256(ProductArgs p, Epilogue epilogue)
	{
		typedef MfmaTraits<T> Traits;
		typedef typename Traits::acc_vec acc_vec;
		constexpr int WAVES = 8, LOADS = PanelLoads<T, SA, WAVES>::COUNT;
		constexpr int A0 = 0, B0 = 1, B1 = 2, A1 = 3; /* panels of a slot */
		constexpr int SLOT = 4 * PANEL_BYTES;
		extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
		int tile_m, tile_n;
		tile_of_block(p, tile_m, tile_n);
		const int first_chunk = blockIdx.y * p.chunks_per_part;
		const int chunks = min(p.chunks_per_part, p.chunks - first_chunk);
		const int wave = wave_number(), wave_m = wave >> 2, wave_n = wave & 3;

		PanelLoads<T, SA, WAVES> a_loads[2];
		PanelLoads<T, SB, WAVES> b_loads[2];
		PanelWalk<T, SA> a_walk[2];
		PanelWalk<T, SB> b_walk[2];
#pragma unroll
		for (int h = 0; h < 2; h++)
		{
			const int m = tile_m * 256 + h * PANEL;
			a_loads[h].begin(p.a.extent - m, p.a.row_bytes, 0);
			a_walk[h].begin(p.a, m, first_chunk, chunks);
			const int n = PAIRED ? tile_n * PANEL : tile_n * 256 + h * PANEL;
			b_loads[h].begin(p.b.extent - n, p.b.row_bytes, 0);
			b_walk[h].begin(p.b, n, first_chunk, chunks);
			if (PAIRED && h == 1)
				b_walk[h].base += p.b.pair_bytes;
		}
		const auto request_a = [&](int chunk, auto half) __attribute__((always_inline))
		{
			constexpr int h = decltype(half)::value;
			a_loads[h].request(a_walk[h].base, a_walk[h].left, lds + (chunk & 1) * SLOT + (h == 0 ? A0 : A1) * PANEL_BYTES);
			a_walk[h].advance();
		};
		const auto request_b = [&](int chunk, auto half) __attribute__((always_inline))
		{
			constexpr int h = decltype(half)::value;
			b_loads[h].request(b_walk[h].base, b_walk[h].left, lds + (chunk & 1) * SLOT + (h == 0 ? B0 : B1) * PANEL_BYTES);
			b_walk[h].advance();
		};
		typedef std::integral_constant<int, 0> zero;
		typedef std::integral_constant<int, 1> one;
		typedef std::integral_constant<int, 2> two;

		PanelFragments<T, SA> a_place[2];
		PanelFragments<T, SB> b_place;
		a_place[0].begin(2 * wave_m);
		a_place[1].begin(2 * wave_m + 1);
		b_place.begin(wave_n);
		uint4_t fa[2][4], fb0[4], fb1[4];
		const auto read_a = [&](int chunk, int panel, int kk) __attribute__((always_inline))
		{
			const uint8_t *src = lds + (chunk & 1) * SLOT + panel * PANEL_BYTES;
#pragma unroll
			for (int i = 0; i < 2; i++)
				fa[i][kk] = a_place[i].read(src, kk);
		};
		const auto read_b = [&](int chunk, int panel, int kk, uint4_t (&regs)[4]) __attribute__((always_inline))
		{
			regs[kk] = b_place.read(lds + (chunk & 1) * SLOT + panel * PANEL_BYTES, kk);
		};

		acc_vec acc[4][2];
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int j = 0; j < 2; j++)
#pragma unroll
				for (int r = 0; r < 16; r++)
					acc[i][j][r] = 0;

		for (int c = 0; c < 2; c++)
			if (c < chunks)
			{
				request_a(c, zero());
				request_b(c, zero());
				request_b(c, one());
				request_a(c, one());
			}
		if (chunks > 1)
			wait_vmcnt<5 * LOADS>();
		else
			wait_vmcnt<LOADS>();
		barrier_no_fence();
		if (chunks > 0)
		{
#pragma unroll
			for (int kk = 0; kk < 4; kk++)
			{
				read_a(0, A0, kk);
				read_b(0, B0, kk, fb0);
				read_b(0, B1, kk, fb1);
			}
		}
		/* one chunk: whether there is a next one, and whether there is one after it */
		const auto process_chunk = [&](int c, auto one_more, auto two_more) __attribute__((always_inline))
		{
			constexpr bool NEXT = decltype(one_more)::value, AFTER = decltype(two_more)::value;
			const auto multiply = [&](int kk, const uint4_t (&regs)[4], auto row, auto column) __attribute__((always_inline))
			{
#pragma unroll
				for (int i = 0; i < 2; i++)
					Traits::mma(regs[kk], fa[i][kk], acc[decltype(row)::value + i][decltype(column)::value]);
			};
			/* A0 with both halves of B. Behind A1 of this chunk: all of the next one. This wavefront's reads of A0, B0 and B1 are complete before anyone may overwrite them */
			wait_lgkmcnt<0>();
			wait_vmcnt<NEXT ? 4 * LOADS : 0>();
			barrier_no_fence();
#pragma unroll
			for (int kk = 0; kk < 4; kk++)
			{
				multiply(kk, fb0, zero(), zero());
				multiply(kk, fb1, zero(), one());
				__builtin_amdgcn_sched_barrier(0);
				read_a(c, A1, kk);
				if constexpr (AFTER)
				{
					if (kk == 0)
						request_a(c + 2, zero());
					if (kk == 1)
						request_b(c + 2, zero());
					if (kk == 2)
						request_b(c + 2, one());
				}
				__builtin_amdgcn_sched_barrier(0);
			}
			/* A1 with both halves of B. Behind A0, B0 and B1 of the next chunk: its A1, and three panels of the one after it */
			if constexpr (NEXT)
			{
				wait_lgkmcnt<0>();
				wait_vmcnt<AFTER ? 4 * LOADS : LOADS>();
				barrier_no_fence();
			}
#pragma unroll
			for (int kk = 0; kk < 4; kk++)
			{
				multiply(kk, fb0, two(), zero());
				multiply(kk, fb1, two(), one());
				__builtin_amdgcn_sched_barrier(0);
				if constexpr (NEXT)
				{
					read_a(c + 1, A0, kk);
					read_b(c + 1, B0, kk, fb0);
					read_b(c + 1, B1, kk, fb1);
				}
				if constexpr (AFTER)
				{
					if (kk == 0)
						request_a(c + 2, one());
				}
				__builtin_amdgcn_sched_barrier(0);
			}
		};
		int c = 0;
		for (; c + 2 < chunks; c++)
			process_chunk(c, std::true_type(), std::true_type());
		if (c + 1 < chunks)
			process_chunk(c++, std::true_type(), std::false_type());
		if (c < chunks)
			process_chunk(c, std::false_type(), std::false_type());

		epilogue.template tile<256, 256>(acc, TilePlace<256, 256> { tile_m, tile_n, static_cast<int>(blockIdx.y), wave_m, wave_n }, lds, p.rows);
	}

	template<typename T, Side SA, Side SB, bool PAIRED, int BM, int SLOTS, typename Epilogue>
	__global__ __launch_bounds__(256, SLOTS == 1 ? 4 : 2) void kernel_product_128(ProductArgs p, Epilogue epilogue)
	{
		typedef MfmaTraits<T> Traits;
		typedef typename Traits::acc_vec acc_vec;
		constexpr int WAVES = 4, A_BYTES = BM * 128, SLOT = A_BYTES + PANEL_BYTES, BLOCKS = BM / 64;
		extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
		int tile_m, tile_n;
		tile_of_block(p, tile_m, tile_n);
		const int first_chunk = blockIdx.y * p.chunks_per_part;
		const int chunks = min(p.chunks_per_part, p.chunks - first_chunk);
		const int wave = wave_number(), wave_m = wave >> 1, wave_n = wave & 1;

		PanelLoads<T, SA, WAVES, PANEL, BM> a_loads;
		PanelLoads<T, SB, WAVES, PAIRED ? 64 : PANEL> b_loads;
		PanelWalk<T, SA> a_walk;
		PanelWalk<T, SB> b_walk;
		const int m0 = tile_m * BM, n0 = tile_n * (PAIRED ? 64 : PANEL);
		a_loads.begin(p.a.extent - m0, p.a.row_bytes, 0);
		a_walk.begin(p.a, m0, first_chunk, chunks);
		b_loads.begin(p.b.extent - n0, p.b.row_bytes, p.b.pair_bytes);
		b_walk.begin(p.b, n0, first_chunk, chunks);
		const auto request = [&](int chunk) __attribute__((always_inline))
		{
			uint8_t *slot = lds + chunk % SLOTS * SLOT;
			a_loads.request(a_walk.base, a_walk.left, slot);
			b_loads.request(b_walk.base, b_walk.left, slot + A_BYTES);
			a_walk.advance();
			b_walk.advance();
		};
		/* block (i, j): rows i 64 + wave_m 32, columns j 64 + wave_n 32 */
		PanelFragments<T, SA> a_place[BLOCKS];
		PanelFragments<T, SB> b_place[2];
#pragma unroll
		for (int i = 0; i < BLOCKS; i++)
			a_place[i].begin(2 * i + wave_m);
#pragma unroll
		for (int j = 0; j < 2; j++)
			b_place[j].begin(2 * j + wave_n);
		acc_vec acc[BLOCKS][2];
#pragma unroll
		for (int i = 0; i < BLOCKS; i++)
#pragma unroll
			for (int j = 0; j < 2; j++)
#pragma unroll
				for (int r = 0; r < 16; r++)
					acc[i][j][r] = 0;
		if (chunks > 0)
			request(0);
		for (int c = 0; c < chunks; c++)
		{
			wait_lgkmcnt<0>(); /* this wavefront's reads of the chunk before are complete before anyone may overwrite its place */
			if constexpr (SLOTS == 1)
				if (c > 0)
				{
					barrier_no_fence();
					request(c);
				}
			wait_vmcnt<0>();
			barrier_no_fence();
			if constexpr (SLOTS == 2)
				if (c + 1 < chunks)
					request(c + 1);
			const uint8_t *slot = lds + c % SLOTS * SLOT;
#pragma unroll
			for (int kk = 0; kk < 4; kk++)
			{
				uint4_t fa[BLOCKS], fb[2];
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
					fa[i] = a_place[i].read(slot, kk);
#pragma unroll
				for (int j = 0; j < 2; j++)
					fb[j] = b_place[j].read(slot + A_BYTES, kk);
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
#pragma unroll
					for (int j = 0; j < 2; j++)
						Traits::mma(fb[j], fa[i], acc[i][j]);
			}
		}
		epilogue.template tile<BM, 128>(acc, TilePlace<BM, 128> { tile_m, tile_n, static_cast<int>(blockIdx.y), wave_m, wave_n }, lds, p.rows);
	}
	/* slots, or what an epilogue lays out there: Epilogue::lds<BM, BN>() bytes */
	template<typename Epilogue>
	constexpr int product_lds(int tile, int slots)
	{
		return tile == 256 ? std::max(8 * PANEL_BYTES, Epilogue::template lds<256, 256>())
				: tile == 128 ? std::max(2 * slots * PANEL_BYTES, Epilogue::template lds<128, 128>()) : std::max(slots * (PANEL_BYTES + 64 * 128), Epilogue::template lds<64, 128>());
	}
	constexpr int LDS_OF_A_UNIT = 160 * 1024;

	/* how a product is cut: tiles of `tile` rows and as many columns (at least 128), `parts` along k. A workspace is sized by the same rule, so it asks no device */
	struct ProductPlan
	{
			int tile, slots, tiles_m, tiles_n, chunks, parts, chunks_per_part;
	};
	/*
	 * The cheapest of the tile sizes and up to 16 parts, by what they take: a compute unit works off its tiles one after the other (two of 128x128 side by side take as long as one after the other), a tile takes
	 * so long per chunk and something for its beginning and end, and parts have to be added up. Microseconds on a full chip, fp16 / fp32: a chunk of 256x256 1.7 / 7.8 (1.2 where at most half of the units have
	 * a tile: what they read then comes faster), of 128x128 0.6 / 2.05 (its operands' way out of the L2 bounds it in fp16: 32 KB, 30 bytes per clock and unit), and where there are four workgroups to
	 * every unit, which one slot each lets in, 0.5 / 2.15 and hardly any beginning and end. Measured, two sides each: dx of 4096 x 2048, k = 16384, fp16 (128 tiles of 256x256) whole 313, in 2 parts 228, 128x128 tiles 310; dW of
	 * 11008 x 2048, k = 8192, fp16 (344 tiles) 388, 385, 379; 2048 x 1024, k = 8192, fp16 143, 87, 79, 128x128 in 2 parts 53; dW of 5462 x 1000, k = 1111, fp32 270, 160, 147, 128x128 in 2 parts 127. 57600 rows
	 * -> 2 x 1024 columns fp16, 256x256 / 128x128 with two slots / with one: k = 256 118 / 118 / 105, both projections kept 146 / 146 / 121, k = 512 160 / 179 / 157, k = 1024 264 / 298 / 277; 512 rows, k = 1024 -> 2 x 4096
	 * 26 / 17 / 20; fp32 57600 rows, k = 256 -> 2 x 1024 589 / 551 / 520, 8192 rows, k = 2048 -> 2 x 2048 1011 / 1071 / 1100.
	 * 64x128 tiles, fp32 with A in rows: half a tile is half the work there, so the last turn costs less and few rows are padded less (901 rows, k = 520 -> 10007 117 -> 109, 64 rows, k = 1024 -> 30000 75 -> 46); in fp16 they would read
	 * more operands per product, which bounds even 128x128.
	 * columns: of the result (of one of the two matrices where the operand is paired)
	 */
	inline ProductPlan plan_product(int rows, int columns, bool paired, int depth, int element_size, bool may_split, bool a_in_rows = true, double *cost_out = nullptr)
	{
		constexpr int UNITS = 256;
		const bool half = element_size == 2;
		const int chunks = ceil_div(depth, 128 / element_size);
		ProductPlan best { 256, 2, 0, 0, chunks, 1, std::max(1, chunks) };
		double least = 0.0;
		for (int tile : { 256, 128, 64 })
		{
			if (tile == 64 && (half || !a_in_rows))
				continue;
			const int width = std::max(tile, 128);
			const int tiles_m = ceil_div(rows, tile), tiles_n = ceil_div(columns, paired ? width / 2 : width);
			const double tiles = static_cast<double>(tiles_m) * tiles_n;
			const int most = (may_split && tiles < 2 * UNITS) ? std::max(1, std::min(16, chunks / 4)) : 1;
			for (int parts = 1; parts <= most; parts++)
			{
				const int per_part = std::max(1, ceil_div(chunks, parts));
				if (parts > 1 && ceil_div(chunks, per_part) != parts)
					continue;
				const double work = tiles * parts / UNITS;
				double cost;
				int slots = 2;
				if (tile == 256)
					cost = std::ceil(work) * (7.0 + per_part * (half ? (work <= 0.5 ? 1.2 : 1.7) : 7.8));
				else if (tile == 64)
					cost = std::ceil(work) * (3.0 + per_part * 1.1);
				else
				{
					cost = std::ceil(work) * (4.0 + per_part * (half ? 0.6 : 2.05));
					const double one_slot = work * (1.8 + per_part * (half ? 0.5 : 2.15));
					if (work >= 4.0 && parts == 1 && per_part <= 32 && one_slot < cost)
					{
						slots = 1;
						cost = one_slot;
					}
				}
				if (parts > 1)
					cost += 6.0 + 8e-6 / 5.0 * parts * rows * (paired ? 2.0 : 1.0) * columns; /* written and read at 5 TB/s */
				if (least == 0.0 || cost < least)
				{
					least = cost;
					best = ProductPlan { tile, slots, tiles_m, tiles_n, chunks, parts, per_part };
				}
			}
		}
		if (cost_out != nullptr)
			*cost_out = least;
		return best;
	}
	/*
	 * A product whose last turn would leave most compute units idle, in two: the rows of whole turns, and the rest, which is split along k. dW of 11008 x 2048, k = 8192, fp16 (344 tiles: 32 rows of 8 tiles and 11 that
	 * are cut in two) whole 388 us, so 330.
	 */
	struct TwoPlans
	{
			ProductPlan first, rest;
			int first_rows; /* the rest may be none */
	};
	inline TwoPlans plan_in_turns(int rows, int columns, int depth, int element_size, bool a_in_rows)
	{
		constexpr int UNITS = 256;
		double whole, first, rest;
		TwoPlans best { plan_product(rows, columns, false, depth, element_size, true, a_in_rows, &whole), ProductPlan { }, rows };
		for (int tile : { 256, 128 })
		{
			const int tiles_n = ceil_div(columns, tile), turns = static_cast<int>(static_cast<long long>(ceil_div(rows, tile)) * tiles_n / UNITS);
			if (turns < 1 || turns > 8 || tiles_n > UNITS)
				continue;
			const int first_rows = turns * UNITS / tiles_n * tile;
			if (first_rows >= rows)
				continue;
			TwoPlans two { plan_product(first_rows, columns, false, depth, element_size, false, a_in_rows, &first), plan_product(rows - first_rows, columns, false, depth, element_size, true, a_in_rows, &rest), first_rows };
			if (first + rest + 3.0 < 0.95 * whole)
			{
				whole = first + rest + 3.0;
				best = two;
			}
		}
		return best;
	}
	/* a launch has less than 2^32 threads along x: 2^23 tiles of 256x256 (2^21 tokens against 2^18 classes) are one more than that, and go out in two. Whole groups of rows of tiles where there is room for one */
	inline int tile_rows_of_a_launch(const ProductPlan &plan)
	{
		const int threads = plan.tile == 256 ? 512 : 256;
		const long long rows = 0xffffffffll / threads / plan.tiles_n;
		MLHIP_REQUIRE(rows > 0, "product too large");
		if (rows >= plan.tiles_m)
			return plan.tiles_m;
		return static_cast<int>(rows > TILE_GROUP ? rows / TILE_GROUP * TILE_GROUP : rows);
	}
	template<typename T, Side SA, Side SB, bool PAIRED, typename Epilogue>
	inline void launch_product(hipStream_t stream, const ProductPlan &plan, const Operand &a, const Operand &b, int rows, const Epilogue &epilogue)
	{
		if (plan.tiles_m == 0 || plan.tiles_n == 0)
			return;
		MLHIP_REQUIRE(plan.parts <= 65535 && a.row_bytes < (1u << 22) && b.row_bytes < (1u << 22), "product too large");
		static_assert(product_lds<Epilogue>(256, 2) <= LDS_OF_A_UNIT && product_lds<Epilogue>(128, 2) <= LDS_OF_A_UNIT / 2 && product_lds<Epilogue>(128, 1) <= LDS_OF_A_UNIT / 4,
				"tiles must fit the LDS of a compute unit");
		const int most = tile_rows_of_a_launch(plan);
		for (int first = 0; first < plan.tiles_m; first += most)
		{
			const int tiles_m = std::min(most, plan.tiles_m - first);
			const ProductArgs args { a, b, rows, first, tiles_m, plan.tiles_n, plan.chunks, plan.chunks_per_part };
			const dim3 grid(static_cast<unsigned int>(tiles_m) * plan.tiles_n, plan.parts);
			if (plan.tile == 256)
			{
				constexpr int bytes = product_lds<Epilogue>(256, 2);
				auto kernel = kernel_product_256<T, SA, SB, PAIRED, Epilogue>;
				ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
				hipLaunchKernelGGL(kernel, grid, dim3(512), bytes, stream, args, epilogue);
			}
			else if (plan.tile == 64)
			{
				if constexpr (sizeof(T) == 4 && SA == Side::ROWS)
				{
					constexpr int bytes = product_lds<Epilogue>(64, 2);
					auto kernel = kernel_product_128<T, SA, SB, PAIRED, 64, 2, Epilogue>;
					ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
					hipLaunchKernelGGL(kernel, grid, dim3(256), bytes, stream, args, epilogue);
				}
				else
					fail_logic("HIP backend: tiles of 64 rows are for fp32 rows");
			}
			else if (plan.slots == 2)
			{
				constexpr int bytes = product_lds<Epilogue>(128, 2);
				auto kernel = kernel_product_128<T, SA, SB, PAIRED, 128, 2, Epilogue>;
				ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
				hipLaunchKernelGGL(kernel, grid, dim3(256), bytes, stream, args, epilogue);
			}
			else
			{
				constexpr int bytes = product_lds<Epilogue>(128, 1);
				auto kernel = kernel_product_128<T, SA, SB, PAIRED, 128, 1, Epilogue>;
				ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
				hipLaunchKernelGGL(kernel, grid, dim3(256), bytes, stream, args, epilogue);
			}
			MLHIP_CHECK(hipGetLastError());
		}
	}

	/* out[m][n] = scale * sum + beta * out[m][n] */
	template<typename Out>
	struct StoreEpilogue
	{
			Out *out;
			int columns;
			float beta;
			const float *scale; /* on the device; null: 1 */

			template<int BM, int BN>
			static constexpr int lds()
			{
				return std::max(Stage<float, BN>::bytes(rows_at_a_time(BM)), sizeof(Out) == 2 ? Stage<Out, BN>::bytes(BM) : 0);
			}
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				const float factor = scale != nullptr ? *scale : 1.0f;
				if (sizeof(Out) == 2 && beta == 0.0f)
				{
					/* rounded in registers: the whole tile in one go */
					const Stage<Out, BN> stage { reinterpret_cast<Out*>(lds) };
					__syncthreads();
#pragma unroll
					for (int i = 0; i < TilePlace<BM, BN>::BLOCKS; i++)
#pragma unroll
						for (int j = 0; j < 2; j++)
#pragma unroll
							for (int q = 0; q < 4; q++)
							{
								const Acc &v = acc[i][j];
								stage.put(at.row(i), at.column(j) + at.lane_column(q), v[4 * q] * factor, v[4 * q + 1] * factor, v[4 * q + 2] * factor, v[4 * q + 3] * factor);
							}
					__syncthreads();
					stage.template copy<BM, TilePlace<BM, BN>::THREADS>(out, columns, at.tile_m * BM, rows, at.tile_n * BN, columns);
				}
				else
					sums_in_rows<BM, BN>(acc, at, lds, rows, columns, [&](int m, int n, const float *sums, int there) __attribute__((always_inline))
					{
						Out *dst = out + static_cast<size_t>(m) * columns + n;
						float v[4];
#pragma unroll
						for (int e = 0; e < 4; e++)
							v[e] = sums[e] * factor;
						if (there == 4)
						{
							if (beta != 0.0f)
							{
								Elements<Out, 4> old;
								old.load(dst);
#pragma unroll
								for (int e = 0; e < 4; e++)
									v[e] = fmaf(beta, old[e], v[e]);
							}
							store_nearest<4>(dst, v);
						}
						else
#pragma unroll
							for (int e = 0; e < 4; e++)
								if (e < there)
									dst[e] = static_cast<Out>(beta != 0.0f ? fmaf(beta, static_cast<float>(dst[e]), v[e]) : v[e]);
					});
			}
	};
	/* partial[part][m][n] = sum, or += sum: [parts][rows][columns] in fp32 */
	struct PartEpilogue
	{
			float *partial;
			size_t part_stride;
			int columns;
			bool add;

			template<int BM, int BN>
			static constexpr int lds()
			{
				return Stage<float, BN>::bytes(rows_at_a_time(BM));
			}
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				float *out = partial + at.part * part_stride;
				sums_in_rows<BM, BN>(acc, at, lds, rows, columns, [&](int m, int n, const float *sums, int there) __attribute__((always_inline))
				{
					float *dst = out + static_cast<size_t>(m) * columns + n;
					if (there == 4)
					{
						float v[4] = { sums[0], sums[1], sums[2], sums[3] };
						if (add)
						{
							Elements<float, 4> old;
							old.load(dst);
#pragma unroll
							for (int e = 0; e < 4; e++)
								v[e] += old[e];
						}
						store_nearest<4>(dst, v);
					}
					else
						for (int e = 0; e < there; e++)
							dst[e] = add ? dst[e] + sums[e] : sums[e];
				});
			}
	};
	/* out = scale * (sum of the parts) + beta * out, parts in order */
	template<typename Out>
	__global__ __launch_bounds__(256) void kernel_join_parts(const float *partial, int parts, size_t count, Out *out, float beta, const float *scale)
	{
		const float factor = scale != nullptr ? *scale : 1.0f;
		for (size_t i = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) * 4; i < count; i += static_cast<size_t>(gridDim.x) * 1024)
		{
			const size_t at = (count >= 4 && i + 4 > count) ? count - 4 : i;
			const int skip = static_cast<int>(i - at);
			if (count >= 4)
			{
				float v[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
				for (int p = 0; p < parts; p++)
				{
					Elements<float, 4> x;
					x.load(partial + p * count + at);
#pragma unroll
					for (int e = 0; e < 4; e++)
						v[e] += x[e];
				}
				Elements<Out, 4> old;
				if (beta != 0.0f)
					old.load(out + at);
#pragma unroll
				for (int e = 0; e < 4; e++)
					v[e] = beta != 0.0f ? fmaf(beta, old[e], v[e] * factor) : v[e] * factor;
				store_nearest<4>(out + at, v, skip);
			}
			else
				for (size_t j = i; j < count; j++)
				{
					float v = 0.0f;
					for (int p = 0; p < parts; p++)
						v += partial[p * count + j];
					v *= factor;
					out[j] = static_cast<Out>(beta != 0.0f ? fmaf(beta, static_cast<float>(out[j]), v) : v);
				}
		}
	}
	template<typename Out>
	inline void launch_join_parts(hipStream_t stream, const float *partial, int parts, size_t count, Out *out, float beta, const float *scale)
	{
		const size_t groups = std::min<size_t>((count + 1023) / 1024, 4096);
		if (groups > 0)
			hipLaunchKernelGGL((kernel_join_parts<Out>), dim3(static_cast<unsigned int>(groups)), dim3(256), 0, stream, partial, parts, count, out, beta, scale);
		MLHIP_CHECK(hipGetLastError());
	}
	/*
	 * out [rows][columns] = scale * A B + beta * out; `partial` holds parts * rows * columns floats where the plan has parts
	 */
	template<typename T, typename Out, Side SA, Side SB>
	inline void product_to(hipStream_t stream, const ProductPlan &plan, const Operand &a, const Operand &b, int rows, int columns, Out *out, float beta, const float *scale, float *partial)
	{
		if (plan.parts == 1)
			launch_product<T, SA, SB, false>(stream, plan, a, b, rows, StoreEpilogue<Out> { out, columns, beta, scale });
		else
		{
			const size_t count = static_cast<size_t>(rows) * columns;
			launch_product<T, SA, SB, false>(stream, plan, a, b, rows, PartEpilogue { partial, count, columns, false });
			launch_join_parts(stream, partial, plan.parts, count, out, beta, scale);
		}
	}
	inline size_t part_bytes(const ProductPlan &plan, int rows, int columns)
	{
		return plan.parts > 1 ? sizeof(float) * plan.parts * static_cast<size_t>(rows) * columns : 0;
	}
	template<typename T, typename Out, Side SA, Side SB>
	inline void product_to(hipStream_t stream, const TwoPlans &plans, const Operand &a, const Operand &b, int rows, int columns, Out *out, float beta, const float *scale, float *partial)
	{
		const int first = plans.first_rows;
		Operand head = a, rest = a;
		if (first < rows)
			head.extent = first; /* a multiple of the tile's rows, so of 16 bytes too */
		product_to<T, Out, SA, SB>(stream, plans.first, head, b, first, columns, out, beta, scale, partial);
		if (first >= rows)
			return;
		rest.base += (SA == Side::ROWS) ? first * a.row_bytes : first * sizeof(T);
		rest.extent -= first;
		product_to<T, Out, SA, SB>(stream, plans.rest, rest, b, rows - first, columns, out + static_cast<size_t>(first) * columns, beta, scale, partial);
	}
	inline size_t part_bytes(const TwoPlans &plans, int rows, int columns)
	{
		return plans.first_rows >= rows ? part_bytes(plans.first, rows, columns)
				: std::max(part_bytes(plans.first, plans.first_rows, columns), part_bytes(plans.rest, rows - plans.first_rows, columns));
	}

	/*
	 * Rows of `columns` elements copied to rows that are whole 16-byte pieces, zeros behind the last element: what the panels' loads ask of an operand whose rows end anywhere. A thread writes a piece, which it
	 * reads in one go, at whatever address; pieces of a launch are counted with 32 bits while they fit (split_index).
	 */
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_pad_rows(const T *src, T *dst, size_t rows, int columns, int pieces)
	{
		constexpr int N = 16 / sizeof(T);
		typedef typename Elements<T, N>::vec_t vec_t;
		const size_t count = rows * pieces;
		for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<size_t>(gridDim.x) * 256)
		{
			int piece;
			const size_t row = split_index(i, pieces, piece);
			const T *from = src + row * columns + piece * N;
			const int there = columns - piece * N;
			Elements<T, N> v;
			if (there >= N)
				v.load(from);
			else
#pragma unroll
				for (int e = 0; e < N; e++)
					v.raw[e] = e < there ? from[e] : static_cast<T>(0.0f);
			*reinterpret_cast<vec_t*>(dst + i * N) = v.raw;
		}
	}
	template<typename T>
	inline int padded_columns(int columns)
	{
		return static_cast<int>(round_up(columns, 16 / sizeof(T)));
	}
	template<typename T>
	inline const T* pad_rows(hipStream_t stream, const T *src, T *space, size_t rows, int columns)
	{
		const int padded = padded_columns<T>(columns);
		if (padded == columns)
			return src;
		const int pieces = padded * static_cast<int>(sizeof(T)) / 16;
		const size_t groups = std::min<size_t>((rows * pieces + 255) / 256, 16384);
		if (groups > 0)
			hipLaunchKernelGGL((kernel_pad_rows<T>), dim3(static_cast<unsigned int>(groups)), dim3(256), 0, stream, src, space, rows, columns, pieces);
		MLHIP_CHECK(hipGetLastError());
		return space;
	}
} /* namespace mlhip */

#endif /* MINML_AMD_PRODUCT_TILES_HPP_ */

/*
 * cross_entropy.hip — the softmax cross entropy of the rows of a last dense layer over many classes (a vocabulary), from the layer's input, and its gradients. The logits are never kept.
 *
 *   z = x W^T + b,   lse[i] = log sum_j exp z[i, j],   loss[i] = lse[i] - z[i, target[i]]        rows whose target is no class: loss 0, no gradient
 *   d[i, j] = (exp(z[i, j] - lse[i]) - [j = target[i]]) dloss[i]
 *   dx = d W,   dW = d^T x,   db[j] = sum_i d[i, j]
 *
 * Forward: a tile's logits stay in the accumulators; every row of the tile leaves its largest logit and the sum of exponentials about it, and a second launch joins these pairs. A few rows stream
 * the weights past themselves instead (few_rows.hpp) and memory bounds it; else the matrix cores do.
 * Backward: the classes are taken in pieces of as many as make d 256 MB, so that it stays in the last-level cache between its makers and users and does not grow with the vocabulary, as the 8 bytes of a row and a tile of
 * the forward pass do, and the padded copy of the weights where their rows are no multiple of 16 bytes. For each
 * piece the logits are made again, which costs a quarter of the operations and spares rows x classes of memory; the epilogue turns them into d; then d is multiplied with the piece's weights, added to
 * dx in fp32, and with x, which gives the piece's rows of dW.
 * d is stored in the tensors' type. In fp16 a probability of one class in 100 000 would be subnormal, so d is scaled by 2^15 / s with s the power of two above the largest |dloss|: of that loss's row probabilities down to
 * 2^-28 keep their 11 bits, of a row whose dloss is 2^-k of it down to 2^(k - 28); what is smaller is off by 2^-39 of the largest |dloss| at most. The products' results are scaled back, exactly, in fp32. What the rounding of
 * d, half a step per element, does to dx is given back (GradientEpilogue); in dW it counts as much as the rounding of dW itself; db is summed before it.
 * fp16: 7 rows of 2048 x 65536 classes 50 us (5.3 TB/s); 4096 rows of 1024 x 50001 430 us (0.98 PFLOP/s), of 2048 x 65536 950 us (1.16); the gradients of the latter 2.98 ms, in two pieces of d 576 us each (0.95 PFLOP/s, a
 * fourth of it the epilogue), dx 470 (1.17), dW 462 (1.19), and 30 us to join the parts of dx.
 */
#include "few_rows.hpp"
#include "product_tiles.hpp"

#include <limits>

namespace
{
	using namespace mlhip;

	/* of one row and some classes: the largest logit and the sum of exp(z - largest). Nothing there: (-inf, 0) */
	struct Partial
	{
			float top, sum;
	};
	/*
	 * exp(z - top) by the hardware's exponential in fp32, too: the rounding of its argument costs |z - top| 2^-24 of a term, and of their sum the mean of that over the probabilities, which is at most the logarithm of the
	 * number of classes: lse is off by 7e-7 for 65536 of them, about as much as its own rounding to fp32.
	 */
	__device__ __forceinline__ float exp_about(float z, float top)
	{
		/* infinities: exp(inf - inf) is 1 here, so that a row with a logit of +inf has lse = +inf, and one of -inf alone -inf */
		return z == top ? 1.0f : __expf(z - top);
	}
	/* NaN passes: the sum becomes NaN */
	__device__ __forceinline__ Partial join(const Partial &a, const Partial &b)
	{
		const float top = fmaxf(a.top, b.top);
		const float from_a = (a.sum == 0.0f) ? 0.0f : a.sum * exp_about(a.top, top);
		const float from_b = (b.sum == 0.0f) ? 0.0f : b.sum * exp_about(b.top, top);
		return Partial { top, from_a + from_b };
	}
	template<int N>
	__device__ __forceinline__ Partial partial_of(const float (&z)[N], const bool (&there)[N])
	{
		float top = -std::numeric_limits<float>::infinity();
#pragma unroll
		for (int e = 0; e < N; e++)
			top = there[e] ? fmaxf(top, z[e]) : top;
		float sum = 0.0f;
#pragma unroll
		for (int e = 0; e < N; e++)
			sum += (there[e] && !(z[e] == -std::numeric_limits<float>::infinity())) ? exp_about(z[e], top) : 0.0f;
		return Partial { top, sum };
	}
	template<int LANES>
	__device__ __forceinline__ Partial lanes_join(Partial p)
	{
#pragma unroll
		for (int offset = LANES / 2; offset >= 1; offset >>= 1)
			p = join(p, Partial { __shfl_xor(p.top, offset), __shfl_xor(p.sum, offset) });
		return p;
	}

	/* ---- forward ------------------------------------------------------------------------------------------------------------ */
	/* a wavefront's share of the bias, and of what lies behind the last class */
	template<typename T, int BM, int BN>
	struct TileColumns
	{
			float bias[2][16];
			int first[2]; /* column of the tile of the wavefront's blocks, counted from the first class */

			__device__ __forceinline__ void begin(const TilePlace<BM, BN> &at, const T *values, int classes)
			{
#pragma unroll
				for (int j = 0; j < 2; j++)
				{
					first[j] = at.tile_n * BN + at.column(j);
					load_lane_bias(bias[j], values, first[j], classes);
				}
			}
			__device__ __forceinline__ int column(int j, int r) const
			{
				return first[j] + TilePlace<BM, BN>::lane_column(r / 4) + r % 4;
			}
			/* f(j, r) for the register that holds class n, in the lane that holds it; most rows have their class in another tile */
			template<typename F>
			__device__ __forceinline__ void at_class(int n, F &&f) const
			{
#pragma unroll
				for (int j = 0; j < 2; j++)
				{
					const int c = n - first[j];
					if (c >= 0 && c < 32 && ((c >> 2) & 1) == ((threadIdx.x >> 5) & 1))
#pragma unroll
						for (int r = 0; r < 16; r++)
							if (column(j, r) == n)
								f(j, r);
				}
			}
	};
	template<typename T>
	struct LossEpilogue
	{
			const T *bias;
			const int *targets;
			Partial *partials; /* [rows][column tiles] */
			float *target_logits;
			int classes, tiles_n;

			template<int BM, int BN>
			static constexpr int lds()
			{
				return (BN / 64) * BM * static_cast<int>(sizeof(Partial));
			}
			/* in registers: a lane has 32 columns of every of its rows, the lane 32 further the other 32 of the wavefront; the wavefronts of a row meet in LDS */
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				constexpr int BLOCKS = TilePlace<BM, BN>::BLOCKS, WAVES_N = BN / 64;
				constexpr float NOTHING = -std::numeric_limits<float>::infinity();
				TileColumns<T, BM, BN> columns;
				columns.begin(at, bias, classes);
				int target[BLOCKS];
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
				{
					const int m = at.tile_m * BM + at.row(i);
					target[i] = m < rows ? targets[m] : -1;
				}
				const bool edge = (at.tile_n + 1) * BN > classes;
				Partial *meeting = reinterpret_cast<Partial*>(lds); /* [WAVES_N][BM] */
				__syncthreads();
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
				{
					float z[2][16];
#pragma unroll
					for (int j = 0; j < 2; j++)
#pragma unroll
						for (int r = 0; r < 16; r++)
						{
							z[j][r] = acc[i][j][r] + columns.bias[j][r];
							if (edge)
								z[j][r] = columns.column(j, r) < classes ? z[j][r] : NOTHING;
						}
					if (target[i] >= 0 && target[i] < classes)
						columns.at_class(target[i], [&](int j, int r) __attribute__((always_inline))
						{
							target_logits[at.tile_m * BM + at.row(i)] = z[j][r];
						});
					float top = NOTHING;
#pragma unroll
					for (int j = 0; j < 2; j++)
#pragma unroll
						for (int r = 0; r < 16; r++)
							top = fmaxf(top, z[j][r]);
					const float about = top == NOTHING ? 0.0f : top; /* a row of -inf alone: a sum of zeros */
					float sum = 0.0f;
#pragma unroll
					for (int j = 0; j < 2; j++)
#pragma unroll
						for (int r = 0; r < 16; r++)
							sum += __expf(z[j][r] - about); /* not exp2 of a product and a sum: the type's lowest value, which masks, has no product */
					if (top == -NOTHING) /* infinite logits are all that counts */
					{
						sum = 0.0f;
#pragma unroll
						for (int j = 0; j < 2; j++)
#pragma unroll
							for (int r = 0; r < 16; r++)
								sum += z[j][r] == top ? 1.0f : (z[j][r] < top ? 0.0f : z[j][r]);
					}
					const Partial p = join(Partial { top, sum }, Partial { __shfl_xor(top, 32), __shfl_xor(sum, 32) });
					if ((threadIdx.x & 32) == 0)
						meeting[at.wave_n * BM + at.row(i)] = p;
				}
				__syncthreads();
				const int row = threadIdx.x, m = at.tile_m * BM + row;
				if (row < BM && m < rows)
				{
					Partial p = meeting[row];
#pragma unroll
					for (int w = 1; w < WAVES_N; w++)
						p = join(p, meeting[w * BM + row]);
					partials[static_cast<size_t>(m) * tiles_n + at.tile_n] = p;
				}
			}
	};
	constexpr int FEW_CLASSES = 32; /* of a workgroup of the few-rows kernel */
	template<typename T, int MB, bool STREAM>
	__global__ __launch_bounds__(256) void kernel_loss_few_rows(const T *x, const T *w, const T *bias, const int *targets, int rows, int features, int classes, Partial *partials,
			float *target_logits)
	{
		extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
		float (*sums)[2][16 * MB][16] = reinterpret_cast<float (*)[2][16 * MB][16]>(lds);
		const int n0 = blockIdx.x * FEW_CLASSES;
		const T *first = w + static_cast<size_t>(n0) * features;
		const bool second = n0 + 16 < classes; /* else the first block stands in for it */
		const int last_first = min(15, classes - 1 - n0), last_second = second ? min(15, classes - 1 - n0 - 16) : last_first;
		const T *next = second ? first + static_cast<size_t>(16) * features : first;
		if constexpr (STREAM)
			few_rows_stream<T, MB>(x, rows, first, next, last_first, last_second, features, lds);
		else
			few_rows_sums<T, MB>(x, rows, first, next, last_first, last_second, features, sums);
		const int c = threadIdx.x & 15;
		for (int row = threadIdx.x >> 4; row < 16 * MB; row += 16)
			if (row < rows)
			{
				const int target = targets[row];
				float z[2];
				bool there[2];
#pragma unroll
				for (int i = 0; i < 2; i++)
				{
					const int n = n0 + 16 * i + c;
					there[i] = n < classes;
					z[i] = sums[0][i][row][c] + ((bias != nullptr && there[i]) ? static_cast<float>(bias[n]) : 0.0f);
					if (there[i] && n == target)
						target_logits[row] = z[i];
				}
				const Partial p = lanes_join<16>(partial_of(z, there));
				if (c == 0)
					partials[static_cast<size_t>(row) * gridDim.x + blockIdx.x] = p;
			}
	}
	/* THREADS threads to a row: a wavefront where there are rows enough, else a workgroup, each thread with 8 pairs on their way at a time. Workgroups of wavefronts take further rows: 2^26 and more would be too many threads for a launch */
	template<int THREADS>
	__global__ __launch_bounds__(256) void kernel_join_partials(const Partial *partials, int count, const int *targets, const float *target_logits, int rows, int classes, float *loss, float *lse)
	{
		__shared__ Partial waves[4];
		for (int row = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS; row < rows; row += gridDim.x * (256 / THREADS))
		{
			Partial p { -std::numeric_limits<float>::infinity(), 0.0f };
			const Partial *src = partials + static_cast<size_t>(row) * count;
			for (int first = threadIdx.x % THREADS; first < count; first += 8 * THREADS)
			{
				Partial next[8];
#pragma unroll
				for (int u = 0; u < 8; u++)
					next[u] = src[min(first + u * THREADS, count - 1)];
#pragma unroll
				for (int u = 0; u < 8; u++)
					if (first + u * THREADS < count)
						p = join(p, next[u]);
			}
			p = lanes_join<64>(p);
			if constexpr (THREADS > 64)
			{
				if ((threadIdx.x & 63) == 0)
					waves[threadIdx.x >> 6] = p;
				__syncthreads();
				p = join(join(waves[0], waves[1]), join(waves[2], waves[3]));
			}
			if (threadIdx.x % THREADS == 0)
			{
				const float value = p.top + logf(p.sum);
				const int target = targets[row];
				lse[row] = value;
				loss[row] = (target >= 0 && target < classes) ? value - target_logits[row] : 0.0f;
			}
			if (THREADS > 64)
				return; /* one row, `waves` is in use */
		}
	}

	/* ---- backward ----------------------------------------------------------------------------------------------------------- */
	constexpr int SCALE_GROUPS = 256;
	__global__ __launch_bounds__(256) void kernel_largest_gradient(const float *dloss, const int *targets, int rows, int classes, float *largest)
	{
		__shared__ float waves[4];
		float top = 0.0f;
		for (int i = blockIdx.x * 256 + threadIdx.x; i < rows; i += gridDim.x * 256)
		{
			if (targets[i] >= 0 && targets[i] < classes)
				top = larger_finite(top, dloss[i]);
		}
#pragma unroll
		for (int offset = 32; offset >= 1; offset >>= 1)
			top = fmaxf(top, __shfl_xor(top, offset));
		if ((threadIdx.x & 63) == 0)
			waves[threadIdx.x >> 6] = top;
		__syncthreads();
		if (threadIdx.x == 0)
			largest[blockIdx.x] = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
	}
	/* factors[i] = dloss[i] 2^15 / s, 0 for rows without a class; back = s / 2^15 */
	__global__ __launch_bounds__(256) void kernel_row_factors(const float *dloss, const int *targets, int rows, int classes, const float *largest, int groups, float *factors, float *back)
	{
		float top = 0.0f;
		for (int i = threadIdx.x & 63; i < groups; i += 64)
			top = fmaxf(top, largest[i]);
#pragma unroll
		for (int offset = 32; offset >= 1; offset >>= 1)
			top = fmaxf(top, __shfl_xor(top, offset));
		const int exponent = scale_exponent(top);
		for (int i = blockIdx.x * 256 + threadIdx.x; i < rows; i += gridDim.x * 256)
			factors[i] = (targets[i] >= 0 && targets[i] < classes) ? ldexpf(dloss[i], SCALE_BITS - exponent) : 0.0f;
		if (blockIdx.x == 0 && threadIdx.x == 0)
			*back = ldexpf(1.0f, exponent - SCALE_BITS);
	}
	/* both in one launch of one workgroup */
	constexpr int ROWS_OF_ONE_GROUP = 8192;
	__global__ __launch_bounds__(1024) void kernel_row_factors_of_few(const float *dloss, const int *targets, int rows, int classes, float *factors, float *back)
	{
		__shared__ float waves[16];
		float top = 0.0f;
		for (int i = threadIdx.x; i < rows; i += 1024)
		{
			if (targets[i] >= 0 && targets[i] < classes)
				top = larger_finite(top, dloss[i]);
		}
#pragma unroll
		for (int offset = 32; offset >= 1; offset >>= 1)
			top = fmaxf(top, __shfl_xor(top, offset));
		if ((threadIdx.x & 63) == 0)
			waves[threadIdx.x >> 6] = top;
		__syncthreads();
		for (int w = 0; w < 16; w++)
			top = fmaxf(top, waves[w]);
		const int exponent = scale_exponent(top);
		for (int i = threadIdx.x; i < rows; i += 1024)
			factors[i] = (targets[i] >= 0 && targets[i] < classes) ? ldexpf(dloss[i], SCALE_BITS - exponent) : 0.0f;
		if (threadIdx.x == 0)
			*back = ldexpf(1.0f, exponent - SCALE_BITS);
	}
	/* sum + what rounding takes from four elements: they, less what is stored of them, in fp32 (its own roundings are 2^-24 of d). Dot products with minus ones take the halves as they lie in pairs, subnormal ones too: differences element
	 * by element take twice the instructions, and registers that a 256 x 256 tile does not have (d of 4096 x 32768, k = 2048: 2 % longer than without any of this, 581 against 570 us; element by element 5 %) */
	template<typename V>
	__device__ __forceinline__ float add_what_rounding_takes(float sum, const float *v, const V &stored)
	{
		const half2_t minus_ones { static_cast<half_t>(-1.0f), static_cast<half_t>(-1.0f) };
		sum = __builtin_amdgcn_fdot2(half2_t { stored[0], stored[1] }, minus_ones, sum + (v[0] + v[1]), false);
		return __builtin_amdgcn_fdot2(half2_t { stored[2], stored[3] }, minus_ones, sum + (v[2] + v[3]), false);
	}
	/*
	 * d, the sums of its columns for db, and what rounding to fp16 took from its rows. The elements of a row add up to zero by definition, so that what the rows of W have in common has no part in dx; their roundings
	 * do not, and with W's common part ten times the rest dx would be 1.9e-3 off (2.8e-4 without one). What was taken from a row is therefore added up here, in fp32, and given back to the target's class when dx is made,
	 * dx += lost W[target]: the row adds up to zero again, and the target's element, the largest of d by far until a model is sure of something else, counts unrounded. dx is 2.1e-4 off then, as much as its own rounding
	 * costs, and 2.6e-4 where other classes have large probabilities; dW, where nothing cancels, 2.8e-4.
	 */
	template<typename T>
	struct GradientEpilogue
	{
			const T *bias; /* of the piece */
			const int *targets;
			const float *lse, *factors;
			T *d; /* [rows][row_elements], zeros behind the piece's classes */
			float *sums; /* [row tiles][classes of the piece], or null */
			float *lost; /* [rows][lost_tiles], at this piece's first column tile; fp16, or null */
			int lost_tiles;
			int first_class, classes, row_elements; /* classes: of the piece */

			template<int BM, int BN>
			static constexpr int lds()
			{
				return Stage<T, BN>::bytes(sizeof(T) == 2 ? BM : rows_at_a_time(BM));
			}
			/* in registers, rounded there; through LDS to whole rows. The column sums of a wavefront's 64 rows are folded so that each of 32 lanes ends up with one column of each block */
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				constexpr int BLOCKS = TilePlace<BM, BN>::BLOCKS, ROWS = (sizeof(T) == 2) ? BM : rows_at_a_time(BM), PASSES = BM / ROWS, WAVES_N = BN / 64;
				static_assert((2 * BN + WAVES_N * BM) * static_cast<int>(sizeof(float)) <= GradientEpilogue::template lds<BM, BN>(), "the sums meet where the rows were");
				TileColumns<T, BM, BN> columns;
				columns.begin(at, bias, classes);
				const bool edge = (at.tile_n + 1) * BN > classes;
				const Stage<T, BN> stage { reinterpret_cast<T*>(lds) };
				float total[2][16], taken[BLOCKS];
#pragma unroll
				for (int j = 0; j < 2; j++)
#pragma unroll
					for (int r = 0; r < 16; r++)
						total[j][r] = 0.0f;
				int target[BLOCKS];
				float norm[BLOCKS], factor[BLOCKS];
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
				{
					const int m = min(at.tile_m * BM + at.row(i), rows - 1);
					norm[i] = lse[m];
					factor[i] = at.tile_m * BM + at.row(i) < rows ? factors[m] : 0.0f;
					target[i] = factor[i] != 0.0f ? targets[m] - first_class : -1; /* a class then */
					taken[i] = 0.0f;
				}
				static_for<PASSES>([&](auto pass)
				{
					constexpr int PASS = decltype(pass)::value, FIRST = PASS * BLOCKS / PASSES;
					__syncthreads();
#pragma unroll
					for (int i = FIRST; i < FIRST + BLOCKS / PASSES; i++)
					{
						float v[2][16];
#pragma unroll
						for (int j = 0; j < 2; j++)
#pragma unroll
							for (int r = 0; r < 16; r++)
							{
								const float about = acc[i][j][r] + columns.bias[j][r] - norm[i];
								const float p = (sizeof(T) == 2) ? __expf(about) : expf(about); /* the hardware's is 2^-20 off, which fp16 rounds away */
								/* a row without gradient has none, whatever its logits are */
								v[j][r] = factor[i] == 0.0f ? 0.0f : p * factor[i];
								if (edge)
									v[j][r] = columns.column(j, r) < classes ? v[j][r] : 0.0f;
							}
						if (factor[i] != 0.0f)
							columns.at_class(target[i], [&](int j, int r) __attribute__((always_inline))
							{
								v[j][r] -= factor[i];
							});
#pragma unroll
						for (int j = 0; j < 2; j++)
#pragma unroll
							for (int q = 0; q < 4; q++)
							{
								typename Stage<T, BN>::vec4_t stored;
#pragma unroll
								for (int e = 0; e < 4; e++)
									stored[e] = static_cast<T>(v[j][4 * q + e]);
								stage.put(at.row(i) - PASS * ROWS, at.column(j) + at.lane_column(q), stored);
#pragma unroll
								for (int e = 0; e < 4; e++)
									total[j][4 * q + e] += v[j][4 * q + e];
								if constexpr (sizeof(T) == 2)
									taken[i] = add_what_rounding_takes(taken[i], &v[j][4 * q], stored);
							}
					}
					__syncthreads();
					stage.template copy<ROWS, TilePlace<BM, BN>::THREADS>(d, row_elements, at.tile_m * BM + PASS * ROWS, rows, at.tile_n * BN, row_elements);
				});
				const bool of_columns = sums != nullptr, of_rows = sizeof(T) == 2 && lost != nullptr;
				if (!of_columns && !of_rows)
					return;
				float *meeting = reinterpret_cast<float*>(lds); /* of columns: [2 wavefront rows][BN], of rows: [WAVES_N][BM] */
				__syncthreads();
				if (of_columns)
#pragma unroll
					for (int j = 0; j < 2; j++)
					{
						/* lane bits 4 .. 1 choose among the 16 registers, a half of them at a time; bit 0 adds up what is left */
#pragma unroll
						for (int bit = 16; bit >= 2; bit >>= 1)
#pragma unroll
							for (int r = 0; r < bit / 2; r++)
							{
								const bool upper = (threadIdx.x & bit) != 0;
								const float sent = upper ? total[j][r] : total[j][r + bit / 2];
								const float kept = upper ? total[j][r + bit / 2] : total[j][r];
								total[j][r] = kept + __shfl_xor(sent, bit);
							}
						const float sum = total[j][0] + __shfl_xor(total[j][0], 1);
						const int r = (threadIdx.x & 31) >> 1;
						if ((threadIdx.x & 1) == 0)
							meeting[at.wave_m * BN + at.column(j) + TilePlace<BM, BN>::lane_column(r / 4) + r % 4] = sum;
					}
				if (of_rows)
#pragma unroll
					for (int i = 0; i < BLOCKS; i++)
					{
						const float sum = taken[i] + __shfl_xor(taken[i], 32);
						if ((threadIdx.x & 32) == 0)
							meeting[2 * BN + at.wave_n * BM + at.row(i)] = sum;
					}
				__syncthreads();
				const int n = at.tile_n * BN + static_cast<int>(threadIdx.x), m = at.tile_m * BM + static_cast<int>(threadIdx.x);
				if (of_columns && static_cast<int>(threadIdx.x) < BN && n < classes)
					sums[static_cast<size_t>(at.tile_m) * classes + n] = meeting[threadIdx.x] + meeting[BN + threadIdx.x];
				if (of_rows && static_cast<int>(threadIdx.x) < BM && m < rows)
				{
					float sum = 0.0f;
#pragma unroll
					for (int w = 0; w < WAVES_N; w++)
						sum += meeting[2 * BN + w * BM + threadIdx.x];
					lost[static_cast<size_t>(m) * lost_tiles + at.tile_n] = sum;
				}
			}
	};
	/*
	 * dx = back (sum + lost W[target]) + beta dx in fp16, where one product gives all of dx: in the accumulators, so that nothing in fp32 goes to memory. us, so / over fp32 and the launch that joins parts / without
	 * giving back: gradients of 65536 x 1024, 300 classes 383 / 521 / 363, 8192 x 4096, 1000 classes 387 / 442 / 376, 16384 x 2048, 4000 classes 1031 / 1075 / 986 (its rows of W, 67 MB, come from beyond the L2).
	 */
	template<typename T>
	struct InputEpilogue
	{
			T *out;
			int columns;
			float beta;
			const float *back, *lost;
			int lost_tiles;
			const int *targets;
			int classes;
			const T *w;
			int w_elements;

			template<int BM, int BN>
			static constexpr int lds()
			{
				return StoreEpilogue<T>::template lds<BM, BN>();
			}
			/* the rows of weights to LDS, whole rows to neighbouring threads (rows without a class: zeros), from where every lane takes what belongs to its accumulators */
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				typedef Stage<T, BN> TileStage;
				typedef typename Elements<T, TileStage::VECTOR>::vec_t vec_t;
				constexpr int BLOCKS = TilePlace<BM, BN>::BLOCKS, LANES = BN / TileStage::VECTOR, AT_A_TIME = TilePlace<BM, BN>::THREADS / LANES, TURNS = BM / AT_A_TIME;
				const TileStage stage { reinterpret_cast<T*>(lds) };
				const int first = at.tile_m * BM, column = static_cast<int>(threadIdx.x) % LANES * TileStage::VECTOR, row0 = static_cast<int>(threadIdx.x) / LANES;
				int target[TURNS];
				vec_t weights_of[TURNS]; /* all on their way at once: one workgroup has the unit to itself and would wait for each */
#pragma unroll
				for (int u = 0; u < TURNS; u++)
					target[u] = targets[min(first + row0 + u * AT_A_TIME, rows - 1)];
#pragma unroll
				for (int u = 0; u < TURNS; u++)
				{
					weights_of[u] = vec_t(static_cast<T>(0.0f));
					if (target[u] >= 0 && target[u] < classes && at.tile_n * BN + column < columns) /* whole vectors: the rows of the weights are */
						weights_of[u] = *reinterpret_cast<const vec_t*>(w + static_cast<size_t>(target[u]) * w_elements + at.tile_n * BN + column);
				}
				float taken[BLOCKS];
				const float *mine[BLOCKS];
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
				{
					mine[i] = lost + static_cast<size_t>(min(first + at.row(i), rows - 1)) * lost_tiles;
					taken[i] = 0.0f;
				}
				constexpr int AHEAD = 16 / BLOCKS; /* 16 loads on their way at a time */
				for (int t = 0; t < lost_tiles; t += AHEAD)
				{
					float v[AHEAD][BLOCKS];
#pragma unroll
					for (int u = 0; u < AHEAD; u++)
#pragma unroll
						for (int i = 0; i < BLOCKS; i++)
							v[u][i] = mine[i][min(t + u, lost_tiles - 1)];
#pragma unroll
					for (int u = 0; u < AHEAD; u++)
#pragma unroll
						for (int i = 0; i < BLOCKS; i++)
							taken[i] += t + u < lost_tiles ? v[u][i] : 0.0f;
				}
				__syncthreads();
#pragma unroll
				for (int u = 0; u < TURNS; u++)
					*reinterpret_cast<vec_t*>(stage.place + (row0 + u * AT_A_TIME) * TileStage::STRIDE + column) = weights_of[u];
				__syncthreads();
				Acc whole[BLOCKS][2];
#pragma unroll
				for (int i = 0; i < BLOCKS; i++)
#pragma unroll
					for (int j = 0; j < 2; j++)
#pragma unroll
						for (int q = 0; q < 4; q++)
						{
							const typename TileStage::vec4_t weights = *reinterpret_cast<const typename TileStage::vec4_t*>(stage.place + at.row(i) * TileStage::STRIDE + at.column(j) + at.lane_column(q));
#pragma unroll
							for (int e = 0; e < 4; e++)
								whole[i][j][4 * q + e] = fmaf(taken[i], static_cast<float>(weights[e]), acc[i][j][4 * q + e]);
						}
				StoreEpilogue<T> { out, columns, beta, back }.template tile<BM, BN>(whole, at, lds, rows);
			}
	};
	/*
	 * The same where dx comes about in parts or over several pieces of the classes. A wavefront has 256 columns of a row at a time and adds up what the tiles of the row lost by itself; the last 4 columns of a row are moved back to end
	 * with it, as in RowPlace.
	 */
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_join_input(const float *partial, int parts, int rows, int features, int spans, T *dx, float beta, const float *back, const float *lost, int lost_tiles,
			const int *targets, int classes, const T *w, int w_elements)
	{
		const int lane = threadIdx.x & 63;
		const size_t units = static_cast<size_t>(rows) * spans, count = static_cast<size_t>(rows) * features;
		const float scale = *back;
		for (size_t unit = static_cast<size_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); unit < units; unit += static_cast<size_t>(gridDim.x) * 4)
		{
			int span;
			const size_t row = split_index(unit, spans, span);
			float taken = 0.0f;
			for (int t = lane; t < lost_tiles; t += 64)
				taken += lost[row * lost_tiles + t];
			taken = lanes_sum<64>(taken);
			const int target = targets[row];
			const bool given = target >= 0 && target < classes; /* else nothing was lost, and there is no row of weights to look at */
			const T *weights = w + static_cast<size_t>(given ? target : 0) * w_elements;
			const int column = span * 256 + lane * 4;
			if (column >= features)
				continue;
			const float *src = partial + row * features;
			T *dst = dx + row * features;
			if (features >= 4)
			{
				const RowPlace place = place_in_row<4>(column, features);
				float v[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
				for (int p = 0; p < parts; p++)
				{
					Elements<float, 4> x;
					x.load(place.in(src + p * count));
#pragma unroll
					for (int e = 0; e < 4; e++)
						v[e] += x[e];
				}
				Elements<T, 4> of_target, old;
				of_target.load(place.in(weights));
				if (beta != 0.0f)
					old.load(place.in(dst));
#pragma unroll
				for (int e = 0; e < 4; e++)
				{
					v[e] = scale * (given ? fmaf(taken, of_target[e], v[e]) : v[e]);
					if (beta != 0.0f)
						v[e] = fmaf(beta, old[e], v[e]);
				}
				store_nearest<4>(place.in(dst), v, place.skip);
			}
			else
				for (int c = column; c < features; c++)
				{
					float v = 0.0f;
					for (int p = 0; p < parts; p++)
						v += src[p * count + c];
					v = scale * (given ? fmaf(taken, static_cast<float>(weights[c]), v) : v);
					dst[c] = static_cast<T>(beta != 0.0f ? fmaf(beta, static_cast<float>(dst[c]), v) : v);
				}
		}
	}

	/* ---- sizes ---------------------------------------------------------------------------------------------------------------- */
	struct LossShape
	{
			int rows, features, classes, element_size;
	};
	LossShape loss_shape(const mlShape_t &x, const mlShape_t &w, mlDataType_t dtype, const char *name)
	{
		const std::string who(name);
		MLHIP_REQUIRE(dtype == DTYPE_FLOAT16 || dtype == DTYPE_FLOAT32, who + ": unsupported data type");
		MLHIP_REQUIRE(x.rank >= 1 && x.rank <= 6 && w.rank == 2, who + ": the input needs one to six dimensions, the weights must be [classes, features]");
		for (int i = 0; i < x.rank; i++)
			MLHIP_REQUIRE(x.dim[i] >= 0, who + ": negative dimension");
		MLHIP_REQUIRE(w.dim[0] > 0 && w.dim[1] > 0 && w.dim[1] == last_dim(x), who + ": the weights' last dimension must be the input's, and there must be classes and features");
		const size_t rows = volume(x) / w.dim[1];
		MLHIP_REQUIRE(rows <= (1 << 28) && w.dim[0] <= (1 << 28) && w.dim[1] <= (1 << 18), who + ": too many rows, classes or features");
		return LossShape { static_cast<int>(rows), w.dim[1], w.dim[0], size_of(dtype) };
	}
	bool few_rows(const LossShape &s)
	{
		return takes_few_rows(s.rows, static_cast<size_t>(s.classes) * s.features * s.element_size);
	}
	constexpr size_t PIECE_BYTES = size_t(1) << 28;
	/* classes of a piece: whole tiles, all pieces about the same */
	int classes_of_piece(const LossShape &s)
	{
		/* and a row of d below 4 MB, which the panels' offsets ask for */
		const size_t most = std::min<size_t>(1 << 19, std::max<size_t>(256, PIECE_BYTES / (static_cast<size_t>(std::max(s.rows, 1)) * s.element_size) / 256 * 256));
		const size_t pieces = (s.classes + most - 1) / most;
		return static_cast<int>(std::min<size_t>(round_up((s.classes + pieces - 1) / pieces, 256), s.classes));
	}
	ProductPlan logits_plan(const LossShape &s, int classes)
	{
		return plan_product(s.rows, classes, false, s.features, s.element_size, false);
	}
	ProductPlan input_plan(const LossShape &s, int classes)
	{
		return plan_product(s.rows, s.features, false, classes, s.element_size, true);
	}
	ProductPlan weights_plan(const LossShape &s, int classes)
	{
		return plan_product(classes, s.features, false, s.rows, s.element_size, true, false);
	}
	/* columns of tiles of all pieces; a piece's classes are whole tiles, but for the last one's */
	int tile_width(const LossShape &s, int piece)
	{
		return std::max(logits_plan(s, piece).tile, 128);
	}
	struct LossSpace
	{
			size_t x, w, partials, target_logits; /* forward */
			size_t d, dx, parts, sums, lost, factors, scale; /* backward */
			size_t total;
	};
	/* whether dx comes about in fp32 first */
	bool dx_in_parts(const LossShape &s, int piece)
	{
		return piece < s.classes || input_plan(s, piece).parts > 1;
	}
	LossSpace loss_space(const LossShape &s, bool backward)
	{
		LossSpace space { };
		size_t at = 0;
		const auto take = [&](size_t bytes)
		{
			const size_t begin = at;
			at += round_up(bytes, 256);
			return begin;
		};
		if (s.rows > 0)
		{
			const int pieces = 16 / s.element_size;
			const size_t padded = (s.features % pieces == 0) ? 0 : round_up(s.features, pieces) * s.element_size;
			const bool few = few_rows(s);
			/* the forward pass's pieces lie in the same places as far as both have them: one workspace serves both */
			space.x = take(backward || !few ? padded * s.rows : 0);
			space.w = take(backward || !few ? padded * s.classes : 0);
			const size_t begin = at;
			const size_t columns = few ? ceil_div(s.classes, FEW_CLASSES) : logits_plan(s, s.classes).tiles_n;
			space.partials = take(sizeof(Partial) * columns * s.rows);
			space.target_logits = take(sizeof(float) * s.rows);
			if (backward)
			{
				const size_t forward_end = at;
				at = begin;
				const int classes = classes_of_piece(s);
				const ProductPlan input = input_plan(s, classes), weights = weights_plan(s, classes);
				space.d = take(round_up(classes, pieces) * s.element_size * s.rows);
				space.dx = take(dx_in_parts(s, classes) ? sizeof(float) * input.parts * s.rows * s.features : 0);
				space.parts = take(part_bytes(weights, classes, s.features));
				space.sums = take(sizeof(float) * classes * logits_plan(s, classes).tiles_m);
				space.lost = take(s.element_size == 2 ? sizeof(float) * s.rows * ceil_div(s.classes, tile_width(s, classes)) : 0);
				space.factors = take(sizeof(float) * s.rows);
				space.scale = take(sizeof(float) * (SCALE_GROUPS + 1));
				at = std::max(at, forward_end);
			}
		}
		space.total = at;
		return space;
	}

	template<typename T>
	void loss_forward(hipStream_t stream, const LossShape &s, const T *x, const T *w, const T *bias, const int *targets, float *loss, float *lse, uint8_t *workspace)
	{
		const LossSpace space = loss_space(s, false);
		Partial *partials = reinterpret_cast<Partial*>(workspace + space.partials);
		float *target_logits = reinterpret_cast<float*>(workspace + space.target_logits);
		int columns;
		if (few_rows(s))
		{
			columns = ceil_div(s.classes, FEW_CLASSES);
			with_few_rows<T>(s.rows, s.features, [&](auto blocks, auto streamed)
			{
				constexpr int MB = decltype(blocks)::value, bytes = few_rows_lds<MB>(decltype(streamed)::value);
				auto kernel = kernel_loss_few_rows<T, MB, decltype(streamed)::value>;
				ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
				hipLaunchKernelGGL(kernel, dim3(columns), dim3(256), bytes, stream, x, w, bias, targets, s.rows, s.features, s.classes, partials, target_logits);
			});
		}
		else
		{
			const int padded = padded_columns<T>(s.features);
			x = pad_rows(stream, x, reinterpret_cast<T*>(workspace + space.x), s.rows, s.features);
			w = pad_rows(stream, w, reinterpret_cast<T*>(workspace + space.w), s.classes, s.features);
			const ProductPlan plan = logits_plan(s, s.classes);
			columns = plan.tiles_n;
			const Operand a { reinterpret_cast<const uint8_t*>(x), padded * sizeof(T), s.rows, padded };
			const Operand b { reinterpret_cast<const uint8_t*>(w), padded * sizeof(T), s.classes, padded };
			launch_product<T, Side::ROWS, Side::ROWS, false>(stream, plan, a, b, s.rows, LossEpilogue<T> { bias, targets, partials, target_logits, s.classes, columns });
		}
		MLHIP_CHECK(hipGetLastError());
		if (s.rows <= 1024)
			hipLaunchKernelGGL((kernel_join_partials<256>), dim3(s.rows), dim3(256), 0, stream, partials, columns, targets, target_logits, s.rows, s.classes, loss, lse);
		else
			hipLaunchKernelGGL((kernel_join_partials<64>), dim3(std::min(ceil_div(s.rows, 4), 1 << 20)), dim3(256), 0, stream, partials, columns, targets, target_logits, s.rows, s.classes, loss, lse);
		MLHIP_CHECK(hipGetLastError());
	}
	template<typename T>
	void loss_backward(hipStream_t stream, const LossShape &s, const T *x, const T *w, const T *bias, const int *targets, const float *lse, const float *dloss, float beta_dx, T *dx,
			float beta_weights, const mlTensor_t &dw, const mlTensor_t &db, uint8_t *workspace)
	{
		const LossSpace space = loss_space(s, true);
		const int padded = padded_columns<T>(s.features), most = classes_of_piece(s);
		T *d = reinterpret_cast<T*>(workspace + space.d);
		float *partial_dx = reinterpret_cast<float*>(workspace + space.dx), *parts = reinterpret_cast<float*>(workspace + space.parts);
		float *sums = reinterpret_cast<float*>(workspace + space.sums), *factors = reinterpret_cast<float*>(workspace + space.factors);
		float *largest = reinterpret_cast<float*>(workspace + space.scale), *back = largest + SCALE_GROUPS;
		const int groups = std::min(ceil_div(s.rows, 256), SCALE_GROUPS);
		if (s.rows <= ROWS_OF_ONE_GROUP)
			hipLaunchKernelGGL(kernel_row_factors_of_few, dim3(1), dim3(1024), 0, stream, dloss, targets, s.rows, s.classes, factors, back);
		else
		{
			hipLaunchKernelGGL(kernel_largest_gradient, dim3(groups), dim3(256), 0, stream, dloss, targets, s.rows, s.classes, largest);
			hipLaunchKernelGGL(kernel_row_factors, dim3(groups), dim3(256), 0, stream, dloss, targets, s.rows, s.classes, largest, groups, factors, back);
		}
		MLHIP_CHECK(hipGetLastError());
		x = pad_rows(stream, x, reinterpret_cast<T*>(workspace + space.x), s.rows, s.features);
		w = pad_rows(stream, w, reinterpret_cast<T*>(workspace + space.w), s.classes, s.features);
		const size_t row_bytes = padded * sizeof(T), outputs = static_cast<size_t>(s.rows) * s.features;
		const ProductPlan whole_input = input_plan(s, most);
		const bool in_parts = dx_in_parts(s, most);
		const int width = tile_width(s, most), lost_tiles = ceil_div(s.classes, width);
		float *lost = reinterpret_cast<float*>(workspace + space.lost);
		/* the last piece, which may be smaller, is cut by the plans of the others: the workspace is sized by them */
		for (int first = 0; first < s.classes; first += most)
		{
			const int classes = std::min(most, s.classes - first), row_elements = padded_columns<T>(classes);
			const uint8_t *weights = reinterpret_cast<const uint8_t*>(w) + first * row_bytes;
			{
				ProductPlan plan = logits_plan(s, most);
				plan.tiles_n = ceil_div(classes, width);
				const Operand a { reinterpret_cast<const uint8_t*>(x), row_bytes, s.rows, padded };
				const Operand b { weights, row_bytes, classes, padded };
				launch_product<T, Side::ROWS, Side::ROWS, false>(stream, plan, a, b, s.rows, GradientEpilogue<T> { bias != nullptr ? bias + first : nullptr, targets, lse, factors, d,
						db.data != nullptr ? sums : nullptr, dx != nullptr ? lost + first / width : nullptr, lost_tiles, first, classes, row_elements });
				if (db.data != nullptr)
					launch_sum_partials(stream, sums, plan.tiles_m, static_cast<size_t>(classes), static_cast<uint8_t*>(db.data) + static_cast<size_t>(first) * size_of(db.dtype), db.dtype, classes,
							beta_weights, back);
			}
			if (dx != nullptr)
			{
				ProductPlan plan = whole_input; /* a part that has no chunk left adds nothing */
				plan.chunks = ceil_div(classes, 128 / static_cast<int>(sizeof(T)));
				const Operand a { reinterpret_cast<const uint8_t*>(d), row_elements * sizeof(T), s.rows, row_elements };
				const Operand b { weights, row_bytes, padded, classes };
				if (in_parts)
					launch_product<T, Side::ROWS, Side::COLUMNS, false>(stream, plan, a, b, s.rows, PartEpilogue { partial_dx, outputs, s.features, first > 0 });
				else if constexpr (sizeof(T) == 2)
					launch_product<T, Side::ROWS, Side::COLUMNS, false>(stream, plan, a, b, s.rows, InputEpilogue<T> { dx, s.features, beta_dx, back, lost, lost_tiles, targets, s.classes, w, padded });
				else
					launch_product<T, Side::ROWS, Side::COLUMNS, false>(stream, plan, a, b, s.rows, StoreEpilogue<T> { dx, s.features, beta_dx, back });
			}
			if (dw.data != nullptr)
			{
				ProductPlan plan = weights_plan(s, most);
				plan.tiles_m = ceil_div(classes, plan.tile);
				const Operand a { reinterpret_cast<const uint8_t*>(d), row_elements * sizeof(T), row_elements, s.rows };
				const Operand b { reinterpret_cast<const uint8_t*>(x), row_bytes, padded, s.rows };
				const size_t offset = static_cast<size_t>(first) * s.features;
				if (dw.dtype == DTYPE_FLOAT32)
					product_to<T, float, Side::COLUMNS, Side::COLUMNS>(stream, plan, a, b, classes, s.features, ptr<float>(dw) + offset, beta_weights, back, parts);
				else if constexpr (sizeof(T) == 2)
					product_to<T, T, Side::COLUMNS, Side::COLUMNS>(stream, plan, a, b, classes, s.features, ptr<T>(dw) + offset, beta_weights, back, parts);
			}
		}
		if (dx != nullptr && in_parts)
		{
			if constexpr (sizeof(T) == 2)
			{
				const int spans = ceil_div(s.features, 256);
				const size_t groups = std::min<size_t>((static_cast<size_t>(s.rows) * spans + 3) / 4, 1 << 16);
				hipLaunchKernelGGL((kernel_join_input<T>), dim3(static_cast<unsigned int>(groups)), dim3(256), 0, stream, partial_dx, whole_input.parts, s.rows, s.features, spans, dx, beta_dx, back, lost,
						lost_tiles, targets, s.classes, w, padded);
				MLHIP_CHECK(hipGetLastError());
			}
			else
				launch_join_parts(stream, partial_dx, whole_input.parts, outputs, dx, beta_dx, back);
		}
	}

	bool weight_type(const mlTensor_t &t, const mlTensor_t &x)
	{
		return t.dtype == x.dtype || t.dtype == DTYPE_FLOAT32;
	}
	bool per_row(const mlTensor_t &t, const LossShape &s, mlDataType_t dtype)
	{
		return t.dtype == dtype && volume(t) == static_cast<size_t>(s.rows) && (s.rows == 0 || (t.data != nullptr && reinterpret_cast<uintptr_t>(t.data) % 4 == 0));
	}
	LossShape check_loss(const mlTensor_t &x, const mlTensor_t &w, const mlTensor_t &b, const mlTensor_t &targets, const char *name)
	{
		const std::string who(name);
		const LossShape s = loss_shape(shape_of(x), shape_of(w), x.dtype, name);
		MLHIP_REQUIRE(w.dtype == x.dtype, who + ": weights must have the input's type");
		MLHIP_REQUIRE(b.data == nullptr || (b.dtype == x.dtype && volume(b) == static_cast<size_t>(s.classes)), who + ": the bias must be [classes] of the input's type");
		MLHIP_REQUIRE(per_row(targets, s, DTYPE_INT32), who + ": there must be one int32 target per row");
		MLHIP_REQUIRE(s.rows == 0 || (x.data != nullptr && w.data != nullptr), who + ": null pointer");
		MLHIP_REQUIRE(reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && reinterpret_cast<uintptr_t>(w.data) % 16 == 0, who + ": input and weights must be aligned to 16 bytes");
		return s;
	}
	void check_space(const void *workspace, size_t given, size_t needed, const char *name)
	{
		MLHIP_REQUIRE(needed == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && given >= needed),
				std::string(name) + ": the workspace is too small or not aligned to 256 bytes");
	}
}

extern "C"
{
	using namespace mlhip;

	size_t hip_linear_cross_entropy_get_workspace_size(mlShape_t input_shape, mlShape_t weights_shape, mlDataType_t dtype, bool backward)
	try
	{
		return loss_space(loss_shape(input_shape, weights_shape, dtype, "linear_cross_entropy_get_workspace_size"), backward).total;
	}
	catch (...)
	{
		return mlhip::entry_failed<size_t>();
	}

	void hip_linear_cross_entropy_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t b, const mlTensor_t targets, mlTensor_t loss, mlTensor_t lse,
			void *workspace, size_t workspace_size)
	try
	{
		const char *name = "linear_cross_entropy_forward";
		const LossShape s = check_loss(x, w, b, targets, name);
		MLHIP_REQUIRE(per_row(loss, s, DTYPE_FLOAT32) && per_row(lse, s, DTYPE_FLOAT32), "linear_cross_entropy_forward: loss and lse must be fp32 with one element per row");
		if (s.rows == 0)
			return;
		check_space(workspace, workspace_size, loss_space(s, false).total, name);
		require_apart( { loss, lse, Extent(workspace, workspace_size) }, { x, w, b, targets }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			loss_forward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(b), ptr<int>(targets), ptr<float>(loss), ptr<float>(lse), reinterpret_cast<uint8_t*>(workspace));
		else
			loss_forward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(b), ptr<int>(targets), ptr<float>(loss), ptr<float>(lse), reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}

	void hip_linear_cross_entropy_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t b, const mlTensor_t targets, const mlTensor_t lse, const mlTensor_t dloss,
			float beta_dx, mlTensor_t dx, float beta_weights, mlTensor_t dw, mlTensor_t db, void *workspace, size_t workspace_size)
	try
	{
		const char *name = "linear_cross_entropy_backward";
		const LossShape s = check_loss(x, w, b, targets, name);
		MLHIP_REQUIRE(per_row(lse, s, DTYPE_FLOAT32) && per_row(dloss, s, DTYPE_FLOAT32), "linear_cross_entropy_backward: lse and dloss must be fp32 with one element per row");
		MLHIP_REQUIRE(dx.data == nullptr || (dx.dtype == x.dtype && volume(dx) == volume(x)), "linear_cross_entropy_backward: dx must have the input's shape and type");
		MLHIP_REQUIRE(dw.data == nullptr || (weight_type(dw, x) && volume(dw) == volume(w)), "linear_cross_entropy_backward: dw must be [classes, features] of the input's type or fp32");
		MLHIP_REQUIRE(db.data == nullptr || (weight_type(db, x) && volume(db) == static_cast<size_t>(s.classes)), "linear_cross_entropy_backward: db must be [classes] of the input's type or fp32");
		if (dx.data == nullptr && dw.data == nullptr && db.data == nullptr)
			return;
		if (s.rows == 0)
		{
			/* sums over nothing */
			const OnDeviceOf on(context);
			for (const mlTensor_t &t : { dw, db })
				if (t.data != nullptr)
				{
					if (t.dtype == DTYPE_FLOAT16)
						launch_join_parts<half_t>(on.stream, nullptr, 0, volume(t), ptr<half_t>(t), beta_weights, nullptr);
					else
						launch_join_parts<float>(on.stream, nullptr, 0, volume(t), ptr<float>(t), beta_weights, nullptr);
				}
			return;
		}
		check_space(workspace, workspace_size, loss_space(s, true).total, name);
		require_apart( { dx, dw, db, Extent(workspace, workspace_size) }, { x, w, b, targets, lse, dloss }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			loss_backward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(b), ptr<int>(targets), ptr<float>(lse), ptr<float>(dloss), beta_dx, ptr<half_t>(dx), beta_weights, dw, db,
					reinterpret_cast<uint8_t*>(workspace));
		else
			loss_backward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(b), ptr<int>(targets), ptr<float>(lse), ptr<float>(dloss), beta_dx, ptr<float>(dx), beta_weights, dw, db,
					reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}

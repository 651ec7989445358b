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
#include "vocabulary_loss.hpp"

namespace
{
	using namespace mlhip;

	/* ---- the goal: one class of every row ----------------------------------------------------------------------------------- */
	struct OneClass
	{
			static constexpr bool ONE = true;
			const int *targets;
			float *target_logits;

			template<int BLOCKS>
			struct Rows
			{
					int target[BLOCKS];

					__device__ __forceinline__ void begin(const OneClass &goal, int i, int m, int rows, int classes)
					{
						const int t = m < rows ? goal.targets[m] : -1;
						target[i] = t < classes ? t : -1;
					}
					template<typename Columns>
					__device__ __forceinline__ void take_row(const OneClass &goal, int i, int m, const Columns &columns, const float (&z)[2][16]) const
					{
						if (target[i] >= 0)
							columns.at_class(target[i], [&](int j, int r) __attribute__((always_inline))
							{
								goal.target_logits[m] = z[j][r];
							});
					}
			};
			__device__ __forceinline__ float scaled(float z) const
			{
				return z;
			}
			__device__ __forceinline__ float less(float z, float norm) const
			{
				return z - norm;
			}
			template<int BM, int BN>
			static constexpr int loss_lds()
			{
				return 0;
			}
			template<int BM, int BN>
			static constexpr int gradient_lds()
			{
				return 0;
			}
			struct Nothing
			{
			};
			template<int BM, int BN>
			__device__ __forceinline__ Nothing begin_loss(const TilePlace<BM, BN>&, int) const
			{
				return Nothing { };
			}
			template<int BM, int BN, typename Acc, typename Columns>
			__device__ __forceinline__ void take_tile(const Acc&, const Columns&, const TilePlace<BM, BN>&, const Nothing&, uint8_t*) const
			{
			}
			template<int BM, int BN>
			__device__ __forceinline__ Nothing begin_gradient(const TilePlace<BM, BN>&, int, const float*) const
			{
				return Nothing { };
			}
			template<int BM, int BN>
			__device__ __forceinline__ void begin_sums(uint8_t*) const
			{
			}
			template<int BM, int BN, int ROWS, typename TileStage>
			__device__ __forceinline__ void correct(const TileStage&, uint8_t*, const TilePlace<BM, BN>&, const Nothing&, int, int) const
			{
			}
			template<int BM, int BN>
			__device__ __forceinline__ float column_sum(float sum, uint8_t*) const
			{
				return sum;
			}
			template<int BM, int BN>
			__device__ __forceinline__ float row_lost(float sum, uint8_t*) const
			{
				return sum;
			}
	};

	/* ---- forward ------------------------------------------------------------------------------------------------------------ */
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
			const Partial p = join_row<THREADS>(partials + static_cast<size_t>(row) * count, count, waves);
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
	template<typename T>
	void loss_forward(hipStream_t stream, const LossShape &s, const T *x, const T *w, const T *bias, const int *targets, float *loss, float *lse, uint8_t *workspace)
	{
		const LossSpace space = loss_space(s, false, few_rows(s), false);
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
			launch_product<T, Side::ROWS, Side::ROWS, false>(stream, plan, a, b, s.rows, LossEpilogue<T, OneClass> { bias, OneClass { targets, target_logits }, partials, s.classes, columns });
		}
		MLHIP_CHECK(hipGetLastError());
		if (s.rows <= 1024)
			hipLaunchKernelGGL((kernel_join_partials<256>), dim3(s.rows), dim3(256), 0, stream, partials, columns, targets, target_logits, s.rows, s.classes, loss, lse);
		else
			hipLaunchKernelGGL((kernel_join_partials<64>), dim3(std::min(ceil_div(s.rows, 4), 1 << 20)), dim3(256), 0, stream, partials, columns, targets, target_logits, s.rows, s.classes, loss, lse);
		MLHIP_CHECK(hipGetLastError());
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
}

extern "C"
{
	using namespace mlhip;

	size_t hip_linear_cross_entropy_get_workspace_size(mlShape_t input_shape, mlShape_t weights_shape, mlDataType_t dtype, bool backward)
	try
	{
		const LossShape s = loss_shape(input_shape, weights_shape, dtype, "linear_cross_entropy_get_workspace_size");
		return loss_space(s, backward, few_rows(s), false).total;
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
		check_space(workspace, workspace_size, loss_space(s, false, few_rows(s), false).total, name);
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
		check_gradients(x, w, s, dx, dw, db, name);
		if (dx.data == nullptr && dw.data == nullptr && db.data == nullptr)
			return;
		if (s.rows == 0)
		{
			const OnDeviceOf on(context);
			sums_over_nothing(on.stream, dw, db, beta_weights);
			return;
		}
		const auto goal = [&](int)
		{
			return OneClass { ptr<int>(targets), nullptr };
		};
		check_space(workspace, workspace_size, loss_space(s, true, few_rows(s), false).total, name);
		require_apart( { dx, dw, db, Extent(workspace, workspace_size) }, { x, w, b, targets, lse, dloss }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			loss_backward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(b), GivenBack<half_t> { ptr<int>(targets), nullptr, nullptr, nullptr }, goal, 1.0f, ptr<float>(lse), ptr<float>(dloss), beta_dx, ptr<half_t>(dx), beta_weights, dw, db, few_rows(s), false,
					reinterpret_cast<uint8_t*>(workspace));
		else
			loss_backward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(b), GivenBack<float> { ptr<int>(targets), nullptr, nullptr, nullptr }, goal, 1.0f, ptr<float>(lse), ptr<float>(dloss), beta_dx, ptr<float>(dx), beta_weights, dw, db, few_rows(s), false,
					reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}

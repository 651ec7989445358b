/*
 * layernorm.hip — layer normalisation over the last dimension and its backward pass.
 *
 *   m = mean_j x[i, j],  v = mean_j (x[i, j] - m)^2,  r = 1 / sqrt(v + epsilon),  n[i, j] = (x[i, j] - m) r
 *   forward:   y[i, j]  = n[i, j] w[j] + b[j]
 *   backward:  g = dy w;  dx[i, j] = r (g[i, j] - mean_j g - n[i, j] mean_j (g n)) + beta dx[i, j]
 *              dw[j] = sum_i dy[i, j] n[i, j],  db[j] = sum_i dy[i, j]
 *
 * Memory bounds both. A row is read once and kept in registers, at most 16 elements to a thread, so the variance is taken about the mean without a second pass over memory, and
 * nothing but x itself has to be kept for the backward pass: the statistics of a row cost less than reading them. 16 to 64 lanes of a wavefront share a row of up to 1024 elements and 256 or
 * 1024 threads a longer one; beyond 16384 elements the row is read again for every step.
 * The sums over the rows stay in the registers of the thread that owns the columns, while its workgroup walks over the rows; every workgroup leaves one row of them in
 * the caller's workspace, and a second launch adds these rows up in a fixed order.
 * Forward 57600 x 256 fp16 11.9 us (5.0 TB/s, launch included); backward 16384 x 4096 fp16 79 us (5.1 TB/s, a large copy moves 5.2), 7001 x 1001 fp32, whose rows begin anywhere, 21 us (4.0 TB/s);
 * beyond 8192 elements a workgroup fills a compute unit and has one row in hand at a time: 4096 x 16384 fp16 115 us (3.5 TB/s), fp32 175 us (4.6 TB/s).
 */
#include "training_utils.hpp"

#include <algorithm>

namespace
{
	using namespace mlhip;

	constexpr int MAX_PARTS = 512; /* workgroups of a backward pass, two per compute unit: what each leaves is written and read once more */
	constexpr int LONGEST_IN_REGISTERS = 16384;
	constexpr int LONGEST_ROW = 1 << 28; /* columns are counted with 32 bits, also one step beyond a row's end, and 8 threads of a launch sum a column */

	/* the threads that share a row, and their sums. LANES <= 64: part of a wavefront; else the whole workgroup, through LDS */
	template<int LANES>
	struct RowSum
	{
			static constexpr int WAVES = LANES / 64;
			float *scratch; /* [2][3][WAVES], the halves in turn: one barrier per sum is enough */
			int turn;

			template<int N>
			__device__ __forceinline__ void operator()(float (&v)[N])
			{
				static_assert(N <= 3, "scratch holds three sums");
#pragma unroll
				for (int i = 0; i < N; i++)
					v[i] = lanes_sum<(LANES < 64 ? LANES : 64)>(v[i]);
				if constexpr (LANES > 64)
				{
					float *slot = scratch + turn * 3 * WAVES;
					turn ^= 1;
					if ((threadIdx.x & 63) == 0)
#pragma unroll
						for (int i = 0; i < N; i++)
							slot[i * WAVES + (threadIdx.x >> 6)] = v[i];
					__syncthreads();
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						v[i] = 0.0f;
#pragma unroll
						for (int w = 0; w < WAVES; w++)
							v[i] += slot[i * WAVES + w];
					}
				}
			}
	};
	/* nothing that the compiler made of the value before stays in registers: it is made again where it is used. Scalar: the same for all lanes */
	template<typename V>
	__device__ __forceinline__ void take_as_new(V &value)
	{
		asm volatile("" : "+v"(value));
	}
	template<typename V>
	__device__ __forceinline__ void take_as_new_scalar(V &value)
	{
		asm volatile("" : "+s"(value));
	}
	template<int LANES>
	constexpr int threads_of()
	{
		return LANES <= 64 ? 256 : LANES;
	}

	/* ------------------------------------------------------------------------------------------------------------------------
	 * forward, rows in registers
	 * ---------------------------------------------------------------------------------------------------------------------- */
	template<typename T, int VEC, int ITEMS, int LANES>
	__global__ __launch_bounds__(threads_of<LANES>()) void kernel_layer_norm_forward(const T *x, T *y, size_t rows, int columns, float epsilon, const T *w, const T *b)
	{
		constexpr int ROWS = threads_of<LANES>() / LANES; /* of a workgroup at a time */
		__shared__ float scratch[LANES > 64 ? 6 * (LANES / 64) : 1];
		RowSum<LANES> row_sum { scratch, 0 };
		const int lane = threadIdx.x % LANES;
		const float inv_columns = 1.0f / static_cast<float>(columns);
		RowPlace place[ITEMS];
		Elements<T, VEC> gamma[ITEMS], shift[ITEMS];
#pragma unroll
		for (int i = 0; i < ITEMS; i++)
		{
			place[i] = place_in_row<VEC>((lane + LANES * i) * VEC, columns);
			if (w != nullptr)
				gamma[i].load(place[i].in(w));
			if (b != nullptr)
				shift[i].load(place[i].in(b));
		}
		for (size_t first = static_cast<size_t>(blockIdx.x) * ROWS; first < rows; first += static_cast<size_t>(gridDim.x) * ROWS)
		{
			/* threads behind the last row work on it again and store nothing */
			const size_t wanted = first + threadIdx.x / LANES, row = min(wanted, rows - 1);
			const T *src = x + row * columns;
			Elements<T, VEC> raw[ITEMS];
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
				raw[i].load(place[i].in(src));
			float sum[1] = { 0.0f };
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					sum[0] += (e >= place[i].skip) ? raw[i][e] : 0.0f;
			row_sum(sum);
			const float mean = sum[0] * inv_columns;
			float square[1] = { 0.0f };
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
#pragma unroll
				for (int e = 0; e < VEC; e++)
				{
					const float d = (e >= place[i].skip) ? raw[i][e] - mean : 0.0f;
					square[0] = fmaf(d, d, square[0]);
				}
			row_sum(square);
			const float r = 1.0f / sqrtf(square[0] * inv_columns + epsilon);
			if (wanted < rows)
			{
				T *dst = y + row * columns;
#pragma unroll
				for (int i = 0; i < ITEMS; i++)
					if (place[i].skip < VEC)
					{
						float out[VEC];
#pragma unroll
						for (int e = 0; e < VEC; e++)
						{
							const float n = (raw[i][e] - mean) * r;
							out[e] = fmaf(n, w != nullptr ? gamma[i][e] : 1.0f, b != nullptr ? shift[i][e] : 0.0f);
						}
						store_nearest<VEC>(place[i].in(dst), out, place[i].skip);
					}
			}
		}
	}

	/* ------------------------------------------------------------------------------------------------------------------------
	 * backward, rows in registers. partial: [gridDim.x][2][columns], the sums of dy n and of dy over the workgroup's rows
	 * ---------------------------------------------------------------------------------------------------------------------- */
	template<typename T, int VEC, int ITEMS, int LANES>
	__global__ __launch_bounds__(threads_of<LANES>()) void kernel_layer_norm_backward(const T *x, const T *dy, T *dx, size_t rows, int columns, float epsilon, float beta,
			const T *w, float *partial)
	{
		constexpr int THREADS = threads_of<LANES>(), ROWS = THREADS / LANES;
		/*
		 * The next row is on its way while this one is summed, where the registers hold both. 1024 threads have 128 registers each: one row at 16 elements a thread, the weights and both sums fit if nothing else is kept
		 * across the row's steps, which the compiler has to be told (it would keep differences and products of the row, addresses of every lane and the tests of `skip`, and spill). us, two rows that spill / so: 4096 x 16384
		 * fp16 164 / 115, fp32 423 / 175 (4.6 TB/s), 4096 x 8200 122 / 86, 352 / 105.
		 */
		constexpr bool AHEAD = LANES < 1024 || VEC * ITEMS < 16;
		/* the workgroup's row groups meet here at the end: all but the first leave their sums, [ROWS - 1][2][LANES * VEC * ITEMS] in pieces of one item */
		__shared__ float scratch[LANES > 64 ? 6 * (LANES / 64) : 2 * THREADS * VEC];
		RowSum<LANES> row_sum { scratch, 0 };
		const int lane = threadIdx.x % LANES;
		const float inv_columns = 1.0f / static_cast<float>(columns);
		RowPlace place[ITEMS];
		Elements<T, VEC> gamma[ITEMS];
		float sum_w[ITEMS][VEC], sum_b[ITEMS][VEC];
#pragma unroll
		for (int i = 0; i < ITEMS; i++)
		{
			place[i] = place_in_row<VEC>((lane + LANES * i) * VEC, columns);
			if (w != nullptr)
				gamma[i].load(place[i].in(w));
#pragma unroll
			for (int e = 0; e < VEC; e++)
				sum_w[i][e] = sum_b[i][e] = 0.0f;
		}
		const size_t step = static_cast<size_t>(gridDim.x) * ROWS;
		size_t first = static_cast<size_t>(blockIdx.x) * ROWS;
		Elements<T, VEC> next_x[ITEMS], next_dy[ITEMS];
		const auto request = [&](size_t group) __attribute__((always_inline))
		{
			size_t offset = min(group + threadIdx.x / LANES, rows - 1) * columns;
			if constexpr (!AHEAD)
				take_as_new_scalar(offset);
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
			{
				next_x[i].load(place[i].in(x + offset));
				next_dy[i].load(place[i].in(dy + offset));
			}
		};
		if (AHEAD && first < rows)
			request(first);
		for (; first < rows; first += step)
		{
			if (!AHEAD)
				request(first);
			const size_t wanted = first + threadIdx.x / LANES;
			const bool there = wanted < rows;
			Elements<T, VEC> raw_x[ITEMS], raw_dy[ITEMS];
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
			{
				raw_x[i] = next_x[i];
				raw_dy[i] = next_dy[i];
				if constexpr (!AHEAD)
					take_as_new(place[i].skip);
			}
			if (AHEAD && first + step < rows)
				request(first + step);
			float sum[1] = { 0.0f };
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					sum[0] += (e >= place[i].skip) ? raw_x[i][e] : 0.0f;
			row_sum(sum);
			const float mean = sum[0] * inv_columns;
			float sums[3] = { 0.0f, 0.0f, 0.0f }; /* of (x - m)^2, g, g (x - m) */
#pragma unroll
			for (int i = 0; i < ITEMS; i++)
			{
#pragma unroll
				for (int e = 0; e < VEC; e++)
				{
					const bool counts = e >= place[i].skip;
					const float d = counts ? raw_x[i][e] - mean : 0.0f;
					const float g = counts ? (w != nullptr ? raw_dy[i][e] * gamma[i][e] : raw_dy[i][e]) : 0.0f;
					sums[0] = fmaf(d, d, sums[0]);
					sums[1] += g;
					sums[2] = fmaf(g, d, sums[2]);
				}
			}
			row_sum(sums);
			const float r = 1.0f / sqrtf(sums[0] * inv_columns + epsilon);
			const float mean_g = sums[1] * inv_columns, mean_gn = sums[2] * r * inv_columns;
			if (there)
			{
				size_t offset = wanted * columns;
				if constexpr (!AHEAD)
					take_as_new_scalar(offset);
				T *dst = dx + offset;
#pragma unroll
				for (int i = 0; i < ITEMS; i++)
				{
					float out[VEC];
					if constexpr (!AHEAD)
					{
						take_as_new(raw_x[i].raw);
						take_as_new(raw_dy[i].raw);
					}
#pragma unroll
					for (int e = 0; e < VEC; e++)
					{
						const float n = (raw_x[i][e] - mean) * r;
						const float g = w != nullptr ? raw_dy[i][e] * gamma[i][e] : raw_dy[i][e];
						out[e] = r * (g - mean_g - n * mean_gn);
						sum_w[i][e] = fmaf(raw_dy[i][e], n, sum_w[i][e]); /* of columns before place.skip too: they are not stored */
						sum_b[i][e] += raw_dy[i][e];
					}
					if (dx != nullptr && place[i].skip < VEC)
					{
						if (beta != 0.0f)
						{
							Elements<T, VEC> old;
							old.load(place[i].in(dst));
#pragma unroll
							for (int e = 0; e < VEC; e++)
								out[e] = fmaf(beta, old[e], out[e]);
						}
						store_nearest<VEC>(place[i].in(dst), out, place[i].skip);
					}
				}
			}
		}
		if (partial == nullptr)
			return;
		float *mine = partial + static_cast<size_t>(blockIdx.x) * 2 * columns;
#pragma unroll
		for (int i = 0; i < ITEMS; i++)
		{
			if constexpr (ROWS > 1)
			{
				/* [2][VEC][THREADS]: neighbouring threads, neighbouring words */
				__syncthreads();
#pragma unroll
				for (int e = 0; e < VEC; e++)
				{
					scratch[e * THREADS + threadIdx.x] = sum_w[i][e];
					scratch[(VEC + e) * THREADS + threadIdx.x] = sum_b[i][e];
				}
				__syncthreads();
				if (threadIdx.x < LANES)
#pragma unroll
					for (int e = 0; e < VEC; e++)
						for (int g = 1; g < ROWS; g++)
						{
							sum_w[i][e] += scratch[e * THREADS + g * LANES + threadIdx.x];
							sum_b[i][e] += scratch[(VEC + e) * THREADS + g * LANES + threadIdx.x];
						}
			}
			if (threadIdx.x < LANES && place[i].skip < VEC)
			{
				store_nearest<VEC>(place[i].in(mine), sum_w[i], place[i].skip);
				store_nearest<VEC>(place[i].in(mine + columns), sum_b[i], place[i].skip);
			}
		}
	}

	/* ------------------------------------------------------------------------------------------------------------------------
	 * rows of more than 16384 elements: one workgroup per row, read again for every step
	 * ---------------------------------------------------------------------------------------------------------------------- */
	template<typename T>
	__device__ __forceinline__ void long_row_statistics(const T *src, int columns, float epsilon, RowSum<256> &row_sum, float &mean, float &r)
	{
		const float inv_columns = 1.0f / static_cast<float>(columns);
		float sum[1] = { 0.0f };
		for (int j = threadIdx.x; j < columns; j += 256)
			sum[0] += static_cast<float>(src[j]);
		row_sum(sum);
		mean = sum[0] * inv_columns;
		sum[0] = 0.0f;
		for (int j = threadIdx.x; j < columns; j += 256)
		{
			const float d = static_cast<float>(src[j]) - mean;
			sum[0] = fmaf(d, d, sum[0]);
		}
		row_sum(sum);
		r = 1.0f / sqrtf(sum[0] * inv_columns + epsilon);
	}
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_layer_norm_forward_long(const T *x, T *y, size_t rows, int columns, float epsilon, const T *w, const T *b)
	{
		__shared__ float scratch[24];
		RowSum<256> row_sum { scratch, 0 };
		for (size_t row = blockIdx.x; row < rows; row += gridDim.x)
		{
			const T *src = x + row * columns;
			float mean, r;
			long_row_statistics(src, columns, epsilon, row_sum, mean, r);
			T *dst = y + row * columns;
			for (int j = threadIdx.x; j < columns; j += 256)
			{
				const float n = (static_cast<float>(src[j]) - mean) * r;
				dst[j] = static_cast<T>(fmaf(n, w != nullptr ? static_cast<float>(w[j]) : 1.0f, b != nullptr ? static_cast<float>(b[j]) : 0.0f));
			}
		}
	}
	/* statistics: [rows][2] */
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_layer_norm_statistics_long(const T *x, size_t rows, int columns, float epsilon, float *statistics)
	{
		__shared__ float scratch[24];
		RowSum<256> row_sum { scratch, 0 };
		for (size_t row = blockIdx.x; row < rows; row += gridDim.x)
		{
			float mean, r;
			long_row_statistics(x + row * columns, columns, epsilon, row_sum, mean, r);
			if (threadIdx.x == 0)
			{
				statistics[2 * row] = mean;
				statistics[2 * row + 1] = r;
			}
		}
	}
	/* a workgroup sums 256 columns of every gridDim.y-th row */
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_layer_norm_sums_long(const T *x, const T *dy, size_t rows, int columns, const float *statistics, float *partial)
	{
		const int j = blockIdx.x * 256 + threadIdx.x;
		if (j >= columns)
			return;
		float sum_w = 0.0f, sum_b = 0.0f;
		for (size_t row = blockIdx.y; row < rows; row += gridDim.y)
		{
			const float g = static_cast<float>(dy[row * columns + j]);
			const float n = (static_cast<float>(x[row * columns + j]) - statistics[2 * row]) * statistics[2 * row + 1];
			sum_w = fmaf(g, n, sum_w);
			sum_b += g;
		}
		partial[static_cast<size_t>(blockIdx.y) * 2 * columns + j] = sum_w;
		partial[(static_cast<size_t>(blockIdx.y) * 2 + 1) * columns + j] = sum_b;
	}
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_layer_norm_backward_long(const T *x, const T *dy, T *dx, size_t rows, int columns, float beta, const T *w, const float *statistics)
	{
		__shared__ float scratch[24];
		RowSum<256> row_sum { scratch, 0 };
		const float inv_columns = 1.0f / static_cast<float>(columns);
		for (size_t row = blockIdx.x; row < rows; row += gridDim.x)
		{
			const T *src = x + row * columns, *grad = dy + row * columns;
			T *dst = dx + row * columns;
			const float mean = statistics[2 * row], r = statistics[2 * row + 1];
			float sums[2] = { 0.0f, 0.0f };
			for (int j = threadIdx.x; j < columns; j += 256)
			{
				const float g = static_cast<float>(grad[j]) * (w != nullptr ? static_cast<float>(w[j]) : 1.0f);
				sums[0] += g;
				sums[1] = fmaf(g, (static_cast<float>(src[j]) - mean) * r, sums[1]);
			}
			row_sum(sums);
			const float mean_g = sums[0] * inv_columns, mean_gn = sums[1] * inv_columns;
			for (int j = threadIdx.x; j < columns; j += 256)
			{
				const float g = static_cast<float>(grad[j]) * (w != nullptr ? static_cast<float>(w[j]) : 1.0f);
				const float n = (static_cast<float>(src[j]) - mean) * r;
				float out = r * (g - mean_g - n * mean_gn);
				if (beta != 0.0f)
					out = fmaf(beta, static_cast<float>(dst[j]), out);
				dst[j] = static_cast<T>(out);
			}
		}
	}

	/* ------------------------------------------------------------------------------------------------------------------------ */
	struct RowForm
	{
			int vec, items, lanes;
	};
	/*
	 * How a row is spread: 16-byte vectors, as few threads as hold the row at 16 elements each. Rows shorter than a vector go element by element (at most 8 lanes of 16 are busy then).
	 */
	template<typename T>
	RowForm row_form(int columns)
	{
		const int widest = 16 / static_cast<int>(sizeof(T));
		if (columns < widest)
			return RowForm { 1, 1, 16 };
		for (int lanes : { 16, 32, 64, 256 })
			for (int items = 1; items * widest <= 16; items *= 2)
				/* one vector to a lane before more lanes; several only where a wavefront, or the workgroup, is not enough */
				if (columns <= lanes * widest * items && (items == 1 || lanes >= 64))
					return RowForm { widest, items, lanes };
		for (int items = 1; items * widest <= 16; items *= 2)
			if (columns <= 1024 * widest * items)
				return RowForm { widest, items, 1024 };
		return RowForm { 0, 0, 0 };
	}
	template<typename T, int VEC, int ITEMS, int LANES>
	void launch_forward_as(hipStream_t stream, const T *x, const T *w, const T *b, T *y, size_t rows, int columns, float epsilon)
	{
		constexpr int ROWS = threads_of<LANES>() / LANES;
		const size_t groups = (rows + ROWS - 1) / ROWS;
		const unsigned int grid = static_cast<unsigned int>(std::min<size_t>(groups, 8192));
		hipLaunchKernelGGL((kernel_layer_norm_forward<T, VEC, ITEMS, LANES>), dim3(grid), dim3(threads_of<LANES>()), 0, stream, x, y, rows, columns, epsilon, w, b);
	}
	template<typename T, int VEC, int ITEMS, int LANES>
	void launch_backward_as(hipStream_t stream, const T *x, const T *w, const T *dy, T *dx, size_t rows, int columns, float epsilon, float beta, float *partial, int parts)
	{
		hipLaunchKernelGGL((kernel_layer_norm_backward<T, VEC, ITEMS, LANES>), dim3(parts), dim3(threads_of<LANES>()), 0, stream, x, dy, dx, rows, columns, epsilon, beta, w, partial);
	}
	/* calls f(vec, items, lanes) with the form as compile-time constants */
	template<typename T, typename F>
	void with_form(const RowForm &form, F &&f)
	{
		constexpr int V = 16 / static_cast<int>(sizeof(T));
		typedef std::integral_constant<int, 1> one;
		typedef std::integral_constant<int, V> widest;
		const auto with_lanes = [&](auto vec, auto items)
		{
			if constexpr (decltype(items)::value == 1)
			{
				if (form.lanes == 16)
					return f(vec, items, std::integral_constant<int, 16>());
				if (form.lanes == 32)
					return f(vec, items, std::integral_constant<int, 32>());
			}
			if (form.lanes == 64)
				return f(vec, items, std::integral_constant<int, 64>());
			if (form.lanes == 256)
				return f(vec, items, std::integral_constant<int, 256>());
			return f(vec, items, std::integral_constant<int, 1024>());
		};
		if (form.vec == 1)
			f(one(), one(), std::integral_constant<int, 16>());
		else if (form.items == 1)
			with_lanes(widest(), one());
		else if (form.items == 2)
			with_lanes(widest(), std::integral_constant<int, 2>());
		else
		{
			if constexpr (V * 4 <= 16)
				with_lanes(widest(), std::integral_constant<int, 4>());
		}
	}
	template<typename T>
	int parts_of(size_t rows, int columns)
	{
		if (columns > LONGEST_IN_REGISTERS)
			return static_cast<int>(std::min<size_t>(rows, 64));
		const RowForm form = row_form<T>(columns);
		const int at_a_time = form.lanes <= 64 ? 256 / form.lanes : 1;
		return static_cast<int>(std::min<size_t>((rows + at_a_time - 1) / at_a_time, MAX_PARTS));
	}
	template<typename T>
	void layer_norm_forward(hipStream_t stream, const mlTensor_t &x, const mlTensor_t &w, const mlTensor_t &b, const mlTensor_t &y, float epsilon)
	{
		const int columns = last_dim(x);
		const size_t rows = volume(x) / columns;
		if (columns > LONGEST_IN_REGISTERS)
			hipLaunchKernelGGL((kernel_layer_norm_forward_long<T>), dim3(static_cast<unsigned int>(std::min<size_t>(rows, 2048))), dim3(256), 0, stream, ptr<T>(x), ptr<T>(y), rows, columns,
					epsilon, ptr<T>(w), ptr<T>(b));
		else
			with_form<T>(row_form<T>(columns), [&](auto vec, auto items, auto lanes)
			{
				launch_forward_as<T, decltype(vec)::value, decltype(items)::value, decltype(lanes)::value>(stream, ptr<T>(x), ptr<T>(w), ptr<T>(b), ptr<T>(y), rows, columns, epsilon);
			});
		MLHIP_CHECK(hipGetLastError());
	}
	template<typename T>
	void layer_norm_backward(hipStream_t stream, const mlTensor_t &x, const mlTensor_t &w, const mlTensor_t &dy, float beta_dx, const mlTensor_t &dx, float beta_weights,
			const mlTensor_t &dw, const mlTensor_t &db, float *workspace, float epsilon)
	{
		const int columns = last_dim(x);
		const size_t rows = volume(x) / columns;
		const bool sums = dw.data != nullptr || db.data != nullptr;
		const int parts = parts_of<T>(rows, columns);
		float *partial = workspace;
		if (rows > 0 && columns > LONGEST_IN_REGISTERS)
		{
			float *statistics = workspace + static_cast<size_t>(parts) * 2 * columns;
			const unsigned int grid = static_cast<unsigned int>(std::min<size_t>(rows, 2048));
			hipLaunchKernelGGL((kernel_layer_norm_statistics_long<T>), dim3(grid), dim3(256), 0, stream, ptr<T>(x), rows, columns, epsilon, statistics);
			if (sums) /* before dx is written, which may be where dy or x is */
				hipLaunchKernelGGL((kernel_layer_norm_sums_long<T>), dim3(ceil_div(columns, 256), parts), dim3(256), 0, stream, ptr<T>(x), ptr<T>(dy), rows, columns, statistics, partial);
			if (dx.data != nullptr)
				hipLaunchKernelGGL((kernel_layer_norm_backward_long<T>), dim3(grid), dim3(256), 0, stream, ptr<T>(x), ptr<T>(dy), ptr<T>(dx), rows, columns, beta_dx, ptr<T>(w), statistics);
		}
		else if (rows > 0)
			with_form<T>(row_form<T>(columns), [&](auto vec, auto items, auto lanes)
			{
				launch_backward_as<T, decltype(vec)::value, decltype(items)::value, decltype(lanes)::value>(stream, ptr<T>(x), ptr<T>(w), ptr<T>(dy), ptr<T>(dx), rows, columns, epsilon,
						beta_dx, sums ? partial : nullptr, parts);
			});
		MLHIP_CHECK(hipGetLastError());
		const size_t stride = 2 * static_cast<size_t>(columns);
		if (dw.data != nullptr && db.data != nullptr && dw.dtype == db.dtype)
			launch_sum_partials(stream, partial, parts, stride, dw.data, dw.dtype, columns, beta_weights, nullptr, db.data);
		else
		{
			if (dw.data != nullptr)
				launch_sum_partials(stream, partial, parts, stride, dw.data, dw.dtype, columns, beta_weights);
			if (db.data != nullptr)
				launch_sum_partials(stream, partial + columns, parts, stride, db.data, db.dtype, columns, beta_weights);
		}
	}

	bool same_shape(const mlTensor_t &a, const mlTensor_t &b)
	{
		if (a.rank != b.rank)
			return false;
		for (int i = 0; i < a.rank; i++)
			if (a.dim[i] != b.dim[i])
				return false;
		return true;
	}
	void require_rows(const mlTensor_t &x, const char *name)
	{
		MLHIP_REQUIRE(x.rank >= 1 && x.rank <= 6, std::string(name) + ": the input needs one to six dimensions");
		for (int i = 0; i < x.rank; i++)
			MLHIP_REQUIRE(x.dim[i] >= 0, std::string(name) + ": negative dimension");
		MLHIP_REQUIRE(last_dim(x) <= LONGEST_ROW, std::string(name) + ": rows are too long");
		MLHIP_REQUIRE(x.dtype == DTYPE_FLOAT16 || x.dtype == DTYPE_FLOAT32, std::string(name) + ": unsupported data type");
	}
	void require_weight(const mlTensor_t &t, const mlTensor_t &x, bool may_be_fp32, const char *what)
	{
		if (t.data == nullptr)
			return;
		MLHIP_REQUIRE(volume(t) == static_cast<size_t>(last_dim(x)), std::string(what) + " must have one element per column");
		MLHIP_REQUIRE(t.dtype == x.dtype || (may_be_fp32 && t.dtype == DTYPE_FLOAT32), std::string(what) + ": wrong data type");
	}
}

extern "C"
{
	using namespace mlhip;

	void hip_layer_norm_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t b, mlTensor_t y, float epsilon)
	try
	{
		require_rows(x, "layer_norm_forward");
		MLHIP_REQUIRE(same_shape(x, y) && x.dtype == y.dtype, "layer_norm_forward: input and output must have one shape and type");
		require_weight(w, x, false, "layer_norm_forward: weights");
		require_weight(b, x, false, "layer_norm_forward: bias");
		MLHIP_REQUIRE(epsilon >= 0.0f, "layer_norm_forward: epsilon must not be negative");
		if (volume(x) == 0)
			return;
		MLHIP_REQUIRE(x.data != nullptr && y.data != nullptr, "layer_norm_forward: null pointer");
		require_apart( { y }, { w, b }, "layer_norm_forward", { x });
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			layer_norm_forward<half_t>(on.stream, x, w, b, y, epsilon);
		else
			layer_norm_forward<float>(on.stream, x, w, b, y, epsilon);
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}

	size_t hip_layer_norm_get_workspace_size(mlShape_t shape, mlDataType_t dtype)
	try
	{
		mlTensor_t x = make_tensor(nullptr, dtype, shape);
		require_rows(x, "layer_norm_get_workspace_size");
		if (volume(x) == 0)
			return 0;
		const int columns = last_dim(x);
		const size_t rows = volume(x) / columns;
		const size_t parts = (dtype == DTYPE_FLOAT16) ? parts_of<half_t>(rows, columns) : parts_of<float>(rows, columns);
		return sizeof(float) * (parts * 2 * columns + (columns > LONGEST_IN_REGISTERS ? 2 * rows : 0));
	}
	catch (...)
	{
		return mlhip::entry_failed<size_t>();
	}

	void hip_layer_norm_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t dy, float beta_dx, mlTensor_t dx, float beta_weights, mlTensor_t dw,
			mlTensor_t db, void *workspace, size_t workspace_size, float epsilon)
	try
	{
		require_rows(x, "layer_norm_backward");
		MLHIP_REQUIRE(same_shape(x, dy) && x.dtype == dy.dtype, "layer_norm_backward: input and gradient must have one shape and type");
		MLHIP_REQUIRE(dx.data == nullptr || (same_shape(x, dx) && x.dtype == dx.dtype), "layer_norm_backward: dx must have the input's shape and type");
		require_weight(w, x, false, "layer_norm_backward: weights");
		require_weight(dw, x, true, "layer_norm_backward: gradient of the weights");
		require_weight(db, x, true, "layer_norm_backward: gradient of the bias");
		MLHIP_REQUIRE(epsilon >= 0.0f, "layer_norm_backward: epsilon must not be negative");
		if (last_dim(x) == 0 || (dx.data == nullptr && dw.data == nullptr && db.data == nullptr))
			return;
		if (volume(x) > 0)
		{
			MLHIP_REQUIRE(x.data != nullptr && dy.data != nullptr, "layer_norm_backward: null pointer");
			mlhip::NestedEntryCalls nested;
			MLHIP_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_size >= hip_layer_norm_get_workspace_size(shape_of(x), x.dtype),
					"layer_norm_backward: the workspace is too small or not aligned to 16 bytes");
		}
		require_apart( { dx, dw, db, Extent(workspace, workspace_size) }, { w }, "layer_norm_backward", { x, dy });
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			layer_norm_backward<half_t>(on.stream, x, w, dy, beta_dx, dx, beta_weights, dw, db, reinterpret_cast<float*>(workspace), epsilon);
		else
			layer_norm_backward<float>(on.stream, x, w, dy, beta_dx, dx, beta_weights, dw, db, reinterpret_cast<float*>(workspace), epsilon);
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}

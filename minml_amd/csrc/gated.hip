/*
 * gated.hip — the gated dense layer of a transformer's feed-forward half, and its backward pass.
 *
 *   g = x Wg^T + bg,  u = x Wu^T + bu,  y = a(g) u           a: sigmoid, relu, silu (g sigmoid(g)), gelu (g P(g), P the normal distribution)
 *   dg = dy u a'(g),  du = dy a(g),  d = [dg | du]
 *   dx = d W,  dW = d^T x,  db = sum_rows d                   W = [Wg; Wu], stored as [2, hidden, features]
 *
 * Forward: one launch. A tile's columns are half gate, half up of the same hidden units, so the epilogue has both projections of an element and neither goes to memory, unless the backward pass is to have
 * them (`projections`, in the tensors' type). The weights of few rows are streamed past them (few_rows.hpp). Where there are too few tiles for the chip the product is split along the
 * features, and the launch that adds the parts up applies the gate.
 * Backward: one pass over dy and the projections makes d and the partial sums of db (bound by memory), then two products (bound by the matrix cores). The matrix cores take operands of the tensors' type, so d is stored
 * in it, in fp16 scaled where it would leave the type's range (shift_of). Its rounding, half a step per element, adds as much to dx and dW as their own rounding does (2.9e-4 off instead of 2.1e-4; dx of few
 * rows 2.1e-4: keeps_low_part); keeping all of d would double both products. db is summed before the rounding.
 * fp16: 1 row of 4096 -> 8192 23.5 us (5.7 TB/s); 57600 x 256 -> 1024 with gelu, bias and the projections kept 133 us (2.9 TB/s, matrix cores 20 % busy: four chunks of k make a tile mostly beginning and end);
 * backward of 8192 x 2048 -> 5504 713 us (1.04 PFLOP/s): d 79 us (5.8 TB/s), 4 to see that it needs no scale, dx 300 us (1.23 PFLOP/s), dW 335 us.
 */
#include "few_rows.hpp"
#include "product_tiles.hpp"

#include <limits>

namespace
{
	using namespace mlhip;

	/*
	 * sigmoid(g), and sigmoid(-g) = 1 - sigmoid(g), of one exponential that does not overflow and without the difference, in which the slope of the sigmoid's right half would lose its digits (all of them from g = 17 on).
	 * exp and 1 / x for gates whose results are rounded to fp16 are the hardware's own, 2^-21 off at most for |x| < 8, where 2^-11 is rounded away; fp32 takes the library's.
	 */
	struct Sigmoid
	{
			float value, complement;
	};
	template<typename T>
	__device__ __forceinline__ Sigmoid sigmoid_of(float g)
	{
		float e, larger;
		if constexpr (sizeof(T) == 2)
		{
			e = __expf(-fabsf(g));
			larger = __builtin_amdgcn_rcpf(1.0f + e);
		}
		else
		{
			e = expf(-fabsf(g));
			larger = 1.0f / (1.0f + e);
		}
		const float smaller = e * larger;
		return g >= 0.0f ? Sigmoid { larger, smaller } : Sigmoid { smaller, larger };
	}
	/*
	 * The normal distribution's integral up to -|g|, 0.5 erfc(z) with z = |g| / sqrt 2. For fp16 0.5 erfc(z) exp(z^2) is t times a polynomial of degree 5 in t = 1 / (1 + 0.43 z), the form of Hastings' approximations of the error
	 * function, with coefficients of the smallest largest relative error over z = 0 .. 7, 2.5e-6 (a linear program over a grid of z gives them): the tail, where gelu is small, is as exact as the rest, with a dozen instructions
	 * instead of the 60 of the library's erfc, which fp32 takes.
	 */
	template<typename T>
	__device__ __forceinline__ float normal_tail(float g)
	{
		if constexpr (sizeof(T) == 2)
		{
			const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.43f * 0.70710678118654752f, 1.0f));
			float poly = fmaf(t, -0.078892514f, 0.21006414f);
			poly = fmaf(t, poly, -0.012823527f);
			poly = fmaf(t, poly, 0.14469013f);
			poly = fmaf(t, poly, 0.11523368f);
			poly = fmaf(t, poly, 0.12172684f);
			return t * poly * __builtin_amdgcn_exp2f(g * g * -0.72134752044448170f); /* exp(-g^2 / 2) */
		}
		else
			return 0.5f * erfcf(fabsf(g) * 0.70710678118654752f);
	}
	/* a(g) and, if asked, its derivative */
	template<typename T, bool SLOPE>
	__device__ __forceinline__ void gate_of(int gate, float g, float &a, float &slope)
	{
		switch (gate)
		{
			case GATE_SIGMOID:
			{
				const Sigmoid s = sigmoid_of<T>(g);
				a = s.value;
				if (SLOPE)
					slope = s.value * s.complement;
				break;
			}
			case GATE_RELU:
				a = (g > 0.0f || g != g) ? g : 0.0f; /* NaN stays */
				if (SLOPE)
					slope = g > 0.0f ? 1.0f : 0.0f;
				break;
			case GATE_SILU:
			{
				const Sigmoid s = sigmoid_of<T>(g);
				a = g * s.value;
				if (SLOPE)
					slope = s.value * fmaf(g, s.complement, 1.0f);
				break;
			}
			default: /* GATE_GELU */
			{
				const float tail = normal_tail<T>(g);
				a = fmaf(-fminf(fabsf(g), 3.0e38f), tail, fmaxf(g, 0.0f)); /* g P(g) for either sign, +inf for +inf */
				if (SLOPE)
					slope = fmaf(g * 0.39894228040143268f, (sizeof(T) == 2) ? __expf(-0.5f * g * g) : expf(-0.5f * g * g), g < 0.0f ? tail : 1.0f - tail);
				break;
			}
		}
	}

	/* ---- forward ------------------------------------------------------------------------------------------------------------ */
	template<typename T>
	struct GatedEpilogue
	{
			T *y, *projections;
			const T *bias;
			int hidden, gate;

			template<int BM, int BN>
			static constexpr int lds()
			{
				return Stage<T, BN / 2>::bytes(sizeof(T) == 2 ? BM : std::min(BM, PANEL));
			}
			/*
			 * The gate is applied in registers (blocks (i, 0) and (i, 1) hold both projections of an element). The results leave one after the other through the same place in LDS: y, then both projections
			 * where they are kept.
			 */
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				constexpr int ROWS = (sizeof(T) == 2) ? BM : std::min(BM, PANEL), PASSES = BM / ROWS, BLOCKS = TilePlace<BM, BN>::BLOCKS / PASSES;
				const Stage<T, BN / 2> stage { reinterpret_cast<T*>(lds) };
				const int n0 = at.tile_n * (BN / 2);
				float shift[2][16];
#pragma unroll
				for (int j = 0; j < 2; j++)
					load_lane_bias(shift[j], bias != nullptr ? bias + j * hidden : nullptr, n0 + at.wave_n * 32, hidden);
				static_for<PASSES>([&](auto pass)
				{
					constexpr int first = decltype(pass)::value * BLOCKS;
					const int m0 = at.tile_m * BM + decltype(pass)::value * ROWS;
					const auto put = [&](auto value) __attribute__((always_inline))
					{
						__syncthreads();
#pragma unroll
						for (int i = first; i < first + BLOCKS; i++)
#pragma unroll
							for (int q = 0; q < 4; q++)
								stage.put(at.row(i) - decltype(pass)::value * ROWS, at.wave_n * 32 + at.lane_column(q), value(i, 4 * q), value(i, 4 * q + 1), value(i, 4 * q + 2), value(i, 4 * q + 3));
						__syncthreads();
					};
					const auto projection = [&](int i, int j, int r) __attribute__((always_inline))
					{
						return acc[i][j][r] + shift[j][r];
					};
					const auto gated = [&](auto kind) __attribute__((always_inline))
					{
						put([&](int i, int r) __attribute__((always_inline))
						{
							float a, unused;
							gate_of<T, false>(decltype(kind)::value, projection(i, 0, r), a, unused);
							return a * projection(i, 1, r);
						});
					};
					switch (gate) /* once per tile, not once per element */
					{
						case GATE_SIGMOID:
							gated(std::integral_constant<int, GATE_SIGMOID>());
							break;
						case GATE_RELU:
							gated(std::integral_constant<int, GATE_RELU>());
							break;
						case GATE_SILU:
							gated(std::integral_constant<int, GATE_SILU>());
							break;
						default:
							gated(std::integral_constant<int, GATE_GELU>());
							break;
					}
					stage.template copy<ROWS, TilePlace<BM, BN>::THREADS>(y, hidden, m0, rows, n0, hidden);
					if (projections != nullptr)
						static_for<2>([&](auto matrix)
						{
							put([&](int i, int r) __attribute__((always_inline))
							{
								return projection(i, decltype(matrix)::value, r);
							});
							stage.template copy<ROWS, TilePlace<BM, BN>::THREADS>(projections + decltype(matrix)::value * hidden, 2 * static_cast<size_t>(hidden), m0, rows, n0, hidden);
						});
				});
			}
	};
	/* the sums of a split product: [part][row][2][hidden] */
	struct GatedPartEpilogue
	{
			float *partial;
			size_t part_stride;
			int hidden;

			template<int BM, int BN>
			static constexpr int lds()
			{
				return Stage<float, BN / 2>::bytes(std::min(BM, PANEL));
			}
			template<int BM, int BN, typename Acc>
			__device__ __forceinline__ void tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const TilePlace<BM, BN> &at, uint8_t *lds, int rows) const
			{
				constexpr int ROWS = std::min(BM, PANEL), BLOCKS = ROWS / 64;
				const Stage<float, BN / 2> stage { reinterpret_cast<float*>(lds) };
				static_for<BM / ROWS>([&](auto half)
				{
					static_for<2>([&](auto matrix)
					{
						constexpr int h = decltype(half)::value, j = decltype(matrix)::value;
						__syncthreads();
#pragma unroll
						for (int i = h * BLOCKS; i < (h + 1) * BLOCKS; i++)
#pragma unroll
							for (int q = 0; q < 4; q++)
								stage.put(at.row(i) - h * ROWS, at.wave_n * 32 + at.lane_column(q), acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
						__syncthreads();
						stage.template copy<ROWS, TilePlace<BM, BN>::THREADS>(partial + at.part * part_stride + j * hidden, 2 * static_cast<size_t>(hidden), at.tile_m * BM + h * ROWS, rows,
								at.tile_n * (BN / 2), hidden);
					});
				});
			}
	};
	template<typename T>
	__device__ __forceinline__ void finish_element(float g, float u, size_t row, int n, const T *bias, T *y, T *projections, int hidden, int gate)
	{
		if (bias != nullptr)
		{
			g += static_cast<float>(bias[n]);
			u += static_cast<float>(bias[hidden + n]);
		}
		float a, unused;
		gate_of<T, false>(gate, g, a, unused);
		y[row * hidden + n] = static_cast<T>(a * u);
		if (projections != nullptr)
		{
			projections[row * 2 * hidden + n] = static_cast<T>(g);
			projections[(row * 2 + 1) * hidden + n] = static_cast<T>(u);
		}
	}
	template<typename T>
	__global__ __launch_bounds__(256) void kernel_gate_parts(const float *partial, int parts, size_t part_stride, int rows, int hidden, const T *bias, T *y, T *projections, int gate)
	{
		const size_t count = static_cast<size_t>(rows) * hidden;
		for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<size_t>(gridDim.x) * 256)
		{
			int n;
			const size_t row = split_index(i, hidden, n);
			float g = 0.0f, u = 0.0f;
			for (int p = 0; p < parts; p++)
			{
				const float *src = partial + p * part_stride + row * 2 * hidden + n;
				g += src[0];
				u += src[hidden];
			}
			finish_element(g, u, row, n, bias, y, projections, hidden, gate);
		}
	}
	template<typename T, int MB, bool STREAM>
	__global__ __launch_bounds__(256) void kernel_gated_few_rows(const T *x, const T *w, T *y, int rows, int hidden, int features, const T *bias, T *projections, int gate)
	{
		extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
		const int n0 = blockIdx.x * 16, last = min(15, hidden - 1 - n0);
		const T *first = w + static_cast<size_t>(n0) * features, *second = w + (static_cast<size_t>(hidden) + n0) * features;
		float (*sums)[2][16 * MB][16] = reinterpret_cast<float (*)[2][16 * MB][16]>(lds);
		if constexpr (STREAM)
			few_rows_stream<T, MB>(x, rows, first, second, last, last, features, lds);
		else
			few_rows_sums<T, MB>(x, rows, first, second, last, last, features, sums);
		for (int i = threadIdx.x; i < 16 * MB * 16; i += 256)
		{
			const int row = i >> 4, n = i & 15;
			if (row < rows && n <= last)
				finish_element(sums[0][0][row][n], sums[0][1][row][n], row, n0 + n, bias, y, projections, hidden, gate);
		}
	}

	/* ---- backward: d and the sums of its columns ------------------------------------------------------------------------------ */
	/*
	 * Whether what fp16 leaves of d is kept beside it, as more rows of d, and multiplied with the weights like them. dx is 2.1e-4 off then (in norm, against 64 bits), which its own rounding costs; else 2.9e-4, two roundings:
	 * a relative error of every term is the same error of their sum, however many terms it has. This is a matter of cost alone. Up to 64 rows both parts lie in the 128 rows of one tile and the weights are read once; further
	 * on dx takes another product. us without / with, 2048 -> 5504: 1 row 40 / 43, 64 rows 45 / 52; 65 rows 47 / 57, 256 rows 65 / 85, 2048 rows 287 / 309, 8192 rows 732 / 1101. dw, a sum over the rows, would need x
	 * twice, and has two roundings for any number of rows.
	 */
	bool keeps_low_part(int rows, int element_size)
	{
		return element_size == 2 && rows <= 64;
	}
	/* what rounding x to the type leaves; nothing of what is infinite there, so that infinities stay what they are (inf - inf is no number) */
	template<typename T>
	__device__ __forceinline__ float low_part(float x)
	{
		const float high = static_cast<float>(static_cast<T>(x));
		return fabsf(high) <= std::numeric_limits<float>::max() ? x - high : 0.0f;
	}
	/*
	 * d is in memory as d 2^shift. In fp16 dy u a'(g) may pass the type's largest value, 65504, where dx, a sum of such terms with weights, does not; and gradients of losses that nobody scaled, 1e-5 or so, are subnormal
	 * there (dw 2.8e-3 off instead of 3e-4, also where it is asked for in fp32). With its largest element between 2^-3 and 2^15 d stays as it is: elements down to 2^-11 of the largest are normal numbers then, and
	 * those below are off by at most 2^-22 of it. Else the largest is brought just below 2^15, and what the products give is scaled back in fp32, exactly.
	 */
	__device__ __forceinline__ int shift_of(float top)
	{
		const int exponent = scale_exponent(top);
		return (top == 0.0f || (exponent >= -2 && exponent <= SCALE_BITS)) ? 0 : SCALE_BITS - exponent;
	}
	/*
	 * d [rows][row_elements] holds dg at column n and du at column hidden + n, zeros from 2 hidden on. A workgroup has 256 hidden units (32 threads of 8) and 8 rows at a time of its share of the rows;
	 * partial [gridDim.y][2 hidden] takes the sums over its rows. What rounding leaves goes `low` elements further, if that is not 0.
	 * Scaling takes two launches, because only the first one finds out what the largest element is: it leaves that of every workgroup in `largest` (fp16; null: no one asks). The second one (AGAIN) reads the `groups` of them,
	 * writes `back` = 2^-shift, and is done if there is nothing to scale, as is usual (3 us); else it makes d once more, as many bytes as the first time.
	 */
	template<typename T, bool AGAIN>
	__global__ __launch_bounds__(256) void kernel_gated_gradient(const T *projections, const T *dy, T *d, int rows, int hidden, int row_elements, int gate, float *partial, size_t low, float *largest,
			int groups, float *back)
	{
		__shared__ float sums[AGAIN ? 1 : 2][8][32 * 8 + 8];
		__shared__ float waves[4];
		/* of the workgroup's threads */
		const auto largest_of = [&](float v) __attribute__((always_inline))
		{
#pragma unroll
			for (int offset = 32; offset >= 1; offset >>= 1)
				v = fmaxf(v, __shfl_xor(v, offset));
			if ((threadIdx.x & 63) == 0)
				waves[threadIdx.x >> 6] = v;
			__syncthreads();
			return fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
		};
		float top = 0.0f, factor = 1.0f;
		if constexpr (AGAIN)
		{
			for (int i = threadIdx.x; i < groups; i += 256)
				top = fmaxf(top, largest[i]);
			const int shift = shift_of(largest_of(top));
			if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
				*back = ldexpf(1.0f, -shift);
			if (shift == 0)
				return;
			factor = ldexpf(1.0f, shift);
		}
		const int group = threadIdx.x & 31, first_row = threadIdx.x >> 5;
		const int n = blockIdx.x * 256 + group * 8;
		float sum[2][8];
#pragma unroll
		for (int i = 0; i < 2; i++)
#pragma unroll
			for (int e = 0; e < 8; e++)
				sum[i][e] = 0.0f;
		const auto gradient = [&](int e, float g, float u, float v, float &dg, float &du) __attribute__((always_inline))
		{
			float a, slope;
			gate_of<T, true>(gate, g, a, slope);
			dg = v * u * slope;
			du = v * a;
			if constexpr (AGAIN)
			{
				dg *= factor;
				du *= factor;
			}
			else
			{
				sum[0][e] += dg;
				sum[1][e] += du;
				if constexpr (sizeof(T) == 2)
					top = larger_finite(larger_finite(top, dg), du);
			}
		};
		for (int row = blockIdx.y * 8 + first_row; row < rows; row += gridDim.y * 8)
		{
			const T *kept = projections + static_cast<size_t>(row) * 2 * hidden + n;
			const T *grad = dy + static_cast<size_t>(row) * hidden + n;
			T *dst = d + static_cast<size_t>(row) * row_elements + n;
			const int there = min(hidden - n, 8);
			if (there == 8)
			{
				Elements<T, 8> g, u, v;
				g.load(kept);
				u.load(kept + hidden);
				v.load(grad);
				float dg[8], du[8];
#pragma unroll
				for (int e = 0; e < 8; e++)
					gradient(e, g[e], u[e], v[e], dg[e], du[e]);
				store_nearest<8>(dst, dg);
				store_nearest<8>(dst + hidden, du);
				if (low != 0)
				{
#pragma unroll
					for (int e = 0; e < 8; e++)
					{
						dg[e] = low_part<T>(dg[e]);
						du[e] = low_part<T>(du[e]);
					}
					store_nearest<8>(dst + low, dg);
					store_nearest<8>(dst + low + hidden, du);
				}
			}
			else
			{
#pragma unroll
				for (int e = 0; e < 8; e++)
					if (e < there)
					{
						float dg, du;
						gradient(e, static_cast<float>(kept[e]), static_cast<float>(kept[hidden + e]), static_cast<float>(grad[e]), dg, du);
						dst[e] = static_cast<T>(dg);
						dst[hidden + e] = static_cast<T>(du);
						if (low != 0)
						{
							dst[low + e] = static_cast<T>(low_part<T>(dg));
							dst[low + hidden + e] = static_cast<T>(low_part<T>(du));
						}
					}
			}
			if (n == 0)
				for (int j = 2 * hidden; j < row_elements; j++)
				{
					d[static_cast<size_t>(row) * row_elements + j] = static_cast<T>(0.0f);
					d[static_cast<size_t>(row) * row_elements + low + j] = static_cast<T>(0.0f);
				}
		}
		if constexpr (!AGAIN)
		{
			if (sizeof(T) == 2 && largest != nullptr)
			{
				const float of_all = largest_of(top);
				if (threadIdx.x == 0)
					largest[blockIdx.y * gridDim.x + blockIdx.x] = of_all;
			}
			if (partial == nullptr)
				return;
#pragma unroll
			for (int i = 0; i < 2; i++)
#pragma unroll
				for (int e = 0; e < 8; e++)
					sums[i][first_row][group * 8 + e] = sum[i][e];
			__syncthreads();
			const int column = blockIdx.x * 256 + threadIdx.x;
			if (column < hidden)
#pragma unroll
				for (int i = 0; i < 2; i++)
				{
					float total = 0.0f;
#pragma unroll
					for (int r = 0; r < 8; r++)
						total += sums[i][r][threadIdx.x];
					partial[static_cast<size_t>(blockIdx.y) * 2 * hidden + i * hidden + column] = total;
				}
		}
	}

	/* ---- sizes ---------------------------------------------------------------------------------------------------------------- */
	struct GatedShape
	{
			int rows, features, hidden, element_size;
			mlDataType_t dtype;
	};
	GatedShape gated_shape(const mlShape_t &x, const mlShape_t &w, mlDataType_t dtype, const char *name)
	{
		const std::string who(name);
		MLHIP_REQUIRE(dtype == DTYPE_FLOAT16 || dtype == DTYPE_FLOAT32, who + ": unsupported data type");
		MLHIP_REQUIRE(x.rank >= 1 && x.rank <= 6 && w.rank == 3 && w.dim[0] == 2, who + ": the input needs one to six dimensions, the weights must be [2, hidden, features]");
		for (int i = 0; i < x.rank; i++)
			MLHIP_REQUIRE(x.dim[i] >= 0, who + ": negative dimension");
		MLHIP_REQUIRE(w.dim[1] >= 0 && w.dim[2] >= 0 && w.dim[2] == last_dim(x), who + ": the weights' last dimension must be the input's");
		MLHIP_REQUIRE(w.dim[2] > 0, who + ": no features");
		const size_t rows = volume(x) / w.dim[2];
		MLHIP_REQUIRE(rows <= 0x3fffffff && w.dim[1] <= (1 << 18) && w.dim[2] <= (1 << 18) && static_cast<size_t>(w.dim[1]) * w.dim[2] * size_of(dtype) <= (size_t(1) << 30),
				who + ": too many rows, hidden units or features");
		return GatedShape { static_cast<int>(rows), w.dim[2], w.dim[1], size_of(dtype), dtype };
	}
	bool few_rows(const GatedShape &s)
	{
		return takes_few_rows(s.rows, 2 * static_cast<size_t>(s.hidden) * s.features * s.element_size);
	}
	int gradient_parts(const GatedShape &s)
	{
		/* about 8 workgroups of 256 threads per compute unit */
		return std::max(1, std::min(ceil_div(s.rows, 8), 2048 / std::max(1, ceil_div(s.hidden, 256))));
	}
	int gradient_groups(const GatedShape &s)
	{
		return ceil_div(s.hidden, 256) * gradient_parts(s);
	}
	ProductPlan forward_plan(const GatedShape &s)
	{
		return plan_product(s.rows, s.hidden, true, s.features, s.element_size, true);
	}
	TwoPlans input_plan(const GatedShape &s)
	{
		return plan_in_turns(s.rows, s.features, 2 * s.hidden, s.element_size, true);
	}
	/* of d with its low part */
	ProductPlan split_input_plan(const GatedShape &s)
	{
		return plan_product(2 * s.rows, s.features, false, 2 * s.hidden, s.element_size, true);
	}
	TwoPlans weights_plan(const GatedShape &s)
	{
		return plan_in_turns(2 * s.hidden, s.features, s.rows, s.element_size, false);
	}
	/* the pieces of a workspace, each aligned to 256 bytes */
	struct GatedSpace
	{
			size_t x, w, parts, d, sums, largest, total;
	};
	GatedSpace gated_space(const GatedShape &s, bool backward)
	{
		GatedSpace space;
		size_t at = 0;
		const auto take = [&](size_t bytes)
		{
			const size_t begin = at;
			at += round_up(bytes, 256);
			return begin;
		};
		const int pieces = 16 / s.element_size;
		const size_t padded = (s.features % pieces == 0) ? 0 : round_up(s.features, pieces) * s.element_size;
		const bool tiles = backward || !few_rows(s);
		space.x = take(tiles ? padded * s.rows : 0);
		space.w = take(tiles ? padded * 2 * s.hidden : 0);
		if (backward)
		{
			const bool low = keeps_low_part(s.rows, s.element_size);
			const size_t for_input = low ? sizeof(float) * split_input_plan(s).parts * 2 * s.rows * s.features : part_bytes(input_plan(s), s.rows, s.features);
			space.parts = take(std::max(for_input, part_bytes(weights_plan(s), 2 * s.hidden, s.features)));
			space.d = take(round_up(2 * s.hidden, pieces) * s.element_size * s.rows * (low ? 2 : 1));
			space.sums = take(sizeof(float) * 2 * s.hidden * gradient_parts(s));
			space.largest = take(s.element_size == 2 ? sizeof(float) * (gradient_groups(s) + 1) : 0);
		}
		else
		{
			space.parts = take(tiles ? part_bytes(forward_plan(s), s.rows, 2 * s.hidden) : 0);
			space.d = space.sums = space.largest = at;
		}
		space.total = at;
		return space;
	}

	template<typename T>
	void gated_forward(hipStream_t stream, const GatedShape &s, const T *x, const T *w, const T *bias, T *y, T *projections, int gate, uint8_t *workspace)
	{
		if (few_rows(s))
		{
			with_few_rows<T>(s.rows, s.features, [&](auto blocks, auto streamed)
			{
				constexpr int MB = decltype(blocks)::value, bytes = few_rows_lds<MB>(decltype(streamed)::value);
				auto kernel = kernel_gated_few_rows<T, MB, decltype(streamed)::value>;
				ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
				hipLaunchKernelGGL(kernel, dim3(ceil_div(s.hidden, 16)), dim3(256), bytes, stream, x, w, y, s.rows, s.hidden, s.features, bias, projections, gate);
			});
			MLHIP_CHECK(hipGetLastError());
			return;
		}
		const GatedSpace space = gated_space(s, false);
		const size_t row_bytes = static_cast<size_t>(padded_columns<T>(s.features)) * sizeof(T);
		x = pad_rows(stream, x, reinterpret_cast<T*>(workspace + space.x), s.rows, s.features);
		w = pad_rows(stream, w, reinterpret_cast<T*>(workspace + space.w), 2 * static_cast<size_t>(s.hidden), s.features);
		const Operand a { reinterpret_cast<const uint8_t*>(x), row_bytes, s.rows, padded_columns<T>(s.features) };
		const Operand b { reinterpret_cast<const uint8_t*>(w), row_bytes, s.hidden, padded_columns<T>(s.features), row_bytes * s.hidden };
		const ProductPlan plan = forward_plan(s);
		if (plan.parts == 1)
			launch_product<T, Side::ROWS, Side::ROWS, true>(stream, plan, a, b, s.rows, GatedEpilogue<T> { y, projections, bias, s.hidden, gate });
		else
		{
			float *partial = reinterpret_cast<float*>(workspace + space.parts);
			const size_t stride = static_cast<size_t>(s.rows) * 2 * s.hidden, count = static_cast<size_t>(s.rows) * s.hidden;
			launch_product<T, Side::ROWS, Side::ROWS, true>(stream, plan, a, b, s.rows, GatedPartEpilogue { partial, stride, s.hidden });
			hipLaunchKernelGGL((kernel_gate_parts<T>), dim3(static_cast<unsigned int>(std::min<size_t>((count + 255) / 256, 8192))), dim3(256), 0, stream, partial, plan.parts, stride, s.rows,
					s.hidden, bias, y, projections, gate);
			MLHIP_CHECK(hipGetLastError());
		}
	}
	template<typename T>
	void gated_backward(hipStream_t stream, const GatedShape &s, const T *x, const T *w, const T *projections, const T *dy, float beta_dx, T *dx, float beta_weights,
			const mlTensor_t &dw, const mlTensor_t &db, int gate, uint8_t *workspace)
	{
		const GatedSpace space = gated_space(s, true);
		const int both = 2 * s.hidden, row_elements = padded_columns<T>(both), padded = padded_columns<T>(s.features);
		T *d = reinterpret_cast<T*>(workspace + space.d);
		float *sums = reinterpret_cast<float*>(workspace + space.sums), *partial = reinterpret_cast<float*>(workspace + space.parts);
		const int parts = gradient_parts(s);
		const bool with_low = keeps_low_part(s.rows, s.element_size) && dx != nullptr;
		const size_t low = with_low ? static_cast<size_t>(s.rows) * row_elements : 0;
		float *back = nullptr; /* what takes d's scale back */
		if (s.rows > 0 && s.hidden > 0)
		{
			const dim3 grid(ceil_div(s.hidden, 256), parts);
			const int groups = gradient_groups(s);
			float *largest = reinterpret_cast<float*>(workspace + space.largest);
			const bool scaled = sizeof(T) == 2 && (dx != nullptr || dw.data != nullptr); /* else nothing reads d */
			hipLaunchKernelGGL((kernel_gated_gradient<T, false>), grid, dim3(256), 0, stream, projections, dy, d, s.rows, s.hidden, row_elements, gate, db.data != nullptr ? sums : nullptr, low,
					scaled ? largest : nullptr, groups, static_cast<float*>(nullptr));
			MLHIP_CHECK(hipGetLastError());
			if constexpr (sizeof(T) == 2)
				if (scaled)
				{
					back = largest + groups;
					hipLaunchKernelGGL((kernel_gated_gradient<T, true>), dim3(grid.x, ceil_div(parts, 2)), dim3(256), 0, stream, projections, dy, d, s.rows, s.hidden, row_elements, gate,
							static_cast<float*>(nullptr), low, largest, groups, back);
					MLHIP_CHECK(hipGetLastError());
				}
		}
		if (db.data != nullptr)
			launch_sum_partials(stream, sums, s.rows > 0 ? parts : 0, static_cast<size_t>(both), db.data, db.dtype, both, beta_weights);
		const Operand d_rows { reinterpret_cast<const uint8_t*>(d), row_elements * sizeof(T), with_low ? 2 * s.rows : s.rows, row_elements };
		if (dx != nullptr && s.rows > 0)
		{
			w = pad_rows(stream, w, reinterpret_cast<T*>(workspace + space.w), static_cast<size_t>(both), s.features);
			const Operand b { reinterpret_cast<const uint8_t*>(w), padded * sizeof(T), padded, both };
			if (with_low)
			{
				/* [part][d, its low part][rows][features]: twice as many parts to add up */
				const ProductPlan plan = split_input_plan(s);
				const size_t outputs = static_cast<size_t>(s.rows) * s.features;
				launch_product<T, Side::ROWS, Side::COLUMNS, false>(stream, plan, d_rows, b, 2 * s.rows, PartEpilogue { partial, 2 * outputs, s.features, false });
				launch_join_parts(stream, partial, 2 * plan.parts, outputs, dx, beta_dx, back);
			}
			else
				product_to<T, T, Side::ROWS, Side::COLUMNS>(stream, input_plan(s), d_rows, b, s.rows, s.features, dx, beta_dx, back, partial);
		}
		if (dw.data != nullptr)
		{
			x = pad_rows(stream, x, reinterpret_cast<T*>(workspace + space.x), s.rows, s.features);
			const Operand a { reinterpret_cast<const uint8_t*>(d), row_elements * sizeof(T), row_elements, s.rows };
			const Operand b { reinterpret_cast<const uint8_t*>(x), padded * sizeof(T), padded, s.rows };
			if (dw.dtype == DTYPE_FLOAT32)
				product_to<T, float, Side::COLUMNS, Side::COLUMNS>(stream, weights_plan(s), a, b, both, s.features, ptr<float>(dw), beta_weights, back, partial);
			else if constexpr (sizeof(T) == 2)
				product_to<T, T, Side::COLUMNS, Side::COLUMNS>(stream, weights_plan(s), a, b, both, s.features, ptr<T>(dw), beta_weights, back, partial);
		}
	}
	void require_like(const mlTensor_t &t, const mlTensor_t &x, int last, const char *what)
	{
		MLHIP_REQUIRE(t.dtype == x.dtype && t.rank == x.rank && last_dim(t) == last, std::string(what) + ": shape or type");
		for (int i = 0; i + 1 < x.rank; i++)
			MLHIP_REQUIRE(t.dim[i] == x.dim[i], std::string(what) + ": shape");
	}
	void require_workspace(const void *workspace, size_t given, size_t needed, const char *name)
	{
		MLHIP_REQUIRE(needed == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && given >= needed),
				std::string(name) + ": the workspace is too small or not aligned to 256 bytes");
	}
	bool aligned_16(const mlTensor_t &t)
	{
		return reinterpret_cast<uintptr_t>(t.data) % 16 == 0;
	}
}

extern "C"
{
	using namespace mlhip;

	size_t hip_gated_dense_get_workspace_size(mlShape_t input_shape, mlShape_t weights_shape, mlDataType_t dtype, bool backward)
	try
	{
		return gated_space(gated_shape(input_shape, weights_shape, dtype, "gated_dense_get_workspace_size"), backward).total;
	}
	catch (...)
	{
		return mlhip::entry_failed<size_t>();
	}

	void hip_gated_dense_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t b, mlTensor_t y, mlTensor_t projections, mlGate_t gate, void *workspace,
			size_t workspace_size)
	try
	{
		const char *name = "gated_dense_forward";
		const GatedShape s = gated_shape(shape_of(x), shape_of(w), x.dtype, name);
		MLHIP_REQUIRE(gate >= GATE_SIGMOID && gate <= GATE_GELU, "gated_dense_forward: unknown gate");
		MLHIP_REQUIRE(w.dtype == x.dtype, "gated_dense_forward: weights must have the input's type");
		MLHIP_REQUIRE(b.data == nullptr || (b.dtype == x.dtype && volume(b) == 2 * static_cast<size_t>(s.hidden)), "gated_dense_forward: the bias must be [2, hidden] of the input's type");
		require_like(y, x, s.hidden, "gated_dense_forward: output");
		MLHIP_REQUIRE(projections.data == nullptr || (projections.dtype == x.dtype && volume(projections) == 2 * static_cast<size_t>(s.hidden) * s.rows && last_dim(projections) == s.hidden),
				"gated_dense_forward: the projections must be [.., 2, hidden] of the input's type");
		if (s.rows == 0 || s.hidden == 0)
			return;
		MLHIP_REQUIRE(x.data != nullptr && w.data != nullptr && y.data != nullptr, "gated_dense_forward: null pointer");
		MLHIP_REQUIRE(aligned_16(x) && aligned_16(w), "gated_dense_forward: input and weights must be aligned to 16 bytes");
		require_workspace(workspace, workspace_size, gated_space(s, false).total, name);
		require_apart( { y, projections, Extent(workspace, workspace_size) }, { x, w, b }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			gated_forward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(b), ptr<half_t>(y), ptr<half_t>(projections), gate, reinterpret_cast<uint8_t*>(workspace));
		else
			gated_forward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(b), ptr<float>(y), ptr<float>(projections), gate, reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}

	void hip_gated_dense_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t projections, const mlTensor_t dy, float beta_dx, mlTensor_t dx,
			float beta_weights, mlTensor_t dw, mlTensor_t db, mlGate_t gate, void *workspace, size_t workspace_size)
	try
	{
		const char *name = "gated_dense_backward";
		const GatedShape s = gated_shape(shape_of(x), shape_of(w), x.dtype, name);
		MLHIP_REQUIRE(gate >= GATE_SIGMOID && gate <= GATE_GELU, "gated_dense_backward: unknown gate");
		MLHIP_REQUIRE(w.dtype == x.dtype, "gated_dense_backward: weights must have the input's type");
		require_like(dy, x, s.hidden, "gated_dense_backward: gradient");
		MLHIP_REQUIRE(projections.dtype == x.dtype && volume(projections) == 2 * static_cast<size_t>(s.hidden) * s.rows && (s.rows == 0 || last_dim(projections) == s.hidden),
				"gated_dense_backward: the projections must be [.., 2, hidden] of the input's type");
		if (dx.data != nullptr)
			require_like(dx, x, s.features, "gated_dense_backward: dx");
		const auto weight_type = [&](const mlTensor_t &t)
		{
			return t.dtype == x.dtype || t.dtype == DTYPE_FLOAT32;
		};
		MLHIP_REQUIRE(dw.data == nullptr || (weight_type(dw) && volume(dw) == volume(w)), "gated_dense_backward: dw must be [2, hidden, features] of the input's type or fp32");
		MLHIP_REQUIRE(db.data == nullptr || (weight_type(db) && volume(db) == 2 * static_cast<size_t>(s.hidden)), "gated_dense_backward: db must be [2, hidden] of the input's type or fp32");
		if (dx.data == nullptr && dw.data == nullptr && db.data == nullptr)
			return;
		if (s.hidden == 0 && (dx.data == nullptr || s.rows == 0))
			return;
		MLHIP_REQUIRE(s.hidden > 0, "gated_dense_backward: no hidden units");
		MLHIP_REQUIRE(s.rows == 0 || (x.data != nullptr && w.data != nullptr && projections.data != nullptr && dy.data != nullptr), "gated_dense_backward: null pointer");
		MLHIP_REQUIRE(aligned_16(x) && aligned_16(w), "gated_dense_backward: input and weights must be aligned to 16 bytes");
		require_workspace(workspace, workspace_size, gated_space(s, true).total, name);
		require_apart( { dx, dw, db, Extent(workspace, workspace_size) }, { x, w, projections, dy }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			gated_backward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(projections), ptr<half_t>(dy), beta_dx, ptr<half_t>(dx), beta_weights, dw, db, gate,
					reinterpret_cast<uint8_t*>(workspace));
		else
			gated_backward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(projections), ptr<float>(dy), beta_dx, ptr<float>(dx), beta_weights, dw, db, gate,
					reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}

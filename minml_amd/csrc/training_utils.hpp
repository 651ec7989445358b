/*
 * training_utils.hpp — what the operators with a backward pass share: element access for rows of any length and alignment, results rounded to nearest,
 * and the sums that become gradients of weights.
 *
 * These operators have no counterpart whose bits they reproduce, so fp16 results are rounded to nearest (half a step, 2^-11 of the value) and not towards
 * zero as the inference path does after the reference: a gradient that is rounded towards zero is too small in every element, and a training run adds that up.
 */
#ifndef MINML_AMD_TRAINING_UTILS_HPP_
#define MINML_AMD_TRAINING_UTILS_HPP_

#include "common.hpp"
#include "device_utils.hpp"

#include <initializer_list>
#include <limits>

namespace mlhip
{
	/* a call's device is its context's, whichever is current when it is made; the caller's comes back at its end */
	class OnDeviceOf
	{
			int before = 0, device;
		public:
			const hipStream_t stream;
			explicit OnDeviceOf(mlContext_t context) :
					device(get(context)->device_index),
					stream(stream_of(context))
			{
				MLHIP_CHECK(hipGetDevice(&before));
				if (before != device)
					MLHIP_CHECK(hipSetDevice(device));
			}
			~OnDeviceOf()
			{
				if (before != device)
					(void) hipSetDevice(before);
			}
			OnDeviceOf(const OnDeviceOf&) = delete;
			OnDeviceOf& operator=(const OnDeviceOf&) = delete;
	};
	/* memory that a call reads or writes */
	struct Extent
	{
			const uint8_t *begin;
			size_t bytes;

			Extent(const void *data, size_t size) :
					begin(static_cast<const uint8_t*>(data)),
					bytes(data == nullptr ? 0 : size)
			{
			}
			Extent(const mlTensor_t &t) :
					Extent(t.data, volume(t) * size_of(t.dtype))
			{
			}
			bool meets(const Extent &other) const
			{
				return bytes > 0 && other.bytes > 0 && begin < other.begin + other.bytes && other.begin < begin + bytes;
			}
	};
	/* results may lie over nothing else of the call; but the first one may be exactly one of the inputs that may be overwritten */
	inline void require_apart(std::initializer_list<Extent> results, std::initializer_list<Extent> inputs, const char *name, std::initializer_list<Extent> replaceable = { })
	{
		for (const Extent *r = results.begin(); r != results.end(); r++)
		{
			for (const Extent *other = results.begin(); other != r; other++)
				MLHIP_REQUIRE(!r->meets(*other), std::string(name) + ": results overlap");
			for (const Extent &input : inputs)
				MLHIP_REQUIRE(!r->meets(input), std::string(name) + ": a result overlaps an input");
			for (const Extent &input : replaceable)
				MLHIP_REQUIRE(!r->meets(input) || (r == results.begin() && r->begin == input.begin && r->bytes == input.bytes), std::string(name) + ": a result overlaps an input");
		}
	}

	/* VEC consecutive elements that need no more alignment than one of them: one memory instruction all the same (global memory takes any address) */
	template<typename T, int VEC>
	struct Elements
	{
			typedef T vec_t __attribute__((ext_vector_type(VEC)));
			typedef vec_t unaligned_t __attribute__((aligned(sizeof(T))));
			vec_t raw;

			__device__ __forceinline__ void load(const T *p)
			{
				raw = *reinterpret_cast<const unaligned_t*>(p);
			}
			__device__ __forceinline__ float operator[](int e) const
			{
				return static_cast<float>(raw[e]);
			}
	};
	template<typename T>
	struct Elements<T, 1>
	{
			T raw;

			__device__ __forceinline__ void load(const T *p)
			{
				raw = *p;
			}
			__device__ __forceinline__ float operator[](int) const
			{
				return static_cast<float>(raw);
			}
	};
	/* VEC results rounded to nearest; those before `skip` are left out (the first ones of the vector that ends a row, see RowPlace) */
	template<int VEC, typename T>
	__device__ __forceinline__ void store_nearest(T *p, const float (&v)[VEC], int skip = 0)
	{
		if (skip == 0)
		{
			if constexpr (VEC == 1)
				*p = static_cast<T>(v[0]);
			else
			{
				typename Elements<T, VEC>::vec_t tmp;
#pragma unroll
				for (int e = 0; e < VEC; e++)
					tmp[e] = static_cast<T>(v[e]);
				*reinterpret_cast<typename Elements<T, VEC>::unaligned_t*>(p) = tmp;
			}
		}
		else
		{
#pragma unroll
			for (int e = 0; e < VEC; e++)
				if (e >= skip)
					p[e] = static_cast<T>(v[e]);
		}
	}
	/*
	 * Where the vector that begins at column j of a row of `columns` (>= VEC) elements lies. The vector that would pass the row's end is moved back to end with it; its first `skip`
	 * elements belong to the vector before it and count for nothing here. So every load is a whole vector inside its row, for any length, and none stands under a test.
	 */
	struct RowPlace
	{
			int start, skip;

			/* a scalar base and 32 bits of offset where the row is the same for the whole wavefront (rows that go by RowPlace are below 2^31 bytes) */
			template<typename T>
			__device__ __forceinline__ T* in(T *row) const
			{
				typedef typename std::conditional<std::is_const<T>::value, const char, char>::type byte;
				return reinterpret_cast<T*>(reinterpret_cast<byte*>(row) + static_cast<uint32_t>(start) * static_cast<uint32_t>(sizeof(T)));
			}
	};
	template<int VEC>
	__device__ __forceinline__ RowPlace place_in_row(int j, int columns)
	{
		const int start = min(j, columns - VEC);
		return RowPlace { start, min(j - start, VEC) };
	}

	/* sum over the LANES (a power of two) neighbouring lanes that share a row; every lane gets it */
	template<int LANES>
	__device__ __forceinline__ float lanes_sum(float v)
	{
#pragma unroll
		for (int offset = LANES / 2; offset >= 1; offset >>= 1)
			v += __shfl_xor(v, offset);
		return v;
	}

	/*
	 * out[j] = scale * (sum over `parts` rows of partial[.][stride], column j) + beta * out[j]: the second half of every sum over rows. The first half leaves one row of sums per workgroup, here 8
	 * threads to a column add up every eighth of them and meet in LDS: a fixed order, so the same bits every time, which additions by atomic operations would not give.
	 */
	template<typename Out>
	__global__ __launch_bounds__(256) void kernel_sum_partials(const float *partial, int parts, size_t stride, Out *out, int columns, float beta, const float *scale, Out *second)
	{
		__shared__ float sums[8][33];
		if (blockIdx.y == 1) /* the columns behind the first ones, for another result */
		{
			partial += columns;
			out = second;
		}
		const int c = threadIdx.x & 31, group = threadIdx.x >> 5;
		const int j = blockIdx.x * 32 + c;
		float sum = 0.0f;
		if (j < columns)
		{
			const float *src = partial + j;
			int p = group;
			for (; p + 56 < parts; p += 64)
			{
				float v[8];
#pragma unroll
				for (int u = 0; u < 8; u++)
					v[u] = src[static_cast<size_t>(p + 8 * u) * stride];
#pragma unroll
				for (int u = 0; u < 8; u++)
					sum += v[u];
			}
			for (; p < parts; p += 8)
				sum += src[static_cast<size_t>(p) * stride];
		}
		sums[group][c] = sum;
		__syncthreads();
		if (group == 0 && j < columns)
		{
#pragma unroll
			for (int g = 1; g < 8; g++)
				sum += sums[g][c];
			if (scale != nullptr)
				sum *= *scale;
			out[j] = static_cast<Out>(beta != 0.0f ? fmaf(beta, static_cast<float>(out[j]), sum) : sum);
		}
	}
	/* out: the gradient of a weight, of the tensors' type or fp32. scale: on the device, or null for 1. second: null, or a result of the same type for the next `columns` columns */
	inline void launch_sum_partials(hipStream_t stream, const float *partial, int parts, size_t stride, void *out, mlDataType_t dtype, int columns, float beta,
			const float *scale = nullptr, void *second = nullptr)
	{
		if (columns == 0)
			return;
		const dim3 grid(ceil_div(columns, 32), second != nullptr ? 2 : 1);
		if (dtype == DTYPE_FLOAT16)
			hipLaunchKernelGGL((kernel_sum_partials<half_t>), grid, dim3(256), 0, stream, partial, parts, stride, reinterpret_cast<half_t*>(out), columns, beta, scale,
					reinterpret_cast<half_t*>(second));
		else
			hipLaunchKernelGGL((kernel_sum_partials<float>), grid, dim3(256), 0, stream, partial, parts, stride, reinterpret_cast<float*>(out), columns, beta, scale,
					reinterpret_cast<float*>(second));
		MLHIP_CHECK(hipGetLastError());
	}
	constexpr int SCALE_BITS = 15; /* a gradient that is scaled has its largest element just below 2^15: fp16 ends at 2^16 */
	/* the exponent of the power of two above the largest element */
	__device__ __forceinline__ int scale_exponent(float top)
	{
		int exponent = 0;
		if (top > 0.0f)
			(void) frexpf(top, &exponent);
		return max(exponent, -100); /* so that the way back is a normal number */
	}
	/* the larger of top and |v| where v is finite, else top (inf * 0 is no number, and a maximum passes over those): rows that are not finite have no say in the scale of the others */
	__device__ __forceinline__ float larger_finite(float top, float v)
	{
		return fmaxf(top, fmaf(v, 0.0f, fabsf(v)));
	}
	inline size_t round_up(size_t n, size_t to)
	{
		return (n + to - 1) / to * to;
	}
} /* namespace mlhip */

#endif /* MINML_AMD_TRAINING_UTILS_HPP_ */

// Entry points of the 4-bit matrix operators (mx_q4_*, include/mx_capi.h): argument checks, device, dispatch on type.
#include <cuda.h>

#include <algorithm>

#include "mx_internal.h"
#include "q4.h"
#include "q4_gemm.h"
#include "q4_ptx.cuh"

namespace mx {
namespace q4 {
namespace {

constexpr int MOST = 1 << 30;  // of rows, columns, vectors and a group's columns: indexes stay inside int32

bool is_vector_type(int dtype) { return dtype == MX_FP16 || dtype == MX_BF16; }

// Everything that can be said of the matrix without looking at device memory.
bool valid(const mx_q4_matrix *m) {
    if (!m || m->n_rows < 0 || m->n_cols < 0 || m->group <= 0 || m->group % 32 ||
        m->n_rows > MOST || m->n_cols > MOST || m->group > MOST || !is_vector_type(m->dtype) ||
        m->device < 0 || m->res_cap < 0)
        return false;
    if (m->n_rows > 0 && m->n_cols > 0) {
        if (!m->codes || !m->scales || (uintptr_t)m->codes % 16 || m->code_ld % 16 ||
            m->code_ld < ((long long)m->n_cols + 1) / 2)
            return false;
    }
    if ((uintptr_t)m->scales % 2 || (uintptr_t)m->res_val % 2 || (uintptr_t)m->res_row_ptr % 4 ||
        (uintptr_t)m->res_col_ind % 4)
        return false;
    if (m->res_row_ptr && m->res_cap > 0 && (!m->res_col_ind || !m->res_val)) return false;
    return true;
}

// n rows of `cols` values of `bytes` each, ld apart
bool valid_rows(const void *p, long long n, long long cols, long long ld, int bytes) {
    if (n == 0 || cols == 0) return true;
    return p && (uintptr_t)p % bytes == 0 && ld >= cols;
}

template <typename V>
Matrix<V> view(const mx_q4_matrix &m) {
    return {m.n_rows,
            m.n_cols,
            m.group,
            (int)(((long long)m.n_cols + m.group - 1) / m.group),
            m.code_ld,
            static_cast<const uint8_t *>(m.codes),
            static_cast<const V *>(m.scales),
            static_cast<const uint8_t *>(m.zeros),
            m.res_row_ptr,
            m.res_col_ind,
            static_cast<const V *>(m.res_val),
            m.res_row_ptr ? m.res_cap : 0};
}

// Whether the calling thread has a context.  The runtime gives it one at its first launch or allocation, which is too late
// for the tensor maps: those ask the driver.
bool has_context() {
    using Current = CUresult (*)(CUcontext *);
    static const Current current = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuCtxGetCurrent", &p, 4000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<Current>(p);
    }();
    CUcontext c = nullptr;
    return current && current(&c) == CUDA_SUCCESS && c;
}

// The matrix's GPU for the length of a call; the thread's own device comes back afterwards.
struct OnDevice {
    int before = -1, status = MX_OK;
    explicit OnDevice(int device) {
        int n = 0;
        if (cudaGetDeviceCount(&n) != cudaSuccess || n <= 0)
            status = MX_ERR_NO_DEVICE;
        else if (device >= n)
            status = MX_ERR_INVALID;
        else if (cudaGetDevice(&before) != cudaSuccess)
            status = MX_ERR_CUDA;
        else if ((before != device || !has_context()) && cudaSetDevice(device) != cudaSuccess)
            status = MX_ERR_CUDA;
        if (before == device) before = -1;
        if (status != MX_OK) cudaGetLastError();
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

int done(cudaError_t e) {
    if (e == cudaSuccess) return MX_OK;
    cudaGetLastError();
    return MX_ERR_CUDA;
}

struct Flags {
    int *flag[4];
};
cudaError_t late_flags(Flags &f) {
    const cudaError_t e[4] = {late_flag(&f.flag[0]), late_flag_few(&f.flag[1]), late_flag_quant(&f.flag[2]),
                              late_flag_grad(&f.flag[3])};
    return *std::max_element(e, e + 4);  // cudaSuccess is the least
}

// *late: whether a flag is set; none is afterwards
__global__ void late_kernel(Flags f, int *late) {
    if (atomicExch(f.flag[threadIdx.x], 0)) *late = 1;
}

// one thread that waits for a barrier at which nobody arrives
__global__ void wait_in_vain_kernel(int *flag, uint32_t polls) {
    __shared__ uint64_t bar;
    mbar_init(smem_addr(&bar), 1);
    if (!mbar_wait(smem_addr(&bar), 0, polls ? polls : polls_for(0))) *flag = 1;
}

// *bad is set when row pointers or columns are not ascending and in range
__global__ void check_kernel(int n_rows, int n_cols, int cap, const int *ptr, const int *col, int *bad) {
    const long long stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i <= n_rows; i += stride) {
        const int b = ptr[i];
        if ((i == 0 && b != 0) || b < 0 || b > cap) {
            *bad = 1;
            continue;
        }
        if (i == n_rows) continue;
        const int e = ptr[i + 1];
        if (e < b || e > cap) {
            *bad = 1;
            continue;
        }
        int last = 0;
        for (int k = b; k < e; ++k) {
            const int c = col[k];
            if (c < last || c >= n_cols) *bad = 1;
            last = c;
        }
    }
}

}  // namespace
}  // namespace q4
}  // namespace mx

using namespace mx;
using namespace mx::q4;

// runs `call` with V = the matrix's type
#define MX_Q4_TYPED(m, call)                    \
    ((m)->dtype == MX_FP16 ? [&] {              \
        using V = __half;                       \
        return call;                            \
    }()                                         \
                           : [&] {              \
                                 using V = __nv_bfloat16; \
                                 return call;   \
                             }())

extern "C" {

int mx_q4_quantize(const mx_q4_matrix *m, int w_dtype, const void *w, long long ld_w, float threshold, void *stream) {
    if (!valid(m) || (!is_vector_type(w_dtype) && w_dtype != MX_FP32) ||
        !valid_rows(w, m->n_rows, m->n_cols, ld_w, w_dtype == MX_FP32 ? 4 : 2))
        return MX_ERR_INVALID;
    OnDevice on(m->device);
    if (on.status != MX_OK) return on.status;
    return done(MX_Q4_TYPED(m, quantize<V>(*m, w_dtype, w, ld_w, threshold, static_cast<cudaStream_t>(stream))));
}

int mx_q4_expand(const mx_q4_matrix *m, void *w, long long ld_w, void *stream) {
    if (!valid(m) || !valid_rows(w, m->n_rows, m->n_cols, ld_w, 2)) return MX_ERR_INVALID;
    OnDevice on(m->device);
    if (on.status != MX_OK) return on.status;
    if (m->n_rows == 0 || m->n_cols == 0) return MX_OK;
    return done(MX_Q4_TYPED(m, expand<V>(view<V>(*m), static_cast<V *>(w), ld_w, static_cast<cudaStream_t>(stream))));
}

int mx_q4_product(const mx_q4_matrix *m, int n_vec, const void *x, long long ld_x, void *y, long long ld_y,
                  void *stream) {
    if (!valid(m) || n_vec < 0 || n_vec > MOST || !valid_rows(x, n_vec, m->n_cols, ld_x, 2) ||
        !valid_rows(y, n_vec, m->n_rows, ld_y, 2))
        return MX_ERR_INVALID;
    OnDevice on(m->device);
    if (on.status != MX_OK) return on.status;
    if (n_vec == 0 || m->n_rows == 0) return MX_OK;
    return done(MX_Q4_TYPED(m, product<V>(view<V>(*m), n_vec, static_cast<const V *>(x), ld_x, static_cast<V *>(y), ld_y,
                                          static_cast<cudaStream_t>(stream))));
}

int mx_q4_product_t(const mx_q4_matrix *m, int n_vec, const void *dy, long long ld_dy, void *dx, long long ld_dx,
                    void *stream) {
    if (!valid(m) || n_vec < 0 || n_vec > MOST || !valid_rows(dy, n_vec, m->n_rows, ld_dy, 2) ||
        !valid_rows(dx, n_vec, m->n_cols, ld_dx, 2))
        return MX_ERR_INVALID;
    OnDevice on(m->device);
    if (on.status != MX_OK) return on.status;
    if (n_vec == 0 || m->n_cols == 0) return MX_OK;
    return done(MX_Q4_TYPED(m, product_t<V>(view<V>(*m), n_vec, static_cast<const V *>(dy), ld_dy, static_cast<V *>(dx),
                                            ld_dx, static_cast<cudaStream_t>(stream))));
}

int mx_q4_grad(const mx_q4_matrix *m, int n_vec, const void *x, long long ld_x, const void *dy, long long ld_dy,
               void *d_scales, void *d_res_val, void *stream) {
    if (!valid(m) || n_vec < 0 || n_vec > MOST || !valid_rows(x, n_vec, m->n_cols, ld_x, 2) ||
        !valid_rows(dy, n_vec, m->n_rows, ld_dy, 2) || (uintptr_t)d_scales % 2 || (uintptr_t)d_res_val % 2 ||
        (d_res_val && !m->res_row_ptr))
        return MX_ERR_INVALID;
    OnDevice on(m->device);
    if (on.status != MX_OK) return on.status;
    if (m->n_rows == 0 || m->n_cols == 0 || (!d_scales && !d_res_val)) return MX_OK;
    return done(MX_Q4_TYPED(m, grad<V>(view<V>(*m), n_vec, static_cast<const V *>(x), ld_x, static_cast<const V *>(dy),
                                       ld_dy, static_cast<V *>(d_scales), static_cast<V *>(d_res_val),
                                       static_cast<cudaStream_t>(stream))));
}

int mx_q4_check(const mx_q4_matrix *m, void *stream) {
    if (!valid(m)) return MX_ERR_INVALID;
    OnDevice on(m->device);
    if (on.status != MX_OK) return on.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int *found = nullptr, is[2] = {0, 0};  // the residual is bad, a wait ran out
    Flags flags;
    cudaError_t e = late_flags(flags);
    if (e == cudaSuccess) e = cudaMallocAsync((void **)&found, sizeof(is), s);
    if (e != cudaSuccess) return done(e);
    e = cudaMemsetAsync(found, 0, sizeof(is), s);
    if (e == cudaSuccess && m->res_row_ptr) {
        const int blocks = (int)std::min<long long>(((long long)m->n_rows + 256) / 256, 148 * 8);
        check_kernel<<<blocks, 256, 0, s>>>(m->n_rows, m->n_cols, m->res_cap, m->res_row_ptr, m->res_col_ind, found);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) {
        late_kernel<<<1, 4, 0, s>>>(flags, found + 1);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaMemcpyAsync(is, found, sizeof(is), cudaMemcpyDeviceToHost, s);
    cudaError_t f = cudaFreeAsync(found, s);
    if (e == cudaSuccess) e = f;
    f = cudaStreamSynchronize(s);  // whatever happened: the copy ends in this frame
    if (e == cudaSuccess) e = f;
    if (e != cudaSuccess) return done(e);
    return is[1] ? MX_ERR_TIMEOUT : is[0] ? MX_ERR_INVALID : MX_OK;
}

int mx_q4_wait_in_vain(int device, int which, unsigned polls, void *stream) {
    if (device < 0 || which < 0 || which > 3 || polls > 1u << 16) return MX_ERR_INVALID;
    OnDevice on(device);
    if (on.status != MX_OK) return on.status;
    Flags flags;
    cudaError_t e = late_flags(flags);
    if (e != cudaSuccess) return done(e);
    wait_in_vain_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(flags.flag[which], polls);
    return done(cudaGetLastError());
}

}  // extern "C"

/*
 * gsx_hip.h - C ABI of the gfx950 (MI355X) backend library libgsx_hip.so.
 *
 * This is the layer the gsx backend vtables call (gsx/src/gsx-impl.h:229-533 for the vtables,
 * gsx/src/gsx-cuda/internal.h:274-675 for the launcher layer it replaces): plain device
 * pointers, sizes and a hipStream_t, C linkage, no C++ or framework types. All device work is
 * enqueued on the given stream in order; nothing here synchronises the host except where a
 * function says so. Every call returns 0 on success, a hipError_t value (> 0) for a HIP
 * runtime error, or a negative GSX_HIP_ERROR_* code; gsx_hip_last_error_message() names the
 * failing condition (thread-local, static storage).
 *
 * Conventions shared with gsx (gsx/include/gsx/gsx-render.h:64-140, gsx-base.h:191-216):
 *   Gaussians: mean3d [N,3], rotation [N,4] (xyzw), logscale [N,3], opacity [N] (logit),
 *   sh0 [N,3], sh1 [N,3,3], sh2 [N,5,3], sh3 [N,7,3], all float32 row-major on the device;
 *   images: float32 CHW [3,H,W]; camera: pinhole, world-to-camera pose, +z forward, y down.
 */
#ifndef GSX_HIP_H
#define GSX_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef HIP_INCLUDE_HIP_HIP_RUNTIME_API_H
typedef struct ihipStream_t* hipStream_t;
typedef struct ihipEvent_t* hipEvent_t;
#endif

typedef int gsx_hip_status;

enum {
    GSX_HIP_SUCCESS = 0,
    GSX_HIP_ERROR_INVALID_ARGUMENT = -1, /* gsx GSX_ERROR_INVALID_ARGUMENT */
    GSX_HIP_ERROR_INVALID_STATE = -2,    /* gsx GSX_ERROR_INVALID_STATE (e.g. backward w/o TRAIN forward) */
    GSX_HIP_ERROR_OUT_OF_RANGE = -3,     /* gsx GSX_ERROR_OUT_OF_RANGE (sizes, gather indices) */
    GSX_HIP_ERROR_OUT_OF_MEMORY = -4,    /* gsx GSX_ERROR_OUT_OF_MEMORY */
    GSX_HIP_ERROR_NOT_SUPPORTED = -5     /* gsx GSX_ERROR_NOT_SUPPORTED */
};

/* Human-readable reason for the last non-zero status returned on this thread. */
const char* gsx_hip_last_error_message(void);

/* ---- device plumbing (replaces the cudaMalloc/cudaMemcpy use of gsx-cuda/buffer.c) -------- */
gsx_hip_status gsx_hip_device_count(int32_t* out_count);
gsx_hip_status gsx_hip_device_name(int32_t device, char* out_name, size_t capacity);
gsx_hip_status gsx_hip_malloc(void** out_ptr, size_t bytes);
gsx_hip_status gsx_hip_free(void* ptr);

/* Stream-ordered caching device allocator (the backend's device buffers, optimizer moments and
 * density-control workspaces; replaces the cudaMalloc / synchronising cudaFree pairs of
 * gsx-cuda/buffer.c and gsx-cuda/optim.c that every gsx_gs_resize commit,
 * gsx/src/gsx-core.c:2811-2869, goes through). A request is rounded up to one of 8 size classes per
 * power of two (at least 512 bytes) and served from cached blocks of its class or the next two
 * when one is free; otherwise hipMalloc (on running out of memory the cache is released and the
 * request retried). pool_free returns a block to the cache behind an event recorded on `stream`
 * (no host synchronisation): reuse on the same stream is ordered by the stream, reuse on another
 * stream waits on that event. Blocks stay cached until gsx_hip_pool_trim (current device; it
 * synchronises the device first) or process exit. Thread-safe. */
typedef struct gsx_hip_pool_stats {
    uint64_t requests;            /* pool_malloc calls */
    uint64_t reuses;              /* requests served from cached blocks */
    uint64_t device_allocations;  /* hipMalloc calls made by the pool */
    uint64_t device_releases;     /* hipFree calls made by the pool (trim, out-of-memory retry) */
    uint64_t bytes_in_use;        /* rounded sizes of the blocks handed out */
    uint64_t bytes_cached;        /* rounded sizes of the cached blocks */
} gsx_hip_pool_stats;
gsx_hip_status gsx_hip_pool_malloc(void** out_ptr, size_t bytes, hipStream_t stream);
gsx_hip_status gsx_hip_pool_free(void* ptr, hipStream_t stream);
gsx_hip_status gsx_hip_pool_trim(void);
gsx_hip_status gsx_hip_pool_get_stats(gsx_hip_pool_stats* out_stats);
gsx_hip_status gsx_hip_memcpy_htod(void* dst, const void* src, size_t bytes);
gsx_hip_status gsx_hip_memcpy_dtoh(void* dst, const void* src, size_t bytes);
gsx_hip_status gsx_hip_memcpy_dtod_async(void* dst, const void* src, size_t bytes, hipStream_t stream);
/* Ordered copy on `stream` between any two of host, pinned host and device memory (the direction
 * is taken from the pointers, hipMemcpyDefault); gsx-cuda/buffer.c's cudaMemcpyAsync uses. */
gsx_hip_status gsx_hip_memcpy_async(void* dst, const void* src, size_t bytes, hipStream_t stream);
gsx_hip_status gsx_hip_set_device(int32_t device);
gsx_hip_status gsx_hip_device_total_memory(int32_t device, size_t* out_bytes);
/* Page-locked host memory (the HOST_PINNED buffer type) and its device-side address. */
gsx_hip_status gsx_hip_host_alloc(void** out_host, size_t bytes);
gsx_hip_status gsx_hip_host_free(void* host);
gsx_hip_status gsx_hip_host_device_pointer(void* host, void** out_device);
gsx_hip_status gsx_hip_stream_create(hipStream_t* out_stream);
gsx_hip_status gsx_hip_stream_destroy(hipStream_t stream);
gsx_hip_status gsx_hip_stream_synchronize(hipStream_t stream);
/* Events (no timing) ordering work between streams: the async dataloader's helper stream and the
 * major stream (gsx-cuda/async_dl.cu orders them by host synchronisation instead). An event
 * never recorded counts as complete. */
gsx_hip_status gsx_hip_event_create(hipEvent_t* out_event);
gsx_hip_status gsx_hip_event_destroy(hipEvent_t event);
gsx_hip_status gsx_hip_event_record(hipEvent_t event, hipStream_t stream);
gsx_hip_status gsx_hip_event_synchronize(hipEvent_t event);
gsx_hip_status gsx_hip_stream_wait_event(hipStream_t stream, hipEvent_t event);
/* Fill `count` floats with `value` (a kernel, not hipMemset, so it is safe under graph capture). */
gsx_hip_status gsx_hip_fill_f32(float* dst, int64_t count, float value, hipStream_t stream);
/* Streaming device copy of `count` floats (16-byte aligned, count % 4 == 0); also the known-size
 * reference kernel against which HBM traffic counters are calibrated. */
gsx_hip_status gsx_hip_copy_f32(float* dst, const float* src, int64_t count, hipStream_t stream);

/* ---- render ---------------------------------------------------------------------------------
 * Replaces gsx_cuda_fastgs_forward_launch / gsx_cuda_fastgs_backward_launch
 * (gsx/src/gsx-cuda/internal.h:545-630) and the renderer vtable behaviour of the CPU oracle
 * (gsx/src/gsx-cpu/render.c:1254-1975). The render context owns every intermediate buffer
 * (pooled, grow-only; the fastgs resize callbacks and per-forward allocations are gone) and
 * the state a TRAIN forward retains for the backward.
 */
typedef struct gsx_hip_camera {
    float fx, fy, cx, cy;   /* gsx_camera_intrinsics (gsx-base.h:191-205) */
    int32_t width, height;
    float rot[4];           /* gsx_camera_pose.rot, world-to-camera quaternion, xyzw */
    float transl[3];        /* gsx_camera_pose.transl */
    float near_plane, far_plane;
    float background[3];
} gsx_hip_camera;

typedef struct gsx_hip_gaussians {
    int64_t count;
    int32_t sh_degree;      /* 0..3; sh1..sh3 required up to this degree, ignored above */
    const float* mean3d;
    const float* rotation;  /* 16-byte aligned (one float4 per Gaussian); the others 4-byte */
    const float* logscale;
    const float* opacity;
    const float* sh0;
    const float* sh1;
    const float* sh2;
    const float* sh3;
} gsx_hip_gaussians;

typedef struct gsx_hip_gaussian_grads {
    float* mean3d;          /* sinks are overwritten, as gsx-cpu/render.c:1537-1550 */
    float* rotation;        /* 16-byte aligned, as gsx_hip_gaussians.rotation; the others 4-byte */
    float* logscale;
    float* opacity;
    float* sh0;
    float* sh1;
    float* sh2;
    float* sh3;
} gsx_hip_gaussian_grads;

typedef struct gsx_hip_render_context gsx_hip_render_context;

typedef struct gsx_hip_render_stats {
    int64_t gaussian_count;
    int64_t visible_count;   /* Gaussians that pass the projection culls (depth-sorted) in the
                                context's last forward, summed on the host when the forward read
                                back its instance count: get_stats reads no device memory */
    int64_t instance_count;  /* (tile, Gaussian) pairs sorted */
    int32_t tile_count;
    int32_t sort_passes;       /* radix passes over the instance tiles */
    int32_t depth_sort_passes; /* radix passes over the per-Gaussian depth keys */
    /* instances are emitted in (depth, index) order of their Gaussians and their tile indices
     * (tile_bits bits) sorted stably with the emission positions as values, which yields the gsx
     * per-tile (depth, index) order */
    int32_t tile_bits;
    int32_t sorted_tile_bytes; /* element size of sorted_tiles (4) */
} gsx_hip_render_stats;

/* Device pointers of the intermediates a forward retains (valid until the next forward). The path keeps
 * tile indices in 16 bits up to 65536 tiles: the first get_buffers after such a forward waits for the
 * device and writes sorted_tiles from them, into memory that the context has. Threads may look at one
 * context at the same time. sorted_tiles is null after a forward that failed before its lists stood. */
typedef struct gsx_hip_render_buffers {
    const uint32_t* sorted_tiles;  /* [instance_count] tile index of each sorted instance */
    const uint32_t* sorted_values; /* [instance_count] emission position of each sorted instance */
    const uint32_t* tile_ranges;   /* [tile_count][2] start, end */
    const float* records;          /* [N][8] geometry then [N][4] colour+depth blend records */
    const uint32_t* tile_counts;   /* [N] tiles touched per Gaussian (0 = culled) */
    const uint32_t* instance_gaussian; /* [instance_count] Gaussian index of each emission position */
    const float* final_transmittance; /* [H*W] */
    const uint32_t* last_contributor; /* [H*W] exclusive end of the last contributing position */
} gsx_hip_render_buffers;

gsx_hip_status gsx_hip_render_context_create(gsx_hip_render_context** out_context);
gsx_hip_status gsx_hip_render_context_destroy(gsx_hip_render_context* context);

/* Forward types (gsx_render_forward_type and borrow_train_state of gsx_render_forward_request,
 * gsx/include/gsx/gsx-render.h:54-58, 101; semantics of gsx/src/gsx-cpu/render.c:263-380,
 * 1406-1440 and gsx/src/gsx-cuda/render.c:551, 662-756). METRIC is not supported (the CPU
 * backend rejects it too, gsx-cpu/render.c:1126-1154). */
enum {
    GSX_HIP_FORWARD_INFERENCE = 0,    /* image only; no state retained */
    GSX_HIP_FORWARD_TRAIN_BORROW = 1, /* borrow_train_state = true: the backward differentiates at
                                         the values the Gaussian arrays hold when it is called */
    GSX_HIP_FORWARD_TRAIN_CLONE = 2   /* borrow_train_state = false: the backward differentiates at
                                         the values of this forward, whatever the caller changes */
};

/* Forward render into out_rgb [3,H,W]. forward_type is a GSX_HIP_FORWARD_* value. A TRAIN forward
 * retains the state for one backward: it copies the Gaussian fields it reads into the context
 * (56 B per Gaussian at SH degree 0, 236 B at degree 3), and, if visible_counter is non-null,
 * adds 1 to it for every visible Gaussian (gsx-cpu/render.c:980-982). The Gaussian arrays are
 * borrowed for the call. One host synchronisation per forward reads the instance count (the GPU
 * keeps working on the depth order meanwhile); a count above 2^32 - 1 (tile, Gaussian)
 * instances fails with GSX_HIP_ERROR_OUT_OF_RANGE before anything is emitted.
 * Precondition: finite inputs (Gaussian fields, and grad_rgb in the backward). The blend kernels
 * evaluate an entry for the 64 pixels of a wave at once, and a pixel that does not take it adds
 * 0 x its colour (or its gradient term): with finite values that changes nothing, but a
 * non-finite colour or image gradient then turns the other pixels of those waves into NaN as
 * well, where the CPU backend leaves them finite. Every pixel the CPU renders finite and this
 * build renders finite is bit-identical. */
gsx_hip_status gsx_hip_render_forward(gsx_hip_render_context* context, const gsx_hip_camera* camera,
                                      const gsx_hip_gaussians* gaussians, int32_t forward_type, float* out_rgb,
                                      float* visible_counter, hipStream_t stream);

/* Backward of the retained TRAIN forward; consumes the state (a second call fails with
 * GSX_HIP_ERROR_INVALID_STATE, as gsx-cpu/render.c:1406-1408, 1973). After a TRAIN_BORROW forward
 * it first compares the caller's Gaussian arrays with the retained copy (one read of both and one
 * host synchronisation) and, if any bit changed, re-runs the forward on the current values before
 * differentiating (the reference CUDA backend re-runs it unconditionally,
 * gsx-cuda/render.c:1451). */
gsx_hip_status gsx_hip_render_backward(gsx_hip_render_context* context, const float* grad_rgb,
                                       const gsx_hip_gaussian_grads* grads, hipStream_t stream);

gsx_hip_status gsx_hip_render_context_get_stats(const gsx_hip_render_context* context,
                                                gsx_hip_render_stats* out_stats);
gsx_hip_status gsx_hip_render_context_get_buffers(const gsx_hip_render_context* context,
                                                  gsx_hip_render_buffers* out_buffers);

/* Per-stage device timing: set_timing(capacity > 0) allocates a ring of `capacity` HIP event
 * sets; each forward (and the following backward) records one set on its launch stream, so a
 * timed loop pays no synchronisation. get_timings synchronises on the recorded events and writes
 * the per-stage average over the recorded sets, in milliseconds, in this order: preprocess,
 * depth_order (depth-key sort, tile counts in depth order, their scan and the instance-count
 * readback), emit, sort, ranges, blend_forward, blend_backward, instance_reduce,
 * projection_backward. set_timing(0) disables timing. */
enum { GSX_HIP_RENDER_STAGE_COUNT = 9 };
gsx_hip_status gsx_hip_render_context_set_timing(gsx_hip_render_context* context, int32_t capacity);
gsx_hip_status gsx_hip_render_context_get_timings(gsx_hip_render_context* context, float* out_ms, int32_t capacity,
                                                  int32_t* out_written);

/* ---- sort / scan ------------------------------------------------------------------------------
 * Replace cub::DeviceScan::ExclusiveSum (fastgs/forward.cu:180-185) and
 * cub::DeviceRadixSort::SortPairs (fastgs/forward.cu:155-161, 214-220). */
size_t gsx_hip_scan_temp_bytes(int64_t n);
gsx_hip_status gsx_hip_scan_exclusive_u32(const uint32_t* in, uint32_t* out, int64_t n, void* temp,
                                          hipStream_t stream);
/* The exclusive scan above without allocation or workspace, for callers that cannot allocate
 * (code under HIP graph capture, serving loops, harnesses that forbid hipMalloc); it has no
 * counterpart in the reference. The partial sums live in a static device array of 256 KiB per
 * GPU (held until the process ends), so n may be at most 67,108,864 (2^26) elements; larger n
 * fails with GSX_HIP_ERROR_OUT_OF_RANGE. Every call on one GPU uses that GPU's array: calls that
 * overlap on one GPU (different streams or host threads) race and must be serialised by the
 * caller. Nothing needs clearing between calls (every partial is written before it is read). */
gsx_hip_status gsx_hip_scan_exclusive_u32_noalloc(const uint32_t* in, uint32_t* out, int64_t n, hipStream_t stream);
size_t gsx_hip_radix_sort_temp_bytes(int64_t n);
/* Stable LSD sort of (key, value) pairs on key bits [begin_bit, end_bit), 8 bits per pass. */
gsx_hip_status gsx_hip_radix_sort_pairs_u64(uint64_t* keys, uint32_t* values, uint64_t* keys_alt,
                                            uint32_t* values_alt, int64_t n, int begin_bit, int end_bit, void* temp,
                                            int* out_result_in_alt, hipStream_t stream);
/* Stable LSD sort of keys alone on bits [begin_bit, end_bit); the other bits travel with the key
 * (the render path packs the emission position below begin_bit). No counterpart in the CUDA
 * backend, which always sorts pairs. */
gsx_hip_status gsx_hip_radix_sort_keys_u64(uint64_t* keys, uint64_t* keys_alt, int64_t n, int begin_bit,
                                           int end_bit, void* temp, int* out_result_in_alt, hipStream_t stream);

/* ---- tensor operations -------------------------------------------------------------------------
 * The element-wise, random, reduce and image-conversion entries of gsx_backend_buffer_i
 * (gsx/src/gsx-impl.h:302-458) that the CUDA backend implements in gsx-cuda/buffer.c and
 * reduce-kernels.cu; semantics of the CPU backend (gsx/src/gsx-cpu/core.c:874-2019). Pointers are
 * device pointers; nothing here synchronises except where stated. */
enum {
    GSX_HIP_DTYPE_F32 = 0,
    GSX_HIP_DTYPE_U8 = 1,
    GSX_HIP_DTYPE_I32 = 2,
    GSX_HIP_DTYPE_BF16 = 3, /* the label-field operators only, as F16 */
    GSX_HIP_DTYPE_F16 = 4
};
enum {                                   /* gsx_impl_unary_op (gsx-impl.h:295-300) */
    GSX_HIP_UNARY_EXP = 0,
    GSX_HIP_UNARY_SIGMOID = 1,
    GSX_HIP_UNARY_SIGMOID_DERIVATIVE = 2,
    GSX_HIP_UNARY_ABS = 3
};
enum {                                   /* gsx_impl_unary/binary_reduce_op (gsx-impl.h:234-243) */
    GSX_HIP_REDUCE_SUM = 0,
    GSX_HIP_REDUCE_MEAN = 1,
    GSX_HIP_REDUCE_MAX = 2,
    GSX_HIP_REDUCE_MSE = 3,
    GSX_HIP_REDUCE_MAE = 4
};
/* Repeat a pattern of 1..64 bytes over `bytes` (memset_tensor / fill_tensor / set_zero). */
gsx_hip_status gsx_hip_fill_pattern(void* dst, size_t bytes, const void* pattern, size_t pattern_bytes,
                                    hipStream_t stream);
/* Element i = pcg32_next_float of draw i of the (state, inc) stream (fill_rand_tensor). */
gsx_hip_status gsx_hip_fill_rand_f32(float* dst, int64_t count, uint64_t state, uint64_t inc, hipStream_t stream);
/* Box-Muller pairs from draws 2k, 2k+1, times sigma (fill_randn_tensor); logf / cosf / sinf are
 * glibc's, bit for bit, so the fill equals the CPU backend's. */
gsx_hip_status gsx_hip_fill_randn_f32(float* dst, int64_t count, uint64_t state, uint64_t inc, float sigma,
                                      hipStream_t stream);
/* fill_randint_tensor: element i = the i-th draw that pcg32_next_uint_bound accepts, mod bound,
 * for u8 (element_bytes 1) or i32 (4) elements. `draws` >= count draws are examined (temp of
 * gsx_hip_fill_randint_temp_bytes(draws)); when out_accepted is non-null the call synchronises
 * the stream and stores how many were accepted (fewer than count: call again with more draws). */
size_t gsx_hip_fill_randint_temp_bytes(int64_t draws);
gsx_hip_status gsx_hip_fill_randint(void* dst, int64_t count, int32_t element_bytes, uint64_t state, uint64_t inc,
                                    uint32_t bound, int64_t draws, void* temp, int64_t* out_accepted,
                                    hipStream_t stream);
/* multinomial_tensor: sample i from draw i and the (non-decreasing, positive-ended) cdf. */
gsx_hip_status gsx_hip_multinomial_i32(int32_t* out, int64_t samples, const float* cdf, int64_t categories,
                                       uint64_t state, uint64_t inc, hipStream_t stream);
/* check_finite_tensor: sets *flag (a device word the caller cleared) to 1 on any inf or NaN. */
gsx_hip_status gsx_hip_check_finite_f32(const float* x, int64_t count, uint32_t* flag, hipStream_t stream);
/* unary_tensor / unary_tensor_inplace (x may equal out); exp through the glibc-exact expf. */
gsx_hip_status gsx_hip_unary_f32(const float* x, float* out, int64_t count, int32_t op, hipStream_t stream);
/* clamp_inplace_tensor for GSX_HIP_DTYPE_*; lo and hi are host pointers to one element. */
gsx_hip_status gsx_hip_clamp_inplace(void* x, int64_t count, int32_t data_type, const void* lo, const void* hi,
                                     hipStream_t stream);
/* unary_reduce_tensor (sum, mean, max over rows of `reduce` elements of x) and
 * binary_reduce_tensor (mse, mae of x - y); out[outer]. Sums run in double in a fixed order;
 * max keeps the CPU's first-occurrence and NaN rules. temp: gsx_hip_reduce_temp_bytes. */
size_t gsx_hip_reduce_temp_bytes(int64_t outer, int64_t reduce);
gsx_hip_status gsx_hip_reduce_f32(const float* x, const float* y, int64_t outer, int64_t reduce, int32_t op,
                                  float* out, void* temp, hipStream_t stream);
/* The dataloader's device layout step (replaces the HWC -> CHW kernels of
 * gsx/src/gsx-cuda/async_dl.cu:45-156): dst [channels, height, width] float32 from a tightly
 * packed HWC (channels 3) or HW (channels 1) payload of u8 (src_is_u8 != 0, values kept, not
 * scaled) or float32 already in device-visible memory. */
gsx_hip_status gsx_hip_dataloader_to_chw_f32(const void* src, int32_t src_is_u8, int64_t channels, int64_t height,
                                            int64_t width, float* dst, hipStream_t stream);
/* image_convert_colorspace (sRGB transfer curves with glibc's powf, bit for bit),
 * image_convert_storage_format (HWC <-> CHW for 1/2/4-byte elements) and
 * image_convert_data_type (f32 <-> u8), gsx/src/extra/gsx-image-impl.h:9-170. */
gsx_hip_status gsx_hip_image_colorspace_f32(const float* src, float* dst, int64_t count, int32_t src_srgb,
                                            int32_t dst_srgb, hipStream_t stream);
gsx_hip_status gsx_hip_image_storage_convert(const void* src, int32_t src_hwc, void* dst, int32_t dst_hwc,
                                             int64_t channels, int64_t height, int64_t width, int32_t element_bytes,
                                             hipStream_t stream);
gsx_hip_status gsx_hip_image_quantize_u8(const float* src, uint8_t* dst, int64_t count, hipStream_t stream);
gsx_hip_status gsx_hip_image_dequantize_u8(const uint8_t* src, float* dst, int64_t count, hipStream_t stream);

/* ---- losses -----------------------------------------------------------------------------------
 * Replace gsx_cuda_loss_*_kernel_launch (gsx/src/gsx-cuda/internal.h:312-369, CHW forms); semantics of
 * gsx/src/gsx-cpu/loss.c:316-709 (accumulate into loss_map / grad_prediction; grad_scale is
 * already normalised as gsx_loss_scale_grad, gsx-tensor-helpers.h:236-244). */
gsx_hip_status gsx_hip_loss_l1_f32_forward_kernel_launch(float* loss_map, const float* prediction,
                                                         const float* target, int64_t total_elements, float scale,
                                                         hipStream_t stream);
gsx_hip_status gsx_hip_loss_l1_f32_backward_kernel_launch(float* grad_prediction, const float* prediction,
                                                          const float* target, int64_t total_elements,
                                                          float grad_scale, hipStream_t stream);
gsx_hip_status gsx_hip_loss_mse_f32_forward_kernel_launch(float* loss_map, const float* prediction,
                                                          const float* target, int64_t total_elements, float scale,
                                                          hipStream_t stream);
gsx_hip_status gsx_hip_loss_mse_f32_backward_kernel_launch(float* grad_prediction, const float* prediction,
                                                           const float* target, int64_t total_elements,
                                                           float grad_scale, hipStream_t stream);
/* SSIM on [outer, channels, H, W] CHW images; ssim_workspace = 3 * outer*channels*H*W floats
 * written by the forward and read by the backward. fuse_l1 != 0 also applies an L1 term of
 * l1_scale (forward) / l1_grad_scale (backward) first, bit-identical to calling the L1
 * launcher before. These are not drop-in replacements of gsx_cuda_loss_ssim_* (gsx-cuda/
 * internal.h:346-369): those take two buffers (ssim_buffer_a/b) and no L1 term; here one
 * workspace holds the three window moments the backward needs. The gsx loss vtable of this
 * library (gsx_amd/plugin/hip_loss.c) owns that workspace per loss context. Limits: at most 65535
 * planes (outer_count * channels) and height * width <= UINT32_MAX, else
 * GSX_HIP_ERROR_OUT_OF_RANGE. */
gsx_hip_status gsx_hip_loss_ssim_chw_f32_forward_kernel_launch(float* loss_map, const float* prediction,
                                                               const float* target, int64_t outer_count,
                                                               int32_t channels, int32_t height, int32_t width,
                                                               float scale, float* ssim_workspace, float l1_scale,
                                                               int fuse_l1, hipStream_t stream);
gsx_hip_status gsx_hip_loss_ssim_chw_f32_backward_kernel_launch(float* grad_prediction, const float* prediction,
                                                                const float* target, int64_t outer_count,
                                                                int32_t channels, int32_t height, int32_t width,
                                                                float grad_scale, const float* ssim_workspace,
                                                                float l1_grad_scale, int fuse_l1,
                                                                hipStream_t stream);

/* ---- optimizer --------------------------------------------------------------------------------
 * Adam, element arithmetic of gsx/src/gsx-cpu/optim.c:712-780; bias corrections
 * 1 - beta^step are computed by the caller in float64 (as the CPU does with pow). */
#define GSX_HIP_ADAM_MAX_GROUPS 16
typedef struct gsx_hip_adam_group {
    float* parameter;
    const float* gradient;
    float* first_moment;
    float* second_moment;
    int64_t count;
    float beta1, beta2, learning_rate, weight_decay, epsilon, max_grad;
    double bias_correction1, bias_correction2;
} gsx_hip_adam_group;

/* Counterpart of gsx_cuda_adam_step_f32_kernel_launch (gsx/src/gsx-cuda/internal.h:296-311),
 * with one difference in the contract: this launcher takes the bias corrections themselves,
 * 1 - beta^step in float64, and divides the moments by them as the CPU backend does
 * (gsx-cpu/optim.c:740-757); the CUDA vtable passes their float inverses instead
 * (gsx-cuda/optim.c:792-793), so a caller ported from there must not pass inverses. The gsx
 * vtable of this library (gsx_amd/plugin/hip_optim.c) calls the multi-group launcher below. */
gsx_hip_status gsx_hip_adam_step_f32_kernel_launch(float* parameter, const float* gradient, float* first_moment,
                                                   float* second_moment, int64_t total_elements, float beta1,
                                                   float beta2, float learning_rate, float weight_decay,
                                                   float epsilon, float max_grad, double bias_correction1,
                                                   double bias_correction2, hipStream_t stream);
/* All groups of one optimizer step in a single launch (the CUDA backend issues one launch
 * per group, gsx/src/gsx-cuda/optim.c:757-796). Above 256 MiB of traffic (28 bytes per element
 * over all groups) the launch reads and writes with non-temporal accesses; the results are the
 * same bits either way. */
gsx_hip_status gsx_hip_adam_step_multi_launch(const gsx_hip_adam_group* groups, int32_t group_count,
                                              hipStream_t stream);

/* AdamW over any number of tensors in one launch (no counterpart in the reference). With t = *steps + 1, all in float32, one
 * rounding for each operation:
 *   g = gradient * grad_scale * grad_factor[0] (null: 1);  m' = beta1 m + (1 - beta1) g;  v' = beta2 v + (1 - beta2) (g g)
 *   p' = p - (rate decay) p - (rate / (1 - beta1^t)) (m' / (sqrt(v') / sqrt(1 - beta2^t) + epsilon))
 * Parameters and gradients are GSX_HIP_DTYPE_F32, BF16 or F16, a parameter rounded to nearest even. bits = 32: first and second
 * are float32 [count]. bits = 8: they hold ceil(count / 128) whole blocks of 128 codes (8-byte aligned) and a float32 scale a
 * block, 0 behind the count:
 *   first:  scale s = max(max |m| * (float)(1/448), 2^-126), code E4M3 of m * (1 / s) (ties to even); stands for code * s
 *   second: scale s = max(max v, 2^-126), ratio y = v * (1 / s) rounded to three bits behind the first (ties to even), code
 *           (bits of y >> 20) - 762 within 1 to 254 for v > 0, 0 for v = 0; stands for ratio * s
 * over a block's finite values; one that is not finite is held as NaN in the first and as 255, +inf, in the second. */
typedef struct gsx_hip_adamw_tensor {
    void* parameter;
    const void* gradient;
    void *first, *second;              /* moments */
    float *first_scale, *second_scale; /* of 8-bit moments */
    int64_t count;
    int32_t parameter_type, gradient_type;
    int32_t bits;  /* 8 or 32 */
    int32_t group; /* of gsx_hip_adamw_step's groups */
} gsx_hip_adamw_tensor;
typedef struct gsx_hip_adamw_group {
    double beta1, beta2, learning_rate, weight_decay, epsilon; /* 0 <= beta < 1, epsilon > 0 as a float, decay >= 0 */
} gsx_hip_adamw_group;

/* The table of a step's tensors: fill writes table_bytes bytes to host memory (8-byte aligned) and *out_chunks, what step is
 * given; the caller copies the table to 8-byte aligned device memory and keeps it there as it is. Nothing that a step writes
 * (parameters, moments, scales) may overlap another tensor's memory or the gradients. table_bytes is 0 where fill would refuse
 * the tensors for anything but an overlap. At most 2^24 - 1 chunks of 2048 elements. */
size_t gsx_hip_adamw_table_bytes(const gsx_hip_adamw_tensor* tensors, int64_t tensor_count);
gsx_hip_status gsx_hip_adamw_table_fill(const gsx_hip_adamw_tensor* tensors, int64_t tensor_count, void* table,
                                        int64_t* out_chunks);
/* One step: counts *steps (on the device) and updates every tensor of the table; those of groups from group_count on stay as
 * they are. `factors` is device memory of 8 * GSX_HIP_ADAM_MAX_GROUPS bytes (8-byte aligned) that steps on one stream may
 * share. Captured into a graph, each replay counts a step, with the capture's groups and grad_scale and with what grad_factor
 * holds then. */
gsx_hip_status gsx_hip_adamw_step(const void* table, int64_t chunks, const gsx_hip_adamw_group* groups, int32_t group_count,
                                  float grad_scale, const float* grad_factor, int64_t* steps, void* factors,
                                  hipStream_t stream);
/* Whole blocks of moments (128 * blocks values) from float32 to their codes and scales, and back. */
gsx_hip_status gsx_hip_moments_hold(const float* first, const float* second, int64_t blocks, uint8_t* first_codes,
                                    float* first_scale, uint8_t* second_codes, float* second_scale, hipStream_t stream);
gsx_hip_status gsx_hip_moments_read(const uint8_t* first_codes, const float* first_scale, const uint8_t* second_codes,
                                    const float* second_scale, int64_t blocks, float* first, float* second,
                                    hipStream_t stream);

/* ---- adaptive density control -----------------------------------------------------------------
 * Replaces the CUDA thrust pipeline (gsx/src/gsx-cuda/adc.cu:757-927) with the semantics of
 * the CPU default/ABSGS refine and opacity reset (gsx/src/gsx-cpu/adc/default.c:160-527,
 * gsx/src/gsx-cpu/adc.c:48-80, 380-559): identical grow/split/prune decisions, row order and
 * rows (the split normals use glibc's logf / cosf bit for bit); split k draws the CPU's pcg32
 * stream advanced by 12 * k draws. */
#define GSX_HIP_ADC_MAX_FIELDS 16
typedef struct gsx_hip_adc_params {
    int32_t algorithm; /* 0 GSX_ADC_ALGORITHM_DEFAULT, 1 GSX_ADC_ALGORITHM_ABSGS */
    float pruning_opacity_threshold;
    float opacity_clamp_value;
    float max_world_scale;
    float max_screen_scale;
    float duplicate_grad_threshold;
    float duplicate_scale_threshold;
    float duplicate_absgrad_threshold;
    float scene_scale;
    int64_t refine_every, start_refine, end_refine, max_num_gaussians, reset_every;
    /* GSX_ADC_ALGORITHM_MCMC (algorithm 2): position noise scale, target growth ratio per
     * refine, and the optimizer's current mean3d learning rate (the noise is scaled by it) */
    float noise_strength;
    float grow_ratio;
    float mean3d_learning_rate;
} gsx_hip_adc_params;

/* Rows of a Gaussian set on the device (the gsx_gs fields, gsx/include/gsx/gsx-core.h:286-308)
 * plus the Adam moments of each parameter field, all nullable except mean3d..sh0. Moment index
 * k follows the field order mean3d, rotation, logscale, opacity, sh0, sh1, sh2, sh3. */
typedef struct gsx_hip_gs_rows {
    int64_t count;
    int32_t sh_degree;
    float *mean3d, *rotation, *logscale, *opacity, *sh0, *sh1, *sh2, *sh3;
    float *grad_acc, *absgrad_acc, *visible_counter, *max_screen_radius;
    float *first_moment[8];
    float *second_moment[8];
} gsx_hip_gs_rows;

typedef struct gsx_hip_adc_context gsx_hip_adc_context;
/* The context owns the split RNG (pcg32 seeded (seed, seed), gsx/src/gsx-cpu/adc.c:466) and
 * the scratch buffers; the RNG advances across steps like the CPU adc object's. */
gsx_hip_status gsx_hip_adc_context_create(gsx_hip_adc_context** out_context, uint64_t seed);
gsx_hip_status gsx_hip_adc_context_destroy(gsx_hip_adc_context* context);
/* One gsx_adc_step at global_step. Growth appends rows in place, so every buffer of `rows` needs
 * `capacity` >= count + (max_num_gaussians - count) rows; when rows are pruned the compacted set
 * is written to `out` (same fields bound) and *out_result_in_out = 1, otherwise the result stays
 * in `rows`. The final count is stored in the result's `count`. out_counts[4] = pruned,
 * duplicated, grown (split), reset, as gsx_adc_result. The host waits once per refine, for the
 * counts (the compaction may still be running when the call returns, ordered on the stream).
 * MCMC (algorithm 2, gsx/src/gsx-cpu/adc/mcmc.c:345-766, dispatched as gsx-cpu/adc.c:515-547):
 * every step before end_refine moves each mean3d by opacity-gated noise shaped by its covariance
 * (6 draws per Gaussian); a refine relocates the rows whose sigmoid(opacity) <= the pruning
 * threshold onto live rows drawn in proportion to opacity and grows the set to
 * min(floor(count * (1 + grow_ratio)), max_num_gaussians) rows drawn the same way (appended in
 * place: `capacity` >= that count), with the opacity / scale correction of the relocated sources.
 * Rows are never removed, so the result stays in `rows`; out_counts = relocated (as pruned), 0,
 * relocated + appended (as grown), reset. The draw weights form their cumulative sums in float
 * in index order, with every rounding of the CPU and Metal backends' sequential sum, on the device;
 * the host waits once per refine, for the number of dead rows. */
gsx_hip_status gsx_hip_adc_step(gsx_hip_adc_context* context, const gsx_hip_adc_params* params, uint64_t global_step,
                                gsx_hip_gs_rows* rows, int64_t capacity, gsx_hip_gs_rows* out,
                                int32_t* out_result_in_out, int64_t* out_counts, hipStream_t stream);

/* Replaces gsx_cuda_gather_rows_kernel_launch (gsx/src/gsx-cuda/internal.h:396-405): out row r
 * = src row src_indices[r]; an index outside [0, src_row_count) sets *out_has_out_of_range
 * (a device int, may be null; the CPU returns GSX_ERROR_OUT_OF_RANGE, gsx-cpu/core.c:1322-1324).
 * No host synchronisation. */
gsx_hip_status gsx_hip_gather_rows_kernel_launch(const void* src, void* dst, int64_t row_bytes, int64_t row_count,
                                                 const int32_t* src_indices, int64_t src_row_count,
                                                 int* out_has_out_of_range, hipStream_t stream);

/* ---- label fields -------------------------------------------------------------------------------
 * Operators of language models beside a Gaussian scene (no counterpart in the reference): each
 * Gaussian or pixel holds the id of a code, the code's row is looked up, a head held in 8-bit blocks
 * turns rows into logits, and a teacher's top logits train them. Row types are GSX_HIP_DTYPE_F32,
 * BF16 or F16; strides count elements from row to row (>= the row's length, which lies
 * contiguously); sums and softmax statistics are float32 and a result is rounded once, to nearest
 * even. Pointers are aligned to their elements. Results do not depend on the order in which workgroups
 * run: two calls on the same inputs give the same bits. `temp` is device memory of the size that the
 * matching *_temp_bytes call gives (16-byte aligned; null where that is 0), used by work on `stream`
 * until the call's work is done; its contents need no initial value. Nothing here synchronises or
 * allocates, and every call may be captured into a graph. A call of no rows does nothing. */

/* out[i, 0..width) = scale * table[ids[i], 0..width). An id outside [0, table_rows) gives a row of zeros; if it is
 * not negative (a negative id stands for "no code"), *out_has_out_of_range (a device int, may be null) is set to 1. */
gsx_hip_status gsx_hip_lookup_forward(const void* table, int32_t table_type, int64_t table_rows, int64_t table_stride,
                                      const int32_t* ids, int64_t count, int64_t width, float scale, void* out,
                                      int32_t out_type, int64_t out_stride, int* out_has_out_of_range,
                                      hipStream_t stream);
/* grad_table[v, :] = scale * sum of grad_out[i, :] over the i with ids[i] = v (ids outside the table are left out). Rows
 * that no id names become 0; with accumulate != 0 the sums are added to what grad_table holds instead, and those rows
 * stay as they are. grad_table is float32 with rows table_stride apart. count may be at most 2^32 - 1,
 * table_rows 2^31 - 1. */
size_t gsx_hip_lookup_backward_temp_bytes(int64_t count, int64_t table_rows, int64_t width);
gsx_hip_status gsx_hip_lookup_backward(const void* grad_out, int32_t grad_type, int64_t grad_stride, const int32_t* ids,
                                       int64_t count, int64_t width, float scale, float* grad_table, int64_t table_rows,
                                       int64_t table_stride, int32_t accumulate, void* temp, hipStream_t stream);

/* Matrices in 8-bit blocks. A row of `cols` values is cut into blocks of 128; a block holds E4M3 values (OCP: 4 exponent
 * bits, 3 mantissa bits, largest 448) and one byte e + 127 for its scale 2^e, with e the least whole number >= -100 such that
 * max |x| <= 448 * 2^e over the block's finite x (e = 0 where that maximum is 0). Each x * 2^-e is rounded to the nearest
 * E4M3 value, ties to even; a non-finite x becomes NaN. Value rows are 16-byte aligned (stride a multiple of 16, >= cols),
 * exponent rows 4-byte aligned (stride a multiple of 4, >= ceil(cols / 128)). Products take values exactly for e from -100 to 119.
 * A row's last 16 bytes of values and 4 of exponents are read whole, but what lies between its last value and its stride is
 * never used as a value; quantize writes zeros there up to the last block's end.
 * transpose != 0 lays out the blocks of src^T (src_cols rows of src_rows values, blocks along src's rows). */
gsx_hip_status gsx_hip_blocks_quantize(const void* src, int32_t src_type, int64_t src_rows, int64_t src_cols,
                                       int64_t src_stride, int32_t transpose, uint8_t* values, int64_t values_stride,
                                       uint8_t* exponents, int64_t exponents_stride, hipStream_t stream);
/* out [m, n] = a b^T for block matrices a [m, k] and b [n, k]; m and n at most 2^31 - 1, k at most 2^27, value strides below
 * 2^28. */
size_t gsx_hip_blocks_matmul_temp_bytes(int64_t m, int64_t n, int64_t k);
gsx_hip_status gsx_hip_blocks_matmul(const uint8_t* a_values, int64_t a_values_stride, const uint8_t* a_exponents,
                                     int64_t a_exponents_stride, const uint8_t* b_values, int64_t b_values_stride,
                                     const uint8_t* b_exponents, int64_t b_exponents_stride, int64_t m, int64_t n,
                                     int64_t k, void* out, int32_t out_type, int64_t out_stride, void* temp,
                                     hipStream_t stream);
/* out [m, n] = blocks(x) w^T: the rows of x [m, k] are quantised as above and multiplied with the block matrix w [n, k].
 * Where that takes a workspace, w's value stride is below 2^28. */
size_t gsx_hip_linear_temp_bytes(int64_t m, int64_t n, int64_t k);
gsx_hip_status gsx_hip_linear_forward(const void* x, int32_t x_type, int64_t x_stride, const uint8_t* w_values,
                                      int64_t w_values_stride, const uint8_t* w_exponents, int64_t w_exponents_stride,
                                      int64_t m, int64_t n, int64_t k, void* out, int32_t out_type, int64_t out_stride,
                                      void* temp, hipStream_t stream);

/* Gradient of linear_forward's weight for the upstream grad_out [m, n]: grad_weight [n, k] (float32) = blocks(grad_out^T)
 * blocks(x^T)^T, both quantised along the m rows that are summed over (at most 2^27). (The gradient of x is linear_forward of
 * grad_out with the transposed weight's blocks.) */
size_t gsx_hip_linear_backward_weight_temp_bytes(int32_t x_type, int32_t grad_type, int64_t m, int64_t n, int64_t k);
gsx_hip_status gsx_hip_linear_backward_weight(const void* x, int32_t x_type, int64_t x_stride, const void* grad_out,
                                              int32_t grad_type, int64_t grad_stride, int64_t m, int64_t n, int64_t k,
                                              float* grad_weight, int64_t weight_stride, void* temp, hipStream_t stream);

/* Matrices in microscaled 4-bit blocks. A row of `cols` values is cut into blocks of 32; a block holds E2M1 values (OCP: 0, 0.5,
 * 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the first one in the low half, and one byte e + 127 for its scale 2^e, with
 * e the least whole number >= -100 such that max |x| <= 6 * 2^e over the block (e = 0 where that maximum is 0). Each x * 2^-e is
 * rounded to the nearest value, ties to the even code. A block that holds anything not finite gets the byte 255 and stands for NaN.
 * Blocks with any byte are read: 0 to 254 for 2^-127 to 2^127, 255 for NaN. Value rows are 16-byte aligned (stride in bytes, a
 * multiple of 16, >= ceil(cols / 2)), exponent rows 4-byte aligned (stride a multiple of 4, >= ceil(cols / 32)). A row's last
 * block and its last 4 exponents are read whole, but what lies behind its last value is never used as one; quantize writes zeros
 * up to the last block's end. */
gsx_hip_status gsx_hip_blocks4_quantize(const void* src, int32_t src_type, int64_t rows, int64_t cols, int64_t src_stride,
                                        uint8_t* values, int64_t values_stride, uint8_t* exponents, int64_t exponents_stride,
                                        hipStream_t stream);
/* out [rows, cols] = what the blocks stand for (exact in float32 and bfloat16 within their range). */
gsx_hip_status gsx_hip_blocks4_expand(const uint8_t* values, int64_t values_stride, const uint8_t* exponents,
                                      int64_t exponents_stride, int64_t rows, int64_t cols, void* out, int32_t out_type,
                                      int64_t out_stride, hipStream_t stream);
/* out [m, n] = a b^T for 4-bit block matrices a [m, k] and b [n, k]; m and n at most 2^31 - 1, k at most 2^27, value strides below
 * 2^28, exponent strides below 2^26. */
size_t gsx_hip_blocks4_matmul_temp_bytes(int64_t m, int64_t n, int64_t k);
gsx_hip_status gsx_hip_blocks4_matmul(const uint8_t* a_values, int64_t a_values_stride, const uint8_t* a_exponents,
                                      int64_t a_exponents_stride, const uint8_t* b_values, int64_t b_values_stride,
                                      const uint8_t* b_exponents, int64_t b_exponents_stride, int64_t m, int64_t n, int64_t k,
                                      void* out, int32_t out_type, int64_t out_stride, void* temp, hipStream_t stream);
/* out [m, n] = blocks(x) w^T: the rows of x [m, k] are quantised to 4-bit blocks as above and multiplied with the 4-bit block
 * matrix w [n, k]. Where that takes a workspace, w's value stride is below 2^28, its exponent stride below 2^26. */
size_t gsx_hip_linear4_temp_bytes(int64_t m, int64_t n, int64_t k);
gsx_hip_status gsx_hip_linear4_forward(const void* x, int32_t x_type, int64_t x_stride, const uint8_t* w_values,
                                       int64_t w_values_stride, const uint8_t* w_exponents, int64_t w_exponents_stride,
                                       int64_t m, int64_t n, int64_t k, void* out, int32_t out_type, int64_t out_stride,
                                       void* temp, hipStream_t stream);

/* Distillation from a teacher's top logits. Row r of `logits` [rows, vocab] is the student's z; teacher_ids and teacher_logits
 * [rows, top] (rows teacher_stride apart, top at most 1024) name the teacher's entries. An entry counts if its id lies in
 * [0, vocab) and its logit is not -inf. With T the temperature (1e-6 to 1e6), p = softmax(t / T) over the entries that
 * count, q = softmax(z / T) over the whole row and w = row_weight[r] (null: 1):
 *   loss[r] = w T^2 sum_k p_k (log p_k - log q_{id_k}),   dz_j = c w T (q_j - sum of p_k over the entries with id_k = j)
 * A row of weight 0 or without an entry that counts has loss 0 and gradient 0 whatever its logits are. A logit of -inf has
 * q = 0. A row of nothing but -inf has no distribution: loss +inf (w > 0), gradient 0. NaN or +inf in a row's logits gives NaN.
 * forward writes loss [rows], row_stats [rows][2] (max z and the sum of exp((z - max z) / T); for the backward) and, with
 * c = grad_scale, the gradient (logits' type); each of the three may be null. backward writes the gradient with
 * c = grad_scale * row_grad[r] (null: 1) from a forward's row_stats of the same logits and temperature. The gradient may not
 * overlap the logits. */
size_t gsx_hip_distill_temp_bytes(int64_t rows, int64_t vocab);
gsx_hip_status gsx_hip_distill_forward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                       int64_t vocab, const int32_t* teacher_ids, const float* teacher_logits,
                                       int64_t teacher_stride, int32_t top, float temperature, const float* row_weight,
                                       float* loss, float* row_stats, void* grad_logits, int64_t grad_stride,
                                       float grad_scale, void* temp, hipStream_t stream);
gsx_hip_status gsx_hip_distill_backward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                        int64_t vocab, const int32_t* teacher_ids, const float* teacher_logits,
                                        int64_t teacher_stride, int32_t top, float temperature, const float* row_weight,
                                        const float* row_stats, const float* row_grad, float grad_scale,
                                        void* grad_logits, int64_t grad_stride, hipStream_t stream);

/* Log probabilities of given labels, entropies and top alternatives. Row r of `logits` [rows, vocab] is z; with T the
 * temperature (1e-6 to 1e6), q = softmax(z / T) and id = ids[r]:
 *   chosen[r] = log q_id (0 where ids is null or id lies outside [0, vocab): a row without a label),
 *   entropy[r] = -sum_j q_j log q_j (a logit of -inf has q = 0 and adds nothing),
 *   top_ids, top_log_probs [rows, top] (contiguous, top at most 64 and vocab): the largest logits and their log q, of equal ones
 *   the lowest index first (-0 equals 0); a logit of -inf is no alternative: where there are fewer, the id is -1 and log q -inf,
 *   row_stats [rows][3]: max z, the sum of exp((z - max z) / T), the entropy; for the gradient,
 *   dz_j = (gl (delta_{j,id} - q_j) - gh q_j (log q_j + entropy)) / T with gl = grad_scale * row_grad[r] (null: 1; 0 for a row
 *   without a label) and gh = entropy_scale * entropy_grad[r] (null: 1), in the logits' type.
 * A row with gl = gh = 0 has gradient 0 whatever its logits are. A row of nothing but -inf has no distribution: chosen -inf (if
 * it has a label), entropy 0, gradient 0, no alternatives. NaN or +inf in a row's logits gives NaN for chosen, entropy and log
 * q; alternatives are then ordered NaN, +inf, the others. Any of chosen, entropy and row_stats may be null, ids too; a gradient
 * from forward (grad_logits not null) needs row_stats. The gradient may not overlap the logits. */
size_t gsx_hip_log_probs_temp_bytes(int64_t rows, int64_t vocab, int32_t top);
gsx_hip_status gsx_hip_log_probs_forward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                         int64_t vocab, const int32_t* ids, float temperature, float* chosen,
                                         float* entropy, float* row_stats, int32_t top, int32_t* top_ids,
                                         float* top_log_probs, void* grad_logits, int64_t grad_stride,
                                         const float* row_grad, float grad_scale, const float* entropy_grad,
                                         float entropy_scale, void* temp, hipStream_t stream);
gsx_hip_status gsx_hip_log_probs_backward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                          int64_t vocab, const int32_t* ids, float temperature, const float* row_stats,
                                          const float* row_grad, float grad_scale, const float* entropy_grad,
                                          float entropy_scale, void* grad_logits, int64_t grad_stride, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GSX_HIP_H */

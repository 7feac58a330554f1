"""ctypes declarations of the C ABI in include/homura_cuda*.h.

GENERATED by homura_b200/gen_cuda_ffi.py; do not edit (the tests run the generator with --check).
"""
from ctypes import (CFUNCTYPE, POINTER, Structure, c_char, c_char_p, c_double, c_float, c_int32, c_int64, c_uint8,
                    c_uint32, c_uint64, c_void_p)

HMC_OK = 0
HMC_OUT_OF_MEMORY = 1
HMC_INVALID = 2
HMC_CUDA_ERROR = 3
HMC_INTERNAL_ERROR = 4
HMC_NAME_LEN = 256
HMC_ARCH_LEN = 64
HMC_BOOL = 0
HMC_U8 = 1
HMC_I8 = 2
HMC_I16 = 3
HMC_I32 = 4
HMC_I64 = 5
HMC_F16 = 6
HMC_BF16 = 7
HMC_F32 = 8
HMC_F64 = 9
HMC_MAX_DIMS = 25
HMC_UNARY_NEG = 0
HMC_UNARY_ABS = 1
HMC_UNARY_SIGN = 2
HMC_UNARY_RELU = 3
HMC_UNARY_EXP = 4
HMC_UNARY_LOG = 5
HMC_UNARY_SQRT = 6
HMC_UNARY_RSQRT = 7
HMC_UNARY_RECIPROCAL = 8
HMC_UNARY_SIN = 9
HMC_UNARY_COS = 10
HMC_UNARY_ERF = 11
HMC_UNARY_TANH = 12
HMC_UNARY_SIGMOID = 13
HMC_UNARY_LOG_SIGMOID = 14
HMC_UNARY_SILU = 15
HMC_UNARY_GELU = 16
HMC_UNARY_GELU_TANH = 17
HMC_UNARY_LOGICAL_NOT = 18
HMC_UNARY_COUNT = 19
HMC_BINARY_ADD = 0
HMC_BINARY_SUB = 1
HMC_BINARY_MUL = 2
HMC_BINARY_DIV = 3
HMC_BINARY_POW = 4
HMC_BINARY_MAXIMUM = 5
HMC_BINARY_MINIMUM = 6
HMC_BINARY_GREATER = 7
HMC_BINARY_GREATER_EQUAL = 8
HMC_BINARY_LESS = 9
HMC_BINARY_LESS_EQUAL = 10
HMC_BINARY_EQUAL = 11
HMC_BINARY_NOT_EQUAL = 12
HMC_BINARY_LOGICAL_AND = 13
HMC_BINARY_LOGICAL_OR = 14
HMC_BINARY_COUNT = 15
HMC_FUSED_SCALED_ADD = 0
HMC_FUSED_LERP = 1
HMC_FUSED_ADDCMUL = 2
HMC_FUSED_ADDCDIV = 3
HMC_REDUCE_SUM = 0
HMC_REDUCE_PROD = 1
HMC_REDUCE_MEAN = 2
HMC_REDUCE_MAX = 3
HMC_REDUCE_MIN = 4
HMC_REDUCE_ALL = 5
HMC_REDUCE_ANY = 6
HMC_RANDOM_INT_TILE = 256
HMC_NOALLOC_SCRATCH_BYTES = 1048576
HMC_MEM_OK = 0
HMC_MEM_OUT_OF_MEMORY = 1
HMC_MEM_FAILED = 2
HMC_COMM_ID_BYTES = 128
HMC_RECURRENCE_SIGMOID = 1
HMC_RECURRENCE_COMPLEMENT = 2
HMC_RECURRENCE_REVERSE = 4
HMC_ACTIVATION_NONE = -1


class hmc_device_properties(Structure):
    _fields_ = [
        ("name", c_char * 256),
        ("arch", c_char * 64),
        ("multiprocessor_count", c_int32),
        ("warp_size", c_int32),
        ("total_memory", c_uint64),
    ]


class hmc_tensor_desc(Structure):
    _fields_ = [
        ("data", c_void_p),
        ("offset", c_int64),
        ("dtype", c_int32),
        ("ndim", c_int32),
        ("sizes", c_int64 * 25),
        ("strides", c_int64 * 25),
    ]


class hmc_adamw_scalars(Structure):
    _fields_ = [
        ("decay", c_double),
        ("lerp_coeff", c_double),
        ("lerp_small", c_int32),
        ("has_decay", c_int32),
        ("beta2", c_double),
        ("one_minus_beta2", c_double),
        ("bias2_sqrt", c_double),
        ("eps", c_double),
        ("neg_step_size", c_double),
    ]


class hmc_adamw_tensor(Structure):
    _fields_ = [
        ("param", c_void_p),
        ("grad", c_void_p),
        ("exp_avg", c_void_p),
        ("exp_avg_sq", c_void_p),
        ("n", c_int64),
    ]


class hmc_abi_info(Structure):
    _fields_ = [
        ("abi_info_size", c_uint32),
        ("properties_size", c_uint32),
        ("properties_align", c_uint32),
        ("properties_offsets", c_uint32 * 5),
        ("status_values", c_int32 * 5),
        ("name_len", c_int32),
        ("arch_len", c_int32),
        ("desc_size", c_uint32),
        ("desc_align", c_uint32),
        ("desc_offsets", c_uint32 * 6),
        ("dtype_values", c_int32 * 10),
        ("max_dims", c_int32),
        ("adamw_scalars_size", c_uint32),
        ("adamw_scalars_align", c_uint32),
    ]


class hmc_memory_ops(Structure):
    _fields_ = [
        ("user", c_void_p),
        ("malloc_fn", CFUNCTYPE(c_int32, c_void_p, c_uint64, POINTER(c_uint64))),
        ("free_fn", CFUNCTYPE(c_int32, c_void_p, c_uint64)),
        ("synchronize_fn", CFUNCTYPE(c_int32, c_void_p)),
    ]


class hmc_memory_stats(Structure):
    _fields_ = [
        ("allocated", c_uint64),
        ("reserved", c_uint64),
        ("peak", c_uint64),
    ]


# name -> (restype, [(argtype, argname), ...])
FUNCTIONS = {
    "hmc_last_error": (c_char_p, []),
    "hmc_device_count": (c_int32, [(POINTER(c_int32), "count")]),
    "hmc_device_properties_get": (c_int32, [(c_int32, "device"), (POINTER(hmc_device_properties), "out")]),
    "hmc_mem_get_info": (c_int32, [(c_int32, "device"), (POINTER(c_uint64), "free_bytes"), (POINTER(c_uint64), "total_bytes")]),
    "hmc_context_create": (c_int32, [(c_int32, "device"), (POINTER(c_void_p), "out")]),
    "hmc_context_destroy": (c_int32, [(c_void_p, "ctx")]),
    "hmc_context_synchronize": (c_int32, [(c_void_p, "ctx")]),
    "hmc_malloc": (c_int32, [(c_int32, "device"), (c_uint64, "nbytes"), (POINTER(c_void_p), "out")]),
    "hmc_free": (c_int32, [(c_int32, "device"), (c_void_p, "ptr")]),
    "hmc_memset": (c_int32, [(c_void_p, "ctx"), (c_void_p, "ptr"), (c_uint8, "value"), (c_uint64, "nbytes")]),
    "hmc_copy_to_host": (c_int32, [(c_void_p, "ctx"), (c_void_p, "dst"), (c_void_p, "src"), (c_uint64, "nbytes")]),
    "hmc_copy_from_host": (c_int32, [(c_void_p, "ctx"), (c_void_p, "dst"), (c_void_p, "src"), (c_uint64, "nbytes")]),
    "hmc_copy_device": (c_int32, [(c_void_p, "ctx"), (c_void_p, "dst"), (c_void_p, "src"), (c_uint64, "nbytes")]),
    "hmc_copy": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "dst"), (POINTER(hmc_tensor_desc), "src")]),
    "hmc_fill": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "dst"), (c_uint64, "bits")]),
    "hmc_unary": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src")]),
    "hmc_binary": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "a"), (POINTER(hmc_tensor_desc), "b")]),
    "hmc_binary_constant": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "a"), (c_uint64, "bits"), (c_int32, "constant_first")]),
    "hmc_binary_scalar": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "a"), (c_double, "s"), (c_int32, "scalar_first")]),
    "hmc_fused": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "a"), (POINTER(hmc_tensor_desc), "b"), (POINTER(hmc_tensor_desc), "c"), (c_double, "coefficient"), (c_int32, "small")]),
    "hmc_where": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "cond"), (POINTER(hmc_tensor_desc), "x"), (POINTER(hmc_tensor_desc), "y")]),
    "hmc_where_constant": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "cond"), (POINTER(hmc_tensor_desc), "x"), (c_uint64, "x_bits"), (POINTER(hmc_tensor_desc), "y"), (c_uint64, "y_bits")]),
    "hmc_reduce_workspace": (c_int32, [(POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (c_int32, "var"), (POINTER(c_int64), "bytes")]),
    "hmc_reduce": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_var": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (c_double, "correction"), (c_int32, "take_sqrt"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_arg_reduce": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "values"), (POINTER(hmc_tensor_desc), "indices"), (POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (c_int32, "is_max"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_softmax_workspace": (c_int32, [(POINTER(hmc_tensor_desc), "src_rows"), (c_int64, "n"), (c_int64, "src_stride"), (POINTER(c_int64), "bytes")]),
    "hmc_softmax": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out_rows"), (POINTER(hmc_tensor_desc), "src_rows"), (c_int64, "n"), (c_int64, "out_stride"), (c_int64, "src_stride"), (c_int32, "log"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_random_uniform": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (c_uint64, "seed"), (c_uint64, "offset"), (c_double, "from"), (c_double, "to")]),
    "hmc_random_normal": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (c_uint64, "seed"), (c_uint64, "offset"), (c_double, "mean"), (c_double, "std")]),
    "hmc_random_int": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (c_uint64, "seed"), (c_uint64, "offset"), (c_uint64, "blocks"), (c_int64, "low"), (c_uint64, "range"), (c_uint64, "threshold"), (c_void_p, "workspace")]),
    "hmc_triangle": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (c_int64, "diagonal"), (c_int32, "upper")]),
    "hmc_flip": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src")]),
    "hmc_addr": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "v1"), (POINTER(hmc_tensor_desc), "v2"), (POINTER(hmc_tensor_desc), "input"), (c_double, "alpha"), (c_double, "beta"), (c_int64, "alpha_int"), (c_int64, "beta_int")]),
    "hmc_exclusive_cumprod": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out_lines"), (POINTER(hmc_tensor_desc), "src_lines"), (c_int64, "n"), (c_int64, "out_stride"), (c_int64, "src_stride"), (c_int32, "reverse")]),
    "hmc_index_check": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "index"), (c_int64, "low"), (c_int64, "high"), (c_int32, "has_exempt"), (c_int64, "exempt"), (POINTER(c_uint64), "slot")]),
    "hmc_index_select": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "index"), (c_int32, "dim"), (c_int32, "wrap_negative")]),
    "hmc_gather": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "index"), (c_int32, "dim")]),
    "hmc_index_overwrite_workspace": (c_int32, [(c_int64, "size"), (POINTER(c_int64), "bytes")]),
    "hmc_index_overwrite": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "positions"), (c_int32, "dim"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_index_add_workspace": (c_int32, [(c_int64, "m"), (c_int64, "size"), (POINTER(c_int64), "bytes")]),
    "hmc_index_add": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "index"), (c_int32, "dim"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_scatter_add_workspace": (c_int32, [(c_int64, "n"), (POINTER(c_int64), "bytes")]),
    "hmc_scatter_add": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "index"), (c_int32, "dim"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_index_positions": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "coord"), (c_int64, "size"), (c_int64, "stride"), (c_int32, "first")]),
    "hmc_mask_workspace": (c_int32, [(c_int64, "n"), (POINTER(c_int64), "bytes"), (POINTER(c_int64), "total_word")]),
    "hmc_mask_count": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "mask"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_mask_coordinates": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "mask"), (c_void_p, "workspace"), (c_int64, "workspace_bytes"), (POINTER(hmc_tensor_desc), "out")]),
    "hmc_reduce_noalloc": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red")]),
    "hmc_binary_promoted": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "a"), (POINTER(hmc_tensor_desc), "b")]),
    "hmc_unary_binary_binary": (c_int32, [(c_void_p, "ctx"), (c_int32, "unary_op"), (c_int32, "first_op"), (c_int32, "second_op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "x"), (POINTER(hmc_tensor_desc), "b"), (POINTER(hmc_tensor_desc), "c")]),
    "hmc_adamw_step": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "param"), (POINTER(hmc_tensor_desc), "grad"), (POINTER(hmc_tensor_desc), "exp_avg"), (POINTER(hmc_tensor_desc), "exp_avg_sq"), (POINTER(hmc_adamw_scalars), "scalars")]),
    "hmc_adamw_step_many_workspace": (c_int32, [(c_int32, "dtype"), (POINTER(hmc_adamw_tensor), "tensors"), (c_int64, "count"), (c_int32, "with_grad_sq"), (POINTER(c_int64), "bytes")]),
    "hmc_adamw_step_many": (c_int32, [(c_void_p, "ctx"), (c_int32, "dtype"), (POINTER(hmc_adamw_tensor), "tensors"), (c_int64, "count"), (POINTER(hmc_adamw_scalars), "scalars"), (POINTER(c_double), "grad_sq"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_host_alloc": (c_int32, [(c_uint64, "nbytes"), (POINTER(c_void_p), "out")]),
    "hmc_host_free": (c_int32, [(c_void_p, "ptr")]),
    "hmc_context_stream": (c_int32, [(c_void_p, "ctx"), (POINTER(c_void_p), "stream")]),
    "hmc_event_create": (c_int32, [(c_void_p, "ctx"), (POINTER(c_void_p), "out")]),
    "hmc_event_record": (c_int32, [(c_void_p, "ctx"), (c_void_p, "ev")]),
    "hmc_event_elapsed_ms": (c_int32, [(c_void_p, "start"), (c_void_p, "stop"), (POINTER(c_float), "ms")]),
    "hmc_event_destroy": (c_int32, [(c_void_p, "ev")]),
    "hmc_built_archs": (c_char_p, []),
    "hmc_abi_check": (None, [(POINTER(hmc_abi_info), "out")]),
    "hmc_test_fail_stream_create": (None, [(c_int32, "n")]),
    "hmc_test_fail_after_probe": (None, [(c_int32, "n")]),
    "hmc_test_fail_properties": (None, [(c_int32, "n")]),
    "hmc_test_fail_data": (None, [(c_int32, "n"), (c_int32, "out_of_memory")]),
    "hmc_test_reduce_plan": (c_int32, [(POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (POINTER(c_int64), "kind"), (POINTER(c_int64), "splits"), (POINTER(c_int64), "chunk")]),
    "hmc_test_softmax_plan": (c_int32, [(POINTER(hmc_tensor_desc), "src_rows"), (c_int64, "n"), (c_int64, "src_stride"), (POINTER(c_int32), "kind"), (POINTER(c_int32), "group"), (POINTER(c_int32), "cache")]),
    "hmc_test_index_value": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "index"), (POINTER(c_uint64), "slot")]),
    "hmc_test_wait_limit": (None, [(c_int32, "polls")]),
    "hmc_test_live_streams": (c_int32, []),
    "hmc_test_current_device": (c_int32, [(POINTER(c_int32), "device")]),
    "hmc_test_set_current_device": (c_int32, [(c_int32, "device")]),
    "hmc_test_fail": (c_int32, [(c_char_p, "message")]),
    "hmc_allocator_create": (c_int32, [(POINTER(hmc_memory_ops), "ops"), (POINTER(c_void_p), "out")]),
    "hmc_allocator_create_cuda": (c_int32, [(c_void_p, "ctx"), (POINTER(c_void_p), "out")]),
    "hmc_allocator_destroy": (c_int32, [(c_void_p, "a")]),
    "hmc_allocator_allocate": (c_int32, [(c_void_p, "a"), (c_uint64, "nbytes"), (POINTER(c_uint64), "addr"), (POINTER(c_uint64), "size")]),
    "hmc_allocator_release": (c_int32, [(c_void_p, "a"), (c_uint64, "addr")]),
    "hmc_allocator_empty_cache": (c_int32, [(c_void_p, "a")]),
    "hmc_allocator_stats": (c_int32, [(c_void_p, "a"), (POINTER(hmc_memory_stats), "out")]),
    "hmc_allocator_reset_peak": (c_int32, [(c_void_p, "a")]),
    "hmc_allocator_rounded": (c_int32, [(c_uint64, "nbytes"), (POINTER(c_uint64), "size"), (POINTER(c_int32), "is_small")]),
    "hmc_allocator_set_callback_error": (None, [(c_char_p, "message")]),
    "hmc_reduce_partial": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(c_double), "partial"), (POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_shard_combine_float": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(c_double), "gathered"), (c_int32, "ranks"), (c_int64, "nout"), (c_int64, "total_count")]),
    "hmc_shard_combine_int": (c_int32, [(c_void_p, "ctx"), (c_int32, "op"), (POINTER(hmc_tensor_desc), "out"), (POINTER(c_int64), "gathered"), (c_int32, "ranks"), (c_int64, "nout")]),
    "hmc_shard_combine_extreme": (c_int32, [(c_void_p, "ctx"), (c_int32, "is_max"), (POINTER(hmc_tensor_desc), "out_values"), (POINTER(hmc_tensor_desc), "out_indices"), (c_void_p, "gathered_values"), (c_int32, "dtype"), (POINTER(c_int64), "gathered_indices"), (POINTER(c_int64), "index_offsets"), (c_int32, "ranks"), (c_int64, "nout")]),
    "hmc_shard_combine_means": (c_int32, [(c_void_p, "ctx"), (POINTER(c_double), "means"), (POINTER(c_double), "gathered"), (c_int32, "ranks"), (c_int64, "nout"), (c_int64, "total_count")]),
    "hmc_var_partial": (c_int32, [(c_void_p, "ctx"), (POINTER(c_double), "partial"), (POINTER(hmc_tensor_desc), "kept"), (POINTER(hmc_tensor_desc), "red"), (POINTER(c_double), "means"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_shard_combine_var": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(c_double), "gathered"), (c_int32, "ranks"), (c_int64, "nout"), (c_int64, "total_count"), (c_double, "correction"), (c_int32, "take_sqrt")]),
    "hmc_comm_unique_id": (c_int32, [(POINTER(c_uint8), "id")]),
    "hmc_comm_create": (c_int32, [(c_void_p, "ctx"), (c_int32, "ranks"), (c_int32, "rank"), (POINTER(c_uint8), "id"), (POINTER(c_void_p), "out")]),
    "hmc_comm_set_timeout": (c_int32, [(c_void_p, "comm"), (c_int64, "milliseconds")]),
    "hmc_comm_destroy": (c_int32, [(c_void_p, "comm")]),
    "hmc_comm_allgather": (c_int32, [(c_void_p, "comm"), (c_void_p, "send"), (c_void_p, "recv"), (c_uint64, "bytes")]),
    "hmc_comm_wait": (c_int32, [(c_void_p, "comm")]),
    "hmc_comm_abort": (c_int32, [(c_void_p, "comm")]),
    "hmc_linear_recurrence": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "gate"), (POINTER(hmc_tensor_desc), "x"), (POINTER(hmc_tensor_desc), "initial"), (POINTER(hmc_tensor_desc), "last"), (c_int32, "flags")]),
    "hmc_linear_recurrence_backward": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "dgate"), (POINTER(hmc_tensor_desc), "dx"), (POINTER(hmc_tensor_desc), "dinitial"), (POINTER(hmc_tensor_desc), "gate"), (POINTER(hmc_tensor_desc), "x"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "initial"), (POINTER(hmc_tensor_desc), "dout"), (POINTER(hmc_tensor_desc), "dlast"), (c_int32, "flags")]),
    "hmc_group_norm_workspace": (c_int32, [(POINTER(hmc_tensor_desc), "src"), (c_int32, "groups"), (c_int32, "backward"), (POINTER(c_int64), "bytes")]),
    "hmc_group_norm": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "weight"), (POINTER(hmc_tensor_desc), "bias"), (POINTER(hmc_tensor_desc), "mean"), (POINTER(hmc_tensor_desc), "rstd"), (c_int32, "groups"), (c_double, "eps"), (c_int32, "activation"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_group_norm_backward": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "dsrc"), (POINTER(hmc_tensor_desc), "dweight"), (POINTER(hmc_tensor_desc), "dbias"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "dout"), (POINTER(hmc_tensor_desc), "mean"), (POINTER(hmc_tensor_desc), "rstd"), (POINTER(hmc_tensor_desc), "weight"), (POINTER(hmc_tensor_desc), "bias"), (c_int32, "groups"), (c_int32, "activation"), (c_void_p, "workspace"), (c_int64, "workspace_bytes")]),
    "hmc_dropout": (c_int32, [(c_void_p, "ctx"), (POINTER(hmc_tensor_desc), "out"), (POINTER(hmc_tensor_desc), "src"), (POINTER(hmc_tensor_desc), "residual"), (c_double, "p"), (c_uint64, "seed"), (c_uint64, "offset")]),
}


def bind(lib, only=None):
    """Sets restype/argtypes on every declared function `lib` exports; returns the names bound."""
    bound = []
    for name, (res, params) in FUNCTIONS.items():
        if only is not None and name not in only:
            continue
        fn = getattr(lib, name, None)
        if fn is None:
            continue
        fn.restype = res
        fn.argtypes = [t for t, _ in params]
        bound.append(name)
    return bound

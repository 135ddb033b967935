"""ctypes view of the training operators' C ABI (include/mr3d.h), for the tests of its refusals."""
import ctypes

P, I, LL, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_size_t


class Matrix(ctypes.Structure):
    _fields_ = [('in_', P), ('out', P), ('rows', LL), ('cols', LL), ('in_row_stride', LL), ('in_col_stride', LL), ('dtype', I), ('reserved', I)]


class LinearCe(ctypes.Structure):
    _fields_ = [(n, P) for n in ('x', 'weight', 'bias', 'labels', 'row_weight', 'avg_factor_dev', 'valid_rows_dev', 'loss', 'dx', 'dweight', 'dbias')] + \
               [(n, LL) for n in ('x_stride', 'weight_stride', 'ignore_index')] + [('avg_factor', F)] + \
               [(n, I) for n in ('rows', 'hidden', 'classes', 'dtype', 'param_dtype', 'want_dx', 'want_dweight', 'want_dbias')]


class Span(ctypes.Structure):
    _fields_ = [('data', P), ('count', LL), ('dtype', I), ('reserved', I)]


def lib():
    import mr3d_amd
    L = mr3d_amd._hip.lib()
    for name, res, args in (('mr3d_linear_cross_entropy_workspace_bytes', Z, [P]), ('mr3d_linear_cross_entropy', I, [P, P, Z, P]),
                            ('mr3d_scale_by', I, [P, I, P, P]), ('mr3d_orthogonalize_workspace_bytes', Z, [P, I]),
                            ('mr3d_orthogonalize', I, [P, I, I, F, F, F, F, P, Z, P]), ('mr3d_layer_norm_workspace_bytes', Z, [LL, I, I]),
                            ('mr3d_layer_norm_forward', I, [P, LL, P, P, P, P, P, LL, I, F, I, I, P]),
                            ('mr3d_layer_norm_backward', I, [P, LL, P, LL, P, P, P, P, P, P, LL, I, I, I, P, Z, P])):
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    return L

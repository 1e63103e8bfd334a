"""ctypes binding of libdp_gbdt (include/dp_gbdt.h).

Mirrors the call sequence the reference trainer issues through the XGBoost C
API (native/class_native_training.cuh:47-70): a DMatrix over borrowed CUDA
fp32 memory, a Booster configured with XGBoosterSetParam, one
XGBoosterUpdateOneIter per round, then the JSON configuration and model.
Device memory is supplied by the caller (here: torch CUDA tensors or raw
pointers); the library itself has no CPU training path and raises if its
shared object is missing.
"""
from __future__ import annotations

import ctypes as C
import json
import math
import pathlib
from typing import Any, Iterable, NamedTuple

HERE = pathlib.Path(__file__).resolve().parent
LIB_PATH = HERE / "libdp_gbdt.so"

EXPORTED = [
    "XGBoostVersion", "XGBuildInfo", "XGBGetLastError", "XGDMatrixCreateFromCudaArrayInterface",
    "XGDMatrixCreateFromDense",
    "XGDMatrixSetInfoFromInterface", "XGDMatrixSetFloatInfo", "XGDMatrixNumRow", "XGDMatrixNumCol",
    "XGDMatrixFree", "XGBoosterCreate", "XGBoosterFree", "XGBoosterSetParam", "XGBoosterUpdateOneIter",
    "XGBoosterTrainOneIter", "XGBoosterBoostedRounds", "XGBoosterSaveJsonConfig", "XGBoosterSaveModel", "XGBoosterSaveModelToBuffer",
    "XGBoosterLoadModelFromBuffer", "XGBoosterLoadModel", "XGBoosterSlice", "XGBoosterGetNumFeature",
    "XGBoosterPredictFromCudaArray",
    "dp_comm_unique_id", "dp_comm_create", "dp_comm_free", "dp_comm_set_timeout", "dp_comm_reduce_scatter_hist", "dp_release_cached_memory", "dp_booster_set_comm", "dp_booster_set_profiling",
    "dp_booster_profile", "dp_booster_margins", "dp_booster_train_margin", "dp_launch_count", "dp_quantile_cuts", "dp_bin_matrix",
    "dp_gradients", "dp_hist_build", "dp_hist_build_noalloc", "dp_probe_hist_atomics", "dp_csv_decode", "dp_csv_shape", "dp_csv_data", "dp_csv_metadata", "dp_csv_copy", "dp_csv_free", "dp_csv_parse_feature", "dp_quantize_gh", "dp_hist_prepare", "dp_hist_run", "dp_hist_free", "dp_eval_splits",
    "dp_log_prob", "dp_log_prob_grad", "dp_policy_loss", "dp_preference_loss", "dp_preference_prepare",
    "dp_preference_run", "dp_preference_free",
]

OBJECTIVE_IDS = {"reg:squarederror": 0, "binary:logistic": 1, "multi:softprob": 2, "multi:softmax": 3}


class DPError(RuntimeError):
    pass


_lib = None


def lib() -> C.CDLL:
    """Loads libdp_gbdt.so (built by `make -C decision-programs_b200`)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise DPError(f"libdp_gbdt.so is missing at {LIB_PATH}; build it with __graft_entry__.build()")
        L = C.CDLL(str(LIB_PATH))
        P, u64, i32, f32, f64 = C.c_void_p, C.c_uint64, C.c_int, C.c_float, C.c_double
        L.XGBoostVersion.restype = None
        L.XGBoostVersion.argtypes = [C.POINTER(i32)] * 3
        L.XGBuildInfo.argtypes = [C.POINTER(C.c_char_p)]
        L.XGBGetLastError.restype = C.c_char_p
        L.XGDMatrixCreateFromCudaArrayInterface.argtypes = [C.c_char_p, C.c_char_p, C.POINTER(P)]
        L.XGDMatrixCreateFromDense.argtypes = [C.c_char_p, C.c_char_p, C.POINTER(P)]
        L.XGDMatrixSetInfoFromInterface.argtypes = [P, C.c_char_p, C.c_char_p]
        L.XGDMatrixSetFloatInfo.argtypes = [P, C.c_char_p, P, u64]
        L.XGDMatrixNumRow.argtypes = [P, C.POINTER(u64)]
        L.XGDMatrixNumCol.argtypes = [P, C.POINTER(u64)]
        L.XGDMatrixFree.argtypes = [P]
        L.XGBoosterCreate.argtypes = [C.POINTER(P), u64, C.POINTER(P)]
        L.XGBoosterFree.argtypes = [P]
        L.XGBoosterSetParam.argtypes = [P, C.c_char_p, C.c_char_p]
        L.XGBoosterUpdateOneIter.argtypes = [P, i32, P]
        L.XGBoosterTrainOneIter.argtypes = [P, P, i32, C.c_char_p, C.c_char_p]
        L.dp_booster_train_margin.argtypes = [P, P, C.POINTER(u64), C.POINTER(u64), C.POINTER(P)]
        L.XGBoosterBoostedRounds.argtypes = [P, C.POINTER(i32)]
        L.XGBoosterSaveJsonConfig.argtypes = [P, C.POINTER(u64), C.POINTER(C.c_char_p)]
        L.XGBoosterSaveModel.argtypes = [P, C.c_char_p]
        L.XGBoosterSaveModelToBuffer.argtypes = [P, C.c_char_p, C.POINTER(u64), C.POINTER(C.c_void_p)]
        L.XGBoosterLoadModelFromBuffer.argtypes = [P, C.c_char_p, u64]
        L.XGBoosterLoadModel.argtypes = [P, C.c_char_p]
        L.XGBoosterSlice.argtypes = [P, i32, i32, i32, C.POINTER(P)]
        L.XGBoosterGetNumFeature.argtypes = [P, C.POINTER(u64)]
        L.XGBoosterPredictFromCudaArray.argtypes = [P, C.c_char_p, C.c_char_p, P, C.POINTER(C.POINTER(u64)),
                                                    C.POINTER(u64), C.POINTER(C.POINTER(f32))]
        L.dp_comm_unique_id.argtypes = [P]
        L.dp_comm_create.argtypes = [P, i32, i32, i32, C.POINTER(P)]
        L.dp_comm_free.argtypes = [P]
        L.dp_comm_set_timeout.argtypes = [P, C.c_int64]
        L.dp_comm_reduce_scatter_hist.argtypes = [P, P, P, u64, P]
        L.dp_release_cached_memory.argtypes = []
        L.dp_booster_set_comm.argtypes = [P, P]
        L.dp_booster_set_profiling.argtypes = [P, i32]
        L.dp_booster_profile.argtypes = [P, C.POINTER(C.c_char_p)]
        L.dp_booster_margins.argtypes = [P, P, u64]
        L.dp_launch_count.restype = u64
        L.dp_launch_count.argtypes = []
        L.dp_quantile_cuts.argtypes = [P, u64, C.c_uint32, u64, i32, P, P, P, P]
        L.dp_bin_matrix.argtypes = [P, u64, C.c_uint32, u64, P, P, P, u64, P]
        L.dp_gradients.argtypes = [i32, i32, P, P, u64, P, P, P]
        L.dp_hist_build.argtypes = [P, u64, C.c_uint32, C.c_int32, P, P, P, P, C.c_int32, f32, f32, P, P]
        L.dp_hist_build_noalloc.argtypes = [P, u64, C.c_uint32, C.c_int32, P, P, P, P, C.c_int32, f32, f32, P, P]
        L.dp_quantize_gh.argtypes = [P, u64, f32, f32, P]
        L.dp_probe_hist_atomics.argtypes = [C.c_uint32, C.POINTER(C.c_double), P]
        L.dp_csv_decode.argtypes = [C.c_char_p, u64, C.c_char_p, C.c_char_p, P, C.POINTER(P)]
        L.dp_csv_shape.argtypes = [P, C.POINTER(u64), C.POINTER(C.c_uint32), C.POINTER(C.c_uint32),
                                   C.POINTER(C.c_int32)]
        L.dp_csv_data.argtypes = [P, C.POINTER(P), C.POINTER(P)]
        L.dp_csv_metadata.argtypes = [P, C.POINTER(C.c_char_p), C.POINTER(C.c_double)]
        L.dp_csv_copy.argtypes = [P, P, P]
        L.dp_csv_free.argtypes = [P]
        L.dp_csv_parse_feature.argtypes = [C.c_char_p, u64, C.POINTER(C.c_float)]
        L.dp_hist_prepare.argtypes = [P, u64, C.c_uint32, C.c_int32, C.c_int32, P, P, P, P, C.c_int32, f32, f32,
                                      P, C.POINTER(P)]
        L.dp_hist_run.argtypes = [P, P]
        L.dp_hist_free.argtypes = [P]
        L.dp_eval_splits.argtypes = [P, C.c_int32, C.c_uint32, P, P, P, f32, f32, f64, f64, f64, f64, P, P, P]
        u32 = C.c_uint32
        margins = [C.c_int32, P, u64, u32, u64]
        L.dp_log_prob.argtypes = margins + [P, P, P, P]
        L.dp_log_prob_grad.argtypes = margins + [P, P, P, P, u64, P, u64, P]
        L.dp_policy_loss.argtypes = margins + [P, P, P, P, P, f32, f32, f32, P, P, P, u64, P, u64, P]
        L.dp_preference_loss.argtypes = [u64, P, u64, P, P, P, f32, f32, P, P, P, P]
        L.dp_preference_prepare.argtypes = [u64, P, u64, P, C.POINTER(P)]
        L.dp_preference_run.argtypes = [P, P, P, P, f32, f32, P, P, P, P]
        L.dp_preference_free.argtypes = [P]
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc != 0:
        raise DPError(lib().XGBGetLastError().decode())


def version() -> tuple[int, int, int]:
    a, b, c = C.c_int(), C.c_int(), C.c_int()
    lib().XGBoostVersion(C.byref(a), C.byref(b), C.byref(c))
    return a.value, b.value, c.value


def build_info() -> dict:
    p = C.c_char_p()
    check(lib().XGBuildInfo(C.byref(p)))
    return json.loads(p.value.decode())


def launch_count() -> int:
    return int(lib().dp_launch_count())


def array_interface(ptr: int, shape: Iterable[int], typestr: str = "<f4", strides=None) -> str:
    """__cuda_array_interface__ JSON as the reference builds it
    (native/class_model_native_adapter.cuh:26)."""
    return json.dumps({"data": [int(ptr), True], "shape": list(shape), "strides": strides, "typestr": typestr,
                       "version": 3, "stream": 1}, separators=(",", ":"))


class DMatrix:
    """Dense fp32 matrix [R][F] (NaN = missing): a borrowed CUDA matrix, or a
    host matrix copied to the current CUDA device (from_host)."""

    def __init__(self, data_ptr: int, rows: int, cols: int, label_ptr: int | None = None, row_stride: int | None = None,
                 missing: float = math.nan, keepalive=None):
        self.handle = C.c_void_p()
        strides = None if row_stride is None else [int(row_stride) * 4, 4]
        cfg = '{"missing":NaN,"nthread":2}' if math.isnan(missing) else json.dumps({"missing": missing, "nthread": 2})
        check(lib().XGDMatrixCreateFromCudaArrayInterface(array_interface(data_ptr, [rows, cols], strides=strides)
                                                          .encode(), cfg.encode(), C.byref(self.handle)))
        self._keep = keepalive
        if label_ptr is not None:
            self.set_label_ptr(label_ptr, rows)

    @classmethod
    def from_torch(cls, x, y=None, missing: float = math.nan) -> "DMatrix":
        """x: CUDA float32 tensor [R, F] (row stride allowed); y: CUDA float32 [R]."""
        assert x.is_cuda and x.dtype.is_floating_point and x.element_size() == 4 and x.dim() == 2
        assert x.stride(1) == 1
        d = cls(x.data_ptr(), x.shape[0], x.shape[1], row_stride=x.stride(0) if x.stride(0) != x.shape[1] else None,
                missing=missing, keepalive=(x, y))
        if y is not None:
            y = y.contiguous()
            d._keep = (x, y)
            d.set_label_ptr(y.data_ptr(), y.shape[0])
        return d

    @classmethod
    def from_host(cls, x, y=None, missing: float = math.nan) -> "DMatrix":
        """x: host float32 [R, F] (numpy array or CPU torch tensor, rows
        contiguous; pinned memory copies fastest); y: host float32 [R].
        Goes through XGDMatrixCreateFromDense."""
        if hasattr(x, "data_ptr"):
            assert not x.is_cuda and x.dim() == 2 and x.element_size() == 4 and x.stride(1) == 1
            ptr, (rows, cols), row_stride = x.data_ptr(), x.shape, x.stride(0)
        else:
            import numpy as np
            assert x.dtype == np.float32 and x.ndim == 2 and x.strides[1] == 4
            ptr, (rows, cols), row_stride = x.ctypes.data, x.shape, x.strides[0] // 4
        d = cls.__new__(cls)
        d.handle = C.c_void_p()
        strides = None if row_stride == cols else [int(row_stride) * 4, 4]
        cfg = '{"missing":NaN,"nthread":2}' if math.isnan(missing) else json.dumps({"missing": missing, "nthread": 2})
        check(lib().XGDMatrixCreateFromDense(array_interface(ptr, [rows, cols], strides=strides).encode(),
                                             cfg.encode(), C.byref(d.handle)))
        d._keep = None  # the library holds its own copy
        if y is not None:
            d.set_label_host(y.numpy() if hasattr(y, "numpy") else y)
        return d

    def set_label_ptr(self, ptr: int, n: int) -> None:
        check(lib().XGDMatrixSetInfoFromInterface(self.handle, b"label", array_interface(ptr, [n]).encode()))

    def set_label_host(self, y) -> None:
        import numpy as np
        y = np.ascontiguousarray(y, dtype=np.float32)
        check(lib().XGDMatrixSetFloatInfo(self.handle, b"label", y.ctypes.data, y.size))

    def num_row(self) -> int:
        n = C.c_uint64()
        check(lib().XGDMatrixNumRow(self.handle, C.byref(n)))
        return n.value

    def num_col(self) -> int:
        n = C.c_uint64()
        check(lib().XGDMatrixNumCol(self.handle, C.byref(n)))
        return n.value

    def free(self) -> None:
        if self.handle:
            check(lib().XGDMatrixFree(self.handle))
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Booster:
    def __init__(self, params: dict | None = None, cache: list[DMatrix] | None = None, handle=None):
        if handle is not None:
            self.handle = handle
        else:
            self.handle = C.c_void_p()
            cache = cache or []
            arr = (C.c_void_p * max(1, len(cache)))(*[d.handle for d in cache])
            check(lib().XGBoosterCreate(arr, len(cache), C.byref(self.handle)))
        for k, v in (params or {}).items():
            self.set_param(k, v)

    def set_param(self, key: str, value) -> None:
        if isinstance(value, (list, tuple)):
            value = json.dumps(list(value))
        elif isinstance(value, bool):
            value = "1" if value else "0"
        check(lib().XGBoosterSetParam(self.handle, key.encode(), str(value).encode()))

    def update(self, dtrain: DMatrix, iteration: int) -> None:
        check(lib().XGBoosterUpdateOneIter(self.handle, iteration, dtrain.handle))

    def boost(self, dtrain: DMatrix, iteration: int, grad, hess) -> None:
        """One round on the caller's gradients and curvatures: CUDA float32
        [rows, outputs] (one output: also [rows]), rows strided as they are."""
        import torch
        _need(grad.is_cuda and hess.is_cuda and grad.dtype == hess.dtype == torch.float32,
              "grad and hess must be CUDA float32 tensors")
        text = [array_interface(t.data_ptr(), list(t.shape), strides=[s * 4 for s in t.stride()]).encode()
                for t in (grad, hess)]
        check(lib().XGBoosterTrainOneIter(self.handle, dtrain.handle, iteration, *text))

    def train_margin(self, dtrain: DMatrix):
        """The training margins of `dtrain` ([rows, outputs] fp32) as a new
        CUDA tensor: the base scores before the first round."""
        import torch
        rows, outputs, ptr = C.c_uint64(), C.c_uint64(), C.c_void_p()
        check(lib().dp_booster_train_margin(self.handle, dtrain.handle, C.byref(rows), C.byref(outputs),
                                            C.byref(ptr)))

        class Borrowed:
            __cuda_array_interface__ = {"data": (ptr.value or 0, False), "shape": (rows.value, outputs.value),
                                        "typestr": "<f4", "version": 3}
        if not rows.value:
            return torch.empty((0, outputs.value), dtype=torch.float32, device="cuda")
        view = torch.as_tensor(Borrowed())
        out = view.clone()
        torch.cuda.current_stream(view.device).synchronize()  # the booster's next call may change them
        return out

    def boosted_rounds(self) -> int:
        n = C.c_int()
        check(lib().XGBoosterBoostedRounds(self.handle, C.byref(n)))
        return n.value

    def save_config(self) -> dict:
        n = C.c_uint64()
        p = C.c_char_p()
        check(lib().XGBoosterSaveJsonConfig(self.handle, C.byref(n), C.byref(p)))
        return json.loads(C.string_at(p, n.value).decode())

    def save_raw(self) -> bytes:
        n = C.c_uint64()
        p = C.c_void_p()
        check(lib().XGBoosterSaveModelToBuffer(self.handle, b'{"format":"json"}', C.byref(n), C.byref(p)))
        return C.string_at(p, n.value)

    def save_model(self, path: str) -> None:
        check(lib().XGBoosterSaveModel(self.handle, str(path).encode()))

    def load_raw(self, raw: bytes) -> None:
        check(lib().XGBoosterLoadModelFromBuffer(self.handle, raw, len(raw)))

    def load_model(self, path: str) -> None:
        check(lib().XGBoosterLoadModel(self.handle, str(path).encode()))

    def slice(self, begin: int, end: int, step: int = 1) -> "Booster":
        out = C.c_void_p()
        check(lib().XGBoosterSlice(self.handle, begin, end, step, C.byref(out)))
        return Booster(handle=out)

    def num_features(self) -> int:
        n = C.c_uint64()
        check(lib().XGBoosterGetNumFeature(self.handle, C.byref(n)))
        return n.value

    def set_comm(self, comm: "Comm") -> None:
        check(lib().dp_booster_set_comm(self.handle, comm.handle))

    def set_profiling(self, on, histograms_only: bool = False) -> None:
        """Mode 1 (on=True): every instrumented launch; histograms_only: mode 2;
        on=False: off.  Enabling resets the counters."""
        mode = 0 if not on else (2 if histograms_only else 1)
        check(lib().dp_booster_set_profiling(self.handle, mode))

    def profile(self) -> dict:
        p = C.c_char_p()
        check(lib().dp_booster_profile(self.handle, C.byref(p)))
        return json.loads(p.value.decode())

    def predict(self, x, margin: bool = False, iteration_begin: int = 0, iteration_end: int = 0,
                strict_shape: bool = True, missing: float = math.nan):
        """XGBoosterPredictFromCudaArray over a CUDA float32 tensor [R, F]
        (row stride allowed).  Returns a new CUDA tensor holding a copy of the
        booster-owned output, shaped as the call reports it."""
        import torch
        assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
        strides = None if x.stride(0) == x.shape[1] else [int(x.stride(0)) * 4, 4]
        cfg = {"type": 1 if margin else 0, "training": False, "iteration_begin": iteration_begin,
               "iteration_end": iteration_end, "strict_shape": strict_shape, "cache_id": 0}
        text = json.dumps(cfg, separators=(",", ":"))[:-1] + (',"missing":NaN}' if math.isnan(missing)
                                                               else f',"missing":{missing!r}}}')
        shape = C.POINTER(C.c_uint64)()
        dims = C.c_uint64()
        out = C.POINTER(C.c_float)()
        check(lib().XGBoosterPredictFromCudaArray(self.handle, array_interface(x.data_ptr(), list(x.shape),
                                                                               strides=strides).encode(),
                                                  text.encode(), None, C.byref(shape), C.byref(dims),
                                                  C.byref(out)))
        dims_t = tuple(shape[i] for i in range(dims.value))
        n = 1
        for d in dims_t:
            n *= d
        res = torch.empty(dims_t, dtype=torch.float32, device=x.device)
        if n:
            from cuda.bindings import runtime as rt
            err, = rt.cudaMemcpy(res.data_ptr(), C.cast(out, C.c_void_p).value, n * 4,
                                 rt.cudaMemcpyKind.cudaMemcpyDeviceToDevice)
            if err != rt.cudaError_t.cudaSuccess:
                raise DPError(f"copy of the prediction failed: {err}")
        return res

    def margins(self, rows: int, outputs: int):
        import numpy as np
        out = np.zeros((rows, outputs), np.float32)
        check(lib().dp_booster_margins(self.handle, out.ctypes.data, out.size))
        return out

    def trees(self) -> list[dict]:
        return json.loads(self.save_raw())["learner"]["gradient_booster"]["model"]["trees"]

    def free(self) -> None:
        if self.handle:
            check(lib().XGBoosterFree(self.handle))
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Comm:
    """NCCL communicator for row-sharded training (one process per GPU)."""

    @staticmethod
    def unique_id() -> bytes:
        buf = C.create_string_buffer(128)
        check(lib().dp_comm_unique_id(buf))
        return buf.raw

    def __init__(self, unique_id: bytes, nranks: int, rank: int, device: int):
        assert len(unique_id) == 128
        self.handle = C.c_void_p()
        check(lib().dp_comm_create(unique_id, nranks, rank, device, C.byref(self.handle)))

    def set_timeout(self, ms: int) -> None:
        """Deadline of every host wait on collectives in flight; a peer that
        stops or fails aborts the communicator and the training call raises."""
        check(lib().dp_comm_set_timeout(self.handle, int(ms)))

    def reduce_scatter_hist(self, send_ptr: int, recv_ptr: int, recv_n: int, stream: int | None = None) -> None:
        """The sharded path's histogram exchange (int64 partial sums)."""
        check(lib().dp_comm_reduce_scatter_hist(self.handle, send_ptr, recv_ptr, recv_n, stream))

    def free(self) -> None:
        if self.handle:
            check(lib().dp_comm_free(self.handle))
            self.handle = C.c_void_p()


class CsvTable:
    """The GPU CSV decoder (dp_csv_decode): the reference's
    decision_programs_csv::decode (native/decision_programs_csv.hpp:36-67).
    `values_ptr` / `labels_ptr` are device pointers owned by this object."""

    def __init__(self, data: bytes, target: str | None = None, header: str = "auto"):
        h = C.c_void_p()
        check(lib().dp_csv_decode(data, len(data), (target or "").encode(), header.encode(), None, C.byref(h)))
        self.handle = h
        rows, feats, classes, hdr = C.c_uint64(), C.c_uint32(), C.c_uint32(), C.c_int32()
        check(lib().dp_csv_shape(h, C.byref(rows), C.byref(feats), C.byref(classes), C.byref(hdr)))
        self.rows, self.features, self.classes, self.header = rows.value, feats.value, classes.value, bool(hdr.value)
        meta, ms = C.c_char_p(), C.c_double()
        check(lib().dp_csv_metadata(h, C.byref(meta), C.byref(ms)))
        m = json.loads(meta.value.decode())
        self.names, self.label_mapping, self.device_ms = m["names"], m["label_mapping"], ms.value
        v, lb = C.c_void_p(), C.c_void_p()
        check(lib().dp_csv_data(h, C.byref(v), C.byref(lb)))
        self.values_ptr, self.labels_ptr = v.value, lb.value

    def to_numpy(self):
        import numpy as np
        values = np.empty((self.rows, self.features), np.float32)
        labels = np.empty(self.rows, np.uint32) if self.labels_ptr else None
        check(lib().dp_csv_copy(self.handle, values.ctypes.data,
                                labels.ctypes.data if labels is not None else None))
        return values, labels

    def free(self) -> None:
        if self.handle:
            check(lib().dp_csv_free(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# ---- losses that learn from choices ------------------------------------------
# Each call runs on the current torch stream of its tensors' device and returns
# new tensors; nothing waits for the GPU (PreferencePairs' construction aside).
# Results are detached: autograd records none of these calls, also where a
# tensor requires a gradient; the gradients returned are what a caller hands on
# (margin.backward(grad), or Booster.boost).

class PolicyLoss(NamedTuple):
    """loss and log_prob [R] fp32; grad [R, K] of the margins' type and hess
    [R, K] fp32, each None when not asked for."""
    loss: Any
    log_prob: Any
    grad: Any
    hess: Any


class PreferenceLoss(NamedTuple):
    """loss [P], grad [R] and hess [R] (None when not asked for), all fp32."""
    loss: Any
    grad: Any
    hess: Any


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise DPError(message)


def _vector(t, n: int, dtype, device, name: str, optional: bool = False, shape=None):
    """`t` as a contiguous tensor of n rows on `device`, checked."""
    if t is None and optional:
        return None
    shape = (n,) if shape is None else shape
    if t.shape != shape:
        raise DPError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise DPError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise DPError(f"{name} must be on {device}, got {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _elsewhere(device) -> bool:
    """Whether a call has to make `device`, its tensors' one, current first."""
    import torch
    _need(device.type == "cuda", "the tensors must be CUDA tensors")
    return device.index != torch.cuda.current_device()


def _stream(device) -> int:
    """The current torch stream of a CUDA device, as the library takes it."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without a Stream object: 0.1 us, not 2
    return raw(device.index) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def _rows_of(t, name: str):
    """(pointer, row stride) of a [R, K] tensor whose classes are adjacent."""
    (rows, classes), (apart, step) = t.shape, t.stride()
    if classes > 1 and step != 1:
        raise DPError(f"{name}: the classes of a row must be adjacent in memory")
    return t.data_ptr(), (apart if rows > 1 else max(classes, apart))


def _margins(margin):
    """The leading arguments of a call on class margins [R, K]."""
    import torch
    _need(margin.dim() == 2, "margin must be [rows, classes]")
    dtype = margin.dtype
    kind = 2 if dtype == torch.bfloat16 else 0 if dtype == torch.float32 else 1
    _need(kind != 1 or dtype == torch.float16, "margin must be float32, float16 or bfloat16")
    ptr, stride = _rows_of(margin, "margin")
    return kind, ptr, margin.shape[0], margin.shape[1], stride


def _grad_out(margin, grad, hess):
    """The gradient and curvature tensors of a call, and their arguments."""
    import torch
    if grad is None or grad is True:
        grad = torch.empty_like(margin)  # (margins whose rows lie apart: without the gaps)
    else:
        _need(isinstance(grad, torch.Tensor) and grad.shape == margin.shape and grad.dtype == margin.dtype and
              grad.device == margin.device, "grad must be a tensor of the margins' shape, type and device")
    if not hess:
        return grad, None, (*_rows_of(grad, "grad"), None, 0)
    hess = torch.empty_like(margin, dtype=torch.float32)
    return grad, hess, (*_rows_of(grad, "grad"), *_rows_of(hess, "hess"))


def log_prob(margin, label):
    """log softmax(margin)[label] of every row ([R] fp32), and the rows' norm
    ([R, 2] fp32: maximum, log-sum) that log_prob_grad takes.  margin: CUDA
    [R, K] float32, float16 or bfloat16 (row stride allowed); label: int32
    [R], rows whose label is not a class are skipped.  Detached from autograd:
    log_prob_grad is the backward pass."""
    import torch
    dev = margin.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return log_prob(margin, label)
    m = _margins(margin)
    rows = m[2]
    label = _vector(label, rows, torch.int32, dev, "label")
    out, norm = torch.empty(rows, dtype=torch.float32, device=dev), torch.empty(rows, 2, dtype=torch.float32, device=dev)
    check(lib().dp_log_prob(*m, label.data_ptr(), out.data_ptr(), norm.data_ptr(), _stream(dev)))
    return out, norm


def log_prob_grad(margin, label, norm, weight, grad=None, hess: bool = False):
    """The backward pass of log_prob: (grad, hess) for `weight` [R] fp32, the
    derivative of a loss by each log-probability.  grad: a tensor to write to
    (the margins themselves included); hess: the diagonal curvature too."""
    import torch
    dev = margin.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return log_prob_grad(margin, label, norm, weight, grad, hess)
    m = _margins(margin)
    rows = m[2]
    label = _vector(label, rows, torch.int32, dev, "label")
    norm = _vector(norm, rows, torch.float32, dev, "norm", shape=(rows, 2))
    weight = _vector(weight, rows, torch.float32, dev, "weight")
    grad, hess, out = _grad_out(margin, grad, hess)
    check(lib().dp_log_prob_grad(*m, label.data_ptr(), norm.data_ptr(), weight.data_ptr(), *out, _stream(dev)))
    return grad, hess


def policy_loss(margin, label, old_log_prob, advantage, ref_log_prob=None, weight=None, clip=(0.2, 0.2),
                kl: float = 0.0, grad=True, hess: bool = False) -> PolicyLoss:
    """Clipped policy loss with a KL term (dp_policy_loss): margin [R, K] as in
    log_prob, label the sampled class; old_log_prob, advantage, ref_log_prob
    (None: no KL term) and weight (None: 1) [R] fp32; clip (low, high).  grad:
    True, a tensor to write to (the margins themselves included), or False for
    the forward pass alone; hess: the diagonal curvature too.  Detached from
    autograd: margin.backward(result.grad) hands the gradient on."""
    import torch
    dev = margin.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return policy_loss(margin, label, old_log_prob, advantage, ref_log_prob, weight, clip, kl, grad, hess)
    m = _margins(margin)
    rows, f32 = m[2], torch.float32
    label = _vector(label, rows, torch.int32, dev, "label")
    old_log_prob = _vector(old_log_prob, rows, f32, dev, "old_log_prob")
    advantage = _vector(advantage, rows, f32, dev, "advantage")
    ref_log_prob = _vector(ref_log_prob, rows, f32, dev, "ref_log_prob", optional=True)
    weight = _vector(weight, rows, f32, dev, "weight", optional=True)
    _need(grad is not False or not hess, "hess is written with a gradient: grad is False")
    loss = torch.empty(rows, dtype=f32, device=dev)
    logp = torch.empty(rows, dtype=f32, device=dev)
    grad, hess, out = (None, None, (None, 0, None, 0)) if grad is False else _grad_out(margin, grad, hess)
    check(lib().dp_policy_loss(*m, label.data_ptr(), old_log_prob.data_ptr(), _ptr(ref_log_prob),
                               advantage.data_ptr(), _ptr(weight), clip[0], clip[1], kl, loss.data_ptr(),
                               logp.data_ptr(), *out, _stream(dev)))
    return PolicyLoss(loss, logp, grad, hess)


def _pair_tensors(score, ref_score, weight, pairs: int, hess: bool):
    import torch
    f32, dev = torch.float32, score.device
    _need(score.dim() == 1, "score must be a vector")
    rows = score.shape[0]
    score = _vector(score, rows, f32, dev, "score")
    ref_score = _vector(ref_score, rows, f32, dev, "ref_score", optional=True)
    weight = _vector(weight, pairs, f32, dev, "weight", optional=True)
    out = PreferenceLoss(torch.empty(pairs, dtype=f32, device=dev), torch.empty(rows, dtype=f32, device=dev),
                         torch.empty(rows, dtype=f32, device=dev) if hess else None)
    return score, ref_score, weight, out


def preference_loss(score, ref_score=None, item_begin=None, weight=None, beta: float = 1.0, smoothing: float = 0.0,
                    hess: bool = False) -> PreferenceLoss:
    """Preference loss over consecutive items (dp_preference_loss): item 2p is
    preferred to item 2p + 1.  score, ref_score: [R] fp32 CUDA; item_begin:
    int64 [2P + 1] offsets into the rows (None: every row is an item); weight:
    [P] fp32.  Detached from autograd: score.backward(result.grad) hands the
    gradient on."""
    import torch
    dev = score.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return preference_loss(score, ref_score, item_begin, weight, beta, smoothing, hess)
    if item_begin is None:
        _need(score.dim() == 1 and score.shape[0] % 2 == 0, "without item offsets score holds pairs of rows")
        pairs = score.shape[0] // 2
    else:
        _need(item_begin.dim() == 1 and item_begin.shape[0] % 2 == 1, "item_begin must hold 2 * pairs + 1 offsets")
        pairs = item_begin.shape[0] // 2
        item_begin = _vector(item_begin, 2 * pairs + 1, torch.int64, dev, "item_begin")
    score, ref_score, weight, out = _pair_tensors(score, ref_score, weight, pairs, hess)
    check(lib().dp_preference_loss(score.shape[0], _ptr(item_begin), pairs, score.data_ptr(), _ptr(ref_score),
                                   _ptr(weight), beta, smoothing, out.loss.data_ptr(), out.grad.data_ptr(),
                                   _ptr(out.hess), _stream(dev)))
    return out


class PreferencePairs:
    """Pairs of rows, checked and laid out once (dp_preference_prepare): pairs
    [P, 2] int32 CUDA (preferred row, other row) over `rows` rows; a row may be
    in any number of pairs."""

    def __init__(self, pairs, rows: int):
        import torch
        self.handle = C.c_void_p()
        self.pairs, self.rows, self.device = pairs.shape[0], int(rows), pairs.device
        _need(self.device.type == "cuda", "the tensors must be CUDA tensors")
        with torch.cuda.device(self.device):
            pairs = _vector(pairs, self.pairs, torch.int32, self.device, "pairs", shape=(self.pairs, 2))
            check(lib().dp_preference_prepare(self.rows, pairs.data_ptr(), self.pairs, _stream(self.device),
                                              C.byref(self.handle)))

    def loss(self, score, ref_score=None, weight=None, beta: float = 1.0, smoothing: float = 0.0,
             hess: bool = False) -> PreferenceLoss:
        """The preference loss of score [rows] fp32, with weight [P].  The runs
        of one plan share its workspace: order them if they are on different
        streams."""
        import torch
        _need(bool(self.handle), "the pairs have been freed")
        if score.shape != (self.rows,):
            raise DPError(f"score must have shape {[self.rows]}, got {list(score.shape)}")
        if score.device != self.device:
            raise DPError(f"score must be on {self.device}, got {score.device}")
        if _elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self.loss(score, ref_score, weight, beta, smoothing, hess)
        score, ref_score, weight, out = _pair_tensors(score, ref_score, weight, self.pairs, hess)
        check(lib().dp_preference_run(self.handle, score.data_ptr(), _ptr(ref_score), _ptr(weight), beta, smoothing,
                                      out.loss.data_ptr(), out.grad.data_ptr(), _ptr(out.hess), _stream(self.device)))
        return out

    def free(self) -> None:
        if self.handle:
            check(lib().dp_preference_free(self.handle))
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def train(params: dict, dtrain: DMatrix, rounds: int, comm: Comm | None = None) -> Booster:
    """The reference's sequence: create, set params, one UpdateOneIter per round."""
    b = Booster(params, [dtrain])
    if comm is not None:
        b.set_comm(comm)
    for i in range(rounds):
        b.update(dtrain, i)
    return b

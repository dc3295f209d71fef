"""What the row-wise entry points would launch, found without a GPU: a process of its own loads the library behind a stand-in for the HIP
runtime that notes the launches (launch_recorder.cpp).  No address that is passed is ever read."""
import ctypes
import json
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIBRARY = os.path.join(os.path.dirname(HERE), "compressgnn_amd", "lib", "libcgnn_hip.so")
TYPES = {"f": 0, "d": 1, "DF16_": 2, "DF16b": 3}  # as the compiler writes them in a kernel's name, and as cgnn_dtype


def _kernel(mangled):
    """(name, values of its template parameters: types as in cgnn_dtype, then numbers)"""
    found = re.match(r"_ZN4cgnn12_GLOBAL__N_1(\d+)(\w+)", mangled)
    if not found:
        return mangled, ()
    length = int(found[1])
    name, rest = found[2][:length], found[2][length:]
    values = re.match(r"I((?:DF16_|DF16b|f|d|L[ib]\d+E)*)E", rest)
    if not values:
        return name, ()
    return name, tuple(TYPES[t] if t else int(n) for t, n in re.findall(r"(DF16_|DF16b|f|d)|L[ib](\d+)E", values[1]))


class _Drop(ctypes.Structure):
    _fields_ = [("seed", ctypes.c_uint64), ("offset", ctypes.c_uint64), ("counter", ctypes.c_void_p), ("kept", ctypes.c_int32)]


def _record(recorder, calls):
    """In the process of its own."""
    stand_in = ctypes.CDLL(recorder, ctypes.RTLD_GLOBAL)
    lib = ctypes.CDLL(LIBRARY)
    lib.cgnn_layer_norm_backward_workspace_bytes.restype = ctypes.c_size_t
    for f in (stand_in.recorded_launches, stand_in.registered_kernels):
        f.restype = ctypes.c_char_p
    i64, at = ctypes.c_int64, ctypes.c_void_p(1 << 20)
    results = []
    for call in calls:
        rows, F, dtype, param = call["rows"], call["F"], call["dtype"], call.get("param", call["dtype"])
        drop = ctypes.byref(_Drop(1, 0, None, call["kept"])) if call.get("kept") is not None else None
        relu = int(call.get("relu", False))
        if call["op"] == "dropout":
            status = lib.cgnn_dropout(i64(rows), i64(F), dtype, at, i64(call.get("ldx", F)), drop, at, None)
        elif call["op"] == "norm":
            status = lib.cgnn_layer_norm(i64(rows), i64(F), dtype, param, at, i64(F), at, at, ctypes.c_double(1e-5), relu, drop, at,
                                         at if call.get("stats") else None, None)
        else:
            need = lib.cgnn_layer_norm_backward_workspace_bytes(i64(rows), i64(F), dtype)
            status = lib.cgnn_layer_norm_backward(i64(rows), i64(F), dtype, param, at, i64(F), at, i64(F), at, at, at, relu, drop,
                                                  at, at, at, at, ctypes.c_size_t(need), None)
        results.append([status, stand_in.recorded_launches().decode()])
    return {"calls": results, "kernels": stand_in.registered_kernels().decode().split()}


def record(directory, calls):
    """([(status, [((kernel, template values), grid, block), ...]), ...] for the calls, all kernels of the library).
    A call: op ("norm", "gradients" or "dropout"), rows, F, dtype; param, relu, kept, stats, ldx where they matter."""
    recorder = os.path.join(str(directory), "launch_recorder.so")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", os.path.join(HERE, "launch_recorder.cpp"), "-o", recorder], check=True)
    done = subprocess.run([sys.executable, os.path.abspath(__file__), recorder], input=json.dumps(calls), stdout=subprocess.PIPE, text=True,
                          check=True, timeout=300)
    answer = json.loads(done.stdout)
    results = []
    for status, text in answer["calls"]:
        launches = []
        for line in text.splitlines():
            name, *numbers = line.split()
            numbers = [int(n) for n in numbers]
            launches.append((_kernel(name), tuple(numbers[:3]), tuple(numbers[3:])))
        results.append((status, launches))
    return results, [_kernel(name) for name in answer["kernels"]]


if __name__ == "__main__":
    json.dump(_record(sys.argv[1], json.load(sys.stdin)), sys.stdout)

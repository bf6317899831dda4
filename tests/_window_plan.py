"""Where mt_attention_paged and mt_attention_sinks place their work (WindowPlan of csrc/f8.hpp), for tests that have to know which
kernel a case runs through."""
import ctypes

import mingtts as mt


class Plan(ctypes.Structure):
    _fields_ = [("waves", ctypes.c_uint32), ("keys", ctypes.c_uint32), ("parts", ctypes.c_uint32), ("run", ctypes.c_uint32),
                ("shared", ctypes.c_bool), ("by_xcd", ctypes.c_bool)]


def window_plan(B, T, hq, hkv, len_max, window=0, sinks=0, cache_t=mt.F16):
    f = mt.load()._ZN2mt11window_planEjjjjjjji
    f.argtypes, f.restype = [ctypes.c_uint32] * 7 + [ctypes.c_int], Plan
    return f(B, T, hq, hkv, len_max, window, sinks, cache_t)


def plan_of(case, len_max=0):
    """That of a Case of _paged_util."""
    kind = {"f32": mt.F32, "f16": mt.F16, "f8": mt.F8}[case.kind]
    return window_plan(case.B, case.T, case.hq, case.hkv, len_max or case.kv.cache_len, case.window, case.sinks, kind)

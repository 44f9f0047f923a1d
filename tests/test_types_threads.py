"""The types of a call's tensors are known to every thread as soon as one of them has been told."""
import importlib.util
import sys

import torch

import clblast_b200
from clblast_b200 import api


def fresh():
    """The module as a process finds it before its first call."""
    spec = importlib.util.spec_from_file_location("clblast_b200._api_again", api.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_first_calls_of_two_threads():
    """A first call is stopped before each of its lines, and a second one made there."""
    x = torch.zeros(2, dtype=torch.bfloat16)
    want = (1016, torch.bfloat16, 32, torch.float32)
    stops = 1
    at = 0
    while at < stops:
        module, seen, count = fresh(), [], 0

        def trace(frame, event, arg):
            nonlocal count
            if frame.f_code.co_filename != api.__file__:
                return None
            if event == "line":
                if count == at:
                    seen.append(module._types(x, None, None, 32))
                count += 1
            return trace

        sys.settrace(trace)
        try:
            first = module._types(x, None, None, 32)
        finally:
            sys.settrace(None)
        assert first == want and all(s == want for s in seen), (at, first, seen)
        stops = max(stops, count)
        at += 1
    assert at > 5

"""on_device in a forked process asks torch.cuda, whose check of the process's state comes before any launch."""

import os

import torch

from table_moe import _native as N


def _child() -> int:
    """0 where on_device lets torch.cuda's refusal through, and takes its answer otherwise."""
    def refuse():
        raise RuntimeError("Cannot re-initialize CUDA in forked subprocess")

    if N._current_device is not torch.cuda.current_device:
        return 1
    N._current_device = refuse
    try:
        N.on_device(torch.device("cuda:0"))
        return 2
    except RuntimeError:
        pass
    N._current_device = lambda: 1
    if N.on_device(torch.device("cuda:1")).__enter__() is not None:
        return 3
    return 0 if isinstance(N.on_device(torch.device("cuda:0")), torch.cuda.device) else 4


def test_on_device_after_a_fork():
    pid = os.fork()
    if pid == 0:
        code = 5
        try:
            code = _child()
        finally:
            os._exit(code)
    assert os.waitstatus_to_exitcode(os.waitpid(pid, 0)[1]) == 0

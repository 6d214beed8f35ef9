"""Which of the operators' kernels a call launches, by the names that torch's
profiler records for the process: a test of a kernel says with it that the kernel
ran."""
import re
import warnings


def kernels_of(call):
    """{kernel name: its template arguments, as texts} of the operators' kernels that
    call() launches."""
    import torch
    from torch.profiler import ProfilerActivity, profile

    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            call()
            torch.cuda.synchronize()
    got = {}
    for e in p.key_averages():
        m = re.search(r"moe::ops::(\w+)(?:<([^>]*)>)?\(", e.key)
        if m:
            got[m.group(1)] = [v.strip() for v in (m.group(2) or "").split(",")]
    return got

"""Which kernels a call runs, by the profiler."""
import re

import torch


def kernels(call):
    """Names of the kernels that ``call`` runs, with their template arguments."""
    from torch.profiler import ProfilerActivity, profile

    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    return {re.sub(r"^.*?(\w+(<[^()]*>)?)\(.*$", r"\1", e.key.replace("(anonymous namespace)::", "")) for e in p.key_averages()
            if e.device_time_total > 0}


def sm_count():
    return torch.cuda.get_device_properties(0).multi_processor_count

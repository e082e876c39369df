"""GPU: the kernel for few queries cuts its work into as many shares as CTAs are resident, whatever their shared memory."""
import json

import pytest
import torch

from test_gpu_int4_weigh import DEV, _cache, _fill, _query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,group,columns,seqs", [(64, 64, 1, 8), (64, 16, 16, 8), (128, 128, 1, 8), (128, 128, 32, 8),
                                                    (128, 64, 16, 8), (128, 32, 16, 8), (256, 256, 1, 8),
                                                    (256, 256, 32, 8), (256, 64, 16, 8), (128, 128, 32, 1024)])
def test_every_share_is_resident(dim, group, columns, seqs, tmp_path):
    c = _cache(pages=4 * seqs, heads=1, dim=dim, group=group, seqs=seqs, blocks=1024)
    _fill(c, [100] * seqs)
    q, lse = _query((seqs, columns, 1, dim), 1, torch.float16), torch.zeros(seqs, columns, 1, device=DEV)
    c.weigh(0, q, lse)
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        c.weigh(0, q, lse)
        torch.cuda.synchronize()
    path = str(tmp_path / "trace.json")
    prof.export_chrome_trace(path)
    runs = [e["args"] for e in json.load(open(path))["traceEvents"] if "weigh_few" in e.get("name", "")]
    if not runs:
        pytest.skip("the profiler shows no kernels here")
    grid, smem = runs[0]["grid"][0], runs[0]["shared memory"]
    sm = torch.cuda.get_device_properties(0)
    per_sm = (228 << 10) // (smem + 1024)                    # 1 KB of each CTA's is the system's
    assert grid <= per_sm * sm.multi_processor_count, (grid, smem, per_sm)

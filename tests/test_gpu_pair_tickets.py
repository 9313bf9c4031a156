"""The pair kernel with every group a ticket: the form in which a call is launched again after a watchdog hit (static groups demoted)."""
import numpy as np
import pytest

import coregex_amd as cx

pytestmark = pytest.mark.gpu
K_PAIR = 21
PAT = "error|warning|fatal|critical"


@pytest.mark.parametrize("n", [1, 3840, 30_721, 122_880, 122_881, 491_521, 3_000_001, 40_000_003])
def test_rows_on_tickets_and_with_the_static_start(oracle, n):
    import torch
    hay = np.ascontiguousarray(cx.synth_pages(3, 0xC0FFEE03, 5, (n + 4095) // 4096).reshape(-1)[:n])
    exp = oracle.Regex(PAT).find_all_index(hay)
    rx = cx.compile(PAT)
    d = torch.from_numpy(hay.copy()).cuda()
    out = torch.zeros((len(exp) + 4, 2), dtype=torch.int64, device="cuda")
    cx.path_reset(0)
    for static in (True, False, False, True):                        # tickets in between and twice: each launch leaves the next one's counter clear
        cx.path_reset(0)
        if not static:
            assert cx._lib.lib().cxg_debug_demote(0, 0) == 0         # as if the look-back's watchdog had fired
        t = cx.Timing()
        out.fill_(-7)
        torch.cuda.synchronize()
        assert rx.find_all_device(d.data_ptr(), n, out.data_ptr(), len(exp) + 4, timing=t) == len(exp)
        assert t.kernels == [K_PAIR]
        assert np.array_equal(out[: len(exp)].cpu().numpy(), exp) and bool((out[len(exp):] == -7).all())
    cx.path_reset(0)

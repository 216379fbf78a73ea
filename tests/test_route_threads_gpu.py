"""Routing from several threads at once, each with its own stream: handles are thread-safe per
stream, whatever the numbers of experts.  The grouping kernel needs more than 48 KB of shared
memory from 187 experts on, and how much depends on E; one thread's call must not take the
permission for it away from another's."""
import threading

import numpy as np
import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def wanted(logits, k):
    experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    flat = experts.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    rows = torch.empty_like(flat)
    rows[order] = torch.arange(flat.numel(), device="cuda")
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"),
                         torch.cumsum(torch.bincount(flat, minlength=logits.shape[1]), 0)])
    return experts, offsets, rows.reshape(-1, k)


@pytest.mark.parametrize("sizes", [(300, 1024, 520, 1024), (187, 256, 200, 256)])
def test_threads_route_over_different_numbers_of_experts(gpu, sizes):
    dev, _, _ = gpu
    T, k, calls = 40, 3, 3000
    state, errors = [], []
    for i, E in enumerate(sizes):
        g = torch.Generator("cuda").manual_seed(100 * i + E)
        logits = torch.randn(T, E, generator=g, device="cuda")
        state.append((E, logits, torch.empty(T, k, device="cuda"),
                      torch.full((T, k), -7, dtype=torch.int32, device="cuda"),
                      torch.empty(E + 1, dtype=torch.int32, device="cuda"),
                      torch.empty(T, k, dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    streams = [dev.stream() for _ in sizes]
    gate = threading.Barrier(len(sizes))

    def work(st, s):
        E, logits, w, e, o, r = s
        ops = qgemm.QuantizedGemmOps(st)
        try:
            gate.wait(60)
            for i in range(calls):
                ops.routeTopK(logits, w, e, o, r, T, E, k)
                if i % 500 == 499:
                    st.sync()
        except Exception as ex:  # noqa: BLE001 - reported by the main thread
            errors.append(f"E={E}: {ex}")

    threads = [threading.Thread(target=work, args=a) for a in zip(streams, state)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for st in streams:
        st.sync()
        st.destroy()
    assert not errors, errors[:3]
    for E, logits, w, e, o, r in state:
        experts, offsets, rows = wanted(logits, k)
        assert torch.equal(e.long(), experts)
        assert torch.equal(o.long(), offsets)
        assert torch.equal(r.long(), rows)
        assert np.isclose(w.sum().item(), T, atol=1e-3)

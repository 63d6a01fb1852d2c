"""GPU tests of the training losses where values cancel, vanish or end: confident rows, a student near
its teacher, exact logits, non-finite rows, the largest sizes, and memory beside the buffers.

Tolerances are bounds, derived before the first run, in the terms of test_gpu_losses.py: u = 2^-24,
logits within 64 u A, so a probability within 128 u A relative. Here they follow |dz| = f |p - q|, the
gradient itself, not f (p + q): a confident row's gradient is the small difference of the two.
  * Classes that no label names: dz = f p, 128 u A relative; bf16 rounds it once, 2^-8.
  * One label: p - 1 is minus the other classes' share, 128 u A relative as well.
  * Several labels: p_i is off by 128 u A p_i, q_i by 16 u q_i (an exponential, a sum of 64, a
    quotient) and by its teacher logit's rounding (8 u A: here it lies near the student's), both by the
    subtraction's rounding.
Products and sums as there: (80 + tiles) u of the sum of the terms' sizes. f32 operands hold nothing
below 2^-38 of the largest of the 128 values they stand beside.
"""
import numpy as np
import pytest

from test_gpu_losses import cuda, grad, make

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rh():
    import rust_ppocrv6_b200 as rh

    rh.load()
    return rh


@pytest.fixture(scope="module")
def ctx(rh):
    c = rh.Context()
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(900, 121, 200), (120, 120, 700), (3000, 33, 130), (257, 80, 2000)])
def test_steps_back_to_back_in_one_workspace(rh, ctx, rows, k, n, dtype):
    """Two steps of other inputs in turn, in one workspace and without a wait between them: each finds
    what its own kernels wrote, never what the other's left at the same addresses."""
    one, two = make(rows, k, n, seed=81), make(rows, k, n, seed=82)
    ka, kb = {}, {}
    want = [{i: v.clone() for i, v in grad(rh, ctx, d, dtype, keep=keep).items()} for d, keep in ((one, ka), (two, kb))]
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    ws = torch.empty(rh.head_grad_workspace_bytes(ctx, dtype, rows, k, n), dtype=torch.uint8, device="cuda")
    runs, st = [], torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(40):
        s = (ka, kb)[i % 2]["s"]
        o = {j: torch.empty_like(v) for j, v in want[i % 2].items()}
        runs.append(o)
        st.wait_stream(torch.cuda.current_stream())
        assert s["x"].dtype == td
        rh.head_cross_entropy_grad_device(ctx, dtype, s["x"].data_ptr(), rows, k, s["w"].data_ptr(), n, s["b"].data_ptr(),
                                          s["t"].data_ptr(), s["g"].data_ptr(),
                                          *[o[j].data_ptr() for j in ("loss", "lse", "da", "dw", "db")], ws.data_ptr(),
                                          ws.numel(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    ctx.sync()
    for i, o in enumerate(runs):
        for j, v in want[i % 2].items():
            assert torch.equal(o[j], v), (i, j)

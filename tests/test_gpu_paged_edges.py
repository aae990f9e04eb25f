"""Steps of packed requests over paged caches where they can go wrong: bits of softmax weights and of small rows and
columns, values that are not finite, steps without sequences, and steps of hundreds of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

import paged_ref as R  # noqa: E402
from test_gpu_paged import _attend, _attn_inputs  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16


# ---- attention: bits of the weights ----------------------------------------------------------------

@pytest.mark.parametrize("rep", [1, 16, 48], ids=["row", "few", "many"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_weights_keep_22_bits(dtype, hd, rep):
    """V rows whose weighted sum cancels: outputs are the weights' last bits. They keep 22 for both types, as the operators
    over one sequence hold them."""
    L = 6
    q, kp, vp, table, plan, _ = _attn_inputs([L - 1] * 32, [1] * 32, 16, rep, 1, hd, dtype, key=("bits", hd, rep), k_size=0.02)
    q[:] = q[:, :1]  # one row of scores for all heads of a sequence
    for b in range(32):
        page = int(table[plan[1][b], 0])
        k = kp[page, 0, :L].double()
        p = torch.softmax(k @ q[b, 0].double() / hd ** 0.5, 0)
        left = torch.zeros(hd, dtype=torch.float64)
        for j in range(L):  # each takes what those before it leave, but for its rounding
            if j:
                vp[page, 0, j] = (-left / p[j]).to(dtype)
            left += p[j] * vp[page, 0, j].double()
    got = _attend(q, kp, vp, table, plan)
    want, size, score = R.attention(q, kp, vp, table, *plan[:3])
    bound = R.attention_bound(want, size, score, dtype, hd, L)
    if dtype is BF16:
        bound -= (2.0 ** -16 - 2.0 ** -22) * size
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())

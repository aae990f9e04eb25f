"""What the calls on packed sequences and paged caches refuse before anything reaches a GPU: through the C ABI with
made-up addresses, and the Python checks on CPU tensors."""
import pytest
import torch

X = 1 << 20


def _lib():
    from mlx_gsq_amd import _lib
    return _lib


PLAN = dict(requests=X, new_tokens=X, lengths=X, held=X, table=X, free_pages=X, n_free=X, sequences=3, n_requests=5, max_pages=7,
            n_pages=20, tokens=9, page_size=16, cu=X, rows=X, lens=X, pos=X, slots=X, stream=None)
ADVANCE = dict(rows=X, lens=X, lengths=X, sequences=3, n_requests=5, stream=None)
RELEASE = dict(requests=X, lengths=X, held=X, table=X, free_pages=X, n_free=X, sequences=3, n_requests=5, max_pages=7, n_pages=20,
               stream=None)
WRITE = dict(q=X, q_stride=1024, q_head_stride=256, k=X, k_stride=128, k_head_stride=128, v=X, v_stride=128, v_head_stride=128,
             q_norm_w=X, k_norm_w=X, inv_freq=X, k_pages=X, v_pages=X, pos=X, slots=X, q_out=X, tokens=9, heads=4, kv_heads=1,
             head_dim=128, rotary_dim=64, n_pages=20, page_size=16, eps=1e-6, dtype=1, stream=None)
ATTN = dict(q=X, gate=None, gate_stride=0, gate_head_stride=0, k_pages=X, v_pages=X, table=X, cu=X, rows=X, lens=X, out=X, work=X,
            tokens=9, sequences=3, n_requests=5, max_pages=7, heads=4, kv_heads=1, head_dim=128, n_pages=20, page_size=16, max_new=9,
            cus=256, dtype=1, stream=None)
GDN = dict(qkv=X, qkv_stride=512, z=X, z_stride=256, ab=X, ab_stride=8, conv_state=X, conv_w=X, ssm_a=X, dt_bias=X, rec_state=X,
           norm_w=X, cu=X, rows=X, lens=X, out=X, out_stride=256, work=X, tokens=9, sequences=3, n_requests=5, key_heads=2,
           value_heads=4, head_k_dim=64, head_v_dim=64, conv_kernel=4, eps=1e-6, max_new=9, dtype=1, stream=None)

STEP = [dict(sequences=1025), dict(sequences=-1), dict(n_requests=0), dict(n_requests=1 << 31), dict(rows=None)]
PAGES = [dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(page_size=0), dict(n_pages=0), dict(n_pages=1 << 31)]
HEADS = [dict(heads=3, kv_heads=2), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=512), dict(heads=65536, kv_heads=1),
         dict(tokens=-1)]


@pytest.mark.parametrize("name,base,changes", [
    ("gsq_page_plan", PLAN, STEP + PAGES + [dict(max_pages=0), dict(max_pages=1 << 27), dict(tokens=-1), dict(tokens=1 << 31),
                                            dict(held=None), dict(pos=None), dict(cu=None), dict(new_tokens=None)]),
    ("gsq_page_advance", ADVANCE, STEP + [dict(lengths=None)]),
    ("gsq_page_release", RELEASE, STEP[:4] + [dict(requests=None), dict(free_pages=None), dict(n_pages=0), dict(max_pages=0)]),
    ("gsq_paged_write", WRITE, PAGES + HEADS + [dict(rotary_dim=3), dict(rotary_dim=130), dict(inv_freq=None), dict(k_pages=X + 8),
                                                dict(q_out=X + 8), dict(eps=float("nan")), dict(eps=-1.0), dict(slots=None),
                                                dict(tokens=1 << 24)]),
    ("gsq_attn_paged", ATTN, STEP + PAGES + HEADS + [dict(max_pages=0), dict(max_pages=1 << 27), dict(q=X + 8), dict(out=X + 2),
                                                     dict(v_pages=X + 4), dict(work=X + 4), dict(cus=0), dict(max_new=-1),
                                                     dict(table=None), dict(cu=None)]),
    ("gsq_gdn_packed", GDN, STEP + [dict(key_heads=3), dict(key_heads=0), dict(head_k_dim=96), dict(head_k_dim=256),
                                    dict(head_v_dim=192), dict(head_v_dim=32), dict(conv_kernel=1), dict(conv_kernel=9),
                                    dict(rec_state=X + 8), dict(work=X + 4), dict(work=None), dict(eps=-1.0), dict(max_new=-1),
                                    dict(tokens=-1), dict(tokens=1 << 20)])],
    ids=["plan", "advance", "release", "write", "attn", "gdn"])
def test_c_refusals(name, base, changes):
    L = _lib()
    fn = getattr(L.lib(), name)
    for change in changes:
        assert fn(*dict(base, **change).values()) == L.GSQ_E_VALUE, change
        assert L.lib().gsq_last_error()
    if "dtype" in base:
        for code in (0, 7):  # 16-bit activations only
            assert fn(*dict(base, dtype=code).values()) == L.GSQ_E_TYPE


def test_c_empty_calls_return():
    L = _lib().lib()
    for fn, base in ((L.gsq_paged_write, WRITE), (L.gsq_attn_paged, ATTN), (L.gsq_gdn_packed, GDN)):
        assert fn(*dict(base, tokens=0).values()) == 0
    assert L.gsq_page_advance(*dict(ADVANCE, sequences=0).values()) == 0
    assert L.gsq_page_release(*dict(RELEASE, sequences=0).values()) == 0


def test_work_sizes():
    L = _lib().lib()
    assert L.gsq_attn_paged_work(9, 3, 4, 1, 128, 7, 16, 9, 256) >= 0
    assert L.gsq_attn_paged_work(9, 3, 4, 3, 128, 7, 16, 9, 256) == -1
    assert L.gsq_gdn_packed_work(9, 3, 2, 4, 64, 64, 4, 9) > 0
    assert L.gsq_gdn_packed_work(9, 3, 2, 4, 63, 64, 4, 9) == -1


def _cpu():
    i32 = torch.zeros(2, dtype=torch.int32)
    q, pages = torch.zeros(3, 4, 64).half(), torch.zeros(5, 2, 16, 64).half()
    return i32, q, pages


def test_python_refusals_on_cpu():
    from mlx_gsq_amd.runtime.kernels import paged
    i32, q, pages = _cpu()
    table, plan = torch.zeros(2, 4, dtype=torch.int32), paged.PagePlan(torch.zeros(3, dtype=torch.int32), i32, i32, i32.long(), i32.long())
    for call in (lambda: paged.page_plan(i32, i32, i32, i32, table, i32, i32[:1], tokens=3, page_size=16),
                 lambda: paged.page_advance(plan, i32), lambda: paged.page_release(i32, i32, i32, table, i32, i32[:1]),
                 lambda: paged.paged_write(q, q[:, :2], q[:, :2], q[0, 0], q[0, 0], i32.double(), pages, pages, plan.pos, plan.slots,
                                           eps=1e-6),
                 lambda: paged.attn_paged(q, pages, pages, table, plan),
                 lambda: paged.gdn_packed(q[0], q[0], q[0], pages, q[0], q[0], q[0], pages, q[0], plan, key_heads=1, value_heads=1,
                                          head_k_dim=32, head_v_dim=64, eps=1e-6)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_tensor_checks():
    """The checks behind the wrappers, which look at shapes, types and strides only."""
    from mlx_gsq_amd.runtime.kernels import paged
    i32, q, pages = _cpu()
    for t, shape in ((i32.long(), (2,)), (i32, (3,)), (torch.zeros(4, dtype=torch.int32)[::2], (2,))):
        with pytest.raises(ValueError, match="int32"):
            paged._int32(shape, t)
    with pytest.raises(ValueError, match="block table"):
        paged._table(i32, i32, i32)
    for k, v, dtype in ((pages[0], pages[0], torch.float16), (pages, pages[:4], torch.float16), (pages, pages, torch.bfloat16),
                        (pages.transpose(1, 2), pages.transpose(1, 2), torch.float16)):
        with pytest.raises(ValueError, match="pages"):
            paged._pages(k, v, dtype)
    assert paged._head_rows(torch.zeros(3, 4, 128).half()[..., :64], 3, 4, 64, torch.float16) == (512, 128)
    with pytest.raises(ValueError, match="inner stride"):
        paged._head_rows(torch.zeros(3, 64, 4).half().transpose(1, 2), 3, 4, 64, torch.float16)
    for args in ((3, 4, 128, torch.float16), (3, 2, 64, torch.float16), (3, 4, 64, torch.bfloat16)):
        with pytest.raises(ValueError, match="share one dtype"):
            paged._head_rows(q, *args)
    bad = paged.PagePlan(torch.zeros(2, dtype=torch.int32), i32, i32, i32.long(), i32.long())
    with pytest.raises(ValueError, match="cu must be"):
        paged._sequences(bad)


def test_calls_refuse_what_autograd_follows():
    from mlx_gsq_amd.runtime.kernels import paged
    i32, q, pages = _cpu()
    plan = paged.PagePlan(torch.zeros(3, dtype=torch.int32), i32, i32, i32.long(), i32.long())
    follow = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="no derivative"):
        paged.attn_paged(follow, pages, pages, i32, plan)
    with pytest.raises(ValueError, match="no derivative"):
        paged.attn_paged(q, pages, pages, i32, plan, gate=follow)
    with pytest.raises(ValueError, match="no derivative"):
        paged.paged_write(follow, q, q, q, q, q, pages, pages, i32, i32, eps=1e-6)

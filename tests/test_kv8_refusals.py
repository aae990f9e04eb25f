"""What the calls on an 8-bit K/V cache and on trees refuse before anything reaches a GPU: through
the C ABI with made-up addresses, and the Python checks on CPU tensors."""
import pytest
import torch

X = 1 << 20


def _lib():
    from mlx_gsq_amd import _lib
    return _lib


WRITE = dict(qg=X, qg_stride=1024, k=X, k_stride=128, v=X, v_stride=128, q_norm_w=X, k_norm_w=X, inv_freq=X, k_cache=X,
             v_cache=X, k_scale=X, v_scale=X, pos=X, n_pos=1, parents=None, n_trees=0, q=X, batch=2, seq=3, heads=4,
             kv_heads=1, head_dim=128, rotary_dim=64, max_len=100, eps=1e-6, dtype=1, stream=None)
READ = dict(k_cache=X, v_cache=X, k_scale=X, v_scale=X, k=X, v=X, heads=4, max_len=100, start=0, n=100, head_dim=128, dtype=1,
            stream=None)
ATTN = dict(q=X, q_stride=512, qg=X, qg_stride=1024, k_cache=X, v_cache=X, k_scale=X, v_scale=X, pos=X, n_pos=1, parents=None,
            n_trees=0, out=X, out_stride=512, work=None, splits=1, batch=2, seq=3, heads=4, kv_heads=1, head_dim=128,
            max_len=100, dtype=1, stream=None)
TREE = dict(qkv=X, qkv_stride=512, z=X, z_stride=256, ab=X, ab_stride=8, conv_state=X, conv_w=X, ssm_a=X, dt_bias=X,
            rec_state=X, norm_w=X, parents=X, n_trees=1, out=X, out_stride=256, batch=2, seq=3, key_heads=2, value_heads=4,
            head_k_dim=64, head_v_dim=64, conv_kernel=4, eps=1e-6, dtype=1, stream=None)

LAYOUT = [dict(heads=3, kv_heads=2), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=512), dict(max_len=0),
          dict(max_len=2), dict(max_len=1 << 31), dict(n_pos=3), dict(n_pos=0), dict(parents=X, n_trees=3),
          dict(parents=X, n_trees=1, seq=65), dict(batch=65536), dict(seq=-1), dict(pos=None), dict(k_scale=None),
          dict(k_cache=X + 8), dict(v_cache=X + 4)]


@pytest.mark.parametrize("name,base,changes", [
    ("gsq_kv8_write", WRITE, LAYOUT + [dict(rotary_dim=3), dict(rotary_dim=130), dict(inv_freq=None), dict(q=X + 8),
                                       dict(eps=float("nan")), dict(eps=-1.0)]),
    ("gsq_attn_kv8", ATTN, LAYOUT + [dict(splits=0), dict(splits=2), dict(splits=65536, work=X), dict(work=X + 4, splits=2),
                                     dict(q=X + 8), dict(q_stride=516), dict(qg=X + 4), dict(qg_stride=1026),
                                     dict(out_stride=514), dict(out=X + 2)]),
    ("gsq_kv8_read", READ, [dict(n=101), dict(start=101, n=0), dict(start=1), dict(start=-1), dict(n=-1), dict(head_dim=100),
                            dict(k_cache=None), dict(v=X + 8), dict(heads=-1), dict(heads=1 << 30, max_len=1 << 20)]),
    ("gsq_gdn_tree", TREE, [dict(seq=65), dict(seq=-1), dict(batch=65536), dict(key_heads=3), dict(key_heads=0),
                            dict(head_k_dim=130), dict(head_k_dim=66), dict(head_v_dim=96), dict(head_v_dim=320),
                            dict(conv_kernel=1), dict(conv_kernel=9), dict(n_trees=3), dict(parents=None), dict(rec_state=None),
                            dict(eps=-1.0)])], ids=["write", "attn", "read", "gdn_tree"])
def test_c_refusals(name, base, changes):
    L = _lib()
    fn = getattr(L.lib(), name)
    for change in changes:
        args = dict(base, **change)
        assert fn(*args.values()) == L.GSQ_E_VALUE, change
        assert L.lib().gsq_last_error()
    assert fn(*dict(base, dtype=7).values()) == L.GSQ_E_TYPE
    if name in ("gsq_kv8_write", "gsq_attn_kv8"):
        assert fn(*dict(base, dtype=0).values()) == L.GSQ_E_TYPE  # 16-bit activations only


def test_c_empty_calls_return():
    L = _lib().lib()
    for fn, base in ((L.gsq_kv8_write, WRITE), (L.gsq_attn_kv8, ATTN), (L.gsq_gdn_tree, TREE)):
        assert fn(*dict(base, batch=0).values()) == 0 and fn(*dict(base, seq=0).values()) == 0
    assert L.gsq_kv8_read(*dict(READ, n=0).values()) == 0 and L.gsq_kv8_read(*dict(READ, heads=0).values()) == 0


def test_python_refusals_on_cpu():
    from mlx_gsq_amd.runtime.kernels import kv8, model_ops
    u, s, p = torch.zeros(1, 1, 8, 64, dtype=torch.uint8), torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int64)
    q, h = torch.zeros(1, 2, 64).half(), torch.zeros(1, 2, 128).half()
    with pytest.raises(ValueError, match="GPU"):
        kv8.attn_kv8(q, h, u, u, s, s, p, heads=1, kv_heads=1, head_dim=64)
    with pytest.raises(ValueError, match="GPU"):
        kv8.kv8_read(u, u, s, s, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        kv8.kv8_write(h, q, q, q[0, 0], q[0, 0], p.double(), u, u, s, s, p, heads=1, kv_heads=1, head_dim=64, rotary_dim=2,
                      eps=1e-6)
    with pytest.raises(ValueError, match="GPU"):
        model_ops.gdn_tree(h, q, q, q, q, s, s, s, q, p.int(), key_heads=1, value_heads=1, head_k_dim=32, head_v_dim=64, eps=1e-6)


def test_tensor_checks():
    """The checks behind the wrappers, which look at shapes, types and strides only."""
    from mlx_gsq_amd.runtime.kernels import kv8
    u, s = torch.zeros(2, 3, 8, 64, dtype=torch.uint8), torch.zeros(2, 3, 8)
    kv8._caches(u, u, s, s)
    for bad in ((u[0], u[0], s, s), (u, u[:, :, :4], s, s), (u, u, s[:1], s), (u, u, s.double(), s),
                (u.transpose(0, 1), u.transpose(0, 1), s.transpose(0, 1), s.transpose(0, 1)),
                (u[:, :, ::2], u[:, :, ::2], s[:, :, ::2], s[:, :, ::2])):
        with pytest.raises(ValueError):
            kv8._caches(*bad)
    with pytest.raises(TypeError):
        kv8._caches(u.to(torch.int8), u, s, s)
    p = torch.zeros(2, dtype=torch.int64)
    t = torch.zeros(2, 5, dtype=torch.int32)
    assert kv8._where(p, None, 2, 5) == (2, 0) and kv8._where(p[:1], t, 2, 5) == (1, 2) and kv8._where(p, t[0], 2, 5) == (2, 1)
    for bad in ((p.int(), None, 2, 5), (torch.zeros(3, dtype=torch.int64), None, 2, 5), (p, t.long(), 2, 5), (p, t, 2, 4),
                (p, t.t().contiguous().t(), 2, 5), (p, torch.zeros(2, 65, dtype=torch.int32), 2, 65),
                (torch.zeros(2, 2, dtype=torch.int64)[:, 0], None, 2, 5)):
        with pytest.raises(ValueError):
            kv8._where(*bad)
    x, half = torch.zeros(2, 5, 64).half(), torch.float16
    assert kv8._row_stride(x, 2, 5, 64, half) == 64 and kv8._row_stride(x[..., :16], 2, 5, 16, half) == 64
    assert kv8._row_stride(x[:, :1], 2, 1, 64, half) == 320 and kv8._row_stride(x[1:], 1, 5, 64, half) == 64
    for bad, n in ((x[..., ::2], 32), (x.transpose(0, 1), 64), (x[:, :4], 64), (x, 32), (x[0], 64), (x.float(), 64)):
        with pytest.raises(ValueError):
            kv8._row_stride(bad, *bad.shape[:2], n, half)
    with pytest.raises(TypeError):
        kv8._dtype_code(x.float())


def test_splits_rule():
    splits = _lib().lib().gsq_attn_kv8_splits
    assert splits(1, 1, 24, 4, 256, 300, 256) == 1 and splits(1, 4096, 24, 4, 256, 4096, 256) == 1
    assert splits(1, 1, 24, 4, 256, 131072, 256) == 128
    for B, S, H, G, hd in ((1, 1, 24, 4, 256), (3, 64, 24, 4, 256), (1, 700, 32, 8, 128), (200, 1, 8, 8, 64), (1, 1, 1, 1, 64)):
        for L in (S, S + 511, 4096, 131072, 10 ** 6):
            n = splits(B, S, H, G, hd, L, 256)
            assert 1 <= n <= 65535 and (n == 1 or n * 256 <= L)
            rows = -(-S * (H // G) // 256) * G * B  # workgroups, at the least
            assert n == 1 or n * rows <= 512
    for bad in ((0, 1, 4, 1, 64, 8, 256), (1, 0, 4, 1, 64, 8, 256), (1, 1, 4, 0, 64, 8, 256), (1, 1, 4, 1, 64, 0, 256),
                (1, 1, 4, 1, 64, 8, 0)):
        assert splits(*bad) == 1


@pytest.mark.parametrize("mode", ["reverse", "forward"])
def test_python_refuses_derivatives(mode):
    """Tensors that autograd follows, one at a time, before anything else is looked at; without a mode that records
    they are as good as others."""
    from contextlib import nullcontext

    from torch.autograd import forward_ad

    from mlx_gsq_amd.runtime.kernels import kv8, model_ops
    p, w, u = torch.zeros(1, dtype=torch.int64), torch.zeros(64).half(), torch.zeros(1, 1, 8, 64, dtype=torch.uint8)
    q, h, s, f = torch.zeros(1, 2, 64).half(), torch.zeros(1, 2, 128).half(), torch.zeros(1, 1, 8), torch.zeros(1).double()
    kw = dict(heads=1, kv_heads=1, head_dim=64)
    calls = [(lambda *t: kv8.kv8_write(*t[:6], u, u, *t[6:], p, rotary_dim=2, eps=1e-6, **kw), [h, q, q, w, w, f, s, s]),
             (lambda *t: kv8.kv8_read(u, u, *t, dtype=torch.float16), [s, s]),
             (lambda *t: kv8.attn_kv8(*t[:2], u, u, *t[2:], p, **kw), [q, h, s, s]),
             (lambda *t: model_ops.gdn_tree(*t, p.int(), key_heads=1, value_heads=1, head_k_dim=32, head_v_dim=64, eps=1e-6),
              [h, q, q, q, q, s, s, s, w])]
    with forward_ad.dual_level() if mode == "forward" else nullcontext():
        for call, args in calls:
            with pytest.raises(ValueError, match="GPU"):
                call(*args)
            for i, t in enumerate(args):
                t = forward_ad.make_dual(t, torch.ones_like(t)) if mode == "forward" else t.clone().requires_grad_()
                changed = args[:i] + [t] + args[i + 1:]
                with pytest.raises(ValueError, match="derivative"):
                    call(*changed)
                if mode == "reverse":
                    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
                        call(*changed)

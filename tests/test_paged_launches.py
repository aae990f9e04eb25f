"""The host side of the calls that serve many requests in one step, on the stand-in for the HIP runtime: their
launches, that they allocate nothing, their LDS limits on every device, and sizes that no launch can count."""
from test_host_launches import run, stub  # noqa: F401  (a fixture)

SIGNATURES = """
V = ctypes.c_int
lib.gsq_page_plan.argtypes = [P] * 7 + [I] * 6 + [P] * 6
lib.gsq_page_advance.argtypes = [P] * 3 + [I] * 2 + [P]
lib.gsq_page_release.argtypes = [P] * 6 + [I] * 4 + [P]
lib.gsq_paged_write.argtypes = [P, I, I] * 3 + [P] * 8 + [I] * 7 + [F, V, P]
lib.gsq_attn_paged_work.argtypes, lib.gsq_attn_paged_work.restype = [I] * 9, I
lib.gsq_attn_paged.argtypes = [P, P, I, I] + [P] * 8 + [I] * 11 + [V, P]
lib.gsq_gdn_packed_work.argtypes, lib.gsq_gdn_packed_work.restype = [I] * 8, I
lib.gsq_gdn_packed.argtypes = [P, I] * 3 + [P] * 10 + [I, P] + [I] * 8 + [F, I, V, P]

def plan(tokens, sequences=4):
    return lib.gsq_page_plan(X, X, X, X, X, X, X, sequences, 8, 600, 5000, tokens, 16, X, X, X, X, X, S)

def write(tokens, hd=256, dtype=F16):
    return lib.gsq_paged_write(X, 24 * 512, 512, X, 4 * hd, hd, X, 4 * hd, hd, X, X, X, X, X, X, X, Y, tokens, 24, 4, hd, 64, 100, 16,
                               1e-6, dtype, S)

def attn(tokens, sequences, pages, most=None, dtype=F16, hd=256, heads=24, kv_heads=4):
    return lib.gsq_attn_paged(X, X, heads * hd, hd, X, X, X, X, X, X, Y, Y + (1 << 36), tokens, sequences, 2000, pages, heads, kv_heads,
                              hd, 100000, 64, tokens if most is None else most, 256, dtype, S)

def gdn(tokens, sequences, most=None, dtype=F16, dk=128, dv=128, hv=48):
    return lib.gsq_gdn_packed(X, 20000, X, 20000, X, 128, X, X, X, X, X, X, X, X, X, Y, 20000, Y + (1 << 36), tokens, sequences, 2000, 16,
                              hv, dk, dv, 4, 1e-6, tokens if most is None else most, dtype, S)
lib.gsq_prepare(S)
stub.stub_clear()
"""


def test_launches(stub):  # noqa: F811
    run(stub, SIGNATURES + """
CALLS = [(lambda: plan(0), 1), (lambda: plan(4096), 1), (lambda: plan(4097), 2), (lambda: plan(20000, 1024), 2),
         (lambda: plan(5, 0), 1), (lambda: lib.gsq_page_advance(X, X, X, 4, 8, S), 1),
         (lambda: lib.gsq_page_release(X, X, X, X, X, X, 4, 8, 600, 5000, S), 1),
         (lambda: write(1), 1), (lambda: write(511), 1), (lambda: write(512, 64, BF16), 1), (lambda: write((1 << 24) - 1, 128), 1),
         (lambda: write(0), 0), (lambda: attn(0, 1, 10), 0),
         # positions of one piece: nothing to merge; more: pieces may be there, whatever the lengths are
         (lambda: attn(1, 1, 4), 1), (lambda: attn(8, 8, 5, 1), 2), (lambda: attn(5000, 5, 80), 2), (lambda: attn(40, 1024, 2000, 1, BF16, 64), 2),
         (lambda: attn(300, 3, 4, dtype=BF16, hd=128), 1),
         # single tokens: convolution and recurrence; chunks and their outputs only where a sequence may have 16 tokens
         (lambda: gdn(32, 32, 1), 2), (lambda: gdn(32, 2, 15), 2), (lambda: gdn(32, 2, 16), 5), (lambda: gdn(524280, 3), 5),
         (lambda: gdn(600, 1, 600, BF16, 32, 256, 16), 5), (lambda: gdn(0, 0), 0)]
for i, (fn, n) in enumerate(CALLS):
    before = stub.stub_launches()
    assert fn() == 0, (i, lib.gsq_last_error())
    assert stub.stub_launches() - before == n, (i, stub.stub_launches() - before)
assert stub.stub_mallocs() == 0
""")


def test_lds_limit_on_every_device(stub):  # noqa: F811
    """Refused before a launch, raised once a device, every time past the devices that are remembered."""
    run(stub, SIGNATURES + """
for i, fn in enumerate((lambda: attn(5000, 5, 80), lambda: attn(8, 8, 5, 1, BF16))):
    stub.stub_clear()
    knob("stub_device", 0)
    knob("stub_attr_fails", 1)
    before = stub.stub_launches()
    assert fn() != 0 and stub.stub_launches() == before, i
    knob("stub_attr_fails", 0)
    for device in (0, 1, 1, 0, 70, 70):
        knob("stub_device", device)
        assert fn() == 0, (i, lib.gsq_last_error())
    assert [stub.stub_attr_device(j) for j in range(stub.stub_attrs())] == [0, 1, 70, 70], i
""")


def test_sizes_no_launch_counts(stub):  # noqa: F811
    """More threads than a launch counts (32 bits along x): refused before anything runs."""
    run(stub, SIGNATURES + """
before = stub.stub_launches()
for fn in (lambda: attn(1 << 24, 1, 20, 1, heads=64, kv_heads=64), lambda: attn(1 << 26, 1, 20, 32, hd=64, heads=31, kv_heads=31)):
    assert fn() != 0 and b"launch" in lib.gsq_last_error(), lib.gsq_last_error()
assert write(1 << 24) != 0 and gdn(524281, 1) != 0
assert stub.stub_launches() == before
assert attn(1 << 22, 1, 20, heads=32, kv_heads=8, hd=128) == 0, lib.gsq_last_error()
assert lib.gsq_attn_paged_work(1 << 31, 1, 24, 4, 256, 100, 64, 1, 256) == -1
# workspaces: what the largest step may need is bounded by the device, not by its tokens
assert lib.gsq_attn_paged_work(1 << 20, 1000, 24, 4, 256, 100000, 64, 1 << 20, 256) < 1 << 27
""")

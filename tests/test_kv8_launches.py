"""The host side of the calls on an 8-bit cache and on trees, on the stand-in for the HIP runtime: their
launches, that they allocate nothing, and their LDS limits on every device."""
from test_host_launches import run, stub  # noqa: F401  (a fixture)


def test_launches_and_attributes(stub):  # noqa: F811
    run(stub, """
V = ctypes.c_int
lib.gsq_kv8_write.argtypes = [P, I, P, I, P, I, P, P, P, P, P, P, P, P, I, P, I, P, I, I, I, I, I, I, I, F, V, P]
lib.gsq_kv8_read.argtypes = [P, P, P, P, P, P, I, I, I, I, I, V, P]
lib.gsq_attn_kv8.argtypes = [P, I, P, I, P, P, P, P, P, I, P, I, P, I, P, I, I, I, I, I, I, I, V, P]
lib.gsq_gdn_tree.argtypes = [P, I, P, I, P, I, P, P, P, P, P, P, P, I, P, I, I, I, I, I, I, I, I, F, V, P]

def write(seq, tree=None):
    return lib.gsq_kv8_write(X, 1024, X, 128, X, 128, X, X, X, X, X, X, X, X, 1, tree, 1 if tree else 0, Y, 2, seq, 4, 1, 128, 64,
                             4096, 1e-6, F16, S)

def attn(seq, splits, dtype=F16, hd=128, heads=24, max_len=8192):
    return lib.gsq_attn_kv8(X, heads * hd, X, 2 * heads * hd, X, X, X, X, X, 1, None, 0, Y, heads * hd, Y + (1 << 28), splits, 1,
                            seq, heads, 4, hd, max_len, dtype, S)

def tree(seq, dtype=F16, dv=128):
    return lib.gsq_gdn_tree(X, 4096, X, 2048, X, 64, X, X, X, X, X, X, X, 1, Y, 2048, 2, seq, 2, 4, 128, dv, 4, 1e-6, dtype, S)

def read():
    return lib.gsq_kv8_read(X, X, X, X, Y, Y, 4, 100, 0, 100, 128, F16, S)

CALLS = [(lambda: write(1), 1), (lambda: write(64, X), 1), (lambda: write(4000), 1), (read, 1), (lambda: attn(1, 1), 1),
         (lambda: attn(1, 8), 2), (lambda: attn(4000, 1), 1), (lambda: attn(4000, 2, BF16, 256), 2), (lambda: attn(4000, 1, F16, 64, 64), 1),
         (lambda: tree(1), 1), (lambda: tree(64), 1), (lambda: tree(20, F32, 256), 1)]
lib.gsq_prepare(S)
stub.stub_clear()
for i, (fn, n) in enumerate(CALLS):
    before = stub.stub_launches()
    assert fn() == 0, (i, lib.gsq_last_error())
    assert stub.stub_launches() - before == n, i
assert stub.stub_mallocs() == 0
# limits: refused before a launch, raised once a device, every time past the devices that are remembered
for i, fn in enumerate((lambda: attn(2, 1, BF16, 64), lambda: attn(4000, 1, BF16, 64, 4), lambda: tree(30, BF16, 64))):
    stub.stub_clear()
    knob("stub_device", 0)
    knob("stub_attr_fails", 1)
    assert fn() != 0 and stub.stub_launches() == 0, i
    knob("stub_attr_fails", 0)
    for device in (0, 1, 1, 0, 70, 70):
        knob("stub_device", device)
        assert fn() == 0, (i, lib.gsq_last_error())
    assert [stub.stub_attr_device(j) for j in range(stub.stub_attrs())] == [0, 1, 70, 70], i
# more threads than a launch counts (32 bits along x): refused before anything runs
stub.stub_clear()
knob("stub_device", 0)
before = stub.stub_launches()
for call in (lambda: attn(400000, 4000, max_len=500000), lambda: attn(400000, 128, max_len=500000)):
    assert call() != 0 and b"launch" in lib.gsq_last_error() and stub.stub_launches() == before
assert lib.gsq_kv8_write(X, 128, X, 64, X, 64, X, X, X, X, X, X, X, X, 1, None, 0, Y, 1, 1 << 24, 1, 1, 64, 0, 1 << 25, 1e-6,
                         F16, S) != 0 and stub.stub_launches() == before
""")

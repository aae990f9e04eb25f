"""The host side of steps of packed requests where it can go wrong, without a GPU: launches of empty steps, sizes of
workspaces, and the decoder's bookkeeping."""
from test_host_launches import run, stub  # noqa: F401  (a fixture)
from test_paged_launches import SIGNATURES


def test_no_launch_is_empty(stub):  # noqa: F811
    """A step without sequences has no workgroup to give a launch over sequences: the convolution and the launch that
    clears the rows run, as many as with a hint of single tokens."""
    run(stub, SIGNATURES + """
for tokens in (1, 16, 100, 5000):
    for most in (None, 1):
        before = stub.stub_launches()
        assert gdn(tokens, 0, most) == 0 and stub.stub_launches() - before == 2, (tokens, most)
    assert lib.gsq_gdn_packed_work(tokens, 0, 16, 48, 128, 128, 4, tokens) == lib.gsq_gdn_packed_work(tokens, 0, 16, 48, 128, 128, 4, 1)
    assert attn(tokens, 0, 80) == 0
""")

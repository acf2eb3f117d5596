"""torch_ops calls are ordered with torch's own work on its default stream."""
import pytest

pytestmark = pytest.mark.gpu


def test_default_stream_order():
    import torch
    import hephaestus_b200.torch_ops as T
    a = torch.randn(8192, 8192, device="cuda")
    x = torch.zeros(1 << 20, device="cuda", dtype=torch.int32)
    m = torch.zeros(64, 1024, device="cuda")
    for _ in range(3):
        x.zero_()
        m.zero_()
        torch.cuda.synchronize()
        b = a
        for _ in range(4):  # some milliseconds of work before x is written
            b = a @ b
        x.fill_(3)
        m[:, 7] = 1.0
        total, scan = T.sum(x), T.cumsum(x)
        value, index = T.argmax_axis(m, 1)
        normed = T.rms_norm(m)
        late = scan[-1] + 0  # torch's next work sees the result
        x.zero_()            # and does not overtake the calls
        assert int(total) == 3 << 20 and int(late) == 3 << 20
        assert bool((index == 7).all()) and bool((value == 1).all())
        # one 1 in 1024: 1 / sqrt(1/1024 + 1e-6), a few fp32 roundings off
        want = (1 / 1024 + 1e-6) ** -0.5
        assert abs(float(normed[0, 7]) - want) < want * 2.0 ** -20

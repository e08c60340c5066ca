"""Layer norm from several host threads at once, a stream each."""
import threading

import pytest

from test_gpu_network_ends import _stream, norm_run, torch, wrap  # noqa: F401

pytestmark = pytest.mark.gpu


def test_layer_norms_of_other_widths_at_the_same_time(nxv, torch):
    """Widths that take one kernel with another amount of shared memory: every call is a valid one, and stays so
    whatever the other threads call in between."""
    from nx_vulkan_b200 import _native
    lib = _native.load()
    widths = [7001, 3501, 6001, 4001, 7003, 3503, 5001, 4501]
    wrong = []

    def work(cols):
        try:
            s = torch.cuda.Stream()
            lib.nxv_set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                torch.manual_seed(cols)
                x, g, b = torch.randn(4, cols, device="cuda"), torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
                want = [t.clone() for t in norm_run(nxv, torch, x, g, b, 1e-5, "f32")]
                outs = [torch.empty_like(t) for t in want]
                hx, hg, hb, *ho = (wrap(nxv, t) for t in (x, g, b, *outs))
                s.synchronize()
                for _ in range(4000):
                    if nxv.layer_norm(hx, hg, hb, 4, cols, 1e-5, out=ho)[0] != "ok":
                        wrong.append((cols, _native.last_error()))
                s.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(outs, want)):
                    wrong.append((cols, "result"))
        except BaseException as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in widths]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, (len(wrong), wrong[0])

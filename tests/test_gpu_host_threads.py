"""Host threads that call the library at the same time, with layers of different
sizes: the shared memory that a launch asks for depends on the number of
experts, and no thread's launch may be refused for another's size."""
import threading

import pytest

torch = pytest.importorskip("torch")

import mail_b200 as mb  # noqa: E402
from mail_b200 import _lib  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run_in_threads(calls, repeats):
    """Each call (returning a status) again and again in a thread of its own."""
    lib = _lib.load()
    failed = []

    def work(call):
        for _ in range(repeats):
            if call() != 0:
                failed.append(lib.moe_last_error().decode())
                return

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[0]
    assert mb.device_error() == 0


@pytest.mark.parametrize("rows", [16, 600])
def test_dense_layers(rows):
    """Pre-routed bf16 layers: swapped operands for few rows an expert, else plain."""
    lib, H, I = _lib.load(), 128, 128
    calls, keep = [], []
    for E in (100, 300):
        g = torch.Generator(device=DEV).manual_seed(E)
        x = torch.randn((rows, H), device=DEV, generator=g).bfloat16()
        w13 = (torch.randn((E, 2 * I, H), device=DEV, generator=g) * H ** -0.5).bfloat16()
        w2 = (torch.randn((E, H, I), device=DEV, generator=g) * I ** -0.5).bfloat16()
        gs = torch.zeros(E, dtype=torch.int32, device=DEV)
        gs[-1] = rows
        want = mb.fused_moe_mlp(x, w13.transpose(1, 2), w2.transpose(1, 2), gs)
        out = torch.empty_like(x)
        size = _lib.query("moe_fused_mlp_workspace_size", rows, H, I, E, _lib.BF16, 128)
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        st = torch.cuda.Stream()
        args = (x.data_ptr(), _lib.BF16, rows, H, w13.data_ptr(), w2.data_ptr(), E, I, gs.data_ptr(), _lib.I32, 128,
                out.data_ptr(), ws.data_ptr(), size, st.cuda_stream)
        calls.append(lambda args=args: lib.moe_fused_mlp(*args))
        keep.append((x, w13, w2, gs, ws, st, out, want))
    run_in_threads(calls, 30000)
    for k in keep:
        assert torch.equal(k[-2], k[-1])


def test_aligning_many_experts():
    lib, T, k = _lib.load(), 40, 4
    calls, keep = [], []
    for E in (400, 1024):
        ids = torch.randint(0, E, (T, k), device=DEV, generator=torch.Generator(device=DEV).manual_seed(E)).int()
        want = mb.moe_align(ids, E, block_m=1)
        cap = int(_lib.query("moe_align_capacity", T * k, E, 1))
        size = _lib.query("moe_align_workspace_size", T, k, E, 1)
        ints = [torch.empty(n, dtype=torch.int32, device=DEV) for n in (
            cap, T * k, E, E + 1, int(_lib.query("moe_tile_table_ints", E, cap)))]
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
        st = torch.cuda.Stream()
        args = (ids.data_ptr(), T, k, E, 1, *(t.data_ptr() for t in ints), ws.data_ptr(), ws.numel(), st.cuda_stream)
        calls.append(lambda args=args: lib.moe_align(*args))
        keep.append((ids, ws, st, ints[1], want["slot_pos"]))
    run_in_threads(calls, 10000)
    for t in keep:
        assert torch.equal(t[-2], t[-1])


def test_tile_schedules_of_many_experts():
    lib, calls, keep = _lib.load(), [], []
    for E in (3200, 4096):
        gs = torch.ones(E, dtype=torch.int64, device=DEV)
        want = mb.build_tile_schedule(gs, E)
        out = [torch.empty_like(t) for t in want[:3]]
        st = torch.cuda.Stream()
        args = (gs.data_ptr(), _lib.I64, E, E, 128, *(t.data_ptr() for t in out), None, st.cuda_stream)
        calls.append(lambda args=args: lib.moe_tile_schedule(*args))
        keep.append((gs, st, out, want))
    run_in_threads(calls, 10000)
    for _, _, out, want in keep:
        assert all(torch.equal(a, b) for a, b in zip(out, want))

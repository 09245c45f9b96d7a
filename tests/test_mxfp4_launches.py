"""What the MXFP4 entries ask of the HIP runtime (no GPU: the runtime's launch functions are stand-ins)."""
from _hip_calls import hip_calls

P = 1 << 20  # an aligned address that nothing reads
BIG = 1 << 40


def _linear(m, k, n, held=False, ldy=None):
    return "amla_mxfp4_linear", [P, P if held else None, m, k, k, P, P, n, P, 0, n, P, BIG, None]


def _grouped(m, k, n, E, held=False):
    return "amla_mxfp4_grouped_linear", [P, P if held else None, m, k, k, P, P, n, E, P, P, 0, n, 1, P, BIG, None]


def _swiglu(m, k, n):
    return "amla_mxfp4_swiglu", [P, m, k, k, P, P, P, P, n, P, P, P, P, BIG, None]


def _moe(m, d, top_k, n, E):
    return "amla_mxfp4_moe_experts", [P, m, d, d, top_k, P, n, E, P, P, P, P, P, P, P, 1, P, BIG, None]


def test_lds_limits_are_never_lowered(tmp_path):
    """A kernel's limit is the process's: a second thread's call may stand between setting and launch."""
    calls = [_linear(8, 16384, 512), _linear(8, 12288, 512), _linear(3, 16384, 512), _linear(16, 7168, 512),
             _linear(6, 12416, 512), _linear(8, 11392, 512), _linear(300, 512, 700), _linear(4096, 1024, 2048),
             _grouped(14, 8192, 512, 4), _grouped(9, 12288, 512, 4), _grouped(500, 640, 512, 4), _swiglu(12, 4096, 2048),
             _swiglu(8, 7168, 2048), _swiglu(400, 512, 512), _moe(8, 7168, 8, 2048, 16), _moe(12, 7168, 8, 2048, 16),
             _moe(300, 512, 2, 512, 4)]
    limit = {}
    launches = 0
    for (name, args), (rc, log) in zip(calls, hip_calls(tmp_path, calls)):
        assert rc == 0, (name, args)
        for what, f, *rest in log:
            if what == "lds":
                assert rest[0] >= limit.get(f, 0), f"{name} {args[2:9]}: limit {limit[f]} lowered to {rest[0]}"
                limit[f] = rest[0]
            else:
                launches += 1
                assert rest[2] <= limit.get(f, 64 * 1024) and rest[2] <= 160 * 1024
    assert launches >= len(calls) and len(limit) >= 6


def test_outputs_beyond_a_grid_are_refused_before_anything_runs(tmp_path):
    """Neither x is quantised nor a schedule made for a call that is refused."""
    n = 2 ** 29 - 1
    calls = [_linear(600, 128, n), _linear(2 ** 31 - 1, 128, 128), _linear(600, 128, n, held=True), _grouped(33, 128, n, 2),
             _grouped(40, 256, n, 1, held=True), _swiglu(2 ** 31 - 1, 128, 128), _moe(4000, 128, 16, 2 ** 24, 512),
             _moe(300, 2 ** 24, 1, 128, 512)]
    for (name, args), (rc, log) in zip(calls, hip_calls(tmp_path, calls)):
        assert rc == -3 and not log, (name, args, rc, log)


def test_largest_grids_hold_fewer_than_2_to_32_threads(tmp_path):
    calls = [_linear(40, 128, 2 ** 29 - 400), _linear(2 ** 30, 128, 100), _grouped(256, 128, 2 ** 27, 2),
             _swiglu(2 ** 27, 128, 128), _moe(65536, 128, 1, 2 ** 18, 512)]
    for (name, args), (rc, log) in zip(calls, hip_calls(tmp_path, calls)):
        assert rc in (0, -3) and (rc == 0) == bool(log), (name, args, rc, log)
        for what, f, *rest in log:
            if what == "launch":
                assert 0 < rest[0] * rest[1] < 2 ** 32, (name, args, rest)

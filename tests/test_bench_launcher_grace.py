"""bench.launch_workers when a worker dies while its peers are still starting."""
import io
import os
import sys
import textwrap
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import bench  # noqa: E402

STUB = textwrap.dedent("""
    import os, sys, time
    if os.environ["RANK"] == "1":
        sys.exit(7)
    time.sleep(0.7)            # a slow start
    open(sys.argv[1], "w").write(str(os.getpid()))
    time.sleep(float(sys.argv[2]))
""")


def _run(tmp_path, stay):
    stub, pidfile = tmp_path / "stub.py", tmp_path / "rank0.pid"
    stub.write_text(STUB)
    t0 = time.monotonic()
    rc = bench.launch_workers(2, [sys.executable, str(stub), str(pidfile), str(stay)], timeout=120, out=io.StringIO())
    return rc, time.monotonic() - t0, pidfile


def test_a_peer_that_is_still_starting_is_heard(tmp_path):
    rc, took, pidfile = _run(tmp_path, 600)
    assert rc == 7 and took < 60 and pidfile.read_text()
    try:
        os.kill(int(pidfile.read_text()), 0)
        assert False, "the peer was left running"
    except ProcessLookupError:
        pass


def test_peers_that_end_are_not_waited_for(tmp_path):
    rc, took, pidfile = _run(tmp_path, 0)
    assert rc == 7 and took < 2.0 + 10.0 and pidfile.read_text()

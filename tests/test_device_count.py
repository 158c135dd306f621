"""The devices are asked for until the runtime has told them: a count that failed once is no answer for the rest
of the process. Runs in a process of its own, whose hipGetDeviceCount is the one below."""
import json
import pathlib
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parent.parent

COUNT = """
static int asked = 0;
int times_asked(void) { return asked; }
int hipGetDeviceCount(int *count) {  /* no device (hipErrorNoDevice) twice, then one */
  *count = ++asked > 2;
  return asked > 2 ? 0 : 100;
}
"""

CALLS = """
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
import h3attn as H
cfg = H.Kv4Cfg(1, 64, 16, 1, 0)
big = H.raw_view(0x1000, 1 << 20)
seen = []
for _ in range(5):
    status = H.lib().h3_kv4_read(ctypes.byref(cfg), 1, 64, 64, big, big, big, big, None)
    seen.append((status, H.last_error(), shim.times_asked()))
print(json.dumps(seen))
"""


def test_a_failed_count_is_asked_again(tmp_path):
    import h3attn as H

    source, shim = tmp_path / "count.c", tmp_path / "count.so"
    source.write_text(COUNT)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(shim), str(source)], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(shim)], capture_output=True, text=True,
                         cwd=ROOT / "h3-hrx_amd", timeout=120)
    assert run.returncode == 0, run.stderr
    seen = json.loads(run.stdout.splitlines()[-1])
    # a call whose bindings could not be looked up is refused, and asks once; once told, none asks again
    assert [asked for _, _, asked in seen] == [1, 2, 3, 3, 3]
    assert [status == H.H3_ERR_NO_DEVICE for status, _, _ in seen] == [True, True, False, False, False]
    assert "no HIP device" in seen[0][1]

"""The build recipe where torch is not installed: the library is for C programs too."""
import os
import subprocess
import sys
import textwrap

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = textwrap.dedent("""
    import os, sys
    sys.modules["torch"] = None                 # import torch raises ImportError
    sys.path.insert(0, sys.argv[1])
    import qmoe_build as B
    out, commands = sys.argv[2], []
    B.BUILD, B.LIB, B.BIND = os.path.join(out, "_build"), os.path.join(out, "lib.so"), os.path.join(out, "torch.so")
    B.nvcc = lambda: "nvcc"
    class Done:
        returncode, stdout, stderr = 0, "", ""
    def run(cmd, **kw):                         # the commands, not run: their outputs are made
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return Done
    B.subprocess.run = run
    B.build()
    objects = [c for c in commands if "-c" in c]
    assert len(objects) == len(B.sources()) > 5 and all(c[0] == "nvcc" for c in commands), commands
    assert os.path.exists(B.LIB) and not os.path.exists(B.BIND)
    commands.clear()
    B.build()                                   # everything is there
    assert not commands, commands
""")


def test_the_library_is_built_without_torch(tmp_path):
    package = os.path.join(REPO, "nemotron-super-8gb_b200")
    r = subprocess.run([sys.executable, "-c", CHILD, package, str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr

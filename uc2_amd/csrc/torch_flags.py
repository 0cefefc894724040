"""prints the compile and link flags of a Python module against the installed torch (see the Makefile)"""
import os
import sysconfig

import torch

root = os.path.dirname(torch.__file__)
print("-I%s/include -I%s -L%s/lib -ltorch_python -ltorch_cpu -lc10" % (root, sysconfig.get_paths()["include"], root))

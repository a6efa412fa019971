// The implementation lives under b200/.
#pragma once
#include "b200/embedding.hxx"

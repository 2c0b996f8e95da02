// Forwarding header: ccglib::quantize::Quantize is defined in <ccglib/b200_api.hpp>.
#pragma once
#include <ccglib/b200_api.hpp>
